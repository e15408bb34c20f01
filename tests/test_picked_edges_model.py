"""Models that attend over chosen pages: what does not depend on the rest of a batch."""
import pytest
import torch

from hartsyinference_b200 import ops
from hartsyinference_b200.engine import LLMEngine, SamplingParams
from hartsyinference_b200.engine.speculative import _forward_chunk, generate_speculative
from hartsyinference_b200.models.llm import transformer as T
from hartsyinference_b200.models.llm.transformer import ForwardBatch
from hartsyinference_b200.ops import _native as N

from .test_picked_model import BOTH, GROUPED, _model, _prompts

gpu = pytest.mark.gpu


def _engine(m, **kw):
    return LLMEngine(m, num_pages=160, page_size=16, max_batch=4, prefill_chunk=512, max_model_len=1024, **kw)


@pytest.mark.parametrize("dev", BOTH)
@pytest.mark.parametrize("kw", [dict(), GROUPED], ids=["plain", "grouped"])
def test_a_short_chunk_chooses_alike_alone_and_beside_a_long_one(dev, kw, monkeypatch):
    """The last ten tokens of a prompt, by themselves and in a batch with another request's hundred: as many runs, and the pages of the first layer, whose
    queries may differ in last bits with the number of rows (one page of the four is allowed to)."""
    m = _model(dev, 4, seed=7, **kw)
    prompt, other = _prompts(310, 130)
    pick, chosen = ops.pick_pages, []
    monkeypatch.setattr(T.ops, "pick_pages", lambda *a, **k: chosen.append((k["run"], pick(*a, **k).cpu())) or chosen[-1][1].to(a[0].device))
    rows = []
    for beside in (False, True):
        e = _engine(m)
        e.replay([("a", prompt[:300], [])])
        chosen.clear()
        e.replay([("a", prompt[300:], [9])] + ([("b", other, [0])] if beside else []))
        run, picked = chosen[0]
        rows.append(picked[:-(-10 // run)])
    assert rows[0].shape == rows[1].shape
    for one, two in zip(rows[0].flatten(0, 1).tolist(), rows[1].flatten(0, 1).tolist()):
        assert len(set(one) ^ set(two)) <= 2
    if dev == "cuda":
        N.check_status()


@pytest.mark.parametrize("draft", [8, 24])
def test_drafts_of_any_length_choose_as_decoded_tokens_do(draft, monkeypatch):
    """On the host verified drafts give the tokens of plain decoding: each of theirs chooses by itself, however many there are."""
    m = _model("cpu", 2, seed=5)
    prompt = torch.randperm(512, generator=torch.Generator().manual_seed(5)).tolist()[:400]      # (whatever comes out, most of it has been there before)
    p = SamplingParams(greedy=True, max_tokens=60, ignore_eos=True)
    runs = []
    pick = ops.pick_pages
    monkeypatch.setattr(T.ops, "pick_pages", lambda q, *a, **k: runs.append((q.shape[0], k["run"])) or pick(q, *a, **k))
    out, stats = generate_speculative(_engine(m), prompt, p, ngram=1, max_draft=draft)
    assert max(n for n, r in runs if n < 400) == draft + 1 and {r for n, r in runs if n < 400} == {1} and any(r > 1 for n, r in runs if n == 400)
    assert out == _engine(m).generate([prompt], p)[0]


@gpu
@pytest.mark.parametrize("kw", [dict(), GROUPED], ids=["plain", "grouped"])
def test_gpu_every_layer_chooses_what_the_host_chooses_for_its_queries_and_bounds(kw, monkeypatch):
    """Inside a model: each layer's own bounds, which are those of its own full pages; the queries that it attends with; and the host's choice for copies of both."""
    from hartsyinference_b200.ops import reference as R
    m = _model("cuda", 4, **kw)
    prompt, other = _prompts(300, 100)
    pick, attend, calls = ops.pick_pages, ops.attn_picked, []

    def checked(q, bounds, table, lens, cu_q=None, **k):
        li = len(calls) % len(m.layers)
        assert bounds.data_ptr() == m.key_bounds[li].data_ptr()
        full = torch.unique(torch.cat([row[:n // 16] for row, n in zip(table.cpu(), lens.tolist())])).long()
        assert torch.equal(bounds.cpu()[full], R.page_bounds(m.kv_cache[li, 0].cpu()[full]))
        got = pick(q, bounds, table, lens, cu_q, **k)
        want = pick(q.cpu(), bounds.cpu(), table.cpu(), lens.cpu(), None if cu_q is None else cu_q.cpu(), **k)
        assert torch.equal(got.cpu(), want)
        calls.append((q.data_ptr(), got, bool((want[:, :, -1] >= 0).any())))
        return got

    def given(q, kc, vc, table, lens, picked, *a, **k):
        assert (q.data_ptr(), id(picked)) == (calls[-1][0], id(calls[-1][1])) and kc.data_ptr() == m.kv_cache[(len(calls) - 1) % len(m.layers), 0].data_ptr()
        return attend(q, kc, vc, table, lens, picked, *a, **k)
    monkeypatch.setattr(T.ops, "pick_pages", checked)
    monkeypatch.setattr(T.ops, "attn_picked", given)
    e = _engine(m, use_cuda_graphs=False)
    for step in ([("a", prompt[:200], [])], [("a", prompt[200:], []), ("b", other, [])], [("a", [7], [0]), ("b", [9], [0])], [("b", [5, 6, 7], [2]), ("a", [3], [0])]):
        e.replay(step)
    N.check_status()
    assert len(calls) == 4 * len(m.layers)


@pytest.mark.parametrize("dev", BOTH)
def test_a_shared_prefix_brings_its_bounds(dev):
    """A sequence that begins with another's pages, and one that has computed them itself: the same hidden states."""
    m = _model(dev, 3, seed=9)
    e = _engine(m)
    prefix, one, two = _prompts(256, 40, 70)
    _forward_chunk(e, 1, prefix, 0)
    _forward_chunk(e, 1, one, 256)
    assert e.kv.fork_prefix(1, 2, 270) == 256
    shared = _forward_chunk(e, 2, two, 256)
    _forward_chunk(e, 3, prefix, 0)
    assert torch.equal(_forward_chunk(e, 3, two, 256), shared)
    tail = [_forward_chunk(e, s, [7], 326) for s in (2, 3)]
    assert torch.equal(*tail)


@pytest.mark.parametrize("dev", BOTH)
@pytest.mark.parametrize("kw", [dict(), dict(mrope_interleaved=True, qk_norm=True)], ids=["sections", "turns"])
def test_a_model_with_positions_on_three_axes(dev, kw, monkeypatch):
    """Its keys are stored by another op than those of one axis: bounded all the same, and with every page among the chosen the hidden states are the model's."""
    m = _model(dev, 40, head_dim=64, mrope_section=(12, 10, 10), **kw)
    ids = torch.randint(0, 512, (300,), generator=torch.Generator().manual_seed(1)).int()
    pos = torch.stack([torch.arange(300) // 20, torch.arange(300) // 5 % 4, torch.arange(300) % 5]).int()
    called = []
    pick = ops.pick_pages
    monkeypatch.setattr(T.ops, "pick_pages", lambda *a, **k: called.append(1) or pick(*a, **k))
    outs = []
    for pages in (40, 0):
        m.attn_pages = pages
        m.alloc_kv(60, 16)
        t = lambda x: x.to(dev)
        for a, z in ((0, 170), (170, 300)):
            b = ForwardBatch(tokens=t(ids[a:z]), positions=t(torch.arange(a, z).int()), slot_mapping=t(torch.arange(a, z)), block_table=t(torch.arange(60).int()[None]),
                             kv_lens=t(torch.tensor([z]).int()), is_decode=False, cu_q=t(torch.tensor([0, z - a]).int()), max_q_len=z - a, positions3=t(pos[:, a:z].contiguous()))
            hidden = m.forward_hidden(b)
        outs.append(hidden.float().cpu())
        if pages:
            from hartsyinference_b200.ops import reference as R
            for li in range(len(m.layers)):
                assert torch.equal(m.key_bounds[li, :18].cpu(), R.page_bounds(m.kv_cache[li, 0, :18].cpu()))
    assert len(called) == 2 * len(m.layers)
    assert torch.nn.functional.cosine_similarity(*outs, dim=-1).min() > 0.999
    if dev == "cuda":
        N.check_status()
