"""Models that attend over chosen pages: the ops together, as an engine runs them."""
import pytest
import torch

from hartsyinference_b200 import config, ops
from hartsyinference_b200.engine import LLMEngine, SamplingParams
from hartsyinference_b200.engine.speculative import generate_speculative
from hartsyinference_b200.models.llm import config as C
from hartsyinference_b200.models.llm import transformer as T
from hartsyinference_b200.models.llm.transformer import DecoderModel, ForwardBatch
from hartsyinference_b200.ops import _native as N

gpu = pytest.mark.gpu
BOTH = ["cpu", pytest.param("cuda", marks=gpu)]
GROUPED = dict(num_heads=8, num_kv_heads=2, head_dim=128, hidden_size=512)


def _model(dev="cpu", attn_pages=0, seed=0, fp8=False, **kw):
    m = DecoderModel(C.tiny("qwen2.5-0.5b", **kw), dev, fp8=fp8, attn_pages=attn_pages)
    m.random_init(seed, std=0.05)
    return m


def _like(m, dev, attn_pages):
    """The same weights on a device, with another number of pages."""
    from .test_kv4_model import _twin
    t = _twin(m, dev, "bf16")
    t.attn_pages = attn_pages
    return t


def _prompts(*lens, seed=2):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 512, (n,), generator=g).tolist() for n in lens]


def _logits(m, steps, chunk=128, limit=1024, **kw):
    """Logits of the last token of every step [(key, tokens)]."""
    e = LLMEngine(m, num_pages=160, page_size=16, max_batch=4, prefill_chunk=chunk, max_model_len=limit, **kw)
    out = [e.replay([(key, tokens, [len(tokens) - 1])]) for key, tokens in steps]
    if m.device.type == "cuda":
        N.check_status()
        assert not e._graphs_disabled
    return torch.cat(out).float().cpu()


@pytest.mark.parametrize("dev", BOTH)
@pytest.mark.parametrize("kw", [dict(), GROUPED, dict(attn_softcap=20.0, sliding_window=40, sliding_window_pattern=2)], ids=["plain", "grouped", "capped"])
def test_with_every_page_among_the_chosen_it_is_the_model(dev, kw, monkeypatch):
    """40 pages between the first and the last two hold all of 600 tokens: the choice runs (the engine's limit is longer) and leaves nothing out."""
    m = _model(dev, 40, **kw)
    called = []
    pick = ops.pick_pages
    monkeypatch.setattr(T.ops, "pick_pages", lambda *a, **k: called.append(k["run"]) or pick(*a, **k))
    prompt, = _prompts(600)
    steps = [("a", prompt[i:i + 128]) for i in range(0, 590, 128)] + [("a", [7]), ("a", [9, 11, 400]), ("a", [8])]
    got = _logits(m, steps, limit=2048)
    assert called and (dev == "cpu" or len(called) > 1)
    want = _logits(_like(m, dev, 0), steps, limit=2048)
    assert torch.nn.functional.cosine_similarity(got, want, dim=-1).min() > 0.999


def test_it_attends_to_what_was_chosen_and_bounds_are_those_of_the_cache(monkeypatch):
    """Long prompts in chunks on the host: every layer's bounds are those of its full pages, and attention sees the chosen pages only: with the others
    made unusable right before it, nothing changes."""
    m = _model("cpu", 3, seed=1)
    prompt, = _prompts(300)
    steps = [("a", prompt[i:i + 60]) for i in range(0, 300, 60)] + [("a", [7]), ("a", [9])]
    want = _logits(m, steps, chunk=64)
    from hartsyinference_b200.ops import reference as R
    pages = 302 // 16
    full = [p for p in range(160) if m.key_bounds[0, p, 0, 128] != 0]
    assert len(full) == pages
    for li in range(len(m.layers)):
        assert torch.equal(m.key_bounds[li, full], R.page_bounds(m.kv_cache[li, 0, full]))
    attend, hidden = ops.attn_picked, []

    def only(q, k, v, table, lens, picked, cu_q=None, **kw):
        seen = set(picked[picked >= 0].tolist())
        gone = [int(table[0, p]) for p in range(-(-int(lens[0]) // 16)) if p not in seen]
        hidden.append(len(gone))
        k, v = k.clone(), v.clone()
        k[gone], v[gone] = float("nan"), float("nan")
        return attend(q, k, v, table, lens, picked, cu_q, **kw)
    monkeypatch.setattr(T.ops, "attn_picked", only)
    assert torch.equal(_logits(m, steps, chunk=64), want) and max(hidden) > 3


@gpu
@pytest.mark.parametrize("kw", [dict(), GROUPED, dict(qk_norm=True, rope_dim=32, rope_style=1)], ids=["plain", "grouped", "normed"])
def test_gpu_logits_are_those_of_the_cpu(kw, monkeypatch):
    """Keys and queries differ in last bits between the two devices, and a page on the edge of a choice may then be another one (the choice itself is held to
    the host's elsewhere, on equal inputs): the host's model attends to the pages that the device's chose. Of what it would choose itself most are the same."""
    m = _model("cuda", 4, **kw)
    prompt, = _prompts(300)
    steps = [("a", prompt[i:i + 100]) for i in range(0, 300, 100)] + [("a", [7]), ("a", [9, 11, 400]), ("a", [8])]
    pick, chosen, same = ops.pick_pages, [], []
    monkeypatch.setattr(T.ops, "pick_pages", lambda *a, **k: chosen.append(pick(*a, **k)) or chosen[-1])
    got = _logits(m, steps, use_cuda_graphs=False)
    left = iter([c.cpu() for c in chosen])

    def given(*a, **k):
        mine, theirs = pick(*a, **k), next(left)
        same.append(float((mine == theirs).float().mean()))
        return theirs
    monkeypatch.setattr(T.ops, "pick_pages", given)
    want = _logits(_like(m, "cpu", 4), steps)
    assert len(same) == len(chosen) > 6 and min(same) > 0.5
    assert torch.nn.functional.cosine_similarity(got, want, dim=-1).min() > 0.995


@gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_gpu_engine_with_graphs_and_without(fp8):
    m = _model("cuda", 6, seed=3, fp8=fp8, **GROUPED)
    p = SamplingParams(greedy=True, ignore_eos=True, max_tokens=20)
    outs = []
    for graphs in (True, False):
        e = LLMEngine(m, num_pages=128, page_size=16, max_batch=4, prefill_chunk=128, max_model_len=1024, use_cuda_graphs=graphs)
        outs.append(e.generate(_prompts(33, 700, 5, 170), p))
        assert e.alive and (not graphs or (len(e._graphs) >= 1 and not e._graphs_disabled))
    N.check_status()
    assert outs[0] == outs[1]


@pytest.mark.parametrize("dev", BOTH)
def test_drafts_that_are_taken_back_leave_no_bounds_behind(dev):
    """Prompt-lookup drafts are written, verified and cut off again: bounds stay those of the cache."""
    m = _model(dev, 3, seed=5)
    part, = _prompts(12, seed=5)
    e = LLMEngine(m, num_pages=64, page_size=16, max_batch=2, prefill_chunk=64, max_model_len=512)
    out, stats = generate_speculative(e, (part * 20)[:200], SamplingParams(greedy=True, max_tokens=24, ignore_eos=True))
    assert len(out) == 24 and stats.drafted > stats.accepted
    if dev == "cpu":
        plain = LLMEngine(m, num_pages=64, page_size=16, max_batch=2, prefill_chunk=64, max_model_len=512)
        want = plain.generate([(part * 20)[:200]], SamplingParams(greedy=True, max_tokens=24, ignore_eos=True))[0]
        assert out[0] == want[0]
    else:
        N.check_status()
    from hartsyinference_b200.ops import reference as R
    bounds, keys = m.key_bounds.cpu(), m.kv_cache[:, 0].cpu()
    full = [p for p in range(64) if bounds[0, p, 0, 2 * m.cfg.head_dim] != 0]
    same = [p for p in full if torch.equal(bounds[:, p], R.page_bounds(keys[:, p]))]
    assert len(full) >= 222 // 16 and len(full) - len(same) <= 1          # (the page at hand may be written again)


def test_the_flag_and_refusals():
    config.set_override("attn_pages", 12)
    try:
        m = DecoderModel(C.tiny(head_dim=64), "cpu")
        assert m.attn_pages == 12 and m.kv_bytes_per_page(16) > DecoderModel(C.tiny(head_dim=64), "cpu", attn_pages=0).kv_bytes_per_page(16)
    finally:
        config.set_override("attn_pages", None)
    assert DecoderModel(C.tiny(), "cpu").attn_pages == 0
    for cfg, kw in ((C.tiny(head_dim=32), dict(attn_pages=4)), (C.tiny(head_dim=64), dict(attn_pages=-1)), (C.tiny(head_dim=64), dict(attn_pages=5000)),
                    (C.tiny(head_dim=64), dict(attn_pages=4, kv_dtype="int4")), (C.PRESETS["deepseek-v3"], dict(attn_pages=4))):
        with pytest.raises(ValueError):
            DecoderModel(cfg, "cpu", **kw)
    with pytest.raises(ValueError):
        _model(attn_pages=4).alloc_kv(4, 8)
    m = _model(attn_pages=4)
    m.alloc_kv(4, 16)
    assert m.kv_cache.numel() * 2 + m.key_bounds.numel() == 4 * m.kv_bytes_per_page(16)
