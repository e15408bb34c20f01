"""Models that attend over chosen pages: what does not depend on the rest of a batch."""
import pytest
import torch

from hartsyinference_b200 import ops
from hartsyinference_b200.engine import LLMEngine, SamplingParams
from hartsyinference_b200.engine.speculative import generate_speculative
from hartsyinference_b200.models.llm import transformer as T
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
