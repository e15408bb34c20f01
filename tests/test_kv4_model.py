"""Models whose K/V cache is held in 4 bits: the ops of that cache together, as an engine runs them."""
from dataclasses import replace

import pytest
import torch

from hartsyinference_b200 import config, ops
from hartsyinference_b200.engine import LLMEngine, SamplingParams
from hartsyinference_b200.models.llm import config as C
from hartsyinference_b200.models.llm import transformer as T
from hartsyinference_b200.models.llm.transformer import DecoderModel, ForwardBatch
from hartsyinference_b200.ops import _native as N
from hartsyinference_b200.ops import reference as R

gpu = pytest.mark.gpu
PLAIN, GROUPED = dict(), dict(num_heads=8, num_kv_heads=2, head_dim=128, hidden_size=512)
CAPPED, NORMED = dict(attn_softcap=20.0, sliding_window=9, sliding_window_pattern=2), dict(qk_norm=True, rope_dim=32, rope_style=1)


def _model(dev="cpu", kv_dtype="int4", seed=0, base="qwen2.5-0.5b", fp8=False, **kw):
    m = DecoderModel(C.tiny(base, **kw), dev, fp8=fp8, kv_dtype=kv_dtype)
    m.random_init(seed, std=0.05)
    return m


def _twin(m, dev, kv_dtype="int4"):
    """The same weights on another device."""
    def move(x):
        if isinstance(x, torch.Tensor):
            return x.to(dev)
        return ops.LinearWeight(move(x.weight), move(x.scale), move(x.bias)) if isinstance(x, ops.LinearWeight) else x
    t = DecoderModel(m.cfg, dev, fp8=m.fp8, kv_dtype=kv_dtype)
    t.embed, t.final_norm, t.lm_head = move(m.embed), move(m.final_norm), move(m.lm_head)
    t.layers = [replace(lw, **{k: move(v) for k, v in vars(lw).items()}) for lw in m.layers]
    return t


def _step(dev, tokens, first, decode=False, page=16):
    """The tokens first .. of one sequence in pages 3, 2, 1, 0."""
    n = len(tokens)
    table = torch.tensor([[3, 2, 1, 0]], dtype=torch.int32)
    pos = torch.arange(first, first + n)
    return ForwardBatch(tokens=tokens.int().to(dev), positions=pos.int().to(dev), slot_mapping=(table[0, pos // page].long() * page + pos % page).to(dev),
                        block_table=table.to(dev), kv_lens=torch.tensor([first + n], dtype=torch.int32, device=dev), is_decode=decode,
                        cu_q=None if decode else torch.tensor([0, n], dtype=torch.int32, device=dev), max_q_len=n, max_kv_len=first + n)


def _logits(m, steps):
    m.alloc_kv(4, 16)
    return torch.cat([m.full_logits(m.forward_hidden(b)).float().cpu() for b in steps])


def _run(m, dev, tokens):
    """A prompt in two chunks, then a decoded token."""
    return _logits(m, [_step(dev, tokens[:33], 0), _step(dev, tokens[33:45], 33), _step(dev, tokens[45:46], 45, True)])


@pytest.mark.parametrize("kw", [PLAIN, GROUPED, CAPPED, NORMED], ids=["plain", "grouped", "capped", "normed"])
def test_it_is_the_model_with_what_the_cache_stands_for(kw, monkeypatch):
    """With keys and values rounded to what 4 bits hold before they go to the bf16 cache, that cache's model gives the same to the bit."""
    m = _model(**kw)
    tokens = torch.randint(0, m.cfg.vocab_size, (46,), generator=torch.Generator().manual_seed(1))
    got = _run(m, "cpu", tokens)
    assert m.kv_cache.dtype == torch.uint8 and m.kv_cache.numel() == 4 * m.kv_bytes_per_page(16)
    two = _twin(m, "cpu", "bf16")
    assert 16 * 2 * m.kv_bytes_per_page(16) == 17 * two.kv_bytes_per_page(16) // 2

    def rope_kv(qkv, positions, hq, hkv, d, k_cache=None, v_cache=None, slot_mapping=None, **k):
        q, key, val = ops.rope_kv4(qkv, positions, hq, hkv, d, want_kv=True, **k)
        for cache, x in ((k_cache, key), (v_cache, val)):
            cache[slot_mapping // 16, :, slot_mapping % 16] = x
        return q, None, None

    monkeypatch.setattr(T.ops, "rope_kv", rope_kv)
    assert torch.equal(_run(two, "cpu", tokens), got)


def test_chunks_and_batches_do_not_change_tokens():
    m = _model(seed=2)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (90, 5, 17)]
    p = SamplingParams(greedy=True, max_tokens=4, ignore_eos=True)
    engine = lambda chunk: LLMEngine(m, num_pages=64, page_size=16, max_batch=4, prefill_chunk=chunk, max_model_len=256)
    want = [engine(256).generate([x], p)[0] for x in prompts]
    assert engine(32).generate(prompts, p) == want


def test_the_flag_and_refusals():
    config.set_override("kv_dtype", "int4")
    try:
        assert DecoderModel(C.tiny(), "cpu").kv_dtype == "int4"
    finally:
        config.set_override("kv_dtype", None)
    assert DecoderModel(C.tiny(), "cpu").kv_dtype == "bf16"
    for cfg, kv in ((C.tiny(), "int8"), (C.tiny(head_dim=32), "int4"), (C.PRESETS["deepseek-v3"], "int4")):
        with pytest.raises(ValueError):
            DecoderModel(cfg, "cpu", kv_dtype=kv)
    with pytest.raises(ValueError):
        _model().alloc_kv(4, 8)


def _biased_case(dev):
    lens, each, hq, hkv, d = [40, 0, 9], [5, 0, 9], 8, 2, 64
    g = torch.Generator().manual_seed(4)
    cache, table = ops.kv4_cache(5, hkv, 16, d, "cpu"), torch.tensor([[4, 0, 2], [-1, -1, -1], [1, -1, -1]], dtype=torch.int32)
    k, v = (torch.randn(5 * 16, hkv, d, generator=g) for _ in range(2))
    R.kv4_store(cache, torch.arange(80), k, v)
    dense = [torch.zeros(5, hkv, 16, d, dtype=torch.bfloat16) for _ in range(2)]
    for x, y in zip(dense, R.kv4_sequence(cache, torch.arange(5), 80)):
        x.copy_(y.view(5, 16, hkv, d).permute(0, 2, 1, 3))
    q = torch.randn(14, hq, d, generator=g).to(torch.bfloat16)
    move = lambda *t: [x.to(dev) for x in t]
    return move(cache, *dense, table, torch.tensor(lens, dtype=torch.int32), q, torch.tensor([0, 5, 5, 14], dtype=torch.int32), torch.randn(hq, generator=g))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("which", ["alibi", "sinks"])
def test_biased_attention_reads_the_cache_back(dev, which):
    cache, k, v, table, lens, q, cu, bias = _biased_case(dev)
    kw = {which: bias, "window": 7}
    got = ops.attn_biased_kv4(q, cache, table, lens, cu, **kw)
    assert torch.equal(got, ops.attn_paged_biased(q, k, v, table, lens, cu, **kw))
    one = lens.clamp(min=1)
    assert torch.equal(ops.attn_biased_kv4(q[:3], cache, table.clamp(min=0), one, None, **kw), ops.attn_paged_biased(q[:3], k, v, table.clamp(min=0), one, None, **kw))


@gpu
@pytest.mark.parametrize("kw", [PLAIN, GROUPED, CAPPED, NORMED, dict(fp8=True, head_dim=128, hidden_size=512)],
                         ids=["plain", "grouped", "capped", "normed", "fp8"])
def test_gpu_logits_are_those_of_the_cpu(kw):
    """As of the bf16 cache's model; a code may differ where a key is on the edge between two, so logits agree to a fraction of a code."""
    m = _model("cuda", **kw)
    tokens = torch.randint(0, m.cfg.vocab_size, (46,), generator=torch.Generator().manual_seed(1))
    got, want = _run(m, "cuda", tokens), _run(_twin(m, "cpu"), "cpu", tokens)
    N.check_status()
    assert torch.nn.functional.cosine_similarity(got, want, dim=-1).min().item() > (0.98 if m.fp8 else 0.995)


@gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_gpu_engine_with_graphs_and_without(fp8):
    """Captured decode steps and eager ones give the same tokens, with prompts in chunks and lengths that cross pages."""
    m = _model("cuda", seed=3, fp8=fp8, **GROUPED)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (33, 700, 5, 17)]
    p = SamplingParams(greedy=True, ignore_eos=True, max_tokens=20)
    outs = []
    for graphs in (True, False):
        e = LLMEngine(m, num_pages=128, page_size=16, max_batch=4, prefill_chunk=128, max_model_len=1024, use_cuda_graphs=graphs)
        outs.append(e.generate(prompts, p))
        assert e.alive and (not graphs or (len(e._graphs) >= 1 and not e._graphs_disabled))
    N.check_status()
    assert outs[0] == outs[1]


def _drafted(dev, n, **kw):
    from hartsyinference_b200.engine.speculative import generate_speculative
    m = _model(dev, seed=5, **kw)
    part = torch.randint(0, 512, (12,), generator=torch.Generator().manual_seed(5)).tolist()
    p = SamplingParams(greedy=True, max_tokens=24, ignore_eos=True)
    engine = lambda: LLMEngine(m, num_pages=96, page_size=16, max_batch=2, prefill_chunk=256, max_model_len=1024)
    prompt = (part * (n // 12 + 1))[:n]
    return (m, prompt, *generate_speculative(engine(), prompt, p), engine().generate([prompt], p)[0])


def test_drafts_are_verified_over_the_cache():
    """Every kept token is the greedy one of a pass over the whole sequence where that decision is no near tie: logits are bf16 numbers below 4, whose
    steps are 2^-6; a step of each of two logits, and of the two ways that hidden states of as many tokens round, are within 0.07."""
    m, prompt, out, stats, plain = _drafted("cpu", 100)
    assert len(out) == len(plain) == 24 and stats.drafted > 0
    for got in (out, plain):
        tokens = torch.tensor(prompt + got)
        m.alloc_kv(8, 16)
        table = torch.arange(8, dtype=torch.int32)[None]
        n = len(tokens)
        rows = m.full_logits(m.forward_hidden(ForwardBatch(
            tokens=tokens.int(), positions=torch.arange(n, dtype=torch.int32), slot_mapping=torch.arange(n), block_table=table, is_decode=False,
            kv_lens=torch.tensor([n], dtype=torch.int32), cu_q=torch.tensor([0, n], dtype=torch.int32), max_q_len=n, max_kv_len=n))).float()[99:-1]
        assert rows.abs().max() < 4
        assert (rows.gather(1, tokens[100:, None])[:, 0] >= rows.amax(1) - 0.07).all()


@gpu
def test_gpu_drafts_are_verified_over_a_long_cache():
    """Passes of up to nine tokens behind 700 others: the kernel that cuts the key axis. Tokens of plain decoding may differ at near ties."""
    assert N.lib().b200_attn_kv4_choice(1, 9, 709, 8, 2, 128, 1, 0, 0.088) == 2
    _, _, out, stats, plain = _drafted("cuda", 700, **GROUPED)
    N.check_status()
    assert len(out) == len(plain) == 24 and stats.drafted > 0 and out[0] == plain[0]


@gpu
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("heads", [dict(), dict(num_heads=16, num_kv_heads=8)], ids=["2", "8"])
def test_gpu_engine_decodes_short_sequences_under_a_long_limit(graphs, heads):
    """An engine for 8192 tokens and a prompt of 17: the tables that decode steps get are as wide as the limit. Logits are those of one pass on the
    CPU to the fraction that two devices' models agree to above."""
    m = _model("cuda", seed=3, **GROUPED | heads)
    tokens = torch.randint(0, 512, (29,), generator=torch.Generator().manual_seed(6))
    e = LLMEngine(m, num_pages=600, page_size=16, max_batch=2, prefill_chunk=128, max_model_len=8192, use_cuda_graphs=graphs)
    stale = [torch.full((n,), float("nan"), device="cuda") for n in (1 << 12, 1 << 14, 1 << 16, 1 << 17, 1 << 18) for _ in range(4)]
    del stale
    got = [e.replay([("a", tokens[:17].tolist(), [16])])]
    got += [e.replay([("a", [x], [0])]) for x in tokens[17:].tolist()]
    assert not graphs or (e._graphs and not e._graphs_disabled)
    N.check_status()
    cpu = _twin(m, "cpu")
    want = _logits(cpu, [_step("cpu", tokens, 0)])[16:]
    assert torch.nn.functional.cosine_similarity(torch.cat(got).cpu(), want, dim=-1).min().item() > 0.995
