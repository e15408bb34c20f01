"""Models that turn by positions on several axes: the decoder of a vision-language model and its vision tower."""
import pytest
import torch

from hartsyinference_b200 import ops
from hartsyinference_b200.models.llm import config as C
from hartsyinference_b200.models.llm.transformer import DecoderModel, ForwardBatch
from hartsyinference_b200.models.vlm import qwen_vl
from hartsyinference_b200.ops import _native as N

gpu = pytest.mark.gpu


def _batch(dev, tokens, positions3, embeds=None, page=16):
    n = tokens.numel()
    return ForwardBatch(tokens=tokens.int().to(dev), positions=torch.arange(n, dtype=torch.int32, device=dev), slot_mapping=torch.arange(n, device=dev),
                        block_table=torch.arange(-(-n // page), dtype=torch.int32, device=dev)[None], kv_lens=torch.tensor([n], dtype=torch.int32, device=dev),
                        is_decode=False, cu_q=torch.tensor([0, n], dtype=torch.int32, device=dev), max_q_len=n, max_kv_len=n, embeds=embeds,
                        positions3=positions3.to(dev))


def test_heads_are_normed_before_they_turn(tmp_path):
    """Norm weights that differ from channel to channel (as trained ones do) against transformers: hidden states of a picture prompt."""
    tr = pytest.importorskip("transformers")
    if not hasattr(tr, "Qwen3VLForConditionalGeneration"):
        pytest.skip("transformers has no Qwen3-VL")
    from transformers.models.qwen3_vl.configuration_qwen3_vl import Qwen3VLConfig
    from hartsyinference_b200.models.llm.loader import load_llm, save_hf_checkpoint
    cfg = Qwen3VLConfig(
        text_config=dict(vocab_size=320, hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=32,
                         max_position_embeddings=512, rope_parameters={"rope_type": "default", "mrope_section": [6, 5, 5], "mrope_interleaved": True, "rope_theta": 100.0}),
        vision_config=dict(depth=1, hidden_size=64, intermediate_size=96, num_heads=4, out_hidden_size=128, patch_size=16, spatial_merge_size=2,
                           temporal_patch_size=2, num_position_embeddings=16, deepstack_visual_indexes=[]),
        image_token_id=318, vision_start_token_id=317, vision_end_token_id=316, video_token_id=315)
    for c in (cfg, cfg.text_config, cfg.vision_config):
        c._attn_implementation = "eager"
    torch.manual_seed(0)
    hf = tr.Qwen3VLForConditionalGeneration(cfg).eval()
    with torch.no_grad():
        for name, p in hf.named_parameters():
            if "q_norm" in name or "k_norm" in name:
                p.copy_(2.5 * torch.rand_like(p) ** 2 + 0.1)
            elif p.ndim >= 2:
                p.mul_(3.0)
    save_hf_checkpoint(cfg.to_dict(), {k: v.detach().to(torch.bfloat16).contiguous() for k, v in hf.state_dict().items()}, tmp_path / "m")
    hf = hf.to(torch.bfloat16).float()
    llm = load_llm(tmp_path / "m", "cpu")
    ids = torch.randint(0, 300, (40,), generator=torch.Generator().manual_seed(1))
    pos, _ = qwen_vl.mrope_positions([1] * 8 + [318] * 24 + [1] * 8, 318, [(4, 6)])
    with torch.no_grad():
        want = hf.model.language_model(input_ids=ids[None], position_ids=pos[:, None].long()).last_hidden_state[0]
    llm.model.alloc_kv(3, 16)
    got = llm.model.forward_hidden(_batch("cpu", ids, pos)).float()
    # two layers of bf16 activations stay within 0.999 of 32 bits; heads turned before their norm ended at 0.44
    assert torch.nn.functional.cosine_similarity(got, want, dim=-1).min() > 0.998


def _model(dev, kv_dtype="bf16", **kw):
    m = DecoderModel(C.tiny("qwen2.5-0.5b", mrope_section=(12, 10, 10), **kw), dev, kv_dtype=kv_dtype)
    m.random_init(0, std=0.05)
    return m


@gpu
@pytest.mark.parametrize("kv_dtype", ["bf16", "int4"])
@pytest.mark.parametrize("kw", [dict(), dict(mrope_interleaved=True, qk_norm=True)], ids=["sections", "turns"])
def test_gpu_logits_are_those_of_the_cpu(kv_dtype, kw):
    from .test_kv4_model import _twin
    m = _model("cuda", kv_dtype, head_dim=64, **kw)
    cpu = _twin(m, "cpu", kv_dtype)
    ids = torch.randint(0, 512, (46,), generator=torch.Generator().manual_seed(1))
    pos, _ = qwen_vl.mrope_positions([1] * 8 + [318] * 24 + [1] * 14, 318, [(4, 6)])
    outs = []
    for model, dev in ((m, "cuda"), (cpu, "cpu")):
        model.alloc_kv(3, 16)
        outs.append(model.full_logits(model.forward_hidden(_batch(dev, ids, pos))).float().cpu())
    N.check_status()
    assert torch.nn.functional.cosine_similarity(*outs, dim=-1).min().item() > 0.995


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_patches_of_a_tower_turn_by_row_and_column(dev, dtype):
    """Against the rotation written out; 32 bits: angles below 40 off by 40 * 2^-24 < 2^-18, values below 6; bf16: two roundings of values below 8 may part by a step, 2^-5."""
    rows, cols = qwen_vl.merge_block_coords(8, 6, 2)
    inv = 1.0 / (10000.0 ** (torch.arange(0, 36, 2, dtype=torch.float32) / 36))
    qkv = torch.randn(48, 3 * 4 * 72, generator=torch.Generator().manual_seed(0)).to(dtype)
    turns = qwen_vl._Turns(rows, cols, inv, torch.device(dev))
    q, k, v = turns(qkv.to(dev), 4)
    fr = torch.cat([rows[:, None].float() * inv, cols[:, None].float() * inv], -1)
    cos, sin = torch.cat([fr, fr], -1).cos()[:, None], torch.cat([fr, fr], -1).sin()[:, None]
    for got, x in zip((q, k, v), qkv.reshape(48, 3, 4, 72).unbind(1)):
        y = x.float()
        want = x if got is v else (y * cos + torch.cat([-y[..., 36:], y[..., :36]], -1) * sin).to(dtype)
        assert got.dtype == dtype and (got.float().cpu() - want.float()).abs().max() <= (0 if got is v else 2.0 ** -15 if dtype == torch.float32 else 2.0 ** -5)
