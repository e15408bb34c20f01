"""Rotary positions on several axes: calls that a model takes in other forms."""
import re
from pathlib import Path

import pytest
import torch

from hartsyinference_b200.models.vlm import qwen_vl
from hartsyinference_b200.ops import _native as N

from .test_rope_axes_model import _batch, _model

gpu = pytest.mark.gpu


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("kv_dtype", ["bf16", "int4"])
def test_a_models_positions_are_whole_numbers_of_any_type_on_any_device(dev, kv_dtype):
    m = _model(dev, kv_dtype, head_dim=64, qk_norm=True)
    ids = torch.randint(0, 512, (46,), generator=torch.Generator().manual_seed(1))
    pos, _ = qwen_vl.mrope_positions([1] * 8 + [318] * 24 + [1] * 14, 318, [(4, 6)])
    outs = []
    for dtype in (torch.int32, torch.int64, torch.int16):
        for where in {"cpu", dev}:
            m.alloc_kv(3, 16)
            b = _batch(dev, ids, pos)
            b.positions3 = pos.to(dtype).to(where)
            outs.append(m.forward_hidden(b))
    assert all(torch.equal(x, outs[0]) for x in outs)
    if dev == "cuda":
        N.check_status()


@pytest.mark.parametrize("name", ["rope_axes", "page_pick", "attn_picked", "attn_picked_tc"])
def test_rules_ask_how_many_processors_there_are(name):
    text = (Path(qwen_vl.__file__).parents[2] / "csrc" / "kernels" / f"{name}.cu").read_text()
    code = "\n".join(line.split("//")[0] for line in text.splitlines())
    assert not re.search(r"\b148\b", code)
