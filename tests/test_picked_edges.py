"""Attention over chosen pages where its parts meet."""
import pytest
import torch

from hartsyinference_b200.ops import _native as N

from .test_picked import Batch

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("hq,hkv,d,run,width", [(24, 1, 128, 5, 40), (8, 8, 64, 24, 7), (16, 2, 128, 16, 3)])
def test_many_blocks_one_after_the_other_end_without_a_wait_that_runs_out(hq, hkv, d, run, width, monkeypatch):
    """Some 100000 blocks of the tiles, of which warps come late to their last product now and then: it must not look like one still to come."""
    monkeypatch.setattr(N.lib(), "b200_attn_picked_form", lambda *a: 1)
    b = Batch([run] * 100, [40 * 16 + run] * 100, hq, hkv, d, 16).to("cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    rows = (run * 100 + 100 * (run - 1)) // run
    picked = torch.rand(rows, hkv, 40, generator=g, device="cuda").argsort(-1)[..., :width].sort(-1).values.int().contiguous()
    want = b.attend(picked, run=run)
    for _ in range(1000 // hkv):
        got = b.attend(picked, run=run)
    N.check_status()
    assert torch.equal(got, want)
