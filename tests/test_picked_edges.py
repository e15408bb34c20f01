"""Attention over chosen pages where its parts meet."""
import math
import re
from pathlib import Path

import pytest
import torch

from hartsyinference_b200 import ops
from hartsyinference_b200.ops import _native as N

from .test_picked import Batch, _attention, _close, _some

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


@pytest.mark.parametrize("dev,tiles", [("cpu", 0), pytest.param("cuda", 0, marks=gpu), pytest.param("cuda", 1, marks=gpu)])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 16), (128, 64), (64, 128)])
@pytest.mark.parametrize("times", [1, 2, 5])
def test_many_values_that_are_not_finite_in_pages_named_several_times(dev, tiles, d, page, times, monkeypatch):
    """A run of 128 queries whose own keys all have an infinite value, each in a channel of its own; its own pages are named up to five times, which makes
    up to 880 such keys. Every query has them in the channels of the keys that it sees, and the other channels are those of finite values."""
    if dev == "cuda":
        monkeypatch.setattr(N.lib(), "b200_attn_picked_form", lambda *a: tiles)
    before = 47
    b = Batch([128], [before + 128], 1, 1, d, page)
    last = (before + 127) // page
    own = list(range(before // page, last + 1))
    picked = torch.tensor([[[0] * (before >= page) + own * times + [last + 1, -1]]], dtype=torch.int32)
    want, bound = _attention(b, picked, 128)
    infinite = torch.zeros(128, d, dtype=torch.bool)
    for t in range(128):
        at = before + t
        b.v[b.table[0, at // page].long(), 0, at % page, t % d] = math.inf
        infinite[t:, t % d] = True
    got = b.to(dev).attend(picked.to(dev), run=128).double().cpu()[:, 0]
    assert (got[infinite] == math.inf).all()
    off = (got - want[:, 0]).abs()
    assert (off[~infinite] <= bound[:, 0][~infinite]).all()


@gpu
@pytest.mark.parametrize("tiles", [0, 1])
@pytest.mark.parametrize("hq,hkv,d,page", [(48, 2, 128, 16), (100, 1, 128, 32), (33, 1, 64, 16), (254, 2, 64, 128), (128, 1, 128, 64)])
def test_single_tokens_of_many_heads_on_a_key_head(hq, hkv, d, page, tiles, monkeypatch):
    """Decoded tokens without cu_q by each of the two kernels: sequences of no keys, one key, ends inside a page and on its border."""
    monkeypatch.setattr(N.lib(), "b200_attn_picked_form", lambda *a: tiles)
    b = Batch([1] * 7, [0, 1, page, page + 1, 700, 333, 2 * page - 1], hq, hkv, d, page, seed=hq)
    picked = _some(b, 1, 9)
    want = _attention(b, picked, 1)
    _close(b.to("cuda").attend(picked.cuda(), step=True), want)
    N.check_status()


@gpu
def test_the_rule_decides_for_single_tokens_too(monkeypatch):
    called = []
    for name in ("b200_attn_picked", "b200_attn_picked_tc"):
        monkeypatch.setattr(N.lib(), name, lambda *a, name=name, call=getattr(N.lib(), name): called.append(name) or call(*a))
    for n, group in ((160, 64), (160, 8), (2, 64)):
        b = Batch([1] * n, [40] * n, group, 1, 128, 16).to("cuda")
        b.attend(torch.arange(132, dtype=torch.int32, device="cuda").expand(n, 1, -1).contiguous(), step=True)
    N.check_status()
    assert called == ["b200_attn_picked_tc", "b200_attn_picked", "b200_attn_picked"]


# (a block of this one has 97 KB of shared memory or more, and one that holds TMEM while it waits for the grid before it has 160: they do not meet on a processor)
ALONE = {"kv4_prefill.cu"}


def test_kernels_let_the_next_one_start_only_once_they_hold_their_tmem():
    """A product that starts early takes its TMEM and then waits for the grid before it; a block of that grid which still has to take its own on the same
    processor would wait for the product. So what allocates TMEM triggers behind the allocation."""
    seen = 0
    for path in sorted((Path(ops.__file__).parents[1] / "csrc" / "kernels").glob("*.cu")):
        for body in path.read_text().split("__global__")[1:]:
            alloc = re.search(r"tmem_alloc\(|tcgen05\.alloc", body)
            trigger = re.search(r"^\s*pdl_trigger\(\);", body, re.M)
            if alloc and trigger and path.name not in ALONE:
                seen += 1
                assert trigger.start() > alloc.start(), path.name
    assert seen >= 4


@pytest.mark.parametrize("name", ["attn_picked_tc", "page_pick"])
def test_a_block_whose_wait_ran_out_leaves_nothing_on_its_way(name):
    """(Read from the sources: no wait of a sound block runs out.) Products are waited for before TMEM is given back; whoever sends tiles stays until the last ones
    have been read, and waits for those on their way where somebody has given up."""
    text = (Path(ops.__file__).parents[1] / "csrc" / "kernels" / f"{name}.cu").read_text()
    products, end = re.search(r"tc_commit\(&bars(->|\.)drain\);\s+mbar_wait\(&bars(->|\.)drain, 0, &none\);", text), text.rindex("tmem_dealloc(")
    assert products and products.start() < end
    given_up = text.index("copies on their way land")
    assert text.index("until the last tiles have been read, or somebody gives up") < given_up < end
    assert re.search(r"mbar_wait\([^;]*_full[^;]*&none\)", text[given_up:end])


def test_a_build_with_other_registers_is_refused():
    """Warps that take more registers wait for those that others give back: 4 warps from 128 to 64, 4 from 128 to 192. The launch asks what the kernel was built with."""
    text = (Path(ops.__file__).parents[1] / "csrc" / "kernels" / "attn_picked_tc.cu").read_text()
    held = int(re.search(r"kTpRegisters = (\d+);", text)[1])
    dec, inc = (int(re.search(rf"setmaxnreg\.{x}\.sync\.aligned\.u32 (\d+);", text)[1]) for x in ("dec", "inc"))
    assert dec + inc == 2 * held
    assert text.index("has.numRegs") < text.index("registers != kTpRegisters) return") < text.index("launch_pdl(attn_picked_tc_kernel")


@gpu
@pytest.mark.parametrize("hq,hkv,d,run", [(8, 1, 128, 16), (14, 2, 64, 18), (64, 1, 128, 2)])
def test_many_runs_under_a_table_too_wide_for_the_tiles(hq, hkv, d, run):
    """A table of 40000 columns, of which a sequence uses 180: its scores have no room beside the tiles, and the other kernel chooses the same pages."""
    b = Batch([2800], [2880], hq, hkv, d, 16, seed=run).fill_bounds()
    assert ((sum(b.each) + run - 1) // run) * hkv > 148
    want = b.pick(top=9, run=run)
    narrow = b.to("cuda").pick(top=9, run=run)
    b.table = torch.cat([b.table, torch.full((1, 40000), -1, dtype=torch.int32, device="cuda")], 1)
    assert torch.equal(narrow.cpu(), want) and torch.equal(b.pick(top=9, run=run).cpu(), want)
    N.check_status()
