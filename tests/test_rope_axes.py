"""Rotary positions on several axes against a plain implementation in 64 bits.

Cosines and sines are off by at most 2^-21 (half a turn in 32 bits, rounded, then the functions' own error), norms by 2^-16 of the value (a
sum of up to 256 squares in 32 bits and its root), products and sums by 2^-23: 2^-15 of |a| + |b| in all, and the result is rounded to bf16, 2^-8 of it."""
import pytest
import torch

from hartsyinference_b200 import ops
from hartsyinference_b200.ops import _native as N

gpu = pytest.mark.gpu


def _inputs(t, hq, hkv, d, pairs, n_axes, seed=0, far=131072):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=g)
    pos = torch.randint(0, far, (n_axes, t), generator=g, dtype=torch.int32)
    axes = torch.randint(0, n_axes, (pairs,), generator=g, dtype=torch.int32)
    freq = (1000000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))).float()
    return qkv.to(torch.bfloat16), pos, axes, freq, (1 + 0.2 * torch.randn(2, d, generator=g)).to(torch.bfloat16)


def _plain(qkv, pos, axes, freq, hq, hkv, d, style, norms, eps=1e-6):
    """(q, k, v) and the bound of each, in 64 bits."""
    x = qkv.double().reshape(qkv.shape[0], -1, d)
    pairs = axes.numel()
    out, bound = x.clone(), 2.0 ** -15 * x.abs()
    for a, b, w in ((0, hq, norms[0]), (hq, hq + hkv, norms[1])):
        y = x[:, a:b]
        if w is not None:
            y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        out[:, a:b], bound[:, a:b] = y, 2.0 ** -15 * y.abs()
        for j in range(pairs):
            i, m = (j, j + pairs) if style == 0 else (2 * j, 2 * j + 1)
            angle = pos[axes[j].long()].double()[:, None] * freq[j].double()
            out[:, a:b, i] = y[..., i] * angle.cos() - y[..., m] * angle.sin()
            out[:, a:b, m] = y[..., m] * angle.cos() + y[..., i] * angle.sin()
            bound[:, a:b, i] = bound[:, a:b, m] = 2.0 ** -15 * (y[..., i].abs() + y[..., m].abs())
    bound = bound + 2.0 ** -8 * (out.abs() + bound)
    return [(z[:, a:b], e[:, a:b]) for z, e in ((out, bound),) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv))]


def _close(got, want):
    off = (got.double().cpu() - want[0]).abs()
    assert torch.isfinite(got).all() and (off <= want[1]).all(), float((off / want[1]).max())


SHAPES = [(28, 4, 128, 64), (16, 16, 80, 40), (3, 3, 72, 36), (5, 1, 64, 16), (2, 2, 128, 24), (3, 1, 70, 35), (4, 2, 256, 128), (6, 2, 34, 5), (2, 1, 96, 0), (9, 3, 128, 60)]


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("hq,hkv,d,pairs", SHAPES)
@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("norm", [False, True])
def test_turns_every_pair_by_its_axis(dev, hq, hkv, d, pairs, style, norm):
    for t, n_axes in ((1, 3), (37, 2), (1300, 3)):
        if dev == "cpu" and t > 100:
            continue
        qkv, pos, axes, freq, w = _inputs(t, hq, hkv, d, pairs, n_axes, seed=t + d)
        norms = (w[0], w[1]) if norm else (None, None)
        want = _plain(qkv, pos, axes, freq, hq, hkv, d, style, norms)
        page = 16
        pages = t // page + 2
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(1))
        at = torch.arange(t) + 5
        slots = order[at // page] * page + at % page
        slots[t // 2] = -1
        kc, vc = (torch.full((pages, hkv, page, d), 7.0, dtype=torch.bfloat16, device=dev) for _ in "kv")
        to = lambda x: None if x is None else x.to(dev)
        q, k, v = ops.rope_axes_kv(to(qkv), to(pos), hq, hkv, d, axes=to(axes), inv_freq=to(freq), k_cache=kc, v_cache=vc, slot_mapping=to(slots), style=style,
                                   q_norm_w=to(norms[0]), k_norm_w=to(norms[1]), want_kv=True)
        for got, ref in zip((q, k, v), want):
            _close(got, ref)
        on = slots >= 0
        for cache, dense in ((kc, k), (vc, v)):
            flat = cache.cpu().transpose(1, 2).reshape(-1, hkv, d)
            assert torch.equal(flat[slots[on]], dense.cpu()[on])
            rest = torch.ones(flat.shape[0], dtype=torch.bool)
            rest[slots[on]] = False
            assert (flat[rest] == 7).all()
        if dev == "cuda":
            N.check_status()


def test_sections_one_after_the_other_and_in_turns():
    assert ops.rope_axes((2, 1, 3)).tolist() == [0, 0, 1, 2, 2, 2]
    assert ops.rope_axes((4, 1, 2), interleaved=True).tolist() == [0, 1, 2, 0, 0, 2, 0]
    assert ops.rope_axes((24, 20, 20), interleaved=True).bincount().tolist() == [24, 20, 20]
    with pytest.raises(ValueError):
        ops.rope_axes((1, 3, 3), interleaved=True)
    with pytest.raises(ValueError):
        ops.rope_axes(())


def test_equal_positions_on_all_axes_are_one_axis():
    """Against the op of one axis in 32 bits: positions below 100, angles off by 100 * 2^-24 a frequency, 2^-17, times two values below 6."""
    qkv, pos, axes, freq, _ = _inputs(9, 4, 2, 64, 32, 1, far=100)
    q, k, v = ops.rope_axes_kv(qkv.float(), pos.expand(3, -1), 4, 2, 64, axes=torch.arange(32, dtype=torch.int32) % 3, inv_freq=freq, want_kv=True)
    want = ops.rope_kv(qkv.float(), pos[0], 4, 2, 64, inv_freq=freq, want_kv=True)
    for a, b in zip((q, k, v), want):
        assert (a - b).abs().max() <= 2.0 ** -13


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(dev):
    qkv, pos, axes, freq, w = (x.to(dev) for x in _inputs(4, 4, 2, 64, 32, 3))
    kw = dict(axes=axes, inv_freq=freq)
    cache = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device=dev)
    slots = torch.zeros(4, dtype=torch.int64, device=dev)
    for args, more in (((qkv, pos[0], 4, 2, 64), kw), ((qkv, pos[:, :3], 4, 2, 64), kw), ((qkv, pos, 4, 1, 64), kw), ((qkv, pos, 4, 2, 63), kw),
                       ((qkv, pos, 4, 2, 64), dict(axes=axes.repeat(2), inv_freq=freq.repeat(2))), ((qkv, pos, 4, 2, 64), dict(axes=axes, inv_freq=freq[:3])),
                       ((qkv, pos, 4, 2, 64), dict(kw, style=2)), ((qkv, pos, 4, 2, 64), dict(kw, k_cache=cache)), ((qkv, pos, 4, 2, 64), dict(kw, slot_mapping=slots)),
                       ((qkv, pos, 4, 2, 64), dict(kw, k_cache=cache, v_cache=cache, slot_mapping=slots[:3])),
                       ((qkv, pos, 4, 2, 64), dict(kw, k_cache=cache[:, :1], v_cache=cache, slot_mapping=slots)), ((qkv, pos, 4, 2, 64), dict(kw, q_norm_w=w[0, :10]))):
        with pytest.raises(ValueError):
            ops.rope_axes_kv(*args, **more)
    empty = ops.rope_axes_kv(qkv[:0], pos[:, :0], 4, 2, 64, **kw, want_kv=True)
    assert [x.shape[0] for x in empty] == [0, 0, 0]


@gpu
def test_a_slot_behind_the_pool_and_an_axis_that_is_none_are_reported():
    from hartsyinference_b200.exceptions import DeviceWaitTimeout
    qkv, pos, axes, freq, _ = (x.cuda() for x in _inputs(4, 4, 2, 64, 32, 3))
    kc, vc = (torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    slots = torch.tensor([0, 32, 5, 1 << 40], device="cuda")
    ops.rope_axes_kv(qkv, pos, 4, 2, 64, axes=axes, inv_freq=freq, k_cache=kc, v_cache=vc, slot_mapping=slots)
    with pytest.raises(DeviceWaitTimeout):
        N.check_status()
    assert int(kc.any(-1).sum()) == 4                       # two tokens of two heads
    ops.rope_axes_kv(qkv, pos, 4, 2, 64, axes=axes + 3, inv_freq=freq)
    with pytest.raises(DeviceWaitTimeout):
        N.check_status()


@gpu
def test_views_streams_and_a_captured_call():
    """Rows that begin off a 16-byte boundary, positions that are a transposed view; a captured call follows its inputs."""
    qkv, pos, axes, freq, _ = (x.cuda() for x in _inputs(50, 4, 2, 64, 32, 3))
    kw = dict(axes=axes, inv_freq=freq, want_kv=True)
    want = ops.rope_axes_kv(qkv, pos, 4, 2, 64, **kw)
    wide = torch.zeros(50, 8 * 64 + 1, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:] = qkv
    got = ops.rope_axes_kv(wide[:, 1:], pos.T.contiguous().T, 4, 2, 64, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x, at = qkv.clone(), pos.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = ops.rope_axes_kv(x, at, 4, 2, 64, **kw)
    x.copy_(qkv.flip(0))
    at.copy_(pos.flip(1))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b.flip(0)) for a, b in zip(held, want))
