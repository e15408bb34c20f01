"""The 4-bit K/V cache: its format, the rotation that stores it, reading it back, and attention over it.

The format and the CPU statements are tested everywhere; the kernels (``gpu``) against a plain implementation in 64 bits, element by element.
A block's scale is max|x| / 7 rounded to 3 bits of mantissa, a code is the nearest multiple of it, so a value is held
within half a scale (largest code: max|x| / s is at most 7 * 17 / 16 = 7.44, which is held as 7)."""
import math

import pytest
import torch

from hartsyinference_b200 import ops
from hartsyinference_b200.ops import reference as R

gpu = pytest.mark.gpu
HEADS = [(14, 2, 64), (8, 1, 128), (3, 3, 64), (40, 2, 128), (28, 4, 128), (33, 1, 64)]


def _normal(*shape, seed=0, dev="cpu"):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dev)


def _values(seed, t, hkv, d):
    """Rows with channels that stand out, blocks of zeros, a block far smaller than its neighbours."""
    x = _normal(t, hkv, d, seed=seed)
    x[..., 3] *= 50
    x[0, 0, 32:64] = 0
    x[t // 2, -1, :32] *= 1e-6
    return x.to(torch.bfloat16).float()


def _tables(lens, page, seed=3, spare=2):
    """Shuffled pages; table entries behind a sequence's last page name none."""
    per = [-(-n // page) for n in lens]
    order = torch.randperm(sum(per) + spare, generator=torch.Generator().manual_seed(seed)).int()
    table, at = torch.full((len(lens), max(max(per), 1) + 1), -7, dtype=torch.int32), 0
    for i, p in enumerate(per):
        table[i, :p] = order[at:at + p]
        at += p
    return table, sum(per) + spare


def _filled(lens, hkv, d, page, seed=0, fill=0xFF):
    """A pool whose unused bytes are all ones (scales that are not numbers), with sequences in it."""
    table, pages = _tables(lens, page)
    cache = ops.kv4_cache(pages, hkv, page, d, "cpu").fill_(fill)
    for i, n in enumerate(lens):
        if n:
            pos = torch.arange(n)
            R.kv4_store(cache, table[i, pos // page].long() * page + pos % page, _values(seed + 2 * i, n, hkv, d), _values(seed + 2 * i + 1, n, hkv, d))
    return cache, table


def _value_scales(cache, table, n):
    """The scale of every value of a sequence, [n, hkv, d] in 64 bits."""
    d = 2 * cache.shape[-1] // 17
    rows = cache[table[:-(-n // (cache.shape[2] * 16))].long()][:, :, :, 1, 8 * d:].unflatten(-1, (16, d // 32))
    return R.kv4_scales(rows, R.KV4_VALUE_EXP).double().permute(0, 2, 3, 1, 4).reshape(-1, cache.shape[1], d // 32)[:n].repeat_interleave(32, -1)


def _plain(q, cache, table, lens, cuts, causal=True, scale=None, softcap=0.0, window=0):
    """Attention in 64 bits: (out, sum of p |v|, sum of p times v's scale)."""
    hq, d = q.shape[1:]
    out, size, scales = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(3))
    for i, n in enumerate(lens):
        a, b = cuts[i], cuts[i + 1]
        if not n or a == b:
            continue
        k, v = (x.double() for x in R.kv4_sequence(cache, table[i], n))
        k, v, c = (x.repeat_interleave(hq // x.shape[1], 1) for x in (k, v, _value_scales(cache, table[i], n)))
        s = torch.einsum("qhd,khd->hqk", q[a:b].double(), k) * (1 / math.sqrt(d) if scale is None else scale)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        pos, key = torch.arange(n - (b - a), n)[:, None], torch.arange(n)[None]
        seen = (key <= pos) if causal else torch.ones(b - a, n, dtype=torch.bool)
        if window > 0:
            seen = seen & (key > pos - window)
        p = torch.nan_to_num(torch.softmax(s.masked_fill(~seen, -math.inf), -1))
        out[a:b], size[a:b], scales[a:b] = (torch.einsum("hqk,khd->qhd", p, x) for x in (v, v.abs(), c))
    return out, size, scales


def _close(got, want, size, scales):
    """A rounding to bf16 (8 bits, the first of them 1) is off by at most half of the last one, 2^-8 of the value. Probabilities are rounded before and
    after the product with a scale: twice 2^-8 of sum p |v|. The result is: 2^-8 of it. Scores are sums of 128 products in 32 bits, of
    which sum |q k| scale is below 2^9 here: off by less than 2^9 * 2^-24 * 2 * 2^3 = 2^-11, and so are probabilities and their sum.
    Values enter as 128 + code, and 136 is taken off again, 16 keys at a time: two sums of at most 143 p s that are cut to 24 bits,
    2 * 2^-22 * 143 < 2^-13 of sum p s with two bits to spare."""
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    bound = 2.0 ** -7 * size + 2.0 ** -8 * want.abs() + 2.0 ** -10 * size + 2.0 ** -13 * scales + 1e-30
    assert (off <= bound).all(), float((off / bound).max())


# ------------------------------------------------------------------------------------------ format (CPU)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("values", [False, True])
def test_every_nibble_of_a_row_has_one_value(d, values):
    places = R.kv4_places(d, values)
    assert places.shape == (16, d) and (places.sort(-1).values == torch.arange(d)).all()


@pytest.mark.parametrize("exp", [R.KV4_KEY_EXP, R.KV4_VALUE_EXP])
def test_values_are_held_within_half_a_scale(exp):
    x = _values(1, 50, 2, 128) * 2.0 ** -3
    code, byte = R.kv4_blocks(x, exp)
    s = R.kv4_scales(byte, exp)
    assert code.min() >= 1 and code.max() <= 15 and byte.min() >= 8 and byte.max() <= 247
    top = x.unflatten(-1, (-1, 32)).abs().amax(-1) / 7
    normal = top >= 2.0 ** (exp - 14)
    assert ((s - top).abs()[normal] <= top[normal] / 16).all()                    # half a step of 3 bits of mantissa
    held = R.kv4_held(x, exp)
    assert ((held - x).abs().unflatten(-1, (-1, 32)) <= 0.5 * s[..., None]).all()
    assert torch.equal(held, held.to(torch.bfloat16).float())                      # a code times a scale is exact in bf16
    assert torch.equal(R.kv4_held(held, exp).abs().unflatten(-1, (-1, 32)).amax(-1) > 0, held.abs().unflatten(-1, (-1, 32)).amax(-1) > 0)


def test_what_is_no_number_and_what_is_too_large():
    x = torch.zeros(1, 1, 64)
    x[0, 0, 0], x[0, 0, 1], x[0, 0, 40] = math.nan, 3.5, math.inf
    held = R.kv4_held(x, R.KV4_KEY_EXP)[0, 0]
    assert held[0] == 0 and held[1] == 3.5 and held[40] == 6720 and held[41] == 0
    assert R.kv4_held(torch.full((32,), 1e30), R.KV4_VALUE_EXP).eq(420).all() and R.kv4_held(torch.full((32,), -6720.0), R.KV4_KEY_EXP).eq(-6720).all()


@pytest.mark.parametrize("d,page", [(64, 16), (128, 32), (128, 128)])
def test_store_and_read_back(d, page):
    lens = [1, 17, 0, 150]
    cache, table = _filled(lens, 2, d, page, seed=4)
    for i, n in enumerate(lens):
        k, v = R.kv4_sequence(cache, table[i], n)
        assert k.shape == (n, 2, d)
        if n:
            assert torch.equal(k, R.kv4_held(_values(4 + 2 * i, n, 2, d), R.KV4_KEY_EXP)) and torch.equal(v, R.kv4_held(_values(5 + 2 * i, n, 2, d), R.KV4_VALUE_EXP))
    cu = torch.tensor([0, 1, 18, 18, 168], dtype=torch.int32)
    k, v = ops.kv4_gather(cache, table, cu, 168)
    assert torch.equal(k[1:18].float(), R.kv4_sequence(cache, table[1], 17)[0]) and torch.equal(v[18:].float(), R.kv4_sequence(cache, table[3], 150)[1])


def _qkv_args(t, hq, hkv, d, page=16, seed=0):
    pages = -(-t // page) + 1
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(seed))[:t]
    if t > 2:
        slots[1] = -1
    return (_normal(t, (hq + 2 * hkv) * d, seed=seed).to(torch.bfloat16), torch.randint(0, 200000, (t,), generator=torch.Generator().manual_seed(seed + 1), dtype=torch.int32),
            ops.kv4_cache(pages, hkv, page, d, "cpu"), slots)


def test_rope_kv4_on_cpu_is_the_rotation_of_the_bf16_cache_in_blocks():
    """At positions that 32-bit angles take well, queries are those of the bf16 form and the cache holds its keys and values."""
    qkv, _, cache, slots = _qkv_args(20, 6, 2, 64)
    pos = torch.arange(20, dtype=torch.int32)
    q, k, v = ops.rope_kv4(qkv, pos, 6, 2, 64, cache=cache, slot_mapping=slots, want_kv=True)
    q2, k2, v2 = ops.rope_kv(qkv, pos, 6, 2, 64, want_kv=True)
    assert (q.float() - q2.float()).abs().max() <= 2.0 ** -7 * q2.abs().max()
    # keys: half a scale of code rounding, and a bf16 rounding of k2
    s = k2.float().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True) / 7 * 17 / 16
    assert ((k.float() - k2.float()).unflatten(-1, (-1, 32)).abs() <= 0.5 * s * 1.01 + 2.0 ** -8 * k2.float().abs().unflatten(-1, (-1, 32))).all()
    assert torch.equal(v.float(), R.kv4_held(v2, R.KV4_VALUE_EXP))


def test_refusals():
    qkv, pos, cache, slots = _qkv_args(4, 4, 2, 64)
    ok = dict(cache=cache, slot_mapping=slots)
    for bad in (lambda: ops.rope_kv4(qkv[:, :-1], pos, 4, 2, 64, **ok), lambda: ops.rope_kv4(qkv, pos, 4, 2, 64, rot=66, **ok),
                lambda: ops.rope_kv4(qkv, pos, 4, 2, 64, rot=7, **ok), lambda: ops.rope_kv4(qkv, pos, 4, 2, 64, style=2, **ok),
                lambda: ops.rope_kv4(qkv, pos[:3], 4, 2, 64, **ok), lambda: ops.rope_kv4(qkv, pos, 4, 2, 64, cache=cache, slot_mapping=slots[:2]),
                lambda: ops.rope_kv4(qkv, pos, 4, 2, 64, slot_mapping=slots), lambda: ops.rope_kv4(qkv, pos, 2, 3, 64, **ok),
                lambda: ops.rope_kv4(qkv, pos, 4, 2, 64, inv_freq=torch.ones(31), **ok), lambda: ops.rope_kv4(qkv, pos, 4, 2, 64, q_norm_w=torch.ones(32), **ok),
                lambda: ops.rope_kv4(qkv, pos, 4, 2, 64, cache=cache.float(), slot_mapping=slots),
                lambda: ops.rope_kv4(qkv, pos, 4, 2, 64, cache=cache.transpose(0, 1), slot_mapping=slots),
                lambda: ops.kv4_cache(4, 2, 8, 64, "cpu"), lambda: ops.kv4_cache(4, 2, 24, 64, "cpu"), lambda: ops.kv4_cache(4, 2, 16, 96, "cpu"), lambda: ops.kv4_cache(4, 2, 16, 256, "cpu")):
        with pytest.raises(ValueError):
            bad()
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    for bad in (lambda: ops.attn_decode_kv4(q[:, :3], cache, table, lens), lambda: ops.attn_decode_kv4(q, cache, table[:1], lens), lambda: ops.attn_decode_kv4(q[:1], cache, table, lens),
                lambda: ops.attn_decode_kv4(q.reshape(2, -1), cache, table, lens), lambda: ops.attn_decode_kv4(torch.zeros(2, 2, 128), cache, table, lens),
                lambda: ops.attn_decode_kv4(q, cache[:, :, 0], table, lens), lambda: ops.attn_prefill_kv4(q, cache, table, lens, cu[:2], 1),
                lambda: ops.attn_prefill_kv4(q, cache, table, lens[:1], cu, 1), lambda: ops.kv4_gather(cache, table, cu[:2], 1), lambda: ops.kv4_gather(cache, table[0], cu, 1)):
        with pytest.raises(ValueError):
            bad()


def test_entry_points_refuse_sizes_before_any_launch():
    """The C entry points themselves: no device is needed, since nothing is launched."""
    from hartsyinference_b200.ops import _native as N
    if not N.available():
        pytest.skip("kernels library not built")
    L, p = N.lib(), 4096
    assert L.b200_rope_kv4(p, p, p, None, None, p, p, None, None, p, 1, 4, 2, 96, 64, 0, 16, 4, 1e-6, None, 0, 0, None, None, None) == -2
    assert L.b200_rope_kv4(p, p, p, None, None, p, p, None, None, p, 1, 4, 2, 64, 64, 0, 24, 4, 1e-6, None, 0, 0, None, None, None) == -2
    assert L.b200_rope_kv4(p, p, p + 8, None, None, p, p, None, None, p, 1, 4, 2, 64, 64, 0, 16, 4, 1e-6, None, 0, 0, None, None, None) == -2
    assert L.b200_rope_kv4(p, p, p, None, None, p, p, None, None, p, 1, 4, 2, 64, 66, 0, 16, 4, 1e-6, None, 0, 0, None, None, None) == -3
    assert L.b200_rope_kv4(p, p, p, None, None, p, p, None, None, None, 1, 4, 2, 64, 64, 0, 16, 4, 1e-6, None, 0, 0, None, None, None) == -3
    assert L.b200_rope_kv4(p + 2, p, p, None, None, p, p, None, None, p, 1, 4, 2, 64, 64, 0, 16, 4, 1e-6, None, 0, 0, None, None, None) == -4
    assert L.b200_kv4_gather(p, p, p, p, p, 1, 1, 2, 64, 8, 1, 1, None, None) == -2
    assert L.b200_kv4_gather(p, p, p, p, p + 2, 1, 1, 2, 64, 16, 1, 1, None, None) == -4
    assert L.b200_attn_kv4(p, p, p, p, p, None, 1, 1, 5, 2, 64, 16, 1, 1, 1, 0, 1.0, 0.0, None, None) == -2
    assert L.b200_attn_kv4(p, p, p, p, p, None, 70000, 1, 4, 2, 64, 16, 1, 1, 1, 0, 1.0, 0.0, None, None) == -3
    assert L.b200_attn_kv4(p, p, p + 8, p, p, None, 1, 1, 4, 2, 64, 16, 1, 1, 1, 0, 1.0, 0.0, None, None) == -4
    assert L.b200_attn_kv4(p, p, p, p, p, None, 1, 1 << 29, 8, 2, 64, 16, 1, 1, 1, 0, 1.0, 0.0, None, None) == -3
    assert L.b200_attn_prefill_kv4(p, p, p, p, p, p, 1, 1, 5, 2, 128, 16, 1, 1, 1, 0, 1.0, 0.0, None, None) == -2
    assert L.b200_attn_prefill_kv4(p, p, p, p, p, p, 70000, 1, 4, 2, 128, 16, 1, 1, 1, 0, 1.0, 0.0, None, None) == -3
    assert L.b200_attn_prefill_kv4(p + 4, p, p, p, p, p, 1, 1, 4, 2, 128, 16, 1, 1, 1, 0, 1.0, 0.0, None, None) == -4
    assert L.b200_attn_prefill_kv4(p, p, p, p, p, p, 1, 1, 4, 2, 64, 16, 1, 1, 1, 0, -1.0, 0.0, None, None) == -5
    assert L.b200_attn_decode_kv4(p, p, p, p, p, 1, 5, 2, 64, 16, 1, 1, 16, 0, 1.0, 0.0, None, 0, None, None) == -2
    assert L.b200_attn_decode_kv4(p, p, p, p, p, 1, 4, 2, 64, 16, 0, 1, 16, 0, 1.0, 0.0, None, 0, None, None) == -2
    assert L.b200_attn_decode_kv4(p, p, p, p, p, 200, 4, 2, 64, 128, 1 << 21, 1, 16, 0, 1.0, 0.0, None, 0, None, None) == -3
    assert L.b200_attn_decode_kv4(p, p, p + 8, p, p, 1, 4, 2, 64, 16, 1, 1, 16, 0, 1.0, 0.0, None, 0, None, None) == -4
    assert L.b200_attn_few_kv4(p, p, p, p, p, None, 1, 2, 4, 2, 64, 16, 1, 1, 16, 0, 1.0, 0.0, None, 0, None, None) == -2
    assert L.b200_attn_few_kv4(p, p, p, p, p, p, 1, 2, 4, 2, 64, 16, 1, 1, 16, 0, 1.0, 0.0, None, 0, None, None) == -6


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 1, 128)])
def test_attention_on_cpu(hq, hkv, d):
    lens, each = [9, 0, 40], [4, 1, 40]
    cache, table = _filled(lens, hkv, d, 16)
    cuts = [0, 4, 5, 45]
    q = _normal(45, hq, d, seed=8).to(torch.bfloat16)
    args = (q, cache, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(cuts, dtype=torch.int32), max(each))
    _close(ops.attn_prefill_kv4(*args, causal=False, window=5), *_plain(q, cache, table, lens, cuts, causal=False, window=5))
    got = ops.attn_prefill_kv4(*args, window=7, softcap=20.0)
    want = _plain(q, cache, table, lens, cuts, window=7, softcap=20.0)
    _close(got, *want)


# ------------------------------------------------------------------------------------------ kernels
def _cuda(*ts):
    return [t.cuda() for t in ts]


@gpu
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("t,rot,style,norm,page", [(1, None, 0, False, 16), (5, 32, 0, True, 16), (37, None, 1, True, 32), (150, 20, 0, False, 128), (1301, None, 0, False, 16),
                                                   (1200, 48, 1, True, 64), (33, 0, 0, True, 16)])
def test_rope_kv4_kernel(hq, hkv, d, t, rot, style, norm, page):
    """Sums are in 64 bits and roundings fixed, so the cache is that of the CPU statement, byte for byte."""
    qkv, pos, cache, slots = _qkv_args(t, hq, hkv, d, page, seed=t)
    w = [(1 + 0.2 * _normal(d, seed=i)).to(torch.bfloat16) if norm else None for i in (5, 6)]
    kw = dict(rot=rot, style=style, theta=500000.0, eps=1e-5, want_kv=True)
    want = ops.rope_kv4(qkv, pos, hq, hkv, d, cache=cache, slot_mapping=slots, q_norm_w=w[0], k_norm_w=w[1], **kw)
    inv = None if rot == 0 else R.rope_inv_freq(d if rot is None else rot, 500000.0).cuda()
    mine = torch.zeros_like(cache, device="cuda")
    got = ops.rope_kv4(qkv.cuda(), pos.cuda(), hq, hkv, d, cache=mine, slot_mapping=slots.cuda(), inv_freq=inv, q_norm_w=None if w[0] is None else w[0].cuda(),
                       k_norm_w=None if w[1] is None else w[1].cuda(), **kw)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    assert torch.equal(mine.cpu(), cache)


@gpu
def test_rope_kv4_leaves_other_slots_and_reports_slots_outside_the_pool():
    from hartsyinference_b200.exceptions import DeviceWaitTimeout
    from hartsyinference_b200.ops import _native as N
    qkv, pos, cache, _ = _qkv_args(6, 4, 2, 64)
    cache.random_(0, 256, generator=torch.Generator().manual_seed(1))
    slots = torch.tensor([3, -1, 17, -5, cache.shape[0] * 16, 1 << 40])
    want = cache.clone()
    ops.rope_kv4(qkv, pos, 4, 2, 64, cache=want, slot_mapping=slots)
    mine = cache.cuda()
    N.check_status()
    ops.rope_kv4(qkv.cuda(), pos.cuda(), 4, 2, 64, cache=mine, slot_mapping=slots.cuda())
    assert torch.equal(mine.cpu(), want)
    with pytest.raises(DeviceWaitTimeout):
        N.check_status()


@gpu
def test_rope_kv4_takes_unsummed_ranges():
    from hartsyinference_b200.ops.core import LinearWeight, SplitSum
    hq, hkv, d = 32, 8, 128
    x, w = _normal(8, 4096, seed=1).to(torch.bfloat16).cuda(), (_normal((hq + 2 * hkv) * d, 4096, seed=2) / 64).to(torch.bfloat16).cuda()
    bias = _normal((hq + 2 * hkv) * d, seed=3).to(torch.bfloat16).cuda()
    part = ops.linear(x, LinearWeight(w, bias=bias), defer=True, defer_bias=True)
    if not isinstance(part, SplitSum):
        pytest.skip("this product is not cut along K")
    pos, slots = torch.arange(8, dtype=torch.int32, device="cuda") * 1000, torch.arange(8, device="cuda")
    rows = ops.rope_kv4(part, pos, hq, hkv, d, rot=0, want_kv=False)[0]                 # the sums, as the kernel reads them
    a, b = ops.kv4_cache(1, hkv, 16, d), ops.kv4_cache(1, hkv, 16, d)
    q1, k1, v1 = ops.rope_kv4(part, pos, hq, hkv, d, cache=a, slot_mapping=slots, want_kv=True)
    full = ops.linear(x, LinearWeight(w, bias=bias))
    assert (rows.reshape(8, -1).float() - full[:, :hq * d].float()).abs().max() <= 2.0 ** -6 * full.float().abs().max()
    q2, k2, v2 = ops.rope_kv4(full, pos, hq, hkv, d, cache=b, slot_mapping=slots, want_kv=True)
    for u, y in ((q1, q2), (k1, k2), (v1, v2)):
        assert ((u.float() - y.float()).norm() / y.float().norm()) < 0.05             # a bf16 step more or less may move a code


@gpu
@pytest.mark.parametrize("hkv,d,page", [(2, 64, 16), (8, 128, 32), (1, 128, 128), (3, 64, 64)])
def test_gather_kernel(hkv, d, page):
    lens = [1, 0, 33, 1000, 16, 0]
    cache, table = _filled(lens, hkv, d, page)
    cu = torch.tensor([0, *lens]).cumsum(0).int()
    want = ops.kv4_gather(cache, table, cu, sum(lens))
    got = ops.kv4_gather(*_cuda(cache, table, cu), sum(lens))
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


CASES = [dict(), dict(window=1), dict(window=17), dict(softcap=15.0), dict(window=300, softcap=30.0), dict(scale=0.3)]


@gpu
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("kw", CASES)
@pytest.mark.parametrize("page", [16, 64])
def test_decode_kernel(hq, hkv, d, kw, page):
    lens = [1, 0, 15, 16, 17, 64, 65, 400, 1777]
    cache, table = _filled(lens, hkv, d, page)
    q = _normal(len(lens), hq, d, seed=9).to(torch.bfloat16)
    want = _plain(q, cache, table, lens, list(range(len(lens) + 1)), **kw)
    dev = _cuda(q, cache, table, torch.tensor(lens, dtype=torch.int32))
    got = ops.attn_decode_kv4(*dev, **kw)
    _close(got, *want)
    for most in (max(lens), 40000):                                                    # how the work is cut
        _close(ops.attn_decode_kv4(*dev, max_kv_len=most, **kw), *want)
    assert torch.equal(got, ops.attn_decode_kv4(*dev, **kw))


@gpu
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("kw", CASES + [dict(causal=False), dict(causal=False, window=17)])
def test_prefill_kernel(hq, hkv, d, kw):
    """Chunks behind nothing and behind a prefix, one token, none, and more queries than keys (the first see nothing)."""
    lens, each = [100, 0, 70, 333, 1, 200, 5], [100, 0, 3, 130, 1, 64, 9]
    cache, table = _filled(lens, hkv, d, 16)
    cuts = torch.tensor([0, *each]).cumsum(0).tolist()
    q = _normal(sum(each), hq, d, seed=9).to(torch.bfloat16)
    want = _plain(q, cache, table, lens, cuts, **kw)
    dev = _cuda(q, cache, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(cuts, dtype=torch.int32))
    got = ops.attn_prefill_kv4(*dev, max(each), **kw)
    _close(got, *want)
    _close(ops.attn_prefill_kv4(*dev, max(each) + 300, max_kv_len=333, **kw), *want)


def _few(q, cache, table, lens, cuts, most, longest, scale=None, softcap=0.0, window=0):
    """The kernel that cuts the key axis, whatever kernel the op would take."""
    from hartsyinference_b200.ops import _native as N
    L, n, hq, d = N.lib(), len(lens), q.shape[1], q.shape[2]
    hkv, page = cache.shape[1], cache.shape[2] * 16
    need = L.b200_attn_few_kv4_workspace(n, most, hq, hkv, d, longest)
    ws, out = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.full_like(q, 7)
    rc = L.b200_attn_few_kv4(q.data_ptr(), cache.data_ptr(), out.data_ptr(), table.data_ptr(), lens.data_ptr(), cuts.data_ptr(), n, most, hq, hkv, d, page,
                             table.shape[1], cache.shape[0], longest, window, 1 / math.sqrt(d) if scale is None else scale, softcap, ws.data_ptr(), need,
                             N.state(q.device).status.data_ptr(), N.stream())
    assert rc > 0
    return out


@gpu
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("kw", CASES)
def test_few_queries_behind_a_long_cache(hq, hkv, d, kw):
    """One query, none, more than keys, parts of columns that a sequence does not fill, sequences without keys."""
    lens, each = [700, 0, 5, 2100, 16, 900, 0, 1033], [3, 2, 7, 17, 0, 1, 0, 2]
    cache, table = _filled(lens, hkv, d, 32)
    cuts = torch.tensor([0, *each]).cumsum(0).tolist()
    q = _normal(sum(each), hq, d, seed=9).to(torch.bfloat16)
    want = _plain(q, cache, table, lens, cuts, **kw)
    dev = _cuda(q, cache, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(cuts, dtype=torch.int32))
    longest = max(lens) if not kw.get("window") else 40000                              # a window would leave one part
    if kw.get("window", 1000) > 600:
        _close(_few(*dev, max(each), longest, **kw), *want)
        _close(_few(*dev, max(each) + 30, 20000, **kw), *want)
    _close(ops.attn_prefill_kv4(*dev, max(each), **kw), *want)


@gpu
def test_few_queries_in_a_window():
    lens, each, kw = [3000, 1500, 611], [5, 3, 9], dict(window=600)
    for hq, hkv, d in HEADS[:4]:
        cache, table = _filled(lens, hkv, d, 64)
        cuts = torch.tensor([0, *each]).cumsum(0).tolist()
        q = _normal(sum(each), hq, d, seed=9).to(torch.bfloat16)
        dev = _cuda(q, cache, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(cuts, dtype=torch.int32))
        _close(_few(*dev, 9, 3000, **kw), *_plain(q, cache, table, lens, cuts, **kw))


@gpu
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("kw", CASES + [dict(causal=False), dict(causal=False, window=17)])
def test_wide_blocks_of_prompts(hq, hkv, d, kw):
    """The kernel of 256 rows a block, whatever kernel the op would take."""
    from hartsyinference_b200.ops import _native as N
    kw = dict(causal=True, scale=1 / math.sqrt(d), softcap=0.0, window=0) | kw
    lens, each = [700, 0, 70, 333, 1, 200, 5, 128], [140, 0, 3, 130, 1, 200, 9, 2]
    cache, table = _filled(lens, hkv, d, 32)
    cuts = torch.tensor([0, *each]).cumsum(0).tolist()
    q = _normal(sum(each), hq, d, seed=9).to(torch.bfloat16)
    qd, c, t, n, cu = _cuda(q, cache, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(cuts, dtype=torch.int32))
    out = torch.full_like(qd, 7)
    rc = N.lib().b200_attn_prefill_kv4(qd.data_ptr(), c.data_ptr(), out.data_ptr(), t.data_ptr(), n.data_ptr(), cu.data_ptr(), len(lens), max(each), hq, hkv, d, 32,
                                       t.shape[1], c.shape[0], int(kw["causal"]), kw["window"], kw["scale"], kw["softcap"], N.state(qd.device).status.data_ptr(), N.stream())
    assert rc == 0
    _close(out, *_plain(q, cache, table, lens, cuts, **kw))


@gpu
@pytest.mark.parametrize("sizes,kernel", [((1, 100, 100), 0), ((1, 2048, 8192), 1), ((16, 5, 4000), 2)])
def test_every_prompt_kernel_is_chosen(sizes, kernel):
    from hartsyinference_b200.ops import _native as N
    assert N.lib().b200_attn_kv4_choice(*sizes, 32, 8, 128, 1, 0, 0.088) == kernel
    assert N.lib().b200_attn_kv4_choice(*sizes, 32, 8, 128, 0, 0, 0.088) < 2
    assert N.lib().b200_attn_kv4_choice(*sizes, 32, 8, 128, 1, 0, -0.088) != 1


@gpu
def test_calls_captured_and_on_two_streams():
    """Two graphs of the same op replayed side by side, with lengths that change between replays, and a call of its own beside them."""
    lens = [1900, 1, 700]
    cache, table = _filled(lens, 2, 128, 16)
    q = [_normal(3, 8, 128, seed=i).to(torch.bfloat16) for i in range(2)]
    dev = _cuda(cache, table, torch.tensor(lens, dtype=torch.int32))
    qd, streams, graphs, outs = _cuda(*q), [torch.cuda.Stream(), torch.cuda.Stream()], [], []
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    run = [lambda x: ops.attn_decode_kv4(x, *dev), lambda x: ops.attn_prefill_kv4(x, *dev, cu, 1)]
    for f, x, st in zip(run, qd, streams):
        with torch.cuda.stream(st):
            f(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(f(x))
        graphs.append(g)
    for now in (lens, [5, 0, 640], lens):
        dev[2].copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        own = run[0](qd[0])
        torch.cuda.synchronize()
        for x, out in zip(q, outs):
            _close(out, *_plain(x, cache, table, now, [0, 1, 2, 3]))
        assert torch.equal(own, outs[0])


@gpu
def test_rows_of_another_layout():
    """Rows with a stride, on an odd address, and integers with a stride; those of another type are refused."""
    lens, hq, hkv, d = [130, 600], 8, 2, 128
    cache, table = _filled(lens, hkv, d, 16)
    wide = _normal(2, 2 * hq, d, seed=3).to(torch.bfloat16)
    q = wide[:, ::2]
    odd = torch.empty(2 * hq * d + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, hq, d)
    odd.copy_(q)
    want = _plain(q, cache, table, lens, [0, 1, 2])
    c, t, n = _cuda(cache, torch.stack([table, table], -1), torch.tensor(lens, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.attn_decode_kv4(odd, c, t[..., 0], n.long())
    for x in (wide.cuda()[:, ::2], odd):
        _close(ops.attn_decode_kv4(x, c, t[..., 0], n), *want)
        _close(ops.attn_prefill_kv4(x, c, t[..., 0], n, torch.tensor([0, 9, 1, 9, 2], dtype=torch.int32, device="cuda")[::2], 1), *want)


@gpu
def test_pages_outside_the_pool_are_reported_and_lengths_cut():
    """An entry that names no page reads as page 0, a length beyond the row's pages ends there; both leave a word in the status."""
    from hartsyinference_b200.exceptions import DeviceWaitTimeout
    from hartsyinference_b200.ops import _native as N
    lens = [40, 1200]
    cache, table = _filled(lens, 2, 128, 16)
    as_read, long = table.clone(), [40, table.shape[1] * 16]
    as_read[(as_read < 0) | (as_read >= cache.shape[0])] = 0
    q = _normal(2, 8, 128, seed=1).to(torch.bfloat16)
    cache.copy_(torch.randint(0, 200, cache.shape, generator=torch.Generator().manual_seed(2), dtype=torch.uint8))      # page 0 and the rest: finite
    cache.view(-1, cache.shape[-1])[:, 64 * 16:] = 100
    want = _plain(q, cache, as_read, long, [0, 1, 2])
    c, t, n = _cuda(cache, table, torch.tensor([40, 1 << 30], dtype=torch.int32))
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for f in (lambda: ops.attn_decode_kv4(q.cuda(), c, t, n), lambda: ops.attn_prefill_kv4(q.cuda(), c, t, n, cu, 1),
              lambda: ops.attn_prefill_kv4(q.cuda(), c, t, n, cu, 1, max_kv_len=16)):
        N.check_status()
        _close(f(), *want)
        with pytest.raises(DeviceWaitTimeout):
            N.check_status()


@gpu
def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes whose used pages lie at its end."""
    hkv, d, page, lens = 8, 128, 64, [70, 900]
    cache, table = _filled(lens, hkv, d, page)
    each = cache[0].numel()
    pages = (1 << 32) // each + cache.shape[0] + 5
    big = torch.empty(pages, *cache.shape[1:], dtype=torch.uint8, device="cuda")
    big[pages - cache.shape[0]:] = cache.cuda()
    moved = torch.where(table >= 0, table + (pages - cache.shape[0]), table)
    q = _normal(2, 32, d, seed=1).to(torch.bfloat16)
    want = _plain(q, cache, table, lens, [0, 1, 2])
    qd, t, n, cu = _cuda(q, moved, torch.tensor(lens, dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32))
    _close(ops.attn_decode_kv4(qd, big, t, n), *want)
    _close(ops.attn_prefill_kv4(qd, big, t, n, cu, 1), *want)
    _close(ops.attn_prefill_kv4(qd, big, t, n, cu, 1, causal=False), *want)
    kv = torch.tensor([0, 70, 970], dtype=torch.int32)
    for a, b in zip(ops.kv4_gather(big, t, kv.cuda(), 970), ops.kv4_gather(cache, table, kv, 970)):
        assert torch.equal(a.cpu(), b)
    qkv, pos, small, _ = _qkv_args(4, 8, hkv, d, page)
    slots = torch.tensor([0, 65, 2, -1])
    ops.rope_kv4(qkv, pos, 8, hkv, d, cache=small, slot_mapping=slots)
    last = pages - small.shape[0]
    big[last:] = 0
    ops.rope_kv4(qkv.cuda(), pos.cuda(), 8, hkv, d, cache=big, inv_freq=R.rope_inv_freq(d, 10000.0).cuda(), slot_mapping=torch.where(slots >= 0, slots + last * page, slots).cuda())
    assert torch.equal(big[last:].cpu(), small)


@gpu
def test_first_token_that_takes_nearly_all_of_the_weight():
    """A first key far ahead of the others whose values are zero: the result is made of probabilities near 2^-20."""
    n, hkv, d = 1500, 2, 128
    k, v = _normal(n, hkv, d, seed=1), _normal(n, hkv, d, seed=2)
    q = _normal(1, 8, d, seed=3).to(torch.bfloat16)
    k[0], v[0] = 0, 0
    k[0, :, :] = q.float().view(hkv, 4, d).mean(1) * 3
    cache, table = ops.kv4_cache(100, hkv, 16, d, "cpu"), torch.arange(99, -1, -1, dtype=torch.int32)[None]
    pos = torch.arange(n)
    R.kv4_store(cache, table[0, pos // 16].long() * 16 + pos % 16, k, v)
    want = _plain(q, cache, table, [n], [0, 1])
    dev = _cuda(cache, table, torch.tensor([n], dtype=torch.int32))
    _close(ops.attn_decode_kv4(q.cuda(), *dev), *want)
    _close(ops.attn_prefill_kv4(q.cuda(), *dev, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 1), *want)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_nothing_to_do(dev):
    """No sequences, no pages, no tokens, and rows that belong to nobody."""
    cache, none = ops.kv4_cache(2, 2, 16, 64, dev), ops.kv4_cache(0, 2, 16, 64, dev)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    q = torch.ones(3, 4, 64, dtype=torch.bfloat16, device=dev)
    table = ints([1], [0], [1])
    assert not ops.attn_decode_kv4(q, none, table, ints(0, 0, 0)).any()
    assert not ops.attn_decode_kv4(q, cache, table[:, :0], ints(0, 0, 0)).any()
    assert ops.attn_decode_kv4(q[:0], cache, table[:0], ints()).shape == (0, 4, 64)
    assert not ops.attn_prefill_kv4(q, none, table, ints(0, 0, 0), ints(0, 1, 2, 3), 1).any()
    assert ops.attn_prefill_kv4(q[:0], cache, table, ints(0, 0, 0), ints(0, 0, 0, 0), 0).shape == (0, 4, 64)
    for k in ops.kv4_gather(cache, table[:0], ints(0), 3) + ops.kv4_gather(none, table, ints(0, 0, 0, 0), 3) + ops.kv4_gather(cache, table, ints(0, 0, 1, 1), 4):
        assert k.shape[1:] == (2, 64) and not k[1:].any()
    assert ops.rope_kv4(torch.ones(0, 8 * 64, dtype=torch.bfloat16, device=dev), ints(), 4, 2, 64, cache=cache)[0].shape == (0, 4, 64)
    with pytest.raises(ValueError):
        ops.attn_prefill_kv4(q, cache, table, ints(1, 1, 1), ints(0, 1, 2, 3), 0)


# ------------------------------------------------------------------------------------------ few units for many blocks
def _parts(q, cache, table, lens, longest, fill, cuts=None, most=1, window=0):
    """The kernels that cut the key axis, with every byte of the workspace set to `fill` before the call."""
    from hartsyinference_b200.ops import _native as N
    L, n, hq, d = N.lib(), lens.numel(), q.shape[1], q.shape[2]
    hkv, page = cache.shape[1], cache.shape[2] * 16
    need = L.b200_attn_decode_kv4_workspace(n, hq, hkv, d, longest) if cuts is None else L.b200_attn_few_kv4_workspace(n, most, hq, hkv, d, longest)
    assert need > 0
    ws, out = torch.full((need,), fill, dtype=torch.uint8, device="cuda"), torch.full_like(q, 7)
    sizes = (hq, hkv, d, page, table.shape[1], cache.shape[0], longest, window, 1 / math.sqrt(d), 0.0, ws.data_ptr(), need, N.state(q.device).status.data_ptr(), N.stream())
    ptrs = [x.data_ptr() for x in (q, cache, out, table, lens)]
    rc = L.b200_attn_decode_kv4(*ptrs, n, *sizes) if cuts is None else L.b200_attn_few_kv4(*ptrs, cuts.data_ptr(), n, most, *sizes)
    assert rc == 2
    return out


FEW_UNITS = [([17], 32, 8, 128, 8192), ([100], 32, 8, 128, 8192), ([300], 32, 8, 128, 8192), ([300], 14, 2, 64, 8192), ([100] * 16, 8, 1, 128, 131072),
             ([700] + [12] * 63, 14, 2, 64, 700), ([1], 8, 1, 128, 131072), ([20, 0, 1], 40, 2, 128, 8192), ([0, 0], 4, 2, 64, 8192), ([1, 0, 2, 16, 33], 24, 1, 64, 40000)]


@gpu
@pytest.mark.parametrize("lens,hq,hkv,d,longest", FEW_UNITS)
@pytest.mark.parametrize("fill", [0xFF, 0x70, 0])                   # as floats: no numbers, 3e29, zeros
def test_fewer_units_than_blocks(lens, hq, hkv, d, longest, fill):
    """Blocks are counted from the longest length that the host knows; where the lengths themselves give fewer units, some blocks have none."""
    cache, table = _filled(lens, hkv, d, 16)
    wide = torch.full((len(lens), -(-longest // 16)), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table[:, :wide.shape[1]]
    q = _normal(len(lens), hq, d, seed=9).to(torch.bfloat16)
    dev = _cuda(q, cache, wide, torch.tensor(lens, dtype=torch.int32))
    want = _plain(q, cache, table, lens, list(range(len(lens) + 1)))
    _close(_parts(*dev, longest, fill), *want)
    _close(_parts(*dev, longest, fill, window=600), *_plain(q, cache, table, lens, list(range(len(lens) + 1)), window=600))
    each = [min(n + 1, 3 - i % 2) if i % 3 else 4 for i, n in enumerate(lens)]          # a query more than keys among them
    cuts = torch.tensor([0, *each]).cumsum(0).tolist()
    q = _normal(sum(each), hq, d, seed=8).to(torch.bfloat16)
    cu = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    got = _parts(q.cuda(), *dev[1:], longest, fill, cu, 4)
    _close(got, *_plain(q, cache, table, lens, cuts))


@gpu
def test_captured_over_a_wide_table_and_short_sequences():
    """A graph made for long sequences and replayed over short ones, in whose memory no number is left by the work before."""
    lens, hkv, d = [5000, 17, 300], 8, 128
    cache, table = _filled(lens, hkv, d, 16)
    q = _normal(3, 32, d, seed=1).to(torch.bfloat16)
    qd, c, t, n = _cuda(q, cache, table, torch.tensor(lens, dtype=torch.int32))
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")

    def run():
        stale = [torch.full((size,), math.nan, device="cuda") for size in (1 << 14, 1 << 17, 1 << 19, 1 << 21)]
        del stale
        return ops.attn_decode_kv4(qd, c, t, n), ops.attn_prefill_kv4(qd, c, t, n, cu, 1)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = run()
    for now in ([17, 1, 0], lens, [0, 0, 0], [100, 16, 33], [1, 0, 0], [5000, 0, 300]):
        n.copy_(torch.tensor(now, dtype=torch.int32))
        g.replay()
        for out in outs + run():
            _close(out, *_plain(q, cache, table, now, [0, 1, 2, 3]))


# ------------------------------------------------------------------------------------------ windows near 2^31
@gpu
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 30])
@pytest.mark.parametrize("causal", [True, False])
def test_windows_wider_than_anything(hq, hkv, d, window, causal):
    """More queries than keys under a window near 2^31, in each kernel: the queries in front of the first key are below 0 already."""
    from hartsyinference_b200.ops import _native as N
    L, lens, each = N.lib(), [5, 700, 1, 0, 40], [17, 9, 20, 3, 90]
    cache, table = _filled(lens, hkv, d, 32)
    cuts = torch.tensor([0, *each]).cumsum(0).tolist()
    q = _normal(sum(each), hq, d, seed=9).to(torch.bfloat16)
    want = _plain(q, cache, table, lens, cuts, causal=causal)
    dev = _cuda(q, cache, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(cuts, dtype=torch.int32))
    _close(ops.attn_prefill_kv4(*dev, max(each), causal=causal, window=window), *want)
    _close(ops.attn_prefill_kv4(*dev, max(each), causal=causal, window=window << 9), *want)
    if causal:
        _close(_few(*dev, max(each), 700, window=window), *want)
    qd, c, t, n, cu = dev
    for run in (L.b200_attn_kv4, L.b200_attn_prefill_kv4):
        out = torch.full_like(qd, 7)
        rc = run(qd.data_ptr(), c.data_ptr(), out.data_ptr(), t.data_ptr(), n.data_ptr(), cu.data_ptr(), len(lens), max(each), hq, hkv, d, 32, t.shape[1],
                 c.shape[0], int(causal), window, 1 / math.sqrt(d), 0.0, N.state(qd.device).status.data_ptr(), N.stream())
        assert rc == 0
        _close(out, *want)
    if causal:
        last = [c - 1 for c in cuts[1:]]
        _close(ops.attn_decode_kv4(qd[last], c, t, n, window=window), *(x[last] for x in want))
    N.check_status()


def test_tables_whose_units_leave_32_bits_are_refused():
    """2^26 units of 24 kv heads: 17 to 24 columns are walked in three parts, 25 to 32 in two, and the units of a sequence are counted in 32 bits."""
    from hartsyinference_b200.ops import _native as N
    if not N.available():
        pytest.skip("kernels library not built")
    L, p = N.lib(), 4096
    decode = lambda columns, max_pages: L.b200_attn_decode_kv4(p, p, p, p, p, 1, 24 * columns, 24, 64, 128, max_pages, 1, 1 << 20, 0, 1.0, 0.0, None, 0, None, None)
    few = lambda columns, max_pages: L.b200_attn_few_kv4(p, p, p, p, p, p, 1, columns, 24, 24, 64, 128, max_pages, 1, 1 << 20, 0, 1.0, 0.0, None, 0, None, None)
    for f in (decode, few):
        assert [f(c, 1 << 23) for c in (16, 17, 20, 24, 25, 32)] == [-5, -3, -3, -3, -5, -5]          # -5: the sizes are taken, no workspace is there
        assert [f(c, 1 << 22) for c in (16, 17, 20, 24, 25, 32)] == [-5] * 6
        assert [f(c, 1 << 24) for c in (16, 17, 20, 24, 25, 32)] == [-5] + [-3] * 5


@gpu
def test_launches_are_counted():
    """A decode call and a few queries behind a long cache are two kernels each, a call of the other kernels one."""
    from hartsyinference_b200.ops import _native as N
    lens = [4000, 3000]
    cache, table = _filled(lens, 8, 128, 16)
    q, c, t, n, cu = _cuda(_normal(10, 32, 128).to(torch.bfloat16), cache, table, torch.tensor(lens, dtype=torch.int32), torch.tensor([0, 5, 10], dtype=torch.int32))
    assert N.lib().b200_attn_kv4_choice(2, 5, table.shape[1] * 16, 32, 8, 128, 1, 0, 128 ** -0.5) == 2
    for call, launches in ((lambda: ops.attn_prefill_kv4(q, c, t, n, cu, 5), 2), (lambda: ops.attn_decode_kv4(q[:2], c, t, n), 2),
                           (lambda: ops.attn_prefill_kv4(q, c, t, n, cu, 5, causal=False), 1), (lambda: ops.attn_decode_kv4(q[:2], c, t[:, :4], n.clamp(max=64)), 1)):
        before = N.launch_count
        call()
        assert N.launch_count - before == launches
    N.check_status()


@gpu
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 1, 128)])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_queries_that_are_no_numbers(hq, hkv, d, softcap):
    """A NaN in a head's query makes that row NaN and no other, capped or not, in every kernel."""
    from hartsyinference_b200.ops import _native as N
    L, lens, each = N.lib(), [900, 40, 600], [3, 40, 1]
    cache, table = _filled(lens, hkv, d, 16)
    cuts = torch.tensor([0, *each]).cumsum(0).tolist()
    q = _normal(sum(each), hq, d, seed=9).to(torch.bfloat16)
    want = _plain(q, cache, table, lens, cuts, softcap=softcap)
    bad = torch.zeros(q.shape[:2], dtype=torch.bool)
    bad[0, 1] = bad[20, hq - 1] = bad[-1, 0] = True
    q[..., 5] = torch.where(bad, math.nan, q[..., 5])
    qd, c, t, n, cu = _cuda(q, cache, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(cuts, dtype=torch.int32))

    def right(out, rows=slice(None)):
        no = bad[rows]
        assert out.cpu()[no].isnan().all()
        _close(out[~no.cuda()], *(x[rows][~no] for x in want))

    right(_few(qd, c, t, n, cu, max(each), 900, softcap=softcap))
    for run in (L.b200_attn_kv4, L.b200_attn_prefill_kv4):
        out = torch.full_like(qd, 7)
        assert run(qd.data_ptr(), c.data_ptr(), out.data_ptr(), t.data_ptr(), n.data_ptr(), cu.data_ptr(), len(lens), max(each), hq, hkv, d, 16, t.shape[1],
                   c.shape[0], 1, 0, 1 / math.sqrt(d), softcap, N.state(qd.device).status.data_ptr(), N.stream()) == 0
        right(out)
    last = [x - 1 for x in cuts[1:]]
    right(ops.attn_decode_kv4(qd[last], c, t, n, softcap=softcap), last)
    short = ops.attn_decode_kv4(qd[[20]], c, t[1:2, :3], n[1:2], softcap=softcap)
    assert short[0, hq - 1].isnan().all() and torch.isfinite(short[0, :hq - 1]).all()


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128)])
def test_decode_into_fp8(dev, hq, hkv, d):
    """The quantised result is that of the bf16 one, for one kernel and for shares."""
    lens = [40, 0, 900]
    cache, table = _filled(lens, hkv, d, 16)
    q = _normal(3, hq, d, seed=2).to(torch.bfloat16).to(dev)
    args = [x.to(dev) for x in (cache, table, torch.tensor(lens, dtype=torch.int32))]
    for n, cut in ((3, slice(None)), (2, slice(0, 4))):
        a = (q[:n], args[0], args[1][:n, cut], args[2][:n])
        want = ops.attn_decode_kv4(*a)
        out, act = ops.attn_decode_kv4(*a, emit_fp8=True)
        none, only = ops.attn_decode_kv4(*a, emit_fp8=True, emit_bf16=False)
        held = ops.quant_fp8_act(want.reshape(n, hq * d))
        assert torch.equal(out, want) and none is None
        for x in (act, only):
            assert torch.equal(x.data.view(torch.uint8), held.data.view(torch.uint8)) and torch.equal(x.scales_fp32(), held.scales_fp32())


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_probabilities_are_rounded_once(d):
    """Two keys, the first with score 0 and a value of zero, the second with a probability of nearly half a step between two bf16: the result differs from
    7 s p / (1 + p) by the rounding of p, at most 2^-8 of it, and its own, 2^-8 again; 2^-12 covers their product (2^-16) and sums and exponentials in 32
    bits. s are scales of every mantissa. A rounding of p s as well would be off by up to 2.5 times 2^-8 here."""
    hkv = 512 // d                                                     # 16 blocks of 32 values: every mantissa twice
    scales = (torch.arange(16) % 8 + 8) / 8.0
    v = torch.zeros(2, hkv, d)
    v[1] = (7 * scales).repeat_interleave(32).view(hkv, d)
    k = torch.zeros(2, hkv, d)
    k[1] = -0.875
    cache, table = ops.kv4_cache(1, hkv, 16, d, "cpu"), torch.zeros(1, 1, dtype=torch.int32)
    R.kv4_store(cache, torch.arange(2), k, v)
    assert all(torch.equal(a, b) for a, b in zip(R.kv4_sequence(cache, table[0], 2), (k, v)))
    c, t, n = _cuda(cache, table, torch.tensor([2], dtype=torch.int32))
    q = torch.ones(1, hkv, d, dtype=torch.bfloat16, device="cuda")
    for j in range(128):
        for part in (-0.49, 0.49):
            p = (128 + j + part) / 256
            want = v[1].double() * p / (1 + p)
            got = ops.attn_decode_kv4(q, c, t, n, scale=-math.log(p) / (0.875 * d))[0].double().cpu()
            assert ((got - want).abs() <= (2.0 ** -7 + 2.0 ** -12) * want).all(), (j, part)
