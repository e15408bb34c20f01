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
    """Probabilities are rounded to bf16 before and after the product with a scale (half a step each, 2^-9 twice, of sum p |v|), the
    result to bf16 (2^-9 of it): 2^-8 of both holds with a half to spare. Scores are sums of 128 products in 32 bits, of
    which sum |q k| scale is below 2^9 here: off by less than 2^9 * 2^-24 * 2 * 2^3 = 2^-11, and so are probabilities and their sum.
    Values enter as 128 + code, and 136 is taken off again, 16 keys at a time: two sums of at most 143 p s that are cut to 24 bits,
    2 * 2^-22 * 143 < 2^-13 of sum p s with two bits to spare."""
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    bound = 2.0 ** -8 * (size + want.abs()) + 2.0 ** -10 * size + 2.0 ** -13 * scales + 1e-30
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


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 1, 128)])
def test_attention_on_cpu(hq, hkv, d):
    lens, each = [9, 0, 40], [4, 1, 40]
    cache, table = _filled(lens, hkv, d, 16)
    cuts = [0, 4, 5, 45]
    q = _normal(45, hq, d, seed=8).to(torch.bfloat16)
    got = ops.attn_prefill_kv4(q, cache, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(cuts, dtype=torch.int32), max(each), window=7, softcap=20.0)
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
@pytest.mark.parametrize("kw", CASES + [dict(causal=False)])
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
