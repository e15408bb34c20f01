"""Workloads of the 4-bit K/V cache: writing it, reading it back, and attention over it.

Four kinds of pass:

``append``   ``ops.rope_kv4``: norm, rotation and 4-bit store of packed q | k | v rows
``gather``   ``ops.rope_kv4`` of new tokens, then ``ops.kv4_gather``: whole sequences as dense keys and values
``decode``   ``ops.attn_decode_kv4``: one query token per sequence
``prefill``  ``ops.attn_prefill_kv4``: ragged chunks of query tokens behind what the cache holds

The cache of a layer is uint8 [pages, kv heads, page / 16, 2, 16 * (d / 2 + d / 32)]: per 16 tokens of one head a plane of keys and one of
values, each 16 rows of d / 2 bytes of codes and then 16 rows of d / 32 scales. Blocks of 32 values share a scale of 5
exponent and 3 mantissa bits, s = max|x| / 7 rounded to them; a code is rint(x / s) + 8. Where a value's four bits lie
in its row is in ``_places``.
"""
from __future__ import annotations

import math

import torch

own = False

K_EXP, V_EXP = -6, -10      # a scale byte b is the half-precision number with bits b << 7, times two to these
THETA = 500000.0


def listed():
    return [
        # one step of 64 chats with a large model
        dict(name="append-step-64", kind="append", tokens=64, hq=64, hkv=8, d=128, rot=128, style=0, norm=False, page=16),
        # the benchmark's prompt chunk of that model
        dict(name="append-chunk-8192", kind="append", tokens=8192, hq=64, hkv=8, d=128, rot=128, style=0, norm=False, page=16),
        # a new prompt of odd length per sequence, read back for attention with a bias that the kernels do not take
        dict(name="gather-small", kind="gather", sequences=3, least=37, most=150, new=29, hq=14, hkv=2, d=64, page=16),
        # the same for a batch of long ragged sequences
        dict(name="gather-ragged", kind="gather", sequences=12, least=700, most=9000, new=64, hq=32, hkv=8, d=128, page=32),
        # a first chat with a small model: latency
        dict(name="decode-short", kind="decode", sequences=1, least=41, most=41, hq=14, hkv=2, d=64, page=16, window=0, softcap=0.0),
        # the benchmark's own step: 64 requests of 2048 tokens and some decoded ones
        dict(name="decode-64x2k", kind="decode", sequences=64, least=2048, most=2304, hq=64, hkv=8, d=128, page=16, window=0, softcap=0.0),
        # one very long document
        dict(name="decode-long", kind="decode", sequences=1, least=131000, most=131000, hq=32, hkv=8, d=128, page=16, window=0, softcap=0.0),
        # a ragged batch through a capped layer with a sliding window
        dict(name="decode-window-cap", kind="decode", sequences=23, least=300, most=9000, hq=32, hkv=8, d=128, page=64, window=4096, softcap=50.0),
        # a few guessed tokens per sequence to be checked at once
        dict(name="prefill-verify", kind="prefill", sequences=16, queries=5, least=2000, most=4000, hq=32, hkv=8, d=128, page=16, window=0, softcap=0.0),
        # short prompts of odd lengths, small model
        dict(name="prefill-short", kind="prefill", sequences=5, queries=97, least=0, most=0, hq=14, hkv=2, d=64, page=16, window=0, softcap=0.0),
        # a chunk of a long prompt on top of what the cache holds already
        dict(name="prefill-8b-long", kind="prefill", sequences=1, queries=2048, least=6144, most=6144, hq=32, hkv=8, d=128, page=16, window=0, softcap=0.0),
        # the benchmark's prompt chunk: four prompts
        dict(name="prefill-70b", kind="prefill", sequences=4, queries=2048, least=0, most=0, hq=64, hkv=8, d=128, page=16, window=0, softcap=0.0),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


HEADS = [(64, 8, 128), (32, 8, 128), (8, 1, 128), (14, 2, 64), (32, 32, 64), (28, 4, 128), (20, 1, 64), (48, 3, 128), (12, 4, 64)]


def draw(rng):
    kind = rng.choice(["append", "append", "gather", "decode", "decode", "decode", "prefill", "prefill", "prefill"])
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice([16, 16, 32, 64])
    heads = dict(hq=hq, hkv=hkv, d=d, page=page)
    if kind == "append":
        return dict(kind=kind, tokens=_log(rng, 1, 8000), rot=rng.choice([d, d, d // 2, 32]), style=rng.choice([0, 0, 1]), norm=rng.random() < 0.3, **heads)
    if kind == "gather":
        n = _log(rng, 1, 24)
        least = _log(rng, 5, 40000 // n)
        return dict(kind=kind, sequences=n, least=least, most=least + _log(rng, 1, 40000 // n), new=_log(rng, 1, 200), **heads)
    window, softcap = rng.choice([(0, 0.0), (0, 0.0), (0, 0.0), (_log(rng, 20, 5000), 0.0), (0, 30.0), (_log(rng, 20, 5000), 50.0)])
    if kind == "decode":
        n = _log(rng, 1, 128)
        top = min(140000, 1000000 // (n * hkv))
        least = _log(rng, 1, top)
        return dict(kind=kind, sequences=n, least=least, most=min(top, least + _log(rng, 1, 3000)), window=window, softcap=softcap, **heads)
    n = _log(rng, 1, 16)
    queries = _log(rng, 2, 4000 // n)
    least = rng.choice([0, _log(rng, 1, 6000)])
    most = least + (_log(rng, 1, 500) if least else 0)
    while n * hq * queries * (queries + most) > 1.0e9:
        queries //= 2
    return dict(kind=kind, sequences=n, queries=queries, least=least, most=most, window=window, softcap=softcap, **heads)


# ------------------------------------------------------------------------------------------ the format
def _places(d, values):
    """Position (in units of 4 bits) of every value of a row, [2, d]: the row of a token t is number (t >> 1) & 1. Keys: words of eight
    values that one lane quarter multiplies, by lane quarter, then by block. Values: words by lane group, then by 64
    values; with 128 of them every other pair of tokens has the lane groups' halves exchanged."""
    c = torch.arange(d)
    if not values:
        p = ((c % 8 // 2) * (d // 32) + c // 32) * 8 + c % 32 // 8 + 4 * (c % 2)
        return torch.stack([p, p])
    g = c % 8
    return torch.stack([((g ^ x) * (d // 64) + c // 64) * 8 + c % 64 // 8 for x in (0, 4 if d == 128 else 0)])


def _blocks(x, exp):
    """x [..., d] in 32 bits -> (codes 1 .. 15, scale bytes [..., d / 32]), both int32."""
    b = torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf).unflatten(-1, (-1, 32))
    f = b.abs().amax(-1)
    f = f / torch.full_like(f, 7) * 2.0 ** -exp           # (a number for a divisor becomes a product with its reciprocal)
    bits = f.view(torch.int32)
    # to three bits of mantissa, ties to even, and the exponent's bias from 127 to 15
    byte = (((bits + 0x7ffff + ((bits >> 20) & 1)) >> 20) - (112 << 3)).clamp(8, 247)
    return (torch.round(b / _scales(byte, exp)[..., None]).clamp(-7, 7) + 8).to(torch.int32).flatten(-2), byte


def _scales(byte, exp):
    """The scales that bytes stand for, in 32 bits."""
    return ((byte + (112 << 3)) << 20).view(torch.float32) * 2.0 ** exp


def _rows(codes, odd, values):
    """codes [n, hkv, d] and (t >> 1) & 1 of every token -> the bytes of its rows [n, hkv, d / 2]."""
    d = codes.shape[-1]
    at = _places(d, values).to(codes.device)[odd][:, None].expand(codes.shape)
    nib = torch.empty_like(codes).scatter_(-1, at, codes)
    return (nib[..., 0::2] | (nib[..., 1::2] << 4)).to(torch.uint8)


def _store(cache, slots, page, k, v):
    """Writes rows of 32-bit values to their slots (below 0: not stored); returns the values that they are held as."""
    n, hkv, d = k.shape
    on = slots >= 0
    s = slots[on]
    pg, unit, t = s // page, s % page // 16, s % 16
    held = []
    for plane, (x, exp) in enumerate(((k, K_EXP), (v, V_EXP))):
        codes, byte = _blocks(x, exp)
        held.append(((codes - 8).float().unflatten(-1, (-1, 32)) * _scales(byte, exp)[..., None]).flatten(-2).to(torch.bfloat16))
        where = cache[:, :, :, plane]
        h = torch.arange(hkv, device=cache.device)[None, :, None]
        first = (pg[:, None, None], h, unit[:, None, None])
        row = (t * (d // 2))[:, None, None] + torch.arange(d // 2, device=cache.device)
        where[(*first, row)] = _rows(codes[on], (t >> 1) & 1, plane == 1)
        row = (16 * (d // 2) + t * (d // 32))[:, None, None] + torch.arange(d // 32, device=cache.device)
        where[(*first, row)] = byte[on].to(torch.uint8)
    return held


def _load(cache, slots, page, d):
    """The values that slots [...] stand for: keys and values [..., hkv, d] in 32 bits."""
    pg, unit, t = slots // page, slots % page // 16, slots % 16
    out = []
    for plane, exp in enumerate((K_EXP, V_EXP)):
        rows = cache[:, :, :, plane].permute(0, 2, 1, 3)[pg, unit]                      # [..., hkv, bytes of a plane]
        row = (t * (d // 2))[..., None, None] + torch.arange(d // 2, device=cache.device)
        both = torch.gather(rows, -1, row.expand(*rows.shape[:-1], -1)).to(torch.int32)
        nib = torch.stack([both & 15, both >> 4], -1).flatten(-2)
        at = _places(d, plane == 1).to(cache.device)[(t >> 1) & 1][..., None, :].expand(nib.shape)
        row = (16 * (d // 2) + t * (d // 32))[..., None, None] + torch.arange(d // 32, device=cache.device)
        byte = torch.gather(rows, -1, row.expand(*rows.shape[:-1], -1)).to(torch.int32)
        codes = torch.gather(nib, -1, at) - 8
        out.append((codes.float().unflatten(-1, (-1, 32)) * _scales(byte, exp)[..., None]).flatten(-2))
    return out


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed, n):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + n)


def _channels(g, hkv, d):
    """How large the channels of keys are: a few stand out, as in trained models."""
    size = torch.empty(hkv, d, device="cuda").normal_(generator=g).mul_(0.5).exp_()
    return torch.where(torch.rand(hkv, d, device="cuda", generator=g) < 0.03, size * 8, size)


def _qkv(case, tokens, g):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    x = torch.empty(tokens, hq + 2 * hkv, d, device="cuda").normal_(generator=g)
    x[:, hq:hq + hkv] *= _channels(g, hkv, d)
    x[:, hq + hkv:] *= 0.3
    return x.to(torch.bfloat16).reshape(tokens, -1)


def _spread(case, seed):
    """Tokens that every sequence holds: spread over the case's range."""
    n = case["sequences"]
    return torch.randint(case["least"], case["most"] + 1, (n,), generator=torch.Generator().manual_seed(case["least"] + 1000003 * n)).tolist()


def _table(lens, page, seed):
    """Page ids of every sequence, shuffled over the pool as a running engine leaves them."""
    pages = [max(1, -(-n // page)) for n in lens]
    order = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(seed + 3)).to(torch.int32)
    table, at = torch.zeros(len(lens), max(pages), dtype=torch.int32), 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    return table.cuda(), at


def _pool(case, pages):
    d = case["d"]
    return torch.zeros(pages, case["hkv"], case["page"] // 16, 2, 16 * (d // 2 + d // 32), dtype=torch.uint8, device="cuda")


def _filled(case, lens, table, pages, seed):
    """A pool whose sequences hold keys and values of a model's sizes."""
    cache, page = _pool(case, pages), case["page"]
    hkv, d, g = case["hkv"], case["d"], _gen(seed, 1)
    size = _channels(g, hkv, d)
    for i, n in enumerate(lens):
        for a in range(0, n, 32768):
            t = torch.arange(a, min(n, a + 32768), device="cuda")
            k = torch.empty(t.numel(), hkv, d, device="cuda").normal_(generator=g) * size
            v = torch.empty(t.numel(), hkv, d, device="cuda").normal_(generator=g) * 0.3
            _store(cache, table[i, t // page].long() * page + t % page, page, k, v)
    return cache


def _freq(rot):
    return (THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().cuda()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    kind, page = case["kind"], case["page"]
    hq, d = case["hq"], case["d"]
    g = _gen(seed, 2)
    if kind == "append":
        t = case["tokens"]
        pages = -(-t // page) + 1
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:t] if t <= 512 else torch.arange(t, device="cuda") + page // 2
        slots = torch.where(torch.rand(t, device="cuda", generator=g) < 0.01, -1, slots)           # padding rows of a batch
        norm = [1 + 0.1 * torch.empty(d, device="cuda").normal_(generator=g) for _ in "qk"] if case["norm"] else [None, None]
        return dict(case=case, qkv=_qkv(case, t, g), positions=torch.randint(0, 131072, (t,), generator=g, device="cuda", dtype=torch.int32), slots=slots,
                    freq=_freq(case["rot"]), q_norm=norm[0] if norm[0] is None else norm[0].to(torch.bfloat16),
                    k_norm=norm[1] if norm[1] is None else norm[1].to(torch.bfloat16), cache=_pool(case, pages))
    lens = _spread(case, seed)
    if kind == "gather":
        old, lens = lens, [n + case["new"] for n in lens]
        table, pages = _table(lens, page, seed)
        pos = torch.cat([torch.arange(a, b) for a, b in zip(old, lens)]).cuda()
        row = torch.arange(len(lens), device="cuda").repeat_interleave(case["new"])
        return dict(case=case, qkv=_qkv(case, pos.numel(), g), positions=pos.to(torch.int32), slots=table[row, pos // page].long() * page + pos % page, freq=_freq(d),
                    q_norm=None, k_norm=None, cache=_filled(case, old, table, pages, seed), table=table, total=sum(lens),
                    cu_kv=torch.nn.functional.pad(_ints(lens).cumsum(0, dtype=torch.int32), (1, 0)))
    queries = case["queries"] if kind == "prefill" else 1
    # a chunk's lengths differ by a whole number from sequence to sequence; a decoded token is counted in `least` and `most`
    n = len(lens)
    each = [queries] * n if kind == "decode" or n == 1 or queries >= 1024 else [max(1, queries + (2 * i - n + 1) * (queries // (2 * n))) for i in range(n)]
    if kind == "prefill":
        lens = [a + b for a, b in zip(lens, each)]
    table, pages = _table(lens, page, seed)
    q = torch.empty(sum(each), hq, d, device="cuda").normal_(generator=g).to(torch.bfloat16)
    state = dict(case=case, q=q, cache=_filled(case, lens, table, pages, seed), table=table, kv_lens=_ints(lens), longest=max(lens))
    if kind == "prefill":
        state.update(cu_q=torch.nn.functional.pad(_ints(each).cumsum(0, dtype=torch.int32), (1, 0)), most=max(each))
    return state


# ------------------------------------------------------------------------------------------ the plain forms
def _turn(x, cos, sin, rot, style):
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if style == 0 else (x[..., 0:rot:2], x[..., 1:rot:2])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([u, v], -1) if style == 0 else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _append(s):
    """Queries, and keys and values as the cache holds them."""
    c = s["case"]
    hq, hkv, d, rot, style = c["hq"], c["hkv"], c["d"], 2 * s["freq"].numel(), c.get("style", 0)
    x = s["qkv"].reshape(-1, hq + 2 * hkv, d).float()
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if s["q_norm"] is not None:
        q = q * (1 / (q.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()).float() * s["q_norm"].float()
        k = k * (1 / (k.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()).float() * s["k_norm"].float()
    angle = s["positions"].double()[:, None, None] * s["freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    k, v = _store(s["cache"], s["slots"], c["page"], _turn(k, cos, sin, rot, style), v)
    return _turn(q, cos, sin, rot, style).to(torch.bfloat16), k, v


def _gather(s):
    c, cu = s["case"], s["cu_kv"].long()
    lens = cu[1:] - cu[:-1]
    row = torch.repeat_interleave(torch.arange(lens.numel(), device=cu.device), lens, output_size=s["total"])
    pos = torch.arange(s["total"], device=cu.device) - cu[row]
    slots = s["table"][row, pos // c["page"]].long() * c["page"] + pos % c["page"]
    return [x.to(torch.bfloat16) for x in _load(s["cache"], slots, c["page"], c["d"])]


def _attention(s, cu_q, most):
    """Padded over sequences: queries [S, most], keys [S, longest]."""
    c = s["case"]
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    n, dev = s["kv_lens"].numel(), s["q"].device
    kpos = torch.arange(s["longest"], device=dev)
    slots = s["table"].long()[:, kpos // page] * page + kpos % page
    lens = s["kv_lens"].long()
    slots = torch.where(kpos < lens[:, None], slots, 0)
    k, v = _load(s["cache"], slots, page, d)                                             # [S, longest, hkv, d]
    qlen = cu_q[1:] - cu_q[:-1]
    i = torch.arange(most, device=dev)
    at = torch.where(i < qlen[:, None], cu_q[:-1, None] + i, 0)                            # [S, most]
    q = s["q"].float()[at].reshape(n, most, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(d ** -0.5)
    if c["softcap"] > 0:
        score.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    score = score.reshape(n, hkv, hq // hkv, most, -1)
    qpos = (lens - qlen)[:, None] + i
    seen = kpos <= qpos[..., None]
    if c["window"] > 0:
        seen &= kpos > qpos[..., None] - c["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    score.div_(score.sum(-1, keepdim=True))
    o = torch.matmul(score.reshape(n, hkv, -1, s["longest"]), v.permute(0, 2, 1, 3)).reshape(n, hq, most, d).permute(0, 2, 1, 3)
    return o[i < qlen[:, None]].to(torch.bfloat16)


def run(state):
    c = state["case"]
    kind = c["kind"]
    if own:
        from hartsyinference_b200 import ops
        if kind in ("append", "gather"):
            q, k, v = ops.rope_kv4(state["qkv"], state["positions"], c["hq"], c["hkv"], c["d"], cache=state["cache"], slot_mapping=state["slots"],
                                   rot=2 * state["freq"].numel(), inv_freq=state["freq"], style=c.get("style", 0), q_norm_w=state["q_norm"],
                                   k_norm_w=state["k_norm"], eps=1e-6, want_kv=kind == "append")
            return (q, k, v) if kind == "append" else (q, *ops.kv4_gather(state["cache"], state["table"], state["cu_kv"], state["total"]))
        kw = dict(softcap=c["softcap"], window=c["window"], max_kv_len=state["longest"])
        if kind == "decode":
            return ops.attn_decode_kv4(state["q"], state["cache"], state["table"], state["kv_lens"], **kw)
        return ops.attn_prefill_kv4(state["q"], state["cache"], state["table"], state["kv_lens"], state["cu_q"], state["most"], **kw)
    if kind == "append":
        return _append(state)
    if kind == "gather":
        q, _, _ = _append(state)
        return (q, *_gather(state))
    if kind == "decode":
        return _attention(state, torch.arange(state["kv_lens"].numel() + 1, device=state["q"].device), 1)
    return _attention(state, state["cu_q"].long(), state["most"])


# ------------------------------------------------------------------------------------------ least work
def work(case):
    hq, hkv, d, kind = case["hq"], case["hkv"], case["d"], case["kind"]
    held = hkv * d * 17 / 16                     # bytes of a token's keys and values in the cache
    if kind == "append":
        t = case["tokens"]
        return dict(bytes=t * ((hq + 2 * hkv) * d * 2 + hq * d * 2 + held + 2 * hkv * d * 2), flops=t * (hq + hkv) * case["rot"] * 3)
    lens = _spread(case, 0)
    if kind == "gather":
        new, total = case["new"] * len(lens), sum(lens) + case["new"] * len(lens)
        return dict(bytes=new * ((2 * hq + 2 * hkv) * d * 2 + held) + total * (held + 4 * hkv * d), flops=total * hkv * d * 4)
    n, queries = len(lens), case.get("queries", 1)
    each = [queries] * n if kind == "decode" or n == 1 or queries >= 1024 else [max(1, queries + (2 * i - n + 1) * (queries // (2 * n))) for i in range(n)]
    pairs = keys = 0
    for m, x in zip(each, lens):
        ctx = x if kind == "prefill" else x - 1
        w = case["window"] or ctx + m
        full = max(0, min(m, w - 1 - ctx))       # queries that see all keys before them
        pairs += full * ctx + full * (full + 1) // 2 + (m - full) * w
        keys += min(ctx + m, w + m - 1)
    return dict(bytes=keys * held + 2 * sum(each) * hq * d * 2, flops=4 * pairs * hq * d)


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def _value_of(plane, d, exp, values):
    """Planes of 16 tokens [..., bytes] -> [..., 16, d] in 64 bits, every value looked up where the description of a row has it."""
    at, high = [], []
    for t in range(16):
        odd = t // 2 % 2
        for c in range(d):
            if values:
                lane = (c + 4) % 8 if odd and d == 128 else c % 8
                word, nibble = lane * (d // 64) + c // 64, c % 64 // 8
            else:
                word, nibble = c % 8 // 2 * (d // 32) + c // 32, c % 32 // 8 + (4 if c % 2 else 0)
            at.append(t * (d // 2) + word * 4 + nibble // 2)
            high.append(nibble % 2 == 1)
    dev = plane.device
    b = plane[..., torch.tensor(at, device=dev)].long()
    code = torch.where(torch.tensor(high, device=dev), b // 16, b % 16) - 8
    byte = plane[..., 8 * d:].long()
    scale = torch.where(byte >= 8, (1 + (byte % 8).double() / 8) * torch.exp2((byte // 8 - 15).double()), (byte % 8).double() / 8 * 2.0 ** -14) * 2.0 ** exp
    return (code.double().unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2).unflatten(-1, (16, d))


def _sequence(state, i, length):
    """Keys and values of sequence i, [length, hkv, d] in 64 bits."""
    c = state["case"]
    d, page = c["d"], c["page"]
    ids = state["table"][i, :-(-length // page)].long()
    units = state["cache"][ids]                                        # [pages, hkv, page / 16, 2, bytes]
    out = []
    for plane, exp in enumerate((K_EXP, V_EXP)):
        x = _value_of(units[:, :, :, plane], d, exp, plane == 1)       # [pages, hkv, page / 16, 16, d]
        out.append(x.permute(0, 2, 3, 1, 4).reshape(-1, c["hkv"], d)[:length])
    return out


def _held(x, exp):
    """What values in 64 bits are held as."""
    b = x.unflatten(-1, (-1, 32))
    f = b.abs().amax(-1) / 7
    e = torch.floor(torch.log2(f.clamp_min(1e-300)))
    e = torch.where(torch.exp2(e + 1) <= f, e + 1, torch.where(torch.exp2(e) > f, e - 1, e))
    s = torch.round(f / torch.exp2(e - 3)) * torch.exp2(e - 3)
    s = s.clamp(2.0 ** (exp - 14), 1.875 * 2.0 ** (exp + 15))
    return (torch.round(b / s[..., None]).clamp(-7, 7) * s[..., None]).flatten(-2)


def _exact_append(s):
    c = s["case"]
    hq, hkv, d, half = c["hq"], c["hkv"], c["d"], s["freq"].numel()
    x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    angle = torch.outer(s["positions"].double(), s["freq"].double())
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    done = []
    for y, w in ((x[:, :hq], s["q_norm"]), (x[:, hq:hq + hkv], s["k_norm"])):
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / d + 1e-6) * w.double()
        if c.get("style", 0) == 0:
            z = torch.complex(y[..., :half], y[..., half:2 * half]) * turn
            y = torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)
        else:
            z = torch.view_as_complex(y[..., :2 * half].reshape(*y.shape[:-1], half, 2).contiguous()) * turn
            y = torch.cat([torch.view_as_real(z).flatten(-2), y[..., 2 * half:]], -1)
        done.append(y)
    return done[0], _held(done[1], K_EXP), _held(x[:, hq + hkv:], V_EXP)


def exact(case, seed):
    state = prepare(case, seed)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    if case["kind"] == "append":
        return _exact_append(state)
    if case["kind"] == "gather":
        q, k, v = _exact_append(state)
        lens, new = (state["cu_kv"][1:] - state["cu_kv"][:-1]).tolist(), case["new"]
        ks, vs = [], []
        for i, n in enumerate(lens):
            ok, ov = _sequence(state, i, n - new)
            ks += [ok, k[i * new:(i + 1) * new]]
            vs += [ov, v[i * new:(i + 1) * new]]
        return q, torch.cat(ks), torch.cat(vs)
    lens = state["kv_lens"].tolist()
    cuts = state["cu_q"].tolist() if case["kind"] == "prefill" else list(range(len(lens) + 1))
    out = torch.empty(cuts[-1], hq, d, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        k, v = _sequence(state, i, n)
        a, b = cuts[i], cuts[i + 1]
        key = torch.arange(n, device="cuda")[None]
        last = torch.arange(n - (b - a), n, device="cuda")[:, None]
        hidden = (key > last) | ((key <= last - case["window"]) if case["window"] > 0 else False)
        for h in range(hq):
            kv = h * hkv // hq
            x = state["q"][a:b, h].double() @ k[:, kv].T / math.sqrt(d)
            if case["softcap"] > 0:
                x = torch.tanh(x / case["softcap"]) * case["softcap"]
            out[a:b, h] = torch.softmax(torch.where(hidden, -math.inf, x), -1) @ v[:, kv]
    return out
