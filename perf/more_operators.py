"""Workloads of long prompts with pictures and film, and of long chats: rotary positions on several axes, and attention over chosen pages.

Three kinds of pass:

``axes``    ``ops.rope_axes_kv``: norm, rotation by positions on several axes and the store of packed q | k | v rows
``pick``    ``ops.key_bounds_`` of the pages that new tokens filled, then ``ops.pick_pages``: the pages that every query attends to
``attend``  ``ops.attn_picked``: attention over chosen pages, at decode, for a few queries and over chunks of prompts

Bounds of the keys of a page and key head are 2 d + 16 bytes: d codes of the largest value of every channel, d of the smallest, an exponent e + 64 and
zeros. e is the smallest with max |value| <= 127 * 2^e, from -50 to 50; codes are ceil(largest / 2^e) and floor(smallest / 2^e). Queries have codes
round(q / 2^e) with an exponent of their own head. The score of a page is the largest 2^(e_q + e_page) * sum_c max(a_c largest_c, a_c smallest_c) of
the queries that choose together: those of the heads of a group, and of `run` neighbouring tokens. Sums are whole numbers below 2^22, so scores are
exact in 32 bits. Kept are the `first` pages, the `last` ones up to the page of a run's first query and all behind it, and of those between the `top`
of the largest score, ties to the lowest index; rows of page numbers in order, then -1.
"""
from __future__ import annotations

import math

import torch

own = False

THETA = 1000000.0


def listed():
    return [
        # a prompt with one small picture
        dict(name="axes-picture", kind="axes", tokens=391, hq=28, hkv=4, d=128, sections="16 24 24", mixed=False, norm=False, store=True, page=16),
        # a chunk of a long film
        dict(name="axes-film-8192", kind="axes", tokens=8192, hq=32, hkv=8, d=128, sections="24 20 20", mixed=True, norm=True, store=True, page=16),
        # rows and columns of a picture's patches in a vision tower, heads of 80, nothing stored
        dict(name="axes-patches", kind="axes", tokens=4900, hq=16, hkv=16, d=80, sections="20 20", mixed=False, norm=False, store=False, page=16),
        # one decode step of sixteen chats
        dict(name="pick-chats", kind="pick", sequences=16, queries=1, run=1, least=2000, most=6000, hq=32, hkv=8, d=128, page=16, top=64, first=1, last=2),
        # one step behind a very long document
        dict(name="pick-long", kind="pick", sequences=1, queries=1, run=1, least=131072, most=131072, hq=64, hkv=8, d=128, page=16, top=128, first=1, last=2),
        # a few guessed tokens of a small model, to be checked at once
        dict(name="pick-guesses", kind="pick", sequences=7, queries=5, run=1, least=900, most=5000, hq=14, hkv=2, d=64, page=32, top=24, first=1, last=1),
        # a chunk of a long prompt on top of what the cache holds: sixteen tokens choose together
        dict(name="pick-chunk", kind="pick", sequences=1, queries=2048, run=16, least=30720, most=30720, hq=64, hkv=8, d=128, page=16, top=128, first=1, last=2),
        # the first tokens of a chat: all of its pages, latency
        dict(name="attend-short", kind="attend", sequences=1, queries=1, run=1, least=41, most=41, hq=14, hkv=2, d=64, page=16, top=32, first=1, last=2, softcap=0.0),
        # one step of 64 long chats
        dict(name="attend-chats-64", kind="attend", sequences=64, queries=1, run=1, least=4000, most=9000, hq=64, hkv=8, d=128, page=16, top=128, first=1, last=2, softcap=0.0),
        # one step behind a very long document
        dict(name="attend-long", kind="attend", sequences=1, queries=1, run=1, least=131001, most=131001, hq=32, hkv=8, d=128, page=16, top=253, first=1, last=2, softcap=0.0),
        # guessed tokens that choose together, in a model that caps its scores
        dict(name="attend-guesses", kind="attend", sequences=16, queries=5, run=5, least=2000, most=7000, hq=32, hkv=8, d=128, page=64, top=30, first=1, last=1, softcap=50.0),
        # a chunk of a long prompt
        dict(name="attend-chunk", kind="attend", sequences=1, queries=2048, run=16, least=30720, most=30720, hq=64, hkv=8, d=128, page=16, top=128, first=1, last=2, softcap=0.0),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


HEADS = [(64, 8, 128), (32, 8, 128), (8, 1, 128), (28, 4, 128), (14, 2, 64), (32, 32, 64), (20, 1, 64), (12, 4, 64), (40, 8, 128)]


def draw(rng):
    kind = rng.choice(["axes", "axes", "pick", "pick", "pick", "attend", "attend", "attend", "attend"])
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice([16, 16, 16, 32, 64])
    if kind == "axes":
        store = rng.random() < 0.7
        if not store:
            hq = hkv = 16
            d = rng.choice([72, 80, 64, 128])
            a = d // 4
            return dict(kind=kind, tokens=_log(rng, 4, 8000), hq=hq, hkv=hkv, d=d, sections=f"{a} {d // 2 - a}", mixed=False, norm=False, store=False, page=16)
        a, b = rng.choice([(d // 8, 3 * d // 16), (3 * d // 16, 5 * d // 32), (d // 4, d // 8)])
        return dict(kind=kind, tokens=_log(rng, 1, 8000), hq=hq, hkv=hkv, d=d, sections=f"{d // 2 - 2 * b} {b} {b}", mixed=d // 2 - 2 * b >= b and rng.random() < 0.5,
                    norm=rng.random() < 0.4, store=True, page=page)
    group = hq // hkv
    shape = rng.choice(["step", "step", "few", "chunk"])
    top = _log(rng, 4, 256 * 16 // page)
    case = dict(kind=kind, hq=hq, hkv=hkv, d=d, page=page, top=top, first=rng.choice([0, 1, 1, 4]), last=rng.choice([1, 2, 2, 5]))
    if kind == "attend":
        case["softcap"] = rng.choice([0.0, 0.0, 0.0, 30.0])
    if shape == "chunk":
        run = rng.choice([r for r in (1, 8, 16, 32) if r * group <= 128])
        queries = _log(rng, 20, 2000 if run >= 8 else 400)
        least = rng.choice([0, _log(rng, 100, 30000)])
        return dict(case, sequences=1, queries=queries, run=run, least=least, most=least)
    n = _log(rng, 1, 48)
    queries = 1 if shape == "step" else rng.randint(2, 9)
    run = 1 if shape == "step" or queries * group > 128 else rng.choice([1, queries])
    cap = min(120000, 500000 // n)
    least = _log(rng, 3, cap)
    return dict(case, sequences=n, queries=queries, run=run, least=least, most=min(cap, least + _log(rng, 1, 4000)))


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed, n):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + n)


def _normal(g, *size):
    return torch.empty(*size, device="cuda").normal_(generator=g)


def _channels(g, hkv, d):
    """How large the channels of keys are: a few stand out, as in trained models."""
    size = _normal(g, hkv, d).mul_(0.5).exp_()
    return torch.where(torch.rand(hkv, d, device="cuda", generator=g) < 0.03, size * 8, size)


def _lens(case):
    """Queries and keys of every sequence; the keys count the queries."""
    n = case["sequences"]
    before = torch.randint(case["least"], case["most"] + 1, (n,), generator=torch.Generator().manual_seed(case["least"] + 1000003 * n)).tolist()
    each = [case["queries"]] * n if n == 1 or case["queries"] == 1 else [max(1, case["queries"] - i % 3) for i in range(n)]
    return each, [a + b for a, b in zip(each, before)]


def _width(case):
    return case["first"] + case["top"] + case["last"] + (case["run"] + case["page"] - 2) // case["page"]


def _table(lens, page, seed):
    """Page ids of every sequence, shuffled over the pool as a running engine leaves them."""
    pages = [-(-n // page) for n in lens]
    order = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(seed + 3)).to(torch.int32)
    table, at = torch.zeros(len(lens), max(pages), dtype=torch.int32), 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    return table.cuda(), at


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sections(case):
    """Pairs that every axis turns."""
    return [int(x) for x in case["sections"].split()]


def _axes_of(sections, mixed):
    """The axis of every pair: sections one after the other, or taking turns while an axis has pairs left, then the first axis."""
    if not mixed:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    got = [0] * sum(sections)
    for j in range(len(got)):
        a = j % len(sections)
        if a and j // len(sections) < sections[a]:
            got[j] = a
    return got


def prepare(case, seed):
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    g = _gen(seed, 2)
    if case["kind"] == "axes":
        t, sections = case["tokens"], _sections(case)
        x = _normal(g, t, hq + 2 * hkv, d)
        x[:, hq:hq + hkv] *= _channels(g, hkv, d)
        pairs = sum(sections)
        if len(sections) == 3:       # film behind some text: frames of 20 rows and 27 columns
            i = torch.arange(t, device="cuda")
            first = 17 + seed % 1000
            pos = torch.stack([first + i // 540, first + i // 27 % 20, first + i % 27])
            freq = THETA ** (-torch.arange(0, 2 * pairs, 2, dtype=torch.float64) / (2 * pairs))
        else:                        # patches of one picture, 70 in a row
            i = torch.arange(t, device="cuda")
            pos = torch.stack([i // 70, i % 70])
            half = sections[0]
            freq = 10000.0 ** (-torch.arange(0, 2 * pairs, 2, dtype=torch.float64) / (2 * pairs) * 2)
            freq = torch.cat([freq[:half], freq[:pairs - half]])
        state = dict(case=case, qkv=x.to(torch.bfloat16).reshape(t, -1), positions=pos.to(torch.int32), freq=freq.float().cuda(), axes=_ints(_axes_of(sections, case["mixed"])),
                     q_norm=None, k_norm=None, k_cache=None, v_cache=None, slots=None)
        if case["norm"]:
            state["q_norm"], state["k_norm"] = ((1 + 0.1 * _normal(g, d)).to(torch.bfloat16) for _ in "qk")
        if case["store"]:
            pages = -(-t // page) + 1
            order = torch.randperm(pages, generator=g, device="cuda")
            at = torch.arange(t, device="cuda") + page // 2
            state["slots"] = order[at // page] * page + at % page
            state["k_cache"], state["v_cache"] = (torch.zeros(pages, hkv, page, d, dtype=torch.bfloat16, device="cuda") for _ in "kv")
        return state
    each, lens = _lens(case)
    table, pages = _table(lens, page, seed)
    q = _normal(g, sum(each), hq, d).to(torch.bfloat16)
    k = _normal(g, pages, hkv, page, d).mul_(_channels(g, hkv, d)[:, None]).to(torch.bfloat16)
    cu = [0]
    for n in each:
        cu.append(cu[-1] + n)
    state = dict(case=case, q=q, k_cache=k, table=table, kv_lens=_ints(lens), cu_q=_ints(cu), each=each, lens=lens, most=max(each))
    if case["kind"] == "pick":
        state["bounds"] = torch.zeros(pages, hkv, 2 * d + 16, dtype=torch.uint8, device="cuda")
        for i, (m, n) in enumerate(zip(each, lens)):       # of the pages that were full before
            _bound(state, i, 0, (n - m) // page)
        return state
    state["v_cache"] = _normal(g, pages, hkv, page, d).mul_(0.3).to(torch.bfloat16)
    rows, runs = _rows(state), -(-state["most"] // case["run"])
    score = torch.rand(len(each), runs, hkv, table.shape[1], generator=g, device="cuda")
    state["picked"] = _keep(state, score)
    assert state["picked"].shape[0] == rows
    return state


# ------------------------------------------------------------------------------------------ the plain forms
def _axes(s):
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    x = s["qkv"].reshape(-1, hq + 2 * hkv, d).float()
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if s["q_norm"] is not None:
        q = q * (1 / (q.square().mean(-1, keepdim=True) + 1e-6).sqrt()) * s["q_norm"].float()
        k = k * (1 / (k.square().mean(-1, keepdim=True) + 1e-6).sqrt()) * s["k_norm"].float()
    angle = s["positions"].double()[s["axes"].long()].T * s["freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half = s["freq"].numel()

    def turn(y):
        a, b = y[..., :half], y[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]], -1).to(torch.bfloat16)

    q, k, v = turn(q), turn(k), v.to(torch.bfloat16)
    if s["k_cache"] is None:
        return q, k, v
    page, off = s["slots"] // c["page"], s["slots"] % c["page"]
    s["k_cache"][page, :, off] = k
    s["v_cache"][page, :, off] = v
    return q, s["k_cache"], s["v_cache"]


def _exponent(top):
    """The smallest e, from -50 to 50, with top <= 127 * 2^e."""
    m, x = torch.frexp(top)
    e = x - 7 + (m * 2 > 127 / 64)
    return torch.where(top > 0, e, -50).clamp(-50, 50).int()


def _bound(s, i, a, b):
    """Bounds of pages a .. b of sequence i."""
    if a >= b:
        return
    ids = s["table"][i, a:b].long()
    k = s["k_cache"][ids].float().nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf)
    high, low = k.amax(2), k.amin(2)
    e = _exponent(torch.maximum(high.abs(), low.abs()).amax(-1))
    f = torch.exp2(-e.float())[..., None]
    codes = torch.cat([torch.ceil(high * f), torch.floor(low * f)], -1).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    s["bounds"][ids] = torch.cat([codes, (e + 64).to(torch.uint8)[..., None], torch.zeros_like(codes[..., :15])], -1)


def _rows(s):
    run = s["case"]["run"]
    return (s["q"].shape[0] + len(s["each"]) * (run - 1)) // run


def _padded(s):
    """Token of query j of sequence i, where it has one: [S, runs * run] and its mask."""
    c = s["case"]
    runs = -(-s["most"] // c["run"])
    j = torch.arange(runs * c["run"], device="cuda")
    cu = s["cu_q"].long()
    on = j < (cu[1:] - cu[:-1])[:, None]
    return torch.where(on, cu[:-1, None] + j, 0), on


def _keep(s, score):
    """Rows of kept pages from scores [S, runs, hkv, pages]."""
    c = s["case"]
    run, page, width = c["run"], c["page"], _width(c)
    n, runs, hkv, pages = score.shape
    cu, lens = s["cu_q"].long(), s["kv_lens"].long()
    count = cu[1:] - cu[:-1]
    r = torch.arange(runs, device="cuda")
    begin = (lens - count)[:, None] + r * run                       # [S, runs] position of a run's first query
    end = torch.minimum(begin + run, lens[:, None]) - 1
    at = torch.arange(pages, device="cuda")
    page0, page1 = (begin // page)[..., None], (end // page)[..., None]
    seen = at <= page1
    between = (at >= c["first"]) & (at <= page0 - c["last"])
    kept = seen & ~between
    score = torch.where(between[:, :, None], score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :min(c["top"], pages)]
    best = torch.zeros_like(score, dtype=torch.bool).scatter_(-1, order, True)
    kept = kept[:, :, None] | (best & between[:, :, None])
    out = torch.full((_rows(s), hkv, width), -1, dtype=torch.int32, device="cuda")
    place = torch.cumsum(kept, -1) - 1
    to = (cu[:-1, None] + torch.arange(n, device="cuda")[:, None] * (run - 1)) // run + r
    on = (r * run < count[:, None])[:, :, None, None] & kept
    i, j, h, p = on.nonzero(as_tuple=True)
    out[to[i, j], h, place[i, j, h, p]] = p.int()
    return out


def _pick(s):
    c = s["case"]
    hq, hkv, d, page, run = c["hq"], c["hkv"], c["d"], c["page"], c["run"]
    for i, (m, n) in enumerate(zip(s["each"], s["lens"])):
        _bound(s, i, (n - m) // page, n // page)
    rows = s["bounds"][s["table"].long()]                            # [S, pages, hkv, bytes]
    codes = rows[..., :2 * d].contiguous().view(torch.int8).float().permute(0, 2, 3, 1)
    factor = torch.exp2(rows[..., 2 * d].float() - 64).permute(0, 2, 1)
    q = s["q"].float().nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf)
    e = _exponent(q.abs().amax(-1))
    a = torch.round(q * torch.exp2(-e.float())[..., None]).clamp(-127, 127)
    a = torch.cat([a.clamp(min=0), a.clamp(max=0)], -1)
    at, on = _padded(s)
    n, m = at.shape
    a = a[at].reshape(n, m, hkv, hq // hkv, 2 * d).permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, 2 * d)
    size = torch.where(on[..., None], torch.exp2(e.float())[at], 0).reshape(n, m, hkv, -1).permute(0, 2, 1, 3).reshape(n, hkv, -1, 1)
    score = torch.matmul(a, codes).mul_(size).reshape(n, hkv, m // run, run, hq // hkv, -1)
    score.masked_fill_(~on.reshape(n, 1, m // run, run, 1, 1), -math.inf)
    score = score.amax((3, 4)) * factor[:, :, None]
    return _keep(s, score.permute(0, 2, 1, 3)), s["bounds"]


def _attend(s):
    c = s["case"]
    hq, hkv, d, page, run = c["hq"], c["hkv"], c["d"], c["page"], c["run"]
    at, on = _padded(s)
    n, m = at.shape
    runs = m // run
    cu = s["cu_q"].long()
    to = (cu[:-1, None] + torch.arange(n, device="cuda")[:, None] * (run - 1)) // run + torch.arange(runs, device="cuda")
    to = torch.where(torch.arange(runs, device="cuda") * run < (cu[1:] - cu[:-1])[:, None], to, 0).flatten()
    picked = s["picked"][to].long()                                  # [S * runs, hkv, width]
    seq = torch.arange(n, device="cuda").repeat_interleave(runs)
    pos = ((s["kv_lens"].long() - (cu[1:] - cu[:-1]))[:, None] + torch.arange(m, device="cuda")).reshape(n * runs, run)
    at, on = at.reshape(n * runs, run), on.reshape(n * runs, run)
    out = torch.zeros_like(s["q"])
    slab = max(1, (1 << 28) // (hkv * picked.shape[2] * page * max(d, run * hq // hkv)))
    head = torch.arange(hkv, device="cuda")[None, :, None]
    for x in range(0, n * runs, slab):
        w = slice(x, x + slab)
        ids = s["table"][seq[w, None, None], picked[w].clamp(min=0)].long()
        k, v = (y[ids, head].flatten(2, 3).float() for y in (s["k_cache"], s["v_cache"]))        # [slab, hkv, keys, d]
        key = (picked[w][..., None] * page + torch.arange(page, device="cuda")).flatten(2)
        key = torch.where(picked[w].repeat_interleave(page, -1) >= 0, key, 1 << 40)
        q = s["q"].float()[at[w]].reshape(-1, run, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4)
        score = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)).mul_(d ** -0.5)
        if c["softcap"] > 0:
            score.div_(c["softcap"]).tanh_().mul_(c["softcap"])
        score = score.reshape(*q.shape[:4], -1)
        score.masked_fill_((key[:, :, None] > pos[w, None, :, None])[:, :, :, None], -math.inf)
        score.sub_(score.amax(-1, keepdim=True)).exp_()
        score.div_(score.sum(-1, keepdim=True))
        o = torch.matmul(score.flatten(2, 3), v).reshape(q.shape).permute(0, 2, 1, 3, 4).reshape(-1, run, hq, d)
        out[at[w][on[w]]] = o[on[w]].to(torch.bfloat16)
    return out


def run(state):
    c = state["case"]
    if own:
        from hartsyinference_b200 import ops
        if c["kind"] == "axes":
            q, k, v = ops.rope_axes_kv(state["qkv"], state["positions"], c["hq"], c["hkv"], c["d"], axes=state["axes"], inv_freq=state["freq"], k_cache=state["k_cache"],
                                       v_cache=state["v_cache"], slot_mapping=state["slots"], q_norm_w=state["q_norm"], k_norm_w=state["k_norm"], eps=1e-6,
                                       want_kv=state["slots"] is None)
            return (q, k, v) if state["slots"] is None else (q, state["k_cache"], state["v_cache"])
        step = c["queries"] == 1
        cu_q = None if step else state["cu_q"]
        if c["kind"] == "pick":
            ops.key_bounds_(state["bounds"], state["k_cache"], state["table"], state["kv_lens"], cu_q, state["most"])
            return ops.pick_pages(state["q"], state["bounds"], state["table"], state["kv_lens"], cu_q, page=c["page"], top=c["top"], first=c["first"], last=c["last"],
                                  run=c["run"]), state["bounds"]
        return ops.attn_picked(state["q"], state["k_cache"], state["v_cache"], state["table"], state["kv_lens"], state["picked"], cu_q, run=c["run"], softcap=c["softcap"])
    return {"axes": _axes, "pick": _pick, "attend": _attend}[c["kind"]](state)


# ------------------------------------------------------------------------------------------ least work
def _runs(case):
    """(first position, tokens) of every run, with its sequence."""
    for i, (m, n) in enumerate(zip(*_lens(case))):
        for a in range(0, m, case["run"]):
            yield i, n - m + a, min(case["run"], m - a)


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["kind"] == "axes":
        t = case["tokens"]
        return dict(bytes=t * ((hq + 2 * hkv) * d * 4 + 4 * len(_sections(case))), flops=t * (hq + hkv) * sum(_sections(case)) * 6)
    each, lens = _lens(case)
    page = case["page"]
    if case["kind"] == "pick":
        flops, widest = 0, [0] * len(each)
        for i, p, t in _runs(case):
            n = max(0, p // page - case["last"] + 1 - case["first"])
            if n > case["top"]:
                flops += 4 * d * n * t * hq
                widest[i] = max(widest[i], n)
        new = sum(n // page - (n - m) // page for m, n in zip(each, lens))
        return dict(bytes=sum(widest) * hkv * (2 * d + 1) + new * hkv * (page * d * 2 + 2 * d) + sum(each) * hq * d * 2, flops=flops)
    pairs, keys = 0, [0] * len(each)
    for i, p, t in _runs(case):
        middle = max(0, p // page - case["last"] + 1 - case["first"])
        left = max(0, middle - case["top"]) * page                    # keys in front of the run that it leaves out
        pairs += sum(p + j + 1 - left for j in range(t))
        keys[i] += p + t - left
    distinct = sum(min(a, n) for a, n in zip(keys, lens))
    return dict(bytes=distinct * hkv * d * 4 + 2 * sum(each) * hq * d * 2, flops=4 * pairs * hq * d)


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_axes(s):
    c = s["case"]
    hq, hkv, d, half = c["hq"], c["hkv"], c["d"], s["freq"].numel()
    x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    axis = torch.tensor(_axes_of(_sections(c), c["mixed"]), device="cuda")
    angle = torch.stack([s["positions"][a].double() * f for a, f in zip(axis.tolist(), s["freq"].tolist())], -1)
    out = x.clone()
    for first, last, w in ((0, hq, s["q_norm"]), (hq, hq + hkv, s["k_norm"])):
        y = x[:, first:last]
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / d + 1e-6) * w.double()
        z = torch.complex(y[..., :half], y[..., half:2 * half]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        out[:, first:last, :half], out[:, first:last, half:2 * half], out[:, first:last, 2 * half:] = z.real, z.imag, y[..., 2 * half:]
    q, k, v = out[:, :hq], out[:, hq:hq + hkv], out[:, hq + hkv:]
    if s["slots"] is None:
        return q, k, v
    pools = []
    for y, pool in ((k, s["k_cache"]), (v, s["v_cache"])):
        flat = torch.zeros(pool.shape[0] * c["page"], hkv, d, dtype=torch.float64, device="cuda")
        flat[s["slots"]] = y
        pools.append(flat.view(-1, c["page"], hkv, d).transpose(1, 2))
    return q, *pools


def _codes(x, top):
    """x / 2^e in 64 bits, and 2^e: the smallest with top <= 127 * 2^e."""
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 127)).clamp(-50, 50)
    e = torch.where((top <= 127 * torch.exp2(e - 1)) & (e > -50), e - 1, torch.where((top > 127 * torch.exp2(e)) & (e < 50), e + 1, e))
    return x / torch.exp2(e)[..., None], torch.exp2(e)


def _exact_pick(s):
    c = s["case"]
    hq, hkv, d, page, width = c["hq"], c["hkv"], c["d"], c["page"], _width(c)
    group = hq // hkv
    out, cu, before = torch.full((_rows(s), hkv, width), -1, dtype=torch.int32), s["cu_q"].tolist(), None
    bounds = torch.zeros_like(s["bounds"], dtype=torch.int64)
    for i, p, t in _runs(c):
        if i != before:
            ids = s["table"][i, :s["lens"][i] // page].long()
            k = s["k_cache"][ids].double()
            high, low = k.max(2).values, k.min(2).values
            top = torch.maximum(high, -low).max(-1).values
            (up, unit), (down, _) = _codes(high, top), _codes(low, top)
            bounds[ids, :, :d], bounds[ids, :, d:2 * d], bounds[ids, :, 2 * d] = up.ceil().long() % 256, down.floor().long() % 256, torch.log2(unit).long() + 64
            up, down, before, row = up.ceil().int(), down.floor().int(), i, (cu[i] + i * (c["run"] - 1)) // c["run"]
        begin = cu[i] + p - (s["lens"][i] - s["each"][i])
        own_page, last_page = p // page, (p + t - 1) // page
        between = list(range(c["first"], max(c["first"], own_page - c["last"] + 1)))
        ends = [x for x in range(last_page + 1) if x < c["first"] or x > own_page - c["last"]]
        for h in range(hkv):
            kept = between
            if len(between) > c["top"]:
                q = s["q"][begin:begin + t, h * group:(h + 1) * group].reshape(-1, d).double()
                a, size = _codes(q, q.abs().max(-1).values)
                a, best = a.round().int(), None
                hi, lo = up[between[0]:between[-1] + 1, h], down[between[0]:between[-1] + 1, h]
                step = max(1, (1 << 28) // (hi.shape[0] * d))
                for x in range(0, a.shape[0], step):
                    y = a[x:x + step, None]
                    total = torch.maximum(y * hi, y * lo).sum(-1).double() * size[x:x + step, None]
                    total = total.max(0).values
                    best = total if best is None else torch.maximum(best, total)
                best = best * unit[between[0]:between[-1] + 1, h]
                kept = (torch.argsort(-best, stable=True)[:c["top"]] + between[0]).tolist()
            got = sorted(set(ends) | set(kept))
            out[row, h, :len(got)] = torch.tensor(got, dtype=torch.int32)
        row += 1
    return out.cuda(), bounds.to(torch.uint8)


def _exact_attend(s):
    c = s["case"]
    hq, hkv, d, page, group = c["hq"], c["hkv"], c["d"], c["page"], c["hq"] // c["hkv"]
    out, cu, before = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), s["cu_q"].tolist(), None
    picked = s["picked"].cpu()
    for i, p, t in _runs(c):
        if i != before:
            before, row = i, (cu[i] + i * (c["run"] - 1)) // c["run"]
        begin = cu[i] + p - (s["lens"][i] - s["each"][i])
        counts = (picked[row] >= 0).sum(-1).tolist()
        for h in range(hkv):
            mine = picked[row, h, :counts[h]].long().cuda()
            ids = s["table"][i, mine].long()
            k, v = (y[ids, h].reshape(-1, d).double() for y in (s["k_cache"], s["v_cache"]))
            key = (mine[:, None] * page + torch.arange(page, device="cuda")).flatten()
            q = s["q"][begin:begin + t, h * group:(h + 1) * group].double()
            score = torch.einsum("tgd,kd->tgk", q, k) / math.sqrt(d)
            if c["softcap"] > 0:
                score = torch.tanh(score / c["softcap"]) * c["softcap"]
            off = key > torch.arange(p, p + t, device="cuda")[:, None, None]
            weight = torch.exp(score - torch.where(off, -math.inf, score).max(-1, keepdim=True).values) * ~off
            out[begin:begin + t, h * group:(h + 1) * group] = torch.einsum("tgk,kd->tgd", weight / weight.sum(-1, keepdim=True), v)
        row += 1
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"axes": _exact_axes, "pick": _exact_pick, "attend": _exact_attend}[case["kind"]](s)
