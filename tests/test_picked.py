"""Attention over chosen pages: bounds of keys, the choice, attention over it.

Bounds and the choice are whole-number arithmetic and have to be equal; attention is held to a plain implementation in 64 bits (bounds in ``_attention``)."""
import math

import pytest
import torch

from hartsyinference_b200 import ops
from hartsyinference_b200.ops import _native as N
from hartsyinference_b200.ops import reference as R

gpu = pytest.mark.gpu
BOTH = ["cpu", pytest.param("cuda", marks=gpu)]


def _normal(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


class Batch:
    """Sequences of ``each`` new tokens, the last of ``lens`` that a shuffled pool holds; what lies behind a sequence's end is NaN, table entries
    behind its last page name none."""

    def __init__(self, each, lens, hq, hkv, d, page, seed=0, extra=1, special=True):
        self.each, self.lens, self.hq, self.hkv, self.d, self.page = each, lens, hq, hkv, d, page
        per = [-(-n // page) for n in lens]
        order = torch.randperm(sum(per) + 2, generator=torch.Generator().manual_seed(seed)).int()
        self.table, at = torch.full((len(lens), max(max(per), 1) + extra), -9, dtype=torch.int32), 0
        self.k, self.v = (torch.full((sum(per) + 2, hkv, page, d), math.nan, dtype=torch.bfloat16) for _ in "kv")
        for i, (n, m) in enumerate(zip(lens, per)):
            self.table[i, :m] = order[at:at + m]
            at += m
            if n:
                pos = torch.arange(n)
                ids = self.table[i, pos // page].long()
                k = _normal(n, hkv, d, seed=seed + 3 * i + 1) * (1 + 7 * (torch.arange(d) % 37 == 3))
                self.k[ids, :, pos % page] = k.to(torch.bfloat16)
                self.v[ids, :, pos % page] = _normal(n, hkv, d, seed=seed + 3 * i + 2).to(torch.bfloat16)
        self.kv_lens = torch.tensor(lens, dtype=torch.int32)
        self.cu_q = torch.tensor([0] + each, dtype=torch.int32).cumsum(0, dtype=torch.int32)
        self.q = _normal(sum(each), hq, d, seed=seed + 100).to(torch.bfloat16)
        self.bounds = ops.key_bounds(self.k.shape[0], hkv, d, "cpu")

    def fill_bounds(self):
        """Of every full page."""
        ops.key_bounds_(self.bounds, self.k, self.table, self.kv_lens, torch.tensor([0] + self.lens).cumsum(0, dtype=torch.int32), max(self.lens + [1]))
        return self

    def to(self, dev):
        for name in ("table", "k", "v", "kv_lens", "cu_q", "q", "bounds"):
            setattr(self, name, getattr(self, name).to(dev))
        return self

    def pick(self, step=False, **kw):
        return ops.pick_pages(self.q, self.bounds, self.table, self.kv_lens, None if step else self.cu_q, page=self.page, **kw)

    def attend(self, picked, step=False, **kw):
        return ops.attn_picked(self.q, self.k, self.v, self.table, self.kv_lens, picked, None if step else self.cu_q, **kw)


# each, lens: single tokens, empty ones, ends inside a page and on its border, chunks, sequences without new tokens, more queries than keys
BATCHES = [([1, 1, 1, 1], [1, 0, 17, 700]), ([5, 0, 3], [300, 40, 3]), ([70], [333]), ([1], [4100]), ([2, 4, 1, 33], [512, 1, 129, 640]), ([0, 9, 0], [0, 900, 16])]
HEADS = [(14, 2, 64), (8, 1, 128), (3, 3, 64), (40, 2, 128), (28, 4, 128), (33, 1, 64), (100, 1, 128)]


# ------------------------------------------------------------------------------------------ bounds
def _bound_by_hand(k):
    """Of keys [page, d]."""
    k = [[0.0 if math.isnan(x) else x for x in row] for row in k.tolist()]
    high, low = [max(c) for c in zip(*k)], [min(c) for c in zip(*k)]
    top = max(max(map(abs, high)), max(map(abs, low)))
    e = next((e for e in range(-50, 50) if top <= 127 * 2.0 ** e), 50)
    cut = lambda x: max(-127, min(127, x))
    up = [cut(math.ceil(x / 2.0 ** e)) if math.isfinite(x) else math.copysign(127, x) for x in high]
    down = [cut(math.floor(x / 2.0 ** e)) if math.isfinite(x) else math.copysign(127, x) for x in low]
    return [int(x) % 256 for x in up + down] + [e + 64] + [0] * 15


@pytest.mark.parametrize("dev", BOTH)
@pytest.mark.parametrize("d,page,hkv", [(64, 16, 3), (128, 16, 1), (128, 32, 2), (64, 64, 1), (128, 128, 2), (64, 128, 3)])
def test_bounds_are_those_of_the_pages_that_new_tokens_filled(dev, d, page, hkv):
    lens, each = [page - 1, page, 5 * page + 3, 0, 3 * page, 4 * page + 1], [1, 1, 2 * page + 9, 0, page, 1]
    b = Batch(each, lens, hkv, hkv, d, page)
    k = b.k[b.table[2, 4]]                                   # a page of odd values: none, one, too large, too small
    k[0], k[0, 3, 5], k[0, 1, 6] = math.nan, math.inf, 1e30
    if hkv > 1:
        k[1] = 0.0
    if hkv > 2:
        k[2] *= 1e-30
    b.to(dev)
    before = b.bounds.fill_(77).clone().cpu()
    ops.key_bounds_(b.bounds, b.k, b.table, b.kv_lens, b.cu_q, max(each))
    got, filled = b.bounds.cpu(), set()
    for i, (m, n) in enumerate(zip(each, lens)):
        for j in range((n - m) // page, n // page):
            at = int(b.table[i, j])
            filled.add(at)
            for h in range(hkv):
                assert got[at, h].tolist() == _bound_by_hand(b.k[at, h].double().cpu()), (i, j, h)
    rest = [x for x in range(got.shape[0]) if x not in filled]
    assert len(filled) == 1 + 3 + 1 and torch.equal(got[rest], before[rest])
    if dev == "cuda":
        N.check_status()


@pytest.mark.parametrize("dev", BOTH)
def test_single_tokens_bound_a_page_when_they_fill_it(dev):
    b = Batch([1, 1, 1], [32, 31, 33], 2, 2, 64, 16).to(dev)
    ops.key_bounds_(b.bounds, b.k, b.table, b.kv_lens)
    assert b.bounds.any(-1).any(-1).sum() == 1 and b.bounds[b.table[0, 1].long()].any()


# ------------------------------------------------------------------------------------------ the choice
def _pick_by_hand(b, top, first, last, run):
    """Rows of kept pages with products in whole numbers, one run at a time."""
    width = first + top + last + (run + b.page - 2) // b.page
    out = torch.full(((b.q.shape[0] + len(b.each) * (run - 1)) // run, b.hkv, width), -1, dtype=torch.int32)
    group, at = b.hq // b.hkv, 0
    for i, (m, n) in enumerate(zip(b.each, b.lens)):
        for r in range(-(-m // run)):
            tokens = [t for t in range(r * run, min(m, (r + 1) * run)) if n - m + t >= 0]
            if not tokens:
                continue
            p0, p1 = n - m + tokens[0], n - m + tokens[-1]
            middle = [x for x in range(p1 // b.page + 1) if x >= first and x <= p0 // b.page - last]
            for h in range(b.hkv):
                best = middle
                if len(middle) > top:
                    rows = b.bounds[b.table[i, middle].long(), h]
                    high, low = rows[:, :b.d].view(torch.int8).long(), rows[:, b.d:2 * b.d].view(torch.int8).long()
                    unit = rows[:, 2 * b.d].double() - 64
                    score = torch.full((len(middle),), -math.inf, dtype=torch.float64)
                    for t in tokens:
                        for x in range(h * group, (h + 1) * group):
                            q = torch.nan_to_num(b.q[at + t, x].double(), nan=0.0, posinf=1e38, neginf=-1e38)
                            peak = float(q.abs().max())
                            e = next((e for e in range(-50, 50) if peak <= 127 * 2.0 ** e), 50)
                            a = torch.round(q / 2.0 ** e).clamp(-127, 127).long()
                            score = torch.maximum(score, torch.maximum(a * high, a * low).sum(-1).double() * 2.0 ** e)
                    score = score * 2.0 ** unit
                    best = [middle[x] for x in sorted(range(len(middle)), key=lambda x: (-float(score[x]), x))[:top]]
                kept = sorted(set(range(p1 // b.page + 1)) - set(middle) | set(best))
                out[(at + i * (run - 1)) // run + r, h, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
        at += m
    return out


@pytest.mark.parametrize("each,lens", BATCHES)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (5, 1, 128)])
@pytest.mark.parametrize("top,first,last,run", [(3, 1, 2, 1), (7, 0, 1, 4), (0, 2, 3, 16), (40, 3, 1, 3)])
def test_the_choice_on_the_host(each, lens, hq, hkv, d, top, first, last, run):
    b = Batch(each, lens, hq, hkv, d, 16, seed=top).fill_bounds()
    got = b.pick(top=top, first=first, last=last, run=run)
    assert torch.equal(got, _pick_by_hand(b, top, first, last, run))


@gpu
@pytest.mark.parametrize("each,lens", BATCHES)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("top,first,last,run,page", [(3, 1, 2, 1, 16), (7, 0, 1, 4, 32), (0, 2, 3, 16, 16), (20, 3, 1, 3, 16), (2, 0, 1, 1, 128), (5, 1, 1, 9, 64)])
def test_the_choice_is_that_of_the_host(each, lens, hq, hkv, d, top, first, last, run, page):
    run = min(run, 128 // (hq // hkv))
    b = Batch(each, lens, hq, hkv, d, page, seed=top).fill_bounds()
    want = b.pick(top=top, first=first, last=last, run=run)
    got = b.to("cuda").pick(top=top, first=first, last=last, run=run)
    assert torch.equal(got.cpu(), want)
    N.check_status()


@gpu
@pytest.mark.parametrize("hq,hkv,d,run", [(14, 2, 64, 18), (8, 1, 128, 16), (28, 4, 128, 5), (100, 1, 128, 1), (33, 1, 64, 3), (40, 2, 128, 6)])
@pytest.mark.parametrize("each,lens", [([2500, 0, 3, 1], [2900, 50, 3000, 1]), ([17, 2600], [17, 2650])])
def test_the_choice_of_many_runs_is_that_of_the_host(each, lens, hq, hkv, d, run):
    """More rows than processors, so that tiles of queries score them: runs in pairs of a sequence, one by themselves at its end, sequences of a token."""
    if run < 16:
        each = [m // (2 if run > 2 else 8) for m in each]
        each = [max(m, 1) if n else 0 for m, n in zip(each, lens)]
    b = Batch(each, lens, hq, hkv, d, 16, seed=run).fill_bounds()
    assert ((sum(each) + len(each) * (run - 1)) // run) * hkv > 148
    want = b.pick(top=9, run=run)
    assert torch.equal(b.to("cuda").pick(top=9, run=run).cpu(), want)
    N.check_status()


@gpu
@pytest.mark.parametrize("front,behind", [(0, 0), (50, 0), (0, 700), (3, 21)])
@pytest.mark.parametrize("run,group", [(5, 4), (16, 4), (16, 2), (21, 6)])
def test_the_choice_of_many_short_sequences_is_that_of_the_host(front, behind, run, group):
    """Sequences of no, one, two and three runs, whole ones and not, and rows of q that no sequence has: rows of no run lie between the others, and are -1 too."""
    each = [(17 * i + i // 5) % (2 * run + 7) if i % 7 else 0 for i in range(60)]
    b = Batch(each, [m + (37 * i) % 300 for i, m in enumerate(each)], 3 * group, 3, 64, 16, seed=run).fill_bounds()
    b.q = torch.cat([b.q[:1].expand(front, -1, -1), b.q, b.q[:1].expand(behind, -1, -1)])
    b.cu_q += front
    want = b.pick(top=4, run=run)
    assert want.shape[0] * 3 > 148 and (want == -1).all(-1).all(-1).sum() > len(each) // 3
    b.to("cuda")
    full_of_sevens = torch.full_like(want, 7, device="cuda")
    del full_of_sevens                               # its memory is likely to be the result's
    assert torch.equal(b.pick(top=4, run=run).cpu(), want)
    N.check_status()


@gpu
@pytest.mark.parametrize("pages,extra,top", [(3000, 0, 100), (9000, 3000, 1), (9000, 0, 2500), (2100, 60000, 300)])
def test_a_long_table_is_shared_by_blocks(pages, extra, top):
    """One sequence; wide tables whose scores no single block holds. Bounds are random bytes."""
    hkv, d, page = 2, 64, 16
    g = torch.Generator().manual_seed(pages)
    b = Batch([1], [5], 2 * hkv, hkv, d, page)
    b.bounds = torch.randint(0, 256, (pages, hkv, 2 * d + 16), generator=g, dtype=torch.uint8)
    b.bounds[..., 2 * d] = torch.randint(58, 62, (pages, hkv), generator=g, dtype=torch.uint8)
    b.table = torch.full((1, pages + extra), -1, dtype=torch.int32)
    b.table[0, :pages] = torch.randperm(pages, generator=g).int()
    b.kv_lens[0] = pages * page - 3
    want = b.pick(step=True, top=top, first=1, last=2)
    assert torch.equal(b.to("cuda").pick(step=True, top=top, first=1, last=2).cpu(), want)
    N.check_status()


@pytest.mark.parametrize("dev", BOTH)
@pytest.mark.parametrize("pages", [70, 2600])
def test_ties_go_to_the_lowest_page(dev, pages):
    b = Batch([1], [5], 4, 2, 64, 16)
    b.bounds = torch.zeros(pages, 2, 144, dtype=torch.uint8)
    b.bounds[..., :64], b.bounds[..., 128] = 9, 64
    b.bounds[41, 1, :64] = 10                              # one page above the others for the second head
    b.table = torch.arange(pages, dtype=torch.int32)[None]
    b.kv_lens[0] = pages * 16
    b.q = b.q.abs()
    got = b.to(dev).pick(step=True, top=6, first=2, last=3).cpu()[0]
    ends = list(range(pages - 3, pages))
    assert got.tolist() == [[0, 1, *range(2, 8), *ends], [0, 1, *range(2, 7), 41, *ends]]


@pytest.mark.parametrize("dev", BOTH)
def test_queries_that_are_no_numbers_and_keys_of_every_size(dev):
    b = Batch([1, 1], [800, 800], 4, 2, 64, 16)
    b.q[0, 0, 3], b.q[0, 1], b.q[1, 2, 5], b.q[1, 3] = math.nan, 0.0, math.inf, 1e-38
    for j in range(40):
        b.k[b.table[0, j].long()] *= 10.0 ** (j - 20)
    b.fill_bounds()
    want = _pick_by_hand(b, 5, 1, 1, 1)
    assert torch.equal(b.to(dev).pick(step=True, top=5, first=1, last=1).cpu(), want)


def test_a_score_is_a_bound_of_the_products():
    """With the query's codes in place of the query: the highest product of a page's keys lies at or below its score."""
    b = Batch([1], [640], 4, 1, 64, 16).fill_bounds()
    q = b.q.float()
    e = R.bounds_exponent(q.abs().amax(-1))
    held = torch.round(q * torch.exp2(-e.float())[..., None]) * torch.exp2(e.float())[..., None]
    ids = b.table[0, :40].long()
    score = R.page_scores(b.q, b.bounds[ids])[0]
    products = torch.einsum("hd,ptd->pth", held[0].double(), b.k[ids, 0].double()).amax((1, 2))
    assert (products <= score.double()).all()


# ------------------------------------------------------------------------------------------ attention
def _attention(b, picked, run, scale=None, softcap=0.0):
    """In 64 bits, with the bound of what the kernels may be off by. Probabilities and the result are rounded to bf16: 2^-8 of sum p |v| and of
    the result. Scores are sums of up to 128 products in 32 bits, 8 or more at a time: off by 2^-19 of sum |q k| scale; a cap's by 2^-20 of it; exponentials by
    2^-20 of themselves. Such an error moves a probability and the sum that divides it: twice."""
    scale = 1 / math.sqrt(b.d) if scale is None else scale
    out, bound = torch.zeros(b.q.shape, dtype=torch.float64), torch.full(b.q.shape, 1e-30, dtype=torch.float64)
    group, at = b.hq // b.hkv, 0
    for i, (m, n) in enumerate(zip(b.each, b.lens)):
        for t in range(m):
            p = n - m + t
            if p < 0:
                continue
            row = (at + i * (run - 1)) // run + t // run
            for h in range(b.hkv):
                pages = [x for x in picked[row, h].tolist() if 0 <= x <= p // b.page]
                keys = torch.tensor([x * b.page + y for x in pages for y in range(b.page) if x * b.page + y <= p], dtype=torch.long)
                if not keys.numel():
                    continue
                ids = b.table[i, keys // b.page].long()
                k, v = (c[ids, h, keys % b.page].double() for c in (b.k, b.v))
                q = b.q[at + t, h * group:(h + 1) * group].double()
                s = q @ k.T * scale
                size = float((q.abs() @ k.abs().T).max()) * abs(scale)
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                w = torch.softmax(s, -1)
                o, a = w @ v, w @ v.abs()
                out[at + t, h * group:(h + 1) * group] = o
                bound[at + t, h * group:(h + 1) * group] += 2.0 ** -8 * 1.02 * (a + o.abs()) + 2 * (2.0 ** -19 * size + 2.0 ** -20 * (softcap + 1)) * a
        at += m
    return out, bound


def _close(got, want):
    out, bound = want
    assert torch.isfinite(got).all()
    off = (got.double().cpu() - out).abs()
    assert (off <= bound).all(), float((off / bound).max())


def _some(b, run, width, seed=0):
    """Rows of random pages, up to the run's last, in order; with entries behind it and none at all among them."""
    g = torch.Generator().manual_seed(seed)
    rows = (b.q.shape[0] + len(b.each) * (run - 1)) // run
    out, at = torch.full((rows, b.hkv, width), -1, dtype=torch.int32), 0
    for i, (m, n) in enumerate(zip(b.each, b.lens)):
        for r in range(-(-m // run)):
            last = max(0, n - m + min(m, (r + 1) * run) - 1) // b.page
            for h in range(b.hkv):
                mine = torch.randperm(last + 1, generator=g)[:max(1, width - 1 - h)].sort().values.int()
                out[(at + i * (run - 1)) // run + r, h, :mine.numel()] = mine
                if mine.numel() < width:
                    out[(at + i * (run - 1)) // run + r, h, mine.numel()] = last + 1 + h
        at += m
    return out


@pytest.mark.parametrize("dev", BOTH)
@pytest.mark.parametrize("each,lens", BATCHES)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("run,page,width,softcap", [(1, 16, 9, 0.0), (4, 32, 40, 0.0), (16, 16, 21, 30.0), (3, 128, 3, 0.0), (1, 64, 200, 5.0)])
def test_attention_over_the_chosen_pages(dev, each, lens, hq, hkv, d, run, page, width, softcap):
    if dev == "cpu" and (page == 16 or d == 128):
        return
    run = min(run, 128 // (hq // hkv))
    b = Batch(each, lens, hq, hkv, d, page, seed=width)
    picked = _some(b, run, width)
    want = _attention(b, picked, run, softcap=softcap)
    _close(b.to(dev).attend(picked.to(dev), run=run, softcap=softcap), want)
    if dev == "cuda":
        N.check_status()


@pytest.mark.parametrize("dev", BOTH)
def test_rows_without_pages_and_queries_in_front_of_their_pages_give_zeros(dev):
    b = Batch([4, 4], [40, 33], 4, 2, 64, 16)
    picked = torch.full((3, 2, 3), -1, dtype=torch.int32)
    picked[1, 0, 0] = 2                                    # the page of position 32 alone: the three queries in front of it see nothing
    got = b.to(dev).attend(picked.to(dev), run=4).cpu()
    assert not got[:7].any() and got[7, :2].any() and not got[7, 2:].any()


@gpu
@pytest.mark.parametrize("each,lens", BATCHES + [([130, 0, 61, 1], [700, 0, 61, 200])])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("page,width", [(16, 30), (32, 5), (64, 9), (128, 7), (16, 1000)])
@pytest.mark.parametrize("tiles", [0, 1])
def test_attention_of_long_runs(each, lens, hq, hkv, d, page, width, tiles, monkeypatch):
    """As many tokens a run as it may have, by each of the two kernels, whichever the rule would take for the size."""
    monkeypatch.setattr(N.lib(), "b200_attn_picked_form", lambda *a: tiles)
    run = 128 // (hq // hkv)
    b = Batch(each, lens, hq, hkv, d, page, seed=width)
    picked = _some(b, run, width)
    want = _attention(b, picked, run)
    _close(b.to("cuda").attend(picked.cuda(), run=run), want)
    N.check_status()


@gpu
@pytest.mark.parametrize("d,page", [(128, 16), (64, 128)])
@pytest.mark.parametrize("tiles", [0, 1])
def test_rows_of_a_long_run_that_begin_with_pages_they_do_not_see(d, page, tiles, monkeypatch):
    """A list that names the run's last page first, one twice, and none between: order does not matter, twice counts twice."""
    monkeypatch.setattr(N.lib(), "b200_attn_picked_form", lambda *a: tiles)
    b = Batch([90], [190], 2, 1, d, page)
    last = 189 // page
    odd = torch.tensor([last, -1, 0, 0, 5000, last - 1], dtype=torch.int32).expand(2, 1, -1).contiguous()
    want = _attention(b, odd, 64)
    _close(b.to("cuda").attend(odd.cuda(), run=64), want)


@pytest.mark.parametrize("dev,tiles", [("cpu", 0), pytest.param("cuda", 0, marks=gpu), pytest.param("cuda", 1, marks=gpu)])
@pytest.mark.parametrize("hq", [3, 8])
def test_values_that_a_query_does_not_see_may_be_anything(dev, tiles, hq, monkeypatch):
    """Infinite and no numbers in a run's own page: they reach the queries that see them and no others."""
    if dev == "cuda":
        monkeypatch.setattr(N.lib(), "b200_attn_picked_form", lambda *a: tiles)
    b = Batch([6], [38], hq, 1, 128, 16)
    want, bound = _attention(b, torch.tensor([[[0, 1, 2]]]), 6)
    b.v[b.table[0, 2].long(), 0, 4, 7] = math.inf          # position 36: the last two queries
    b.v[b.table[0, 2].long(), 0, 5, 9] = math.nan          # position 37: the last query
    b.k[b.table[0, 2].long(), 0, 5, 3] = math.nan
    got = b.to(dev).attend(torch.tensor([[[0, 1, 2]]], dtype=torch.int32, device=dev), run=6).double().cpu()
    off = (got - want).abs() <= bound
    assert off[:4].all() and (dev == "cpu" or got[5].isnan().all())       # (the host's statement gives zeros for a row of no numbers)
    assert (got[4, :, 7] == math.inf).all() and off[4, :, :7].all() and off[4, :, 8:].all()


@pytest.mark.parametrize("dev", BOTH)
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_a_query_that_is_no_number_gives_none(dev, softcap):
    b = Batch([1, 1], [700, 700], 4, 2, 64, 16)
    b.q[0, 1, 5] = math.nan
    got = b.to(dev).attend(_some(b, 1, 40).to(dev), step=True, softcap=softcap).cpu()
    if dev == "cuda":                                      # (the host's statement gives zeros for such a row)
        assert got[0, 1].isnan().all()
    assert torch.isfinite(got[0, [0, 2, 3]]).all() and torch.isfinite(got[1]).all()


# both kernels measured: tiles of 128 rows where they are faster
@pytest.mark.skipif(not N.available(), reason="kernels library not built")
@pytest.mark.parametrize("d,cols,rows,tiles", [(128, 16, 4000, 0), (128, 24, 144, 0), (128, 24, 192, 1), (128, 40, 64, 1), (128, 64, 16, 0), (128, 64, 32, 1), (128, 128, 1024, 1),
                                               (64, 35, 24, 0), (64, 35, 48, 1), (64, 112, 16, 0), (64, 112, 24, 1)])
def test_the_rule_between_the_kernels(d, cols, rows, tiles):
    form = N.lib().b200_attn_picked_form
    assert form(rows // 8, cols, 8, d, 16, 132, 10000, 0.1, 0.0) == tiles
    assert form(1024, 128, 8, d, 16, 1025, 10000, 0.1, 0.0) == form(1024, 128, 8, d, 16, 132, 10000, 0.1, 30.0) == form(1024, 128, 8, d, 16, 132, 10000, 0.0, 0.0) == 0


@pytest.mark.parametrize("dev", BOTH)
def test_all_pages_are_plain_attention(dev):
    """The choice of every page, and the attention of the whole cache beside it: both within their bound of the same values."""
    b = Batch([5, 1, 64], [90, 400, 64], 8, 2, 64, 16).fill_bounds()
    want = _attention(b, torch.arange(30, dtype=torch.int32).expand(70, 2, -1), 1)
    b.to(dev)
    picked = b.pick(top=30, run=4)
    _close(b.attend(picked, run=4), want)
    _close(ops.attn_prefill_paged(b.q, b.k.nan_to_num(), b.v.nan_to_num(), b.table.clamp(min=0), b.kv_lens, b.cu_q, 64), want)


@pytest.mark.parametrize("dev", BOTH)
def test_the_ops_together(dev):
    """As a model runs them: keys are stored chunk by chunk, bounded, chosen from; then single tokens, then a draft that is taken back."""
    hq, hkv, d, page, run = 8, 2, 64, 16, 4
    whole = Batch([0], [330], hq, hkv, d, page)
    kc, vc = (torch.full_like(whole.k, math.nan).to(dev) for _ in "kv")
    bounds, table = ops.key_bounds(kc.shape[0], hkv, d, dev).fill_(0), whole.table.to(dev)
    q = _normal(330, hq, d, seed=9).to(torch.bfloat16)
    k, v = (torch.stack([c[whole.table[0, p // page].long(), :, p % page] for p in range(330)]) for c in (whole.k, whole.v))
    freq = torch.ones(1)
    at = 0
    for count, kept in ((100, 100), (157, 157), (1, 1), (7, 3), (5, 5), (1, 1), (1, 1), (60, 60)):
        b = Batch([count], [at + count], hq, hkv, d, page)
        b.table, b.k, b.v, b.q = whole.table, whole.k, whole.v, q[at:at + count]
        pos = torch.arange(at, at + count)
        slots = (whole.table[0, pos // page].long() * page + pos % page).to(dev)
        drafted = count != kept                            # tokens that are not kept are others than those that follow
        packed = torch.cat([b.q, k[at:at + count] * (3 if drafted else 1), v[at:at + count]], 1).reshape(count, -1).to(dev)
        got_q, _, _ = ops.rope_axes_kv(packed, torch.zeros(1, count, dtype=torch.int32, device=dev), hq, hkv, d, axes=torch.zeros(1, dtype=torch.int32, device=dev),
                                       inv_freq=freq.to(dev), k_cache=kc, v_cache=vc, slot_mapping=slots)
        lens, cu = torch.tensor([at + count], dtype=torch.int32, device=dev), torch.tensor([0, count], dtype=torch.int32, device=dev)
        ops.key_bounds_(bounds, kc, table, lens, cu, count)
        picked = ops.pick_pages(got_q, bounds, table, lens, cu, page=page, top=4, run=run)
        out = ops.attn_picked(got_q, kc, vc, table, lens, picked, cu, run=run)
        if not drafted:
            b.bounds = ops.key_bounds(whole.k.shape[0], hkv, d, "cpu")
            b.fill_bounds()
            assert torch.equal(picked.cpu(), b.pick(top=4, run=run))
            _close(out, _attention(b, picked.cpu(), run))
            at += count
        # a draft is forgotten: its tokens are written again


@gpu
def test_single_tokens_and_their_rows_written_out_are_the_same():
    b = Batch([1, 1, 1], [700, 33, 5], 14, 2, 64, 16).fill_bounds().to("cuda")
    p, r = b.pick(step=True, top=5), b.pick(top=5)
    assert torch.equal(p, r) and torch.equal(b.attend(p, step=True), b.attend(r))


@gpu
def test_a_call_gives_the_same_bits_each_time_on_any_stream_and_captured():
    b = Batch([1, 1, 1], [3000, 800, 40], 14, 2, 64, 16).fill_bounds().to("cuda")

    def run():
        ops.key_bounds_(b.bounds, b.k, b.table, b.kv_lens)
        p = b.pick(step=True, top=40)
        return p, b.attend(p, step=True)
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    lens = b.kv_lens.clone()
    for lens_now in ([2900, 790, 17], lens.tolist()):
        b.kv_lens.copy_(torch.tensor(lens_now, dtype=torch.int32))
        graph.replay()
        now = run()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, now))
    assert all(torch.equal(x, y) for x, y in zip(held, want))


@gpu
def test_offsets_behind_32_bits():
    """Pages behind the first 2^31 values of a pool."""
    pages, hkv, page, d = 2 ** 31 // (2 * 64 * 128) + 300, 2, 64, 128
    k, v = (torch.empty(pages, hkv, page, d, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    b = Batch([1], [800], 4, hkv, d, page).fill_bounds()
    far = (pages - 1 - torch.arange(13)).int()
    ids = b.table[0, :13].long()
    for big, small in ((k, b.k), (v, b.v)):
        big[far.long().cuda()] = small[ids].cuda()
    picked = _some(b, 1, 5)
    want, choice = _attention(b, picked, 1), b.pick(step=True, top=3)
    bounds = torch.zeros(pages, hkv, 2 * d + 16, dtype=torch.uint8, device="cuda")
    b.to("cuda")
    b.table[0, :13] = far.cuda()
    ops.key_bounds_(bounds, k, b.table, b.kv_lens, torch.tensor([0, 800], dtype=torch.int32, device="cuda"), 800)
    assert torch.equal(ops.pick_pages(b.q, bounds, b.table, b.kv_lens, page=page, top=3), choice.cuda())
    _close(ops.attn_picked(b.q, k, v, b.table, b.kv_lens, picked.cuda()), want)


@gpu
def test_pages_outside_the_pool_are_left_out_and_reported():
    from hartsyinference_b200.exceptions import DeviceWaitTimeout
    b = Batch([1], [700], 4, 2, 64, 16).fill_bounds()
    picked = _some(b, 1, 6)
    picked[0, :, 2] = picked[0, :, 1]                      # named twice, with a table entry that is no page
    b.table[0, int(picked[0, 0, 1])] = 10 ** 6
    b.to("cuda")
    assert torch.isfinite(b.attend(picked.cuda(), step=True)).all()
    with pytest.raises(DeviceWaitTimeout):
        N.check_status()
    b.table[0, 7] = -3
    got = b.pick(step=True, top=5)
    assert 7 not in got[0, 0].tolist()
    with pytest.raises(DeviceWaitTimeout):
        N.check_status()
    b.table[0, 42] = 10 ** 6
    b.kv_lens[0] = 43 * 16
    ops.key_bounds_(b.bounds, b.k, b.table, b.kv_lens)
    with pytest.raises(DeviceWaitTimeout):
        N.check_status()


@pytest.mark.parametrize("dev", BOTH)
def test_refusals(dev):
    b = Batch([3, 2], [40, 33], 8, 2, 64, 16).fill_bounds().to(dev)
    rows = b.pick(top=2, run=2)
    bad = [lambda: ops.key_bounds(3, 2, 96, dev),
           lambda: ops.key_bounds_(b.bounds[:-1], b.k, b.table, b.kv_lens, b.cu_q, 3),
           lambda: ops.key_bounds_(b.bounds[..., :-16].contiguous(), b.k, b.table, b.kv_lens, b.cu_q, 3),
           lambda: ops.key_bounds_(b.bounds, b.k[:, :, :8].contiguous(), b.table, b.kv_lens, b.cu_q, 3),
           lambda: ops.key_bounds_(b.bounds, b.k.transpose(1, 2), b.table, b.kv_lens, b.cu_q, 3),
           lambda: ops.key_bounds_(b.bounds, b.k, b.table, b.kv_lens[:1], b.cu_q, 3),
           lambda: ops.key_bounds_(b.bounds, b.k, b.table, b.kv_lens, b.cu_q),
           lambda: b.pick(top=2, run=0), lambda: b.pick(top=2, run=33), lambda: b.pick(top=2, last=0), lambda: b.pick(top=-1), lambda: b.pick(top=5000),
           lambda: b.pick(top=2, step=True),
           lambda: ops.pick_pages(b.q, b.bounds, b.table, b.kv_lens, b.cu_q, page=24, top=2),
           lambda: ops.pick_pages(b.q[:, :7], b.bounds, b.table, b.kv_lens, b.cu_q, page=16, top=2),
           lambda: ops.pick_pages(b.q, b.bounds, b.table, b.kv_lens, b.cu_q[:2], page=16, top=2),
           lambda: b.attend(rows, run=1), lambda: b.attend(rows[:, :1], run=2), lambda: b.attend(rows[..., :0], run=2),
           lambda: ops.attn_picked(b.q, b.k, b.v[:-1], b.table, b.kv_lens, rows, b.cu_q, run=2),
           lambda: ops.attn_picked(b.q[..., :32], b.k, b.v, b.table, b.kv_lens, rows, b.cu_q, run=2),
           lambda: ops.attn_picked(b.q.reshape(5, -1), b.k, b.v, b.table, b.kv_lens, rows, b.cu_q, run=2)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    if dev == "cuda":
        for call in (lambda: b.pick(top=2).long() and ops.attn_picked(b.q.float(), b.k, b.v, b.table, b.kv_lens, rows, b.cu_q, run=2),
                     lambda: ops.pick_pages(b.q, b.bounds, b.table.cpu(), b.kv_lens, b.cu_q, page=16, top=2),
                     lambda: ops.attn_picked(b.q, b.k, b.v, b.table, b.kv_lens, rows.long(), b.cu_q, run=2)):
            with pytest.raises((ValueError, RuntimeError)):
                call()


@pytest.mark.parametrize("dev", BOTH)
@pytest.mark.parametrize("run", [1, 4, 16])
def test_rows_in_front_of_the_first_sequence_and_behind_the_last(dev, run):
    """A padded batch: q has rows that no sequence has. Their rows of pages are -1, and the sequences' results are those without them."""
    b = Batch([9, 1], [300, 170], 8, 2, 64, 16).fill_bounds().to(dev)
    want_p, want = b.pick(top=4, run=run), b.attend(b.pick(top=4, run=run), run=run)
    for front, behind in ((0, 40), (33, 0), (5, 17)):
        q = torch.cat([b.q[:1].expand(front, -1, -1), b.q, b.q[:1].expand(behind, -1, -1)])
        cu = b.cu_q + front
        p = ops.pick_pages(q, b.bounds, b.table, b.kv_lens, cu, page=16, top=4, run=run)
        first = [(int(c) + i * (run - 1)) // run for i, c in enumerate(cu)]
        rows = [x for i, m in enumerate(b.each) for x in range(first[i], first[i] + -(-m // run))]
        was = [x for i, m in enumerate(b.each) for x in range((int(b.cu_q[i]) + i * (run - 1)) // run, (int(b.cu_q[i]) + i * (run - 1)) // run + -(-m // run))]
        assert torch.equal(p[rows], want_p[was])
        rest = [x for x in range(p.shape[0]) if x not in rows]
        assert (p[rest] == -1).all()
        got = ops.attn_picked(q, b.k, b.v, b.table, b.kv_lens, p, cu, run=run)
        assert torch.equal(got[front:front + 10], want)


@pytest.mark.parametrize("dev", BOTH)
def test_empty_batches_and_pools(dev):
    b = Batch([0], [40], 8, 2, 64, 16).to(dev)
    p = b.pick(top=2)
    assert p.shape == (0, 2, 5) and b.attend(p).shape == (0, 8, 64)
    b = Batch([2], [40], 8, 2, 64, 16).to(dev)
    none = ops.pick_pages(b.q, b.bounds[:0], b.table[:, :0], b.kv_lens * 0, b.cu_q, page=16, top=2)
    assert (none == -1).all() and none.shape == (2, 2, 5)
    assert not ops.attn_picked(b.q, b.k[:0], b.v[:0], b.table[:, :0], b.kv_lens * 0, none, b.cu_q).any()
    ops.key_bounds_(b.bounds[:0], b.k[:0], b.table[:, :0], b.kv_lens * 0, b.cu_q, 2)
