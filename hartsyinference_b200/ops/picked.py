"""Attention over pages of the K/V cache that every query chooses by a cheap score.

Beside a layer's pool of keys [pages, hkv, page, d] lies one of their bounds, uint8 ``[pages, hkv, 2 d + 16]`` (:func:`key_bounds`): per page and
key head d codes of every channel's largest value, d of its smallest (signed, rounded away from the page's values), then e + 64 and zeros. e is the smallest exponent
from -50 to 50 with max |value| <= 127 * 2^e; NaN counts as 0. A forward pass stores its keys, bounds the pages that they filled
(:func:`key_bounds_`), chooses (:func:`pick_pages`) and attends (:func:`attn_picked`).

Queries choose in runs of ``run`` neighbouring tokens of a sequence; the rows of runs are packed, run r of sequence s in row
``(cu_q[s] + s * (run - 1)) // run + r`` of ``(tokens + S * (run - 1)) // run`` (``cu_q`` from 0). Pages of 16, 32, 64 or 128 tokens, heads of 64 or 128, any number of query heads per key
head as long as a run has at most 128 of them. CUDA tensors are bf16, block tables and lengths int32; CPU tensors go to the statements here and in :mod:`.reference`.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _native as N
from . import reference as R
from .core import quant_fp8_act
from .kv4 import _dense, _ints, _on

WIDTH = 4096          # pages that a run can choose
_PAGES, _HEADS, _I32, _BF16 = (16, 32, 64, 128), (64, 128), torch.int32, torch.bfloat16


def _plain(x: torch.Tensor, device: int, n: int) -> bool:
    """Whether x is n neighbouring numbers of 32 bits on the device."""
    return x.dtype is _I32 and x.get_device() == device and x.numel() == n and x.is_contiguous()


def key_bounds(pages: int, hkv: int, d: int, device="cuda") -> torch.Tensor:
    """Bounds of an empty pool of one layer."""
    if d not in (64, 128):
        raise ValueError(f"key_bounds: head size 64 or 128, got {d}")
    return torch.zeros(pages, hkv, 2 * d + 16, dtype=torch.uint8, device=device)


def _pool_of(what: str, cache: torch.Tensor, device: int, d: Optional[int] = None) -> tuple:
    """(pages, hkv, page, d) of a pool of keys or values."""
    shape = cache.shape
    if len(shape) != 4 or shape[2] not in _PAGES or shape[3] not in _HEADS or (d is not None and shape[3] != d):
        raise ValueError(f"{what}: pools [pages, hkv, page, d] with pages of 16, 32, 64 or 128 tokens and heads of 64 or 128, got {tuple(shape)}")
    if not cache.is_contiguous() or cache.get_device() != device or (device >= 0 and cache.dtype is not torch.bfloat16):
        raise ValueError(f"{what}: a contiguous pool, bf16 on a device, on that of the other tensors")
    return tuple(shape)


def _bounds_of(what: str, bounds: torch.Tensor, device: int, hkv: int, d: int) -> int:
    if bounds.dtype is not torch.uint8 or bounds.dim() != 3 or bounds.shape[1] != hkv or bounds.shape[2] != 2 * d + 16 or not bounds.is_contiguous() or bounds.get_device() != device:
        raise ValueError(f"{what}: contiguous bounds uint8 [pages, {hkv}, {2 * d + 16}] on the device of the other tensors (key_bounds makes them), got {bounds.dtype} {tuple(bounds.shape)}")
    return bounds.shape[0]


def _batch(what: str, block_table: torch.Tensor, kv_lens: torch.Tensor, cu_q: Optional[torch.Tensor], device: int) -> tuple:
    if block_table.dim() != 2 or kv_lens.numel() != block_table.shape[0] or (cu_q is not None and cu_q.numel() != kv_lens.numel() + 1):
        raise ValueError(f"{what}: block_table [S, pages], kv_lens [S], cu_q [S + 1]")
    return _ints("block_table", block_table, device), _ints("kv_lens", kv_lens, device), _ints("cu_q", cu_q, device)


def _rows(what: str, tokens: int, seqs: int, run: int, group: int, cu_q: Optional[torch.Tensor]) -> int:
    if run < 1 or run * group > 128:
        raise ValueError(f"{what}: a run has 1 to 128 query heads on a key head, got {run} * {group}")
    if cu_q is None and (run != 1 or tokens != seqs):
        raise ValueError(f"{what}: without cu_q one query token per sequence, which chooses by itself; got {tokens} for {seqs}, run {run}")
    return (tokens + seqs * (run - 1)) // run


def _runs(kv_lens: torch.Tensor, cu_q: Optional[torch.Tensor], run: int, most: int):
    """(row, sequence, first query, position, queries) of every run, for CPU tensors."""
    cuts = list(range(kv_lens.numel() + 1)) if cu_q is None else cu_q.tolist()
    for s, n in enumerate(kv_lens.tolist()):
        n, count = min(n, most), cuts[s + 1] - cuts[s]
        for r in range(-(-count // run)):
            yield (cuts[s] + s * (run - 1)) // run + r, s, cuts[s] + r * run, n - count + r * run, min(run, count - r * run)


def key_bounds_(bounds: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None,
                max_q_len: Optional[int] = None) -> torch.Tensor:
    """Bounds of the pages that the last tokens of every sequence filled, written into ``bounds``: ``cu_q[s + 1] - cu_q[s]`` tokens (one without ``cu_q``, at most
    ``max_q_len``) of ``kv_lens[s]`` that the cache holds; ``max_q_len`` is asked for with ``cu_q``, since pages behind it would keep old bounds. Pages that are not full are left as they are: whoever attends
    has them among its last ones. A page that is cut back and filled again is bounded again."""
    device, shape, table = bounds.get_device(), k_cache.shape, block_table.shape
    seqs = kv_lens.numel()
    if cu_q is not None and max_q_len is None:
        raise ValueError("key_bounds_: cu_q with the longest run of new tokens, max_q_len")
    if not (device >= 0 and len(shape) == 4 and len(table) == 2 and table[0] == seqs and shape[2] in _PAGES and shape[3] in _HEADS and bounds.dtype is torch.uint8
            and k_cache.dtype is _BF16 and block_table.dtype is _I32 and kv_lens.dtype is _I32 and (cu_q is None or _plain(cu_q, device, seqs + 1))
            and bounds.shape == (shape[0], shape[1], 2 * shape[3] + 16) and device == k_cache.get_device() == block_table.get_device() == kv_lens.get_device()
            and bounds.is_contiguous() and k_cache.is_contiguous() and block_table.is_contiguous() and kv_lens.is_contiguous()):
        # not the ordinary call: say what is wrong, or make it one
        pages, hkv, page, d = _pool_of("key_bounds_", k_cache, device)
        if _bounds_of("key_bounds_", bounds, device, hkv, d) != pages:
            raise ValueError(f"key_bounds_: bounds of {bounds.shape[0]} pages for a pool of {pages}")
        block_table, kv_lens, cu_q = _batch("key_bounds_", block_table, kv_lens, cu_q, device)
    pages, hkv, page, d = shape
    if device < 0:
        cuts = list(range(seqs + 1)) if cu_q is None else cu_q.tolist()
        for s, n in enumerate(kv_lens.tolist()):
            n, count = min(n, block_table.shape[1] * page), cuts[s + 1] - cuts[s]
            if count > 0 and n > 0:
                ids = block_table[s, max(0, n - count) // page:n // page].long()
                bounds[ids] = R.page_bounds(k_cache[ids])
        return bounds
    to, keys = bounds.data_ptr(), k_cache.data_ptr()
    if (to | keys) % 16:
        raise ValueError("key_bounds_: bounds and pool from 16-byte boundaries")
    if seqs and pages and table[1]:
        with _on(device):
            rc = N.lib().b200_key_bounds(keys, to, block_table.data_ptr(), kv_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), seqs,
                                         max_q_len if cu_q is not None else 1, hkv, d, page, table[1], pages, N.state(bounds.device).status.data_ptr(), N.stream())
            N.check(rc, "b200_key_bounds")
    return bounds


def pick_pages(q: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None, *, page: int,
               top: int, first: int = 1, last: int = 2, run: int = 1) -> torch.Tensor:
    """The pages that queries q [tokens, hq, d] attend to, int32 [rows, hkv, width]: page numbers of the sequence in order, then -1, ``width = first + top + last +
    (run + page - 2) // page``. A run keeps the ``first`` pages, the ``last`` (at least 1) up to that of its first query and all behind it, and of those between the ``top``
    of the largest score, ties to the lowest number. The score is the largest, over the run's queries and the heads of a
    group, of ``2^(e_q + e_page) * sum_c max(a_c high_c, a_c low_c)`` with the query's codes ``a = round(q / 2^e_q)`` (its own
    exponent, as for bounds). Sums are whole numbers below 2^22, so scores are exact and the choice does not depend on how they are computed.
    The queries of a sequence are its last tokens; ``cu_q`` None: one per sequence. Rows of no run are -1."""
    device, shape, rows_of, table = q.get_device(), q.shape, bounds.shape, block_table.shape
    seqs = kv_lens.numel()
    if not (device >= 0 and len(shape) == 3 and len(rows_of) == 3 and len(table) == 2 and table[0] == seqs and shape[2] in _HEADS and page in _PAGES
            and rows_of[2] == 2 * shape[2] + 16 and shape[1] > 0 and rows_of[1] > 0 and shape[1] % rows_of[1] == 0 and q.dtype is _BF16
            and bounds.dtype is torch.uint8 and block_table.dtype is _I32 and kv_lens.dtype is _I32 and (cu_q is None or _plain(cu_q, device, seqs + 1))
            and device == bounds.get_device() == block_table.get_device() == kv_lens.get_device()
            and bounds.is_contiguous() and block_table.is_contiguous() and kv_lens.is_contiguous()):
        if q.dim() != 3 or (device >= 0 and q.dtype is not _BF16) or q.shape[2] not in _HEADS:
            raise ValueError(f"pick_pages: q is [tokens, hq, 64 or 128], bf16 on a device; got {q.dtype} {tuple(q.shape)}")
        hkv = bounds.shape[1] if bounds.dim() == 3 else 0
        if hkv < 1 or shape[1] < 1 or shape[1] % hkv or page not in _PAGES:
            raise ValueError(f"pick_pages: {shape[1]} query heads on {hkv} key heads, pages of 16, 32, 64 or 128 tokens, got {page}")
        _bounds_of("pick_pages", bounds, device, hkv, shape[2])
        block_table, kv_lens, cu_q = _batch("pick_pages", block_table, kv_lens, cu_q, device)
    (tokens, hq, d), (pages, hkv, _) = shape, rows_of
    rows = _rows("pick_pages", tokens, seqs, run, hq // hkv, cu_q)
    width = first + top + last + (run + page - 2) // page
    if top < 0 or first < 0 or last < 1 or width > WIDTH:
        raise ValueError(f"pick_pages: top and first from 0, last from 1, at most {WIDTH} pages together; got {top}, {first}, {last}")
    if device < 0:
        out = torch.full((rows, hkv, width), -1, dtype=torch.int32)
        for row, s, a, begin, count in _runs(kv_lens, cu_q, run, block_table.shape[1] * page):
            end = begin + count - 1
            if end < 0:
                continue
            skip = max(0, -begin)                                # queries in front of the first key see nothing
            middle = max(first, (begin + skip) // page - last + 1)
            kept = list(range(end // page + 1))
            if middle - first > top:
                score = R.page_scores(q[a + skip:a + count], bounds[block_table[s, first:middle].long()])
                best = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :top].sort(-1).values + first
                for h in range(hkv):
                    mine = kept[:first] + best[h].tolist() + kept[middle:]
                    out[row, h, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
            else:
                out[row, :, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
        return out
    out = kv_lens.new_empty((rows, hkv, width))
    with _on(device):
        if pages == 0 or table[1] == 0 or seqs == 0:
            return out.fill_(-1)
        if bounds.data_ptr() % 16:
            raise ValueError("pick_pages: bounds from a 16-byte boundary")
        q = _dense(q)
        rc = N.lib().b200_pick_pages(q.data_ptr(), bounds.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), out.data_ptr(),
                                     seqs, rows, tokens, hq, hkv, d, page, table[1], pages, run, top, first, last, width, N.state(q.device).status.data_ptr(), N.stream())
        N.check(rc, "b200_pick_pages")
    return out


def attn_picked(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, picked: torch.Tensor,
                cu_q: Optional[torch.Tensor] = None, *, run: int = 1, scale: Optional[float] = None, softcap: float = 0.0, emit_fp8: bool = False,
                emit_bf16: bool = True):
    """Causal attention of q [tokens, hq, d] over the pages that :func:`pick_pages` chose (with the same ``cu_q`` and ``run``), [tokens, hq, d]. The
    queries of a sequence are its last tokens; ``cu_q`` None: one per sequence. A query that sees no key gives zeros; rows behind the last sequence's are undefined. Page numbers below 0 or
    behind the run's last query are none; one that is named twice counts twice. With ``emit_fp8`` the result is ``(out, Fp8Act of out.reshape(tokens, hq * d))``
    as of :func:`.core.attn_decode`."""
    device, shape, pool, table, chosen = q.get_device(), q.shape, k_cache.shape, block_table.shape, picked.shape
    seqs = kv_lens.numel()
    if not (device >= 0 and len(shape) == 3 and len(pool) == 4 and len(table) == 2 and len(chosen) == 3 and table[0] == seqs and pool[2] in _PAGES and pool[3] in _HEADS
            and shape[2] == pool[3] and shape[1] > 0 and pool[1] > 0 and shape[1] % pool[1] == 0 and v_cache.shape == pool
            and q.dtype is k_cache.dtype is v_cache.dtype is _BF16 and block_table.dtype is kv_lens.dtype is picked.dtype is _I32 and (cu_q is None or _plain(cu_q, device, seqs + 1))
            and device == k_cache.get_device() == v_cache.get_device() == block_table.get_device() == kv_lens.get_device() == picked.get_device()
            and k_cache.is_contiguous() and v_cache.is_contiguous() and block_table.is_contiguous() and kv_lens.is_contiguous() and picked.is_contiguous()):
        if q.dim() != 3 or (device >= 0 and q.dtype is not _BF16):
            raise ValueError(f"attn_picked: q is [tokens, hq, d], bf16 on a device; got {q.dtype} {tuple(q.shape)}")
        hkv = _pool_of("attn_picked", k_cache, device, shape[2])[1]
        if _pool_of("attn_picked", v_cache, device, shape[2]) != tuple(pool) or hkv < 1 or shape[1] < 1 or shape[1] % hkv:
            raise ValueError(f"attn_picked: pools of keys and of values alike, {shape[1]} query heads on {hkv} key heads")
        block_table, kv_lens, cu_q = _batch("attn_picked", block_table, kv_lens, cu_q, device)
        if picked.dim() != 3:
            raise ValueError(f"attn_picked: picked [rows, {hkv}, width], got {tuple(picked.shape)}")
        picked = _ints("picked", picked, device)
    (tokens, hq, d), (pages, hkv, page, _) = shape, pool
    rows = _rows("attn_picked", tokens, seqs, run, hq // hkv, cu_q)
    width = chosen[2]
    if chosen[0] != rows or chosen[1] != hkv or not 1 <= width <= WIDTH:
        raise ValueError(f"attn_picked: picked [{rows}, {hkv}, 1 to {WIDTH}], got {tuple(chosen)}")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if device < 0:
        out = torch.zeros_like(q)
        for row, s, a, begin, count in _runs(kv_lens, cu_q, run, block_table.shape[1] * page):
            for h in range(hkv):
                heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                mine = [x for x in picked[row, h].tolist() if 0 <= x <= (begin + count - 1) // page and x < block_table.shape[1]]
                key = torch.tensor([x * page + i for x in mine for i in range(page)], dtype=torch.long)
                ids = block_table[s, mine].long()
                for j in range(count):
                    on = key <= begin + j
                    k, v = (c[ids, h].reshape(-1, d)[on][:, None] for c in (k_cache, v_cache))
                    if k.shape[0]:
                        out[a + j, heads] = R.attention(q[a + j:a + j + 1, heads], k, v, scale=scale, softcap=softcap)[0].to(q.dtype)
    else:
        with _on(device):
            q = _dense(q)
            out = torch.empty_like(q)
            if table[1] == 0 or pages == 0:
                out.zero_()
            elif seqs:
                L, status, keys, values = N.lib(), N.state(q.device).status.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
                if (keys | values) % 16:
                    raise ValueError("attn_picked: pools from 16-byte boundaries")
                ptrs = (q.data_ptr(), keys, values, out.data_ptr(), picked.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr())
                cols = run * (hq // hkv)          # (few of them never take the tiles: small calls do without the question)
                if cols > 16 and L.b200_attn_picked_form(rows, cols, hkv, d, page, width, pages, scale, softcap):
                    rc = L.b200_attn_picked_tc(*ptrs, seqs, rows, tokens, hq, hkv, d, page, table[1], pages, run, width, scale, status, N.stream())
                else:
                    rc = L.b200_attn_picked(*ptrs, seqs, rows, tokens, hq, hkv, d, page, table[1], pages, run, width, scale, float(softcap), status, N.stream())
                N.check(rc, "b200_attn_picked")
    if not emit_fp8:
        return out
    if device < 0:
        return out if emit_bf16 else None, quant_fp8_act(out.reshape(tokens, hq * d))
    with _on(device):
        return out if emit_bf16 else None, quant_fp8_act(out.reshape(tokens, hq * d))
