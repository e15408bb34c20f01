"""Ops of a K/V cache held in 4 bits: the rotation that stores it, attention over it, and reading it back.

A layer's pool is uint8 ``[pages, kv heads, page / 16, 2, 16 * (d / 2 + d / 32)]`` (:func:`kv4_cache`): 17 bytes per 32 values
instead of 64. Every 32 neighbouring values of a head share a scale of 8 bits, ``max|x| / 7`` with three bits of mantissa; a value is held
as the nearest multiple of it from -7 to 7. Keys up to 6720 and values up to 420 in magnitude are held so, larger ones and
infinities as the largest multiple, NaN as zero. Head sizes 64 and 128, pages of 16, 32, 64 or 128 tokens, any number
of query heads per key head. CUDA tensors are bf16, block tables and lengths int32; CPU tensors go to the statements in :mod:`.reference`.
"""
from __future__ import annotations

import contextlib
import math
from typing import Optional

import torch

from . import _native as N
from . import reference as R
from .core import Fp8Act, SplitSum, _part_args, quant_fp8_act


def kv4_cache(pages: int, hkv: int, page: int, d: int, device="cuda") -> torch.Tensor:
    """An empty pool of one layer."""
    _layout((pages, hkv, page // 16, 2, 17 * d // 2), page, d)
    return torch.zeros(pages, hkv, page // 16, 2, 17 * d // 2, dtype=torch.uint8, device=device)


def _layout(shape, page: int, d: int) -> None:
    if d not in (64, 128) or page not in (16, 32, 64, 128) or len(shape) != 5 or shape[2] * 16 != page or shape[3] != 2 or 2 * shape[4] != 17 * d:
        raise ValueError(f"4-bit K/V cache: head size 64 or 128 and pages of 16, 32, 64 or 128 tokens, [pages, hkv, page / 16, 2, 17 d / 2]; got {tuple(shape)} for head size {d}")


def _pool(cache: torch.Tensor, d: int, device: int) -> tuple:
    """(pages, kv heads, page) of a pool that an op of this module takes; ``device``: ``get_device()`` of the other tensors."""
    shape = cache.shape
    if cache.dtype is not torch.uint8 or len(shape) != 5 or not cache.is_contiguous() or cache.get_device() != device or (device >= 0 and cache.data_ptr() % 16):
        raise ValueError("4-bit K/V cache: a contiguous uint8 pool on the device of the other tensors (kv4_cache makes one)")
    pages, hkv, units, _, _ = shape
    _layout(shape, units * 16, d)
    return pages, hkv, units * 16


def _dense(x: torch.Tensor) -> torch.Tensor:
    """x as rows that follow one another from a 16-byte boundary."""
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def _ints(what: str, x: Optional[torch.Tensor], device: int, dtype: torch.dtype = torch.int32) -> Optional[torch.Tensor]:
    if x is None:
        return None
    if x.get_device() != device or (device >= 0 and x.dtype is not dtype):
        raise ValueError(f"{what}: {dtype} on the device of the other tensors, got {x.dtype} on {x.device}")
    return x.contiguous()


_HERE = contextlib.nullcontext()


def _on(device: int):
    """Kernels go to the current device's current stream: make it the tensors' device."""
    return _HERE if device == torch._C._cuda_getDevice() else torch.cuda.device(device)


def rope_kv4(qkv, positions: torch.Tensor, hq: int, hkv: int, d: int, *, cache: Optional[torch.Tensor] = None,
             slot_mapping: Optional[torch.Tensor] = None, rot: Optional[int] = None, theta: float = 10000.0,
             inv_freq: Optional[torch.Tensor] = None, style: int = 0, q_norm_w: Optional[torch.Tensor] = None,
             k_norm_w: Optional[torch.Tensor] = None, eps: float = 1e-6, want_kv: bool = False):
    """:func:`.core.rope_kv` for a 4-bit cache: optional QK RMSNorm + rotary embedding on a packed qkv activation
    [T, (hq + 2 hkv) d] (a :class:`SplitSum` too), and keys and values to ``slot_mapping`` int64 [T] (page_index * page + offset, below 0: not
    stored; no slot twice). Returns (q [T, hq, d], k, v): with ``want_kv`` k and v [T, hkv, d] are the values that the cache holds,
    otherwise None. Angles are formed in 64 bits."""
    part = qkv if isinstance(qkv, SplitSum) else None
    x = part.ws if part is not None else qkv
    t = qkv.shape[0]
    rot = d if rot is None else rot
    if len(qkv.shape) != 2 or qkv.shape[1] != (hq + 2 * hkv) * d or hq < 1 or hkv < 1 or not 0 <= rot <= d or rot % 2 or style not in (0, 1):
        raise ValueError(f"rope_kv4: [T, (hq + 2 hkv) d] with an even rotated part of at most d, style 0 or 1; got {tuple(qkv.shape)}, rot {rot}, style {style}")
    if cache is not None:
        pages, heads, page = _pool(cache, d, x.get_device())
        if heads != hkv:
            raise ValueError(f"rope_kv4: a cache of {heads} heads for {hkv}")
    elif slot_mapping is not None:
        raise ValueError("rope_kv4: slots without a cache")
    elif d not in (64, 128):
        raise ValueError(f"rope_kv4: head size 64 or 128, got {d}")
    if positions.numel() != t or (slot_mapping is not None and slot_mapping.numel() != t):
        raise ValueError("rope_kv4: a position and a slot for every token")
    for w in (q_norm_w, k_norm_w):
        if w is not None and (w.numel() != d or w.device != x.device or (w.is_cuda and w.dtype != torch.bfloat16)):
            raise ValueError("rope_kv4: norm weights are bf16 [d] on the device of qkv")
    if rot > 0 and inv_freq is None:
        inv_freq = R.rope_inv_freq(rot, theta, x.device)
    if rot > 0 and (inv_freq.numel() != rot // 2 or inv_freq.device != x.device or inv_freq.dtype != torch.float32):
        raise ValueError("rope_kv4: inv_freq is fp32 [rot / 2] on the device of qkv")
    if not x.is_cuda:
        q, k, v = R.rope64(qkv, positions, hq, hkv, d, inv_freq if rot > 0 else None, style, q_norm_w, k_norm_w, eps)
        held = R.kv4_held(k, R.KV4_KEY_EXP), R.kv4_held(v, R.KV4_VALUE_EXP)
        if cache is not None and slot_mapping is not None:
            R.kv4_store(cache, slot_mapping, k, v)
        return (q.to(qkv.dtype), *(y.to(qkv.dtype) for y in held)) if want_kv else (q.to(qkv.dtype), None, None)
    if part is None and qkv.dtype != torch.bfloat16:
        raise ValueError(f"rope_kv4: bf16 activations, got {qkv.dtype}")
    device = x.get_device()
    positions, slot_mapping = _ints("positions", positions, device), _ints("slot_mapping", slot_mapping, device, torch.int64)
    with _on(device):
        src = None if part is not None else _dense(qkv)
        inv_freq = None if rot == 0 else inv_freq.contiguous()
        q_norm_w, k_norm_w = (None if w is None else w.contiguous() for w in (q_norm_w, k_norm_w))
        q = torch.empty(t, hq, d, dtype=torch.bfloat16, device=x.device)
        k = torch.empty(t, hkv, d, dtype=torch.bfloat16, device=x.device) if want_kv else None
        v = torch.empty_like(k) if want_kv else None
        rc = N.lib().b200_rope_kv4(N.ptr(src), q.data_ptr(), N.ptr(cache), N.ptr(k), N.ptr(v), positions.data_ptr(), N.ptr(slot_mapping),
                                   N.ptr(q_norm_w), N.ptr(k_norm_w), N.ptr(inv_freq), t, hq, hkv, d, rot, style, page if cache is not None else 16,
                                   pages if cache is not None else 0, eps, *_part_args(qkv), N.ptr(part.bias) if part is not None else None,
                                   N.state(x.device).status.data_ptr(), N.stream())
        N.check(rc, "b200_rope_kv4")
    return q, k, v


def kv4_gather(cache: torch.Tensor, block_table: torch.Tensor, cu_kv: torch.Tensor, total: int) -> tuple:
    """The first tokens of sequences as dense bf16 (k, v) [total, hkv, d]: rows ``cu_kv[s]`` .. ``cu_kv[s + 1]`` (int32 [S + 1], from 0) are
    those of block-table row s, ``total`` is the last of them on the host. What the cache stands for is exact in bf16. Rows that belong to
    no sequence are zeros."""
    d = 2 * cache.shape[-1] // 17
    device = cache.get_device()
    pages, hkv, page = _pool(cache, d, device)
    if block_table.dim() != 2 or cu_kv.numel() != block_table.shape[0] + 1 or total < 0:
        raise ValueError("kv4_gather: block_table [S, pages] and cu_kv [S + 1]")
    if not cache.is_cuda or total == 0 or block_table.numel() == 0 or pages == 0:
        k, v = (torch.zeros(total, hkv, d, dtype=torch.bfloat16, device=cache.device) for _ in range(2))
        cuts = [] if cache.is_cuda else cu_kv.tolist()
        for i, (a, b) in enumerate(zip(cuts, cuts[1:])):
            k[a:b], v[a:b] = R.kv4_sequence(cache, block_table[i], b - a)
        return k, v
    k = torch.empty(total, hkv, d, dtype=torch.bfloat16, device=cache.device)
    v = torch.empty_like(k)
    block_table, cu_kv = _ints("block_table", block_table, device), _ints("cu_kv", cu_kv, device)
    with _on(device):
        rc = N.lib().b200_kv4_gather(cache.data_ptr(), block_table.data_ptr(), cu_kv.data_ptr(), k.data_ptr(), v.data_ptr(), block_table.shape[0],
                                     total, hkv, d, page, block_table.shape[1], pages, N.state(cache.device).status.data_ptr(), N.stream())
        N.check(rc, "b200_kv4_gather")
    return k, v


def _attention_args(what: str, q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor) -> tuple:
    device = q.get_device()
    if q.dim() != 3 or (device >= 0 and q.dtype is not torch.bfloat16):
        raise ValueError(f"{what}: q is [tokens, hq, d], bf16 on a device; got {q.dtype} {tuple(q.shape)}")
    _, hq, d = q.shape
    pages, hkv, page = _pool(cache, d, device)
    if hq < 1 or hkv < 1 or hq % hkv:
        raise ValueError(f"{what}: {hq} query heads on {hkv} key heads")
    if block_table.dim() != 2 or block_table.shape[0] != kv_lens.numel():
        raise ValueError(f"{what}: block_table [S, pages] and kv_lens [S]")
    return _ints("block_table", block_table, device), _ints("kv_lens", kv_lens, device), pages, hkv, page


def _on_cpu(q, cache, block_table, kv_lens, cuts, **kw) -> torch.Tensor:
    out = torch.zeros_like(q)
    for i, n in enumerate(kv_lens.tolist()):
        a, b = cuts[i], cuts[i + 1]
        k, v = R.kv4_sequence(cache, block_table[i], n)
        out[a:b] = R.attention(q[a:b], k, v, **kw).to(q.dtype)
    return out


def attn_decode_kv4(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, scale: Optional[float] = None,
                    softcap: float = 0.0, window: int = 0, max_kv_len: Optional[int] = None, emit_fp8: bool = False, emit_bf16: bool = True):
    """One query token per sequence against a 4-bit pool: q [B, hq, d] -> [B, hq, d]. A sequence without keys gives zeros. ``max_kv_len``: the
    longest sequence where the host knows it (the width of the block table otherwise); it only chooses how the work is cut. With
    ``emit_fp8`` the result is ``(out, Fp8Act of out.reshape(B, hq * d))`` as of :func:`.core.attn_decode`."""
    block_table, kv_lens, pages, hkv, page = _attention_args("attn_decode_kv4", q, cache, block_table, kv_lens)
    b, hq, d = q.shape
    if kv_lens.numel() != b:
        raise ValueError("attn_decode_kv4: one query token per sequence")
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    if not q.is_cuda:
        out = _on_cpu(q, cache, block_table, kv_lens, list(range(b + 1)), scale=scale, softcap=softcap, window=window)
    else:
        with _on(q.get_device()):
            q = _dense(q)
            out = torch.empty_like(q)
            if block_table.shape[1] == 0 or pages == 0:
                out.zero_()
            elif b:
                L, longest = N.lib(), block_table.shape[1] * page
                longest = longest if max_kv_len is None else min(max_kv_len, longest)
                # parts of sequences: memory of this call alone, since other streams may be in the same op
                need = L.b200_attn_decode_kv4_workspace(b, hq, hkv, d, longest)
                ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
                rc = L.b200_attn_decode_kv4(q.data_ptr(), cache.data_ptr(), out.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr(), b, hq, hkv, d,
                                            page, block_table.shape[1], pages, longest, min(int(window), 2 ** 31 - 1), float(scale), float(softcap), N.ptr(ws), need,
                                            N.state(q.device).status.data_ptr(), N.stream())
                N.check(min(rc, 0), "b200_attn_decode_kv4", rc)
    if not emit_fp8:
        return out
    with _on(q.get_device()) if q.is_cuda else _HERE:
        return out if emit_bf16 else None, quant_fp8_act(out.reshape(b, hq * d))


def attn_prefill_kv4(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, cu_q: torch.Tensor,
                     max_q_len: int, causal: bool = True, scale: Optional[float] = None, softcap: float = 0.0, window: int = 0,
                     max_kv_len: Optional[int] = None) -> torch.Tensor:
    """Variable-length (chunked) attention over a 4-bit pool: q [total_q, hq, d] packed by ``cu_q`` int32 [S + 1], the keys of sequence s are
    its first ``kv_lens[s]`` tokens, the last of them its last query's own. No sequence has more queries than ``max_q_len``; ``max_kv_len``
    (as of :func:`attn_decode_kv4`) only chooses between three kernels. A query without keys gives zeros; rows behind the last sequence's are undefined. Arguments as of :func:`.core.attn_prefill_paged`."""
    block_table, kv_lens, pages, hkv, page = _attention_args("attn_prefill_kv4", q, cache, block_table, kv_lens)
    if cu_q.numel() != kv_lens.numel() + 1:
        raise ValueError("attn_prefill_kv4: cu_q [S + 1]")
    if q.shape[0] and max_q_len < 1:
        raise ValueError(f"attn_prefill_kv4: at most {max_q_len} queries a sequence")
    cu_q = _ints("cu_q", cu_q, q.get_device())
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    if not q.is_cuda:
        return _on_cpu(q, cache, block_table, kv_lens, cu_q.tolist(), causal=causal, scale=scale, softcap=softcap, window=window)
    with _on(q.get_device()):
        q = _dense(q)
        out = torch.empty_like(q)
        if block_table.shape[1] == 0 or pages == 0:
            return out.zero_()
        L, longest = N.lib(), block_table.shape[1] * page
        longest = longest if max_kv_len is None else min(max_kv_len, longest)
        seqs, most, hq, d, window, scale = kv_lens.numel(), int(max_q_len), q.shape[1], q.shape[2], min(int(window), 2 ** 31 - 1), float(scale)
        ptrs = (q.data_ptr(), cache.data_ptr(), out.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr(), cu_q.data_ptr(), seqs, most)
        sizes, status = (hq, hkv, d, page, block_table.shape[1], pages), N.state(q.device).status.data_ptr()
        kernel = L.b200_attn_kv4_choice(seqs, most, longest, hq, hkv, d, int(causal), window, scale)
        if kernel == 2:                                  # few queries behind a long cache
            need = L.b200_attn_few_kv4_workspace(seqs, most, hq, hkv, d, longest)
            ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
            rc = L.b200_attn_few_kv4(*ptrs, *sizes, longest, window, scale, float(softcap), N.ptr(ws), need, status, N.stream())
            N.check(min(rc, 0), "b200_attn_few_kv4", rc)
        else:
            run = L.b200_attn_prefill_kv4 if kernel else L.b200_attn_kv4
            rc = run(*ptrs, *sizes, int(causal), window, scale, float(softcap), status, N.stream())
            N.check(rc, "b200_attn_prefill_kv4")
    return out


def attn_biased_kv4(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, cu_q: Optional[torch.Tensor],
                    scale: Optional[float] = None, softcap: float = 0.0, window: int = 0, alibi: Optional[torch.Tensor] = None,
                    sinks: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`.core.attn_paged_biased` over a 4-bit pool: causal attention with ALiBi slopes and / or per-head sink logits, which the kernels
    do not take. The sequences are read back (:func:`kv4_gather`) and run through tensor ops. ``cu_q`` None: one query token per sequence."""
    block_table, kv_lens, *_ = _attention_args("attn_biased_kv4", q, cache, block_table, kv_lens)
    n = kv_lens.numel()
    if cu_q is not None and cu_q.numel() != n + 1:
        raise ValueError("attn_biased_kv4: cu_q [S + 1]")
    cuts = list(range(n + 1)) if cu_q is None else cu_q.tolist()
    cu_kv = torch.nn.functional.pad(kv_lens.clamp(min=0).cumsum(0, dtype=torch.int32), (1, 0))
    at = cu_kv.tolist()
    k, v = kv4_gather(cache, block_table, cu_kv, at[-1])
    out = torch.zeros_like(q)
    for i in range(n):
        a, b, u, w = cuts[i], cuts[i + 1], at[i], at[i + 1]
        if a < b and u < w:
            out[a:b] = R.attention(q[a:b], k[u:w], v[u:w], causal=True, scale=scale, softcap=softcap, window=window, alibi=alibi, sinks=sinks).to(q.dtype)
    return out
