"""Rotary positions on several axes: time, row and column of pictures and film."""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _native as N
from . import reference as R
from .kv4 import _dense, _ints, _on


def rope_axes(sections: Sequence[int], interleaved: bool = False, device="cpu") -> torch.Tensor:
    """The axis that turns every pair, int32 [sum(sections)]: ``sections[a]`` pairs for axis a, one axis after the other, or with
    ``interleaved`` in turns (pair j for axis j % A while that one has pairs left, all others for axis 0)."""
    sections = [int(n) for n in sections]
    if not sections or min(sections) < 0:
        raise ValueError(f"rope_axes: a number of pairs for every axis, got {sections}")
    axes = [a for a, n in enumerate(sections) for _ in range(n)]
    if interleaved:
        count = len(sections)
        axes = [j % count if j // count < sections[j % count] else 0 for j in range(len(axes))]
        if any(axes.count(a) != n for a, n in enumerate(sections)):
            raise ValueError(f"rope_axes: sections {sections} do not take turns over {len(axes)} pairs")
    return torch.tensor(axes, dtype=torch.int32, device=device)


def rope_axes_kv(qkv: torch.Tensor, positions: torch.Tensor, hq: int, hkv: int, d: int, *, axes: torch.Tensor, inv_freq: torch.Tensor,
                 k_cache: Optional[torch.Tensor] = None, v_cache: Optional[torch.Tensor] = None, slot_mapping: Optional[torch.Tensor] = None,
                 style: int = 0, q_norm_w: Optional[torch.Tensor] = None, k_norm_w: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 want_kv: bool = False):
    """:func:`.core.rope_kv` with positions on several axes: optional QK RMSNorm, then rotary embedding on a packed qkv activation
    [T, (hq + 2 hkv) d], and the K/V write into the page pool ([pages, hkv, page, d]; ``slot_mapping`` int64 [T], page_index * page + offset, below 0:
    not stored; no slot twice). ``positions`` int32 [A, T]; pair j of the rotated part (the first 2 * len(axes) channels) turns by
    ``positions[axes[j]] * inv_freq[j]``, in angles of 64 bits; ``axes`` int32 as of :func:`rope_axes`, ``inv_freq`` fp32, both [pairs]. Heads of an
    even size up to 256; style 0 pairs channel j with j + pairs, 1 channel 2 j with 2 j + 1. Returns (q [T, hq, d], k [T, hkv, d] or None, v or None)."""
    shape, where, pairs, device = qkv.shape, positions.shape, axes.numel(), qkv.get_device()
    if len(where) != 2 or len(shape) != 2 or where[1] != shape[0]:
        raise ValueError(f"rope_axes_kv: positions [A, T] of qkv [T, (hq + 2 hkv) d], got {tuple(where)} and {tuple(shape)}")
    t = shape[0]
    if hq < 1 or hkv < 1 or shape[1] != (hq + 2 * hkv) * d or not 2 <= d <= 256 or d % 2 or 2 * pairs > d or style not in (0, 1):
        raise ValueError(f"rope_axes_kv: heads of an even size up to 256, at most d / 2 pairs, style 0 or 1; got {tuple(shape)} for {hq} + 2 * {hkv} heads of {d}, {pairs} pairs")
    if where[0] < 1 or inv_freq.numel() != pairs:
        raise ValueError("rope_axes_kv: an axis and a frequency for every pair")
    if (k_cache is None) != (v_cache is None) or (slot_mapping is not None and k_cache is None):
        raise ValueError("rope_axes_kv: caches of keys and of values, and slots only with them")
    if slot_mapping is not None and slot_mapping.numel() != t:
        raise ValueError("rope_axes_kv: a slot for every token")
    pages, page = 0, 1
    if k_cache is not None:
        pool = k_cache.shape
        if (len(pool) != 4 or v_cache.shape != pool or pool[1] != hkv or pool[3] != d or not k_cache.is_contiguous() or not v_cache.is_contiguous()
                or k_cache.get_device() != device or v_cache.get_device() != device or k_cache.dtype is not qkv.dtype or v_cache.dtype is not qkv.dtype):
            raise ValueError("rope_axes_kv: contiguous caches [pages, hkv, page, d] of the type and on the device of qkv")
        pages, page = pool[0], pool[2]
    for w in (q_norm_w, k_norm_w):
        if w is not None and (w.numel() != d or w.get_device() != device or (device >= 0 and w.dtype != torch.bfloat16)):
            raise ValueError("rope_axes_kv: norm weights are bf16 [d] on the device of qkv")
    positions, axes, slot_mapping = _ints("positions", positions, device), _ints("axes", axes, device), _ints("slot_mapping", slot_mapping, device, torch.int64)
    inv_freq = _ints("inv_freq", inv_freq, device, torch.float32)
    if device < 0:
        q, k, v = (x.to(qkv.dtype) for x in R.rope_axes(qkv, positions, hq, hkv, d, axes, inv_freq, style, q_norm_w, k_norm_w, eps))
        if slot_mapping is not None:
            page, on = k_cache.shape[2], slot_mapping >= 0
            at, off = slot_mapping[on].long() // page, slot_mapping[on].long() % page
            k_cache[at, :, off], v_cache[at, :, off] = k[on], v[on]
        return (q.contiguous(), k.contiguous(), v.contiguous()) if want_kv else (q.contiguous(), None, None)
    if qkv.dtype != torch.bfloat16:
        raise ValueError(f"rope_axes_kv: bf16 activations, got {qkv.dtype}")
    with _on(device):
        qkv = _dense(qkv)
        if q_norm_w is not None or k_norm_w is not None:
            q_norm_w, k_norm_w = (None if w is None else w.contiguous() for w in (q_norm_w, k_norm_w))
        q = qkv.new_empty((t, hq, d))
        k = qkv.new_empty((t, hkv, d)) if want_kv else None
        v = qkv.new_empty((t, hkv, d)) if want_kv else None
        rc = N.lib().b200_rope_axes(qkv.data_ptr(), q.data_ptr(), N.ptr(k_cache), N.ptr(v_cache), N.ptr(k), N.ptr(v), positions.data_ptr(), axes.data_ptr(),
                                    inv_freq.data_ptr(), N.ptr(slot_mapping), N.ptr(q_norm_w), N.ptr(k_norm_w), t, where[0], hq, hkv, d, 2 * pairs, style,
                                    page, pages, eps, N.state(qkv.device).status.data_ptr(), N.stream())
        N.check(rc, "b200_rope_axes")
    return q, k, v
