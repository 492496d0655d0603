"""Eviction from a paged cache by attention weight: what attention gave to each
cached token is added up step by step, and a cache that has grown too long is cut
to its first and last tokens and those between that got the most.

Both operators take the 16-bit (or fp32) pools of :mod:`aicas_b200.paged` and the
4-bit ones of :mod:`aicas_b200.paged_int4`.  Weights are fp32 ``[B, Hkv, C]``, a sum for
each slot of each request and key-value head, whose query heads are added up.

A key keeps the rotation of the position that its token was appended with, so a cut
cache is attended to as any other; only slots and positions are no longer the same,
and the caller counts positions by itself (:func:`aicas_b200.paged_rope_kv_append` takes
slots as ``positions`` and angles as ``cos`` and ``sin``).

The reference's caches keep every token (dujunbaoV1/evaluation_wrapper.py:54-112).
"""
from __future__ import annotations

import operator
from typing import Sequence

import torch

from . import _native as nat
from ._hostpath import fast, launch, lengths, pointer, rows_ready, steps
from .ops import _DTYPE_CODES, SUPPORTED_HEAD_DIMS, _reject_grad
from .paged import _ITEM
from .paged_int4 import Int4Pages, _side, _table

_INT32_MAX = 2 ** 31 - 1


def _pages_side(what: str, pages, index: int, dtype: torch.dtype | None):
    """(shape (P, Hkv, page_size, D), steps) of a pool of the framework's float types."""
    if pages.get_device() != index:
        raise ValueError(f"{what} needs CUDA tensors on one device")
    shape = pages.shape
    if len(shape) != 4 or pages.dtype not in _DTYPE_CODES or (dtype is not None and pages.dtype is not dtype):
        raise ValueError(f"{what}: the pages must be [P, Hkv, page_size, D] of fp32, fp16 or bf16, of the query's dtype, "
                         "or Int4Pages")
    if shape[3] not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"{what}: head_dim {shape[3]} is not one of {sorted(SUPPORTED_HEAD_DIMS)}")
    if shape[2] < 8 or shape[2] % 8:
        raise ValueError(f"{what}: page_size must be a positive multiple of 8 (got {shape[2]})")
    s = steps(pages)
    if s[3] != 1:
        raise ValueError(f"{what}: head_dim must be the unit-stride dimension of the pages")
    if pages.requires_grad:
        _reject_grad(pages)
    return shape, s


def _check_weights(what: str, name: str, weights, B: int, Hkv: int, slots: int, index: int) -> tuple[int, int]:
    if weights.dtype is not torch.float32 or weights.ndim != 3 or weights.get_device() != index \
            or weights.shape[:2] != (B, Hkv) or weights.shape[2] < slots:
        raise ValueError(f"{what}: {name} must be a CUDA fp32 [{B}, {Hkv}, C] tensor, C at least the {slots} slots of the "
                         "page table")
    s = steps(weights)
    C = weights.shape[2]
    if (C > 1 and s[2] != 1) or (Hkv > 1 and s[1] < C) or (B > 1 and s[0] < C) \
            or (Hkv > 1 and B > 1 and s[0] < s[1] * Hkv and s[1] < s[0] * B):
        raise ValueError(f"{what}: {name} must have contiguous slots and rows apart from one another")
    return s[0], s[1]


def paged_attention_weights(
    query: torch.Tensor,
    k_pages: torch.Tensor | Int4Pages,
    page_table: torch.Tensor,
    lse: torch.Tensor,
    weights: torch.Tensor,
    *,
    sm_scale: float,
    num_key_value_groups: int,
    kv_lens: torch.Tensor | Sequence[int] | None = None,
    kv_starts: torch.Tensor | Sequence[int] | None = None,
) -> torch.Tensor:
    """Adds to ``weights[b, h, t]`` the softmax weights that the queries of key-value
    head h gave to slot t: ``2^(sm_scale log2(e) q.k_t - lse)``, summed over the heads of
    the group and over a window of S queries.

    query ``[B, Hq, S, D]``, rotated: query s of request b is the token at slot
    ``kv_lens[b] - S + s`` and sees the slots ``[kv_starts[b], kv_lens[b] - S + s]``; with
    S = 1, those of :func:`aicas_b200.paged_gqa_decode_attention`.  lse fp32
    ``[B, Hq, S]`` (or ``[B, Hq]`` where S is 1): the base-2 log-sum-exp that each query's
    attention returned; ``-inf``, of a query that saw nothing, adds nothing.  weights fp32
    ``[B, Hkv, C]``, C at least the page table's slots, updated in place and returned;
    slots outside the range keep what they hold.  ``kv_lens`` and ``kv_starts`` are the
    attention's.  Each slot is summed in one order, so results repeat to the bit."""
    done = fast("weigh", query, k_pages, page_table, lse, weights, sm_scale, num_key_value_groups, kv_lens, kv_starts)
    if done is not None:
        return done
    what = "paged_attention_weights"
    if query.requires_grad or lse.requires_grad or weights.requires_grad:
        _reject_grad(query, lse, weights)
    if query.ndim != 4 or query.device.type != "cuda":
        raise ValueError(f"{what} needs CUDA tensors, query [B, Hq, S, D]")
    B, Hq, S, D = query.shape
    index, dtype, device = query.get_device(), query.dtype, query.device
    if dtype not in _DTYPE_CODES:
        raise ValueError(f"{what}: unsupported dtype {dtype}")
    if isinstance(k_pages, torch.Tensor):
        (P, Hkv, size, dim), ks = _pages_side(what, k_pages, index, dtype)
        group, scales, k_strides, s_strides = 0, 0, ks[:3], (0, 0, 0)
        codes = k_pages.data_ptr()
    else:
        (P, Hkv, size, dim, group), ref = _side(what, k_pages, index, dtype)
        codes, scales, k_strides, s_strides = ref[0], ref[1], ref[2:5], ref[5:8]
    if dim != D:
        raise ValueError(f"{what}: head_dim {D} of the query, {dim} of the pages")
    if num_key_value_groups < 1 or Hq != Hkv * num_key_value_groups:
        raise ValueError("num_q_heads != num_kv_heads * num_key_value_groups")
    page_table, max_pages, table_stride = _table(what, page_table, B, index)
    if lse.ndim == 2 and S == 1:
        lse = lse.unsqueeze(2)
    if lse.shape != (B, Hq, S) or lse.dtype is not torch.float32 or lse.get_device() != index:
        raise ValueError(f"{what}: lse must be a CUDA fp32 [{B}, {Hq}, {S}] tensor")
    wb, wh = _check_weights(what, "weights", weights, B, Hkv, max_pages * size, index)
    query, qi = rows_ready(query, _ITEM[dtype])
    lens = None if kv_lens is None else lengths(kv_lens, B, device)
    starts = None if kv_starts is None else lengths(kv_starts, B, device)
    if B and S and max_pages:
        launch(device, "aicas_paged_weights", nat.PACK_PAGED_WEIGHTS.pack(
            query.data_ptr(), codes, scales, lse.data_ptr(), weights.data_ptr(), page_table.data_ptr(), pointer(lens),
            pointer(starts), *qi[:3], *steps(lse), wb, wh, *k_strides, *s_strides, table_stride,
            B, Hq, Hkv, S, D, group, P, size, max_pages, _DTYPE_CODES[dtype], sm_scale))
    return weights


def paged_kv_evict(
    k_pages: torch.Tensor | Int4Pages,
    v_pages: torch.Tensor | Int4Pages,
    page_table: torch.Tensor,
    weights: torch.Tensor,
    kv_lens: torch.Tensor | Sequence[int],
    *,
    keep: int,
    keep_first: int = 0,
    keep_last: int = 0,
    longer_than: int | None = None,
    kv_lens_out: torch.Tensor | None = None,
    weights_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Cuts every cache of more than ``longer_than`` slots (default ``keep``) to ``keep``
    slots, each key-value head for itself: the first ``keep_first``, the last
    ``keep_last`` and, of those between, the ones of the largest ``weights[b, h, t]``,
    the lower slot where two are equal; NaN is less than every number.

    The kept rows of the keys' and values' pages move to slots ``0 .. keep - 1`` in their
    order, in place; rows behind them stay as they were.  ``weights`` fp32 ``[B, Hkv, C]``
    move along and become 0 behind, in place or, with ``weights_out``, there (a cache that
    is not cut is copied; slots past its length are not written).  ``kv_lens_out`` int32
    ``[B]`` receives the new lengths (``kv_lens`` itself may be passed).  Returns int32
    ``[B, Hkv, keep]``: the slot that slot i was, which for a cache that is not cut is i,
    and -1 past its length.

    A page that a cut request holds must be in one place of one row of the page table:
    pages that requests share have to be copied first.  All slots below ``kv_lens[b]`` are
    tokens here: a request that is attended to from a ``kv_starts[b]`` above 0 has to be
    left out (its masked slots would be kept as its first ones, and others by their weight
    of 0, as many as each head chances to have, and no start would hold for the cut cache)."""
    done = fast("evict", k_pages, v_pages, page_table, weights, kv_lens, keep, keep_first, keep_last, longer_than, kv_lens_out,
                weights_out)
    if done is not None:
        return done
    what = "paged_kv_evict"
    int4 = not isinstance(k_pages, torch.Tensor)
    first = (k_pages[0] if isinstance(k_pages, tuple) and len(k_pages) == 2 else page_table) if int4 else k_pages
    if first.device.type != "cuda" or page_table.ndim != 2:
        raise ValueError(f"{what} needs CUDA tensors, page_table [B, max_pages]")
    index, device, B = first.get_device(), first.device, page_table.shape[0]
    planes, shapes = [], []
    for pages in (k_pages, v_pages):
        if int4:
            shape, ref = _side(what, pages, index, None)
            groups = shape[3] // shape[4]
            planes += [ref[0], *ref[2:5], shape[3] // 2, ref[1], *(2 * s for s in ref[5:8]), 4 * groups]
        else:
            if not isinstance(pages, torch.Tensor):
                raise ValueError(f"{what}: keys' and values' pages must be of one kind")
            shape, s = _pages_side(what, pages, index, None)
            item = _ITEM[pages.dtype]
            planes += [pages.data_ptr(), *(item * x for x in s[:3]), item * shape[3]]
        shapes.append(tuple(shape))
    if shapes[0] != shapes[1]:
        raise ValueError(f"{what}: keys' and values' pages must be of one shape")
    P, Hkv, size = shapes[0][:3]
    page_table, max_pages, table_stride = _table(what, page_table, B, index)
    keep, keep_first, keep_last, longer_than = (
        operator.index(n) for n in (keep, keep_first, keep_last, keep if longer_than is None else longer_than))
    if keep < 1 or keep_first < 0 or keep_last < 0 or keep_first + keep_last > keep or longer_than < keep:
        raise ValueError(f"{what}: keep must be positive, keep_first + keep_last at most keep, and longer_than not below it")
    # no cache is longer than the table: numbers beyond it all mean the same
    longer_than = min(longer_than, _INT32_MAX)
    if keep > _INT32_MAX:
        raise ValueError(f"{what}: keep must be below 2^31")
    slots = max_pages * size
    wb, wh = _check_weights(what, "weights", weights, B, Hkv, slots, index)
    if weights_out is None:
        weights_out = weights
    if weights.requires_grad or weights_out.requires_grad:
        _reject_grad(weights, weights_out)
    ob, oh = _check_weights(what, "weights_out", weights_out, B, Hkv, slots, index)
    at, to = ((t.data_ptr(), t.data_ptr() + 4 * (max(B - 1, 0) * sb + max(Hkv - 1, 0) * sh + slots))
              for t, sb, sh in ((weights, wb, wh), (weights_out, ob, oh)))
    if (at[0], wb, wh) != (to[0], ob, oh) and at[0] < to[1] and to[0] < at[1]:
        raise ValueError(f"{what}: weights_out must be weights or memory apart from it")
    lens = lengths(kv_lens, B, device)
    if lens is None:
        raise ValueError(f"{what}: kv_lens are required")
    if kv_lens_out is not None and (kv_lens_out.shape != (B,) or kv_lens_out.dtype is not torch.int32
                                    or kv_lens_out.get_device() != index or not kv_lens_out.is_contiguous()):
        raise ValueError(f"{what}: kv_lens_out must be a contiguous int32 [{B}] tensor on the device")
    kept = torch.empty_strided((B, Hkv, keep), (Hkv * keep, keep, 1), dtype=torch.int32, device=device)
    if B and Hkv and max_pages:
        count = len(planes) // 5
        planes += [0] * (5 * (nat.EVICT_MAX_PLANES - count))
        launch(device, "aicas_paged_evict", nat.PACK_PAGED_EVICT.pack(
            *planes, weights.data_ptr(), weights_out.data_ptr(), kept.data_ptr(), page_table.data_ptr(), lens.data_ptr(),
            pointer(kv_lens_out), wb, wh, ob, oh, table_stride,
            count, B, Hkv, P, size, max_pages, keep, keep_first, keep_last, longer_than))
    else:
        kept.fill_(-1)
        if kv_lens_out is not None:
            kv_lens_out.zero_()
    return kept
