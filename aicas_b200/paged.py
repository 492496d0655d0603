"""Paged key-value cache: the append with the position rotation on the way, the
single-token attention that reads it, and the pool that hands out the pages.

A pool is a pair of tensors ``[P, Hkv, page_size, D]`` (or any view of that
shape whose strides are multiples of 16 bytes with a contiguous ``D``, so a
``[P, page_size, Hkv, D]`` pool is passed as ``pool.transpose(1, 2)``), and a
page table is an int32 ``[B, max_pages]`` tensor on the device: token ``t`` of
request ``b`` is row ``t % page_size`` of page ``page_table[b, t // page_size]``.
Against the contiguous caches of :func:`aicas_b200.rope_kv_append` and
:func:`aicas_b200.gqa_decode_attention` a request holds only the pages its
tokens fill, not a row of the longest request's capacity.

The reference has contiguous caches only (dujunbaoV1/evaluation_wrapper.py:54-112).
The rules are those of :mod:`aicas_b200.ops`: the caller's current stream, no
host synchronisation, ``ValueError`` for what the kernels cannot take.
"""
from __future__ import annotations

from typing import Sequence

import torch

from . import _native as nat
from .ops import (
    _DTYPE_CODES,
    SUPPORTED_HEAD_DIMS,
    _as_lens,
    _call_in_device,
    _heads_ready,
    _reject_grad,
    _stream_handle,
    _workspace,
)


def _check_pool(what: str, query, k_pages, v_pages, page_table):
    """The pool's shape and strides and the page table, checked against the query."""
    if not (query.is_cuda and k_pages.is_cuda and v_pages.is_cuda and page_table.is_cuda):
        raise ValueError(f"{what} needs CUDA tensors")
    device = query.device
    if k_pages.device != device or v_pages.device != device or page_table.device != device:
        raise ValueError(f"{what}: query, pages and page_table must be on one device")
    shape = k_pages.shape
    if query.ndim != 4 or len(shape) != 4 or v_pages.shape != shape:
        raise ValueError(f"{what}: query must be 4-D and the pages [P, Hkv, page_size, D] of one shape")
    dtype = query.dtype
    if dtype not in _DTYPE_CODES or k_pages.dtype != dtype or v_pages.dtype != dtype:
        raise ValueError(f"{what}: query and pages must share a dtype of fp32, fp16 or bf16")
    if shape[3] != query.shape[3] or shape[3] not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"{what}: head_dim {query.shape[3]} of the query, {shape[3]} of the pages; "
                         f"both must be one of {sorted(SUPPORTED_HEAD_DIMS)}")
    if shape[2] < 8 or shape[2] % 8:
        raise ValueError(f"{what}: page_size must be a positive multiple of 8 (got {shape[2]})")
    ks, vs = k_pages.stride(), v_pages.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError(f"{what}: head_dim must be the unit-stride dimension of the pages")
    if page_table.dtype != torch.int32 or page_table.ndim != 2 or page_table.shape[0] != query.shape[0]:
        raise ValueError(f"{what}: page_table must be an int32 [{query.shape[0]}, max_pages] tensor")
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    return shape, ks, vs, page_table


def _lens(lens, batch: int, device: torch.device) -> torch.Tensor | None:
    if isinstance(lens, torch.Tensor) and lens.dtype == torch.int32 and lens.device == device \
            and lens.shape == (batch,) and lens.is_contiguous():
        return lens
    return _as_lens(lens, batch, device)


def _pointer(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def paged_rope_kv_append(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    positions: torch.Tensor | Sequence[int],
    *,
    num_new: torch.Tensor | Sequence[int] | None = None,
    q_out: torch.Tensor | None = None,
    kv_lens_out: torch.Tensor | None = None,
    q_norm_weight: torch.Tensor | None = None,
    k_norm_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
) -> torch.Tensor:
    """:func:`aicas_b200.rope_kv_append` into a paged cache: rotates q and the new
    k (rotate-half), after the per-head RMSNorm where a weight is given, writes
    k and v of token ``s`` to slot ``positions[b] + s`` of request ``b`` and
    returns the rotated q.

    query ``[B, Hq, S, D]``, key/value ``[B, Hkv, S, D]``, cos/sin ``[B, S, D]``
    (or ``[1, S, D]``), pages ``[P, Hkv, page_size, D]``, page_table int32
    ``[B, max_pages]``, positions int32 ``[B]``.  ``num_new`` (int32 ``[B]``): only
    the first ``num_new[b]`` tokens of row ``b`` are real, the others (padding)
    are rotated but not written.  ``kv_lens_out[b]`` receives the new length.
    Tokens past the page table's end, at negative slots or with a page number
    outside the pool are dropped.

    With fp32 cos/sin norm and rotation are held in fp32 and rounded once; with
    cos/sin of the tensors' 16-bit dtype every operation is rounded, as Hugging
    Face's modules and :func:`rope_kv_append` round, so such a model's keys are
    the same in either cache."""
    _reject_grad(query, key, value)
    shape, ks, vs, page_table = _check_pool("paged_rope_kv_append", query, k_pages, v_pages, page_table)
    device, dtype = query.device, query.dtype
    B, Hq, S, D = query.shape
    Hkv = shape[1]
    if key.shape != (B, Hkv, S, D) or value.shape != key.shape:
        raise ValueError(f"paged_rope_kv_append: key and value must be [{B}, {Hkv}, {S}, {D}]")
    if Hq % Hkv:
        raise ValueError("paged_rope_kv_append: num_q_heads is not a multiple of num_kv_heads")
    if key.dtype != dtype or value.dtype != dtype or key.device != device or value.device != device:
        raise ValueError("paged_rope_kv_append: query, key and value must share dtype and device")
    if cos.ndim != 3 or cos.shape[1:] != (S, D) or cos.shape[0] not in (1, B) or sin.shape != cos.shape:
        raise ValueError("paged_rope_kv_append: cos/sin must be [B, S, D] (or [1, S, D])")
    if cos.dtype not in (dtype, torch.float32) or sin.dtype != cos.dtype:
        raise ValueError("paged_rope_kv_append: cos/sin must have the tensor dtype or fp32")
    if cos.device != device or sin.device != device:
        raise ValueError("paged_rope_kv_append: cos and sin must be on the query's device")
    query, key, value = _heads_ready(query), _heads_ready(key), _heads_ready(value)
    cs = cos.stride()
    eb = cos.element_size()
    if sin.stride() != cs or cs[2] != 1 or cs[0] * eb % 16 or cs[1] * eb % 16 or cos.data_ptr() % 16 \
            or sin.data_ptr() % 16:
        cos, sin = cos.contiguous().clone(), sin.contiguous().clone()
        cs = cos.stride()
    pos = _lens(positions, B, device)
    if pos is None:
        raise ValueError("paged_rope_kv_append: positions are required")
    new = _lens(num_new, B, device)
    if kv_lens_out is not None and (kv_lens_out.shape != (B,) or kv_lens_out.dtype != torch.int32
                                    or kv_lens_out.device != device or not kv_lens_out.is_contiguous()):
        raise ValueError(f"paged_rope_kv_append: kv_lens_out must be a contiguous int32 [{B}] tensor on the device")
    for w in (q_norm_weight, k_norm_weight):
        if w is not None and (w.shape != (D,) or w.dtype != dtype or w.device != device or not w.is_contiguous()):
            raise ValueError("paged_rope_kv_append: norm weights must be contiguous [D] of the tensor dtype")
    if q_out is None:
        q_out = torch.empty((B, S, Hq, D), dtype=dtype, device=device).transpose(1, 2)
    elif q_out.shape != (B, Hq, S, D) or q_out.dtype != dtype or q_out.device != device or q_out.stride(3) != 1:
        raise ValueError(f"paged_rope_kv_append: q_out must be [{B}, {Hq}, {S}, {D}] with a unit-stride head_dim")
    if B == 0 or S == 0:
        if kv_lens_out is not None and B:
            kv_lens_out.copy_(pos.clamp(0, page_table.shape[1] * shape[2]))
        return q_out
    qi, qo, ki, vi = query.stride(), q_out.stride(), key.stride(), value.stride()
    args = nat.PACK_PAGED_APPEND.pack(
        query.data_ptr(), q_out.data_ptr(), key.data_ptr(), value.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), pos.data_ptr(), _pointer(new),
        _pointer(kv_lens_out), _pointer(q_norm_weight), _pointer(k_norm_weight),
        qi[0], qi[1], qi[2], qo[0], qo[1], qo[2], ki[0], ki[1], ki[2], vi[0], vi[1], vi[2],
        cs[0] if cos.shape[0] == B else 0, cs[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], page_table.stride(0),
        B, Hq, Hkv, S, D, shape[0], shape[2], page_table.shape[1], _DTYPE_CODES[dtype], _DTYPE_CODES[cos.dtype], eps)

    def run():
        nat.check(nat.lib().aicas_paged_rope_append(args, _stream_handle(device)), "aicas_paged_rope_append")

    _call_in_device(device, run)
    return q_out


def paged_gqa_decode_attention(
    query: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    *,
    sm_scale: float,
    num_key_value_groups: int,
    kv_lens: torch.Tensor | Sequence[int] | None = None,
    kv_starts: torch.Tensor | Sequence[int] | None = None,
    return_lse: bool = False,
):
    """:func:`aicas_b200.gqa_decode_attention` over a paged cache: one query token
    per request, softmax(sm_scale * q K^T) V over its slots ``[kv_starts[b], kv_lens[b])``.

    query ``[B, Hq, 1, D]``, pages ``[P, Hkv, page_size, D]``, page_table int32
    ``[B, max_pages]`` -> ``[B, Hq, 1, D]``; any whole number of query heads a
    key-value head.  ``kv_lens`` (int32 ``[B]``) defaults to all of the page table's
    slots, ``kv_starts`` to 0 (a sliding window, or the padding of a left-padded
    prompt, otherwise).  Slots outside the range may hold anything, NaN among it.
    A request without a slot gets zeros.  With ``return_lse`` the base-2 log-sum-exp
    ``[B, Hq]`` is returned too.  Page numbers outside the pool read as zeros."""
    _reject_grad(query, k_pages, v_pages)
    shape, ks, vs, page_table = _check_pool("paged_gqa_decode_attention", query, k_pages, v_pages, page_table)
    B, Hq, q_len, D = query.shape
    Hkv = shape[1]
    if q_len != 1:
        raise ValueError("paged_gqa_decode_attention needs q_len == 1")
    if num_key_value_groups < 1 or Hq != Hkv * num_key_value_groups:
        raise ValueError("num_q_heads != num_kv_heads * num_key_value_groups")
    device, dtype = query.device, query.dtype
    query = _heads_ready(query)
    lens = _lens(kv_lens, B, device)
    starts = _lens(kv_starts, B, device)
    out = torch.empty((B, 1, Hq, D), dtype=dtype, device=device).transpose(1, 2)
    lse = torch.empty((B, Hq), dtype=torch.float32, device=device) if return_lse else None
    if B == 0:
        return (out, lse) if return_lse else out
    qi, oi = query.stride(), out.stride()
    args = nat.PACK_PAGED_DECODE.pack(
        query.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), _pointer(lse),
        page_table.data_ptr(), _pointer(lens), _pointer(starts), qi[0], qi[1], oi[0], oi[1],
        ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], page_table.stride(0),
        B, Hq, Hkv, D, shape[0], shape[2], page_table.shape[1], _DTYPE_CODES[dtype], sm_scale)

    def run():
        lib = nat.lib()
        stream = _stream_handle(device)
        nbytes = lib.aicas_paged_decode_workspace_bytes(args)
        ws = _workspace(device, stream, nbytes)
        nat.check(lib.aicas_paged_decode_gqa(args, ws.data_ptr(), ws.numel(), stream), "aicas_paged_decode_gqa")

    _call_in_device(device, run)
    return (out, lse) if return_lse else out
