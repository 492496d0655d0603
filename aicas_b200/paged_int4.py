"""Paged key-value cache in 4 bits: the append that rounds on the way, the
single-token attention that reads the rows as stored, and the read that gives
them back as 16-bit values.

A pool is an :class:`Int4Pages` instead of :mod:`aicas_b200.paged`'s tensor
``[P, Hkv, page_size, D]``: a row (one head of one token) is D codes of 4 bits and
a pair ``(scale, least)`` for each group of 64 elements, or of all D, so that
element d stands for ``scale * code[d] + least``.  A row of 128 takes 68 or 72
bytes, not 256.  Page tables, lengths and strides are :mod:`aicas_b200.paged`'s.

The reference has 16-bit contiguous caches in its served path
(dujunbaoV1/evaluation_wrapper.py:54-112).  The rules are those of
:mod:`aicas_b200.ops`: the caller's current stream, no host synchronisation,
``ValueError`` for what the kernels cannot take.
"""
from __future__ import annotations

import operator
from typing import NamedTuple, Sequence

import torch

from . import _native as nat
from ._hostpath import fast, heads_out, launch, launch_with_workspace, lengths, pointer, rows_ready, steps
from .ops import _DTYPE_CODES, _LINEAR_DTYPES, _WORKSPACES, _reject_grad
from .paged import _new_rows

INT4_HEAD_DIMS = (64, 128)


class Int4Pages(NamedTuple):
    """``codes`` uint8 ``[P, Hkv, page_size, D / 2]`` (even d in the low half of a byte)
    and ``scales`` fp16/bf16 ``[P, Hkv, page_size, D / g, 2]``, the pairs (scale, least)
    of a row's groups.  D is 64 or 128, g is 64 or D.  Rows are contiguous; the strides
    of pages, heads and rows are free (multiples of 16 bytes for the codes)."""

    codes: torch.Tensor
    scales: torch.Tensor

    def dequantize(self) -> torch.Tensor:
        """The fp32 rows ``[..., D]`` that the numbers stand for (any device)."""
        q = torch.stack([self.codes & 15, self.codes >> 4], -1).flatten(-2)
        q = q.unflatten(-1, (self.scales.shape[-2], -1)).float()
        s = self.scales.float()
        return (q * s[..., :1] + s[..., 1:]).flatten(-2)


def _check_group(head_dim: int, group_size: int) -> None:
    if head_dim not in INT4_HEAD_DIMS or group_size not in (64, head_dim):
        raise ValueError(f"4-bit rows need a head_dim of {INT4_HEAD_DIMS} and groups of 64 or head_dim "
                         f"(got {head_dim}, {group_size})")


def int4_pages(num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, group_size: int | None = None, *,
               dtype: torch.dtype, device: torch.device | str) -> Int4Pages:
    """A pool of zeros; ``group_size`` defaults to ``head_dim``."""
    group_size = head_dim if group_size is None else group_size
    _check_group(head_dim, group_size)
    if dtype not in _LINEAR_DTYPES:
        raise ValueError(f"4-bit pages need fp16 or bf16 scales (got {dtype})")
    shape = (num_pages, num_kv_heads, page_size)
    return Int4Pages(torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device=device),
                     torch.zeros(*shape, head_dim // group_size, 2, dtype=dtype, device=device))


def quantize_kv_int4(rows: torch.Tensor, group_size: int | None = None) -> Int4Pages:
    """Codes ``[..., D / 2]`` and scales ``[..., D / g, 2]`` of fp16/bf16 rows ``[..., D]``,
    as :func:`paged_rope_kv_append_int4` writes them: a set-up step in plain torch
    operations, on any device."""
    d = rows.shape[-1]
    group_size = d if group_size is None else group_size
    _check_group(d, group_size)
    if rows.dtype not in _LINEAR_DTYPES:
        raise ValueError(f"quantize_kv_int4 needs fp16 or bf16 rows (got {rows.dtype})")
    x = rows.detach().float().unflatten(-1, (d // group_size, group_size))
    lo = x.amin(-1).to(rows.dtype)
    scale = ((x.amax(-1) - lo.float()) * (1 / 15)).to(rows.dtype)  # on a GPU torch's "/ 15" is this product too
    bad = ~(scale.float().abs() < torch.inf)
    scale, lo = scale.masked_fill(bad, torch.nan), lo.masked_fill(bad, torch.nan)
    step, least = scale.float()[..., None], lo.float()[..., None]
    fine = step >= torch.finfo(torch.float32).tiny
    q = torch.where(fine, (x - least) / torch.where(fine, step, 1.0), 0.0)
    q = q.round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return Int4Pages(q[..., 0::2] | (q[..., 1::2] << 4), torch.stack([scale, lo], -1))


def _side(what: str, pages, index: int, dtype: torch.dtype | None):
    """One side's shape (P, Hkv, page_size, D, g) and packed reference, checked."""
    if not isinstance(pages, tuple) or len(pages) != 2:
        raise ValueError(f"{what}: the pages must be Int4Pages")
    codes, scales = pages
    if codes.get_device() != index or scales.get_device() != index:
        raise ValueError(f"{what} needs CUDA tensors on one device")
    shape, s_shape = codes.shape, scales.shape
    if codes.dtype is not torch.uint8 or len(shape) != 4:
        raise ValueError(f"{what}: codes must be uint8 [P, Hkv, page_size, D / 2]")
    if scales.dtype not in _LINEAR_DTYPES or (dtype is not None and scales.dtype is not dtype):
        raise ValueError(f"{what}: scales must be fp16 or bf16, of the query's dtype")
    if len(s_shape) != 5 or s_shape[:3] != shape[:3] or s_shape[4] != 2 or s_shape[3] < 1 or shape[3] * 2 % s_shape[3]:
        raise ValueError(f"{what}: scales must be [P, Hkv, page_size, D / g, 2] beside codes of {tuple(shape)}")
    dim = shape[3] * 2
    _check_group(dim, dim // s_shape[3])
    if shape[2] < 8 or shape[2] % 8:
        raise ValueError(f"{what}: page_size must be a positive multiple of 8 (got {shape[2]})")
    cs, ss = steps(codes), steps(scales)
    if cs[3] != 1 or ss[4] != 1 or (s_shape[3] > 1 and ss[3] != 2):
        raise ValueError(f"{what}: the codes and the pairs of a row must be contiguous")
    if scales.requires_grad:
        _reject_grad(scales)
    return (*shape[:3], dim, dim // s_shape[3]), (codes.data_ptr(), scales.data_ptr(), *cs[:3], *ss[:3])


def _pools(what: str, like: torch.Tensor, k_pages, v_pages, page_table, batch: int, dtype: torch.dtype | None):
    """((P, Hkv, page_size, D, g), both sides' packed references, the page table, its
    width and stride), checked.  ``like``: a tensor that says the device."""
    index = like.get_device()
    if like.device.type != "cuda":
        raise ValueError(f"{what} needs CUDA tensors")
    shape, k_ref = _side(what, k_pages, index, dtype)
    v_shape, v_ref = _side(what, v_pages, index, dtype)
    if v_shape != shape or k_pages[1].dtype is not v_pages[1].dtype:
        raise ValueError(f"{what}: keys' and values' pages must be of one shape and dtype")
    return shape, (*k_ref, *v_ref), *_table(what, page_table, batch, index)


def _table(what: str, page_table, batch: int, index: int):
    t_shape = page_table.shape
    if page_table.dtype is not torch.int32 or len(t_shape) != 2 or t_shape[0] != batch or page_table.get_device() != index:
        raise ValueError(f"{what}: page_table must be an int32 [{batch}, max_pages] tensor on the device")
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    return page_table, t_shape[1], page_table.stride(0)


def _check_query(what: str, query) -> None:
    if query.ndim != 4:
        raise ValueError(f"{what}: query must be 4-D")
    if query.device.type != "cuda":
        raise ValueError(f"{what} needs CUDA tensors")
    if query.dtype not in _LINEAR_DTYPES:
        raise ValueError(f"{what} needs fp16 or bf16 tensors")


def paged_rope_kv_append_int4(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    k_pages: Int4Pages,
    v_pages: Int4Pages,
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
    """:func:`aicas_b200.paged_rope_kv_append` into a cache of 4-bit rows: the same
    arguments, rotation, rounding, drops and lengths, but for the pages, whose scales
    are of the query's dtype (fp16 or bf16).

    A group's least value, and its range above that times 1/15 (an fp32 product), are
    rounded to that dtype; each element becomes the nearest of the 16 levels.  A group that is all one
    value gets that value, one with an element that is not finite reads back as NaN."""
    done = fast("append_int4", query, key, value, cos, sin, k_pages, v_pages, page_table, positions, num_new, q_out,
                kv_lens_out, q_norm_weight, k_norm_weight, eps)
    if done is not None:
        return done
    if query.requires_grad or key.requires_grad or value.requires_grad:
        _reject_grad(query, key, value)
    what = "paged_rope_kv_append_int4"
    _check_query(what, query)
    B, Hq, S, D = query.shape
    (P, Hkv, size, dim, group), refs, page_table, max_pages, table_stride = _pools(
        what, query, k_pages, v_pages, page_table, B, query.dtype)
    if dim != D:
        raise ValueError(f"{what}: head_dim {D} of the query, {dim} of the pages")
    rows, steps_of_rows, per_request, dtypes, pos, q_out, _held = _new_rows(
        what, query, key, value, cos, sin, Hkv, positions, num_new, q_out, kv_lens_out, q_norm_weight, k_norm_weight)
    if B == 0 or S == 0:
        if kv_lens_out is not None and B:
            kv_lens_out.copy_(pos.clamp(0, max_pages * size))
        return q_out
    launch(query.device, "aicas_paged_append_int4", nat.PACK_PAGED_APPEND_INT4.pack(
        *rows, *refs, page_table.data_ptr(), *per_request, *steps_of_rows, table_stride,
        B, Hq, Hkv, S, D, group, P, size, max_pages, *dtypes, eps))
    return q_out


def paged_kv_read_int4(
    k_pages: Int4Pages,
    v_pages: Int4Pages,
    page_table: torch.Tensor,
    positions: torch.Tensor | Sequence[int],
    seq_len: int,
    *,
    num_tokens: torch.Tensor | Sequence[int] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values ``[B, Hkv, seq_len, D]`` (of the scales' dtype) that the slots
    ``positions[b] + s`` hold: a cached prefix as the 16-bit rows that a model's own
    modules, :func:`aicas_b200.gqa_flash_attention` or another cache take.  Rows past
    ``num_tokens[b]`` (int32 ``[B]``, default all), slots outside the page table and
    pages outside the pool read as zeros."""
    done = fast("read_int4", k_pages, v_pages, page_table, positions, seq_len, num_tokens)
    if done is not None:
        return done
    what = "paged_kv_read_int4"
    if not isinstance(k_pages, tuple) or len(k_pages) != 2 or page_table.ndim != 2:
        raise ValueError(f"{what} needs Int4Pages and a page_table [B, max_pages]")
    B = page_table.shape[0]
    (P, Hkv, size, D, group), refs, page_table, max_pages, table_stride = _pools(
        what, page_table, k_pages, v_pages, page_table, B, None)
    device, dtype = page_table.device, k_pages[1].dtype
    seq_len = operator.index(seq_len)
    if seq_len < 0:
        raise ValueError(f"{what}: seq_len must not be negative")
    pos = lengths(positions, B, device)
    if pos is None:
        raise ValueError(f"{what}: positions are required")
    count = None if num_tokens is None else lengths(num_tokens, B, device)
    shape, strides = (B, Hkv, seq_len, D), (Hkv * seq_len * D, seq_len * D, D, 1)
    k, v = (torch.empty_strided(shape, strides, dtype=dtype, device=device) for _ in range(2))
    if k.numel():
        launch(device, "aicas_paged_read_int4", nat.PACK_PAGED_READ_INT4.pack(
            *refs, k.data_ptr(), v.data_ptr(), page_table.data_ptr(), pos.data_ptr(), pointer(count), *strides[:3],
            table_stride, B, Hkv, seq_len, D, group, P, size, max_pages, _DTYPE_CODES[dtype]))
    return k, v


def paged_gqa_decode_attention_int4(
    query: torch.Tensor,
    k_pages: Int4Pages,
    v_pages: Int4Pages,
    page_table: torch.Tensor,
    *,
    sm_scale: float,
    num_key_value_groups: int,
    kv_lens: torch.Tensor | Sequence[int] | None = None,
    kv_starts: torch.Tensor | Sequence[int] | None = None,
    return_lse: bool = False,
):
    """:func:`aicas_b200.paged_gqa_decode_attention` over a cache of 4-bit rows: the same
    arguments, masks and results, but for the pages, whose scales are of the query's
    dtype (fp16 or bf16).  The codes enter the products as they are; scores, statistics
    and sums are held in fp32 and the result is rounded once."""
    done = fast("decode_int4", query, k_pages, v_pages, page_table, sm_scale, num_key_value_groups, kv_lens, kv_starts,
                return_lse, _WORKSPACES)
    if done is not None:
        return done
    if query.requires_grad:
        _reject_grad(query)
    what = "paged_gqa_decode_attention_int4"
    _check_query(what, query)
    B, Hq, q_len, D = query.shape
    (P, Hkv, size, dim, group), refs, page_table, max_pages, table_stride = _pools(
        what, query, k_pages, v_pages, page_table, B, query.dtype)
    if dim != D:
        raise ValueError(f"{what}: head_dim {D} of the query, {dim} of the pages")
    if q_len != 1:
        raise ValueError(f"{what} needs q_len == 1")
    if num_key_value_groups < 1 or Hq != Hkv * num_key_value_groups:
        raise ValueError("num_q_heads != num_kv_heads * num_key_value_groups")
    device, dtype = query.device, query.dtype
    query, qi = rows_ready(query, 2)
    lens = None if kv_lens is None else lengths(kv_lens, B, device)
    starts = None if kv_starts is None else lengths(kv_starts, B, device)
    out, oi = heads_out(B, Hq, 1, D, dtype, device)
    lse = torch.empty_strided((B, Hq), (Hq, 1), dtype=torch.float32, device=device) if return_lse else None
    if B > 0:
        launch_with_workspace(
            device, "aicas_paged_decode_int4", "aicas_paged_decode_int4_workspace_bytes", nat.PACK_PAGED_DECODE_INT4.pack(
                query.data_ptr(), *refs, out.data_ptr(), pointer(lse), page_table.data_ptr(), pointer(lens),
                pointer(starts), qi[0], qi[1], oi[0], oi[1], table_stride,
                B, Hq, Hkv, D, group, P, size, max_pages, _DTYPE_CODES[dtype], sm_scale))
    return (out, lse) if return_lse else out
