"""Paged key-value cache: the append with the position rotation on the way, the
single-token attention that reads it, and :class:`PagedKVCache`, which owns the
pages and hands them out.

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
from ._hostpath import (fast_append, fast_decode, heads_out, launch, launch_with_workspace, lengths, plain, pointer,
                        rows_ready, steps)
from .ops import _DTYPE_CODES, _WORKSPACES, SUPPORTED_HEAD_DIMS, _reject_grad

_ITEM = {torch.float32: 4, torch.float16: 2, torch.bfloat16: 2}


def _check_pool(what: str, query, k_pages, v_pages, page_table):
    """The pool's shape and strides and the page table, checked against the query."""
    device = query.device
    if device.type != "cuda":
        raise ValueError(f"{what} needs CUDA tensors")
    index = query.get_device()
    if k_pages.get_device() != index or v_pages.get_device() != index or page_table.get_device() != index:
        raise ValueError(f"{what} needs CUDA tensors: query, pages and page_table on one device")
    shape, q_shape = k_pages.shape, query.shape
    if len(q_shape) != 4 or len(shape) != 4 or v_pages.shape != shape:
        raise ValueError(f"{what}: query must be 4-D and the pages [P, Hkv, page_size, D] of one shape")
    dtype = query.dtype
    if dtype not in _DTYPE_CODES or k_pages.dtype is not dtype or v_pages.dtype is not dtype:
        raise ValueError(f"{what}: query and pages must share a dtype of fp32, fp16 or bf16")
    if shape[3] != q_shape[3] or shape[3] not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"{what}: head_dim {q_shape[3]} of the query, {shape[3]} of the pages; "
                         f"both must be one of {sorted(SUPPORTED_HEAD_DIMS)}")
    if shape[2] < 8 or shape[2] % 8:
        raise ValueError(f"{what}: page_size must be a positive multiple of 8 (got {shape[2]})")
    ks, vs = steps(k_pages), steps(v_pages)
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError(f"{what}: head_dim must be the unit-stride dimension of the pages")
    t_shape = page_table.shape
    if page_table.dtype is not torch.int32 or len(t_shape) != 2 or t_shape[0] != q_shape[0]:
        raise ValueError(f"{what}: page_table must be an int32 [{q_shape[0]}, max_pages] tensor")
    ts = page_table.stride()
    if ts[1] != 1:
        page_table = page_table.contiguous()
        ts = page_table.stride()
    return q_shape, shape, ks, vs, page_table, t_shape[1], ts[0]


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
    are rotated but not written.  ``kv_lens_out[b]`` receives the new length, in
    memory of its own (not that of ``positions``, ``num_new`` or the page table).
    Tokens past the page table's end, at negative slots or with a page number
    outside the pool are dropped, but count: the length is ``max(positions[b], 0) +
    num_new[b]``, at most the table's slots, as :func:`rope_kv_append` counts.  A
    request that has nothing to append gets ``num_new[b] = 0``.

    With fp32 cos/sin norm and rotation are held in fp32 and rounded once; with
    cos/sin of the tensors' 16-bit dtype every operation is rounded, as Hugging
    Face's modules and :func:`rope_kv_append` round, so such a model's keys are
    the same in either cache."""
    done = fast_append(query, key, value, cos, sin, k_pages, v_pages, page_table, positions, num_new, q_out, kv_lens_out,
                       q_norm_weight, k_norm_weight, eps)
    if done is not None:
        return done
    if query.requires_grad or key.requires_grad or value.requires_grad:
        _reject_grad(query, key, value)
    what = "paged_rope_kv_append"
    (B, Hq, S, D), shape, ks, vs, page_table, max_pages, table_stride = _check_pool(what, query, k_pages, v_pages,
                                                                                    page_table)
    device, dtype, Hkv = query.device, query.dtype, shape[1]
    if key.shape != (B, Hkv, S, D) or value.shape != (B, Hkv, S, D):
        raise ValueError(f"{what}: key and value must be [{B}, {Hkv}, {S}, {D}]")
    if Hkv == 0 or Hq % Hkv:
        raise ValueError(f"{what}: num_q_heads is not a multiple of num_kv_heads")
    index = query.get_device()
    if key.dtype is not dtype or value.dtype is not dtype or key.get_device() != index or value.get_device() != index:
        raise ValueError(f"{what}: query, key and value must share dtype and device")
    cs_shape, cs_dtype = cos.shape, cos.dtype
    if (cs_shape != (B, S, D) and cs_shape != (1, S, D)) or sin.shape != cs_shape:
        raise ValueError(f"{what}: cos/sin must be [B, S, D] (or [1, S, D])")
    if (cs_dtype is not torch.float32 and cs_dtype is not dtype) or sin.dtype is not cs_dtype:
        raise ValueError(f"{what}: cos/sin must have the tensor dtype or fp32")
    if cos.get_device() != index or sin.get_device() != index:
        raise ValueError(f"{what}: cos and sin must be on the query's device")
    item = _ITEM[dtype]
    query, qi = rows_ready(query, item)
    key, ki = rows_ready(key, item)
    value, vi = rows_ready(value, item)
    cs = steps(cos)
    if steps(sin) != cs or cs[2] != 1 or ((cs[0] | cs[1]) * _ITEM[cs_dtype] | cos.data_ptr() | sin.data_ptr()) & 15:
        cos, sin = plain(cos), plain(sin)
        cs = cos.stride()
    pos = lengths(positions, B, device)
    if pos is None:
        raise ValueError(f"{what}: positions are required")
    new = None if num_new is None else lengths(num_new, B, device)
    if kv_lens_out is not None and (kv_lens_out.shape != (B,) or kv_lens_out.dtype is not torch.int32
                                    or kv_lens_out.get_device() != index or not kv_lens_out.is_contiguous()):
        raise ValueError(f"{what}: kv_lens_out must be a contiguous int32 [{B}] tensor on the device")
    for w in (q_norm_weight, k_norm_weight):
        if w is not None and (w.shape != (D,) or w.dtype is not dtype or w.get_device() != index
                              or not w.is_contiguous()):
            raise ValueError(f"{what}: norm weights must be contiguous [D] of the tensor dtype")
    if q_out is None:
        q_out, qo = heads_out(B, Hq, S, D, dtype, device)
    else:
        qo = steps(q_out)
        if q_out.shape != (B, Hq, S, D) or q_out.dtype != dtype or q_out.device != device or qo[3] != 1:
            raise ValueError(f"{what}: q_out must be [{B}, {Hq}, {S}, {D}] with a unit-stride head_dim")
    if B == 0 or S == 0:
        if kv_lens_out is not None and B:
            kv_lens_out.copy_(pos.clamp(0, max_pages * shape[2]))
        return q_out
    launch(device, "aicas_paged_rope_append", nat.PACK_PAGED_APPEND.pack(
        query.data_ptr(), q_out.data_ptr(), key.data_ptr(), value.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), pos.data_ptr(), pointer(new),
        pointer(kv_lens_out), pointer(q_norm_weight), pointer(k_norm_weight),
        qi[0], qi[1], qi[2], qo[0], qo[1], qo[2], ki[0], ki[1], ki[2], vi[0], vi[1], vi[2],
        cs[0] if cs_shape[0] == B else 0, cs[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], table_stride,
        B, Hq, Hkv, S, D, shape[0], shape[2], max_pages, _DTYPE_CODES[dtype], _DTYPE_CODES[cs_dtype], eps))
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
    done = fast_decode(query, k_pages, v_pages, page_table, sm_scale, num_key_value_groups, kv_lens, kv_starts, return_lse,
                       _WORKSPACES)
    if done is not None:
        return done
    if query.requires_grad or k_pages.requires_grad or v_pages.requires_grad:
        _reject_grad(query, k_pages, v_pages)
    (B, Hq, q_len, D), shape, ks, vs, page_table, max_pages, table_stride = _check_pool(
        "paged_gqa_decode_attention", query, k_pages, v_pages, page_table)
    Hkv = shape[1]
    if q_len != 1:
        raise ValueError("paged_gqa_decode_attention needs q_len == 1")
    if num_key_value_groups < 1 or Hq != Hkv * num_key_value_groups:
        raise ValueError("num_q_heads != num_kv_heads * num_key_value_groups")
    device, dtype = query.device, query.dtype
    query, qi = rows_ready(query, _ITEM[dtype])
    lens = None if kv_lens is None else lengths(kv_lens, B, device)
    starts = None if kv_starts is None else lengths(kv_starts, B, device)
    out, oi = heads_out(B, Hq, 1, D, dtype, device)
    lse = torch.empty_strided((B, Hq), (Hq, 1), dtype=torch.float32, device=device) if return_lse else None
    if B > 0:
        launch_with_workspace(
            device, "aicas_paged_decode_gqa", "aicas_paged_decode_workspace_bytes", nat.PACK_PAGED_DECODE.pack(
                query.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), pointer(lse),
                page_table.data_ptr(), pointer(lens), pointer(starts), qi[0], qi[1], oi[0], oi[1],
                ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], table_stride,
                B, Hq, Hkv, D, shape[0], shape[2], max_pages, _DTYPE_CODES[dtype], sm_scale))
    return (out, lse) if return_lse else out


class PagedKVCache:
    """Page pools of every layer and the host's account of who holds which page.

    ``keys[i]`` / ``values[i]`` are the layers' pools ``[P, Hkv, page_size, D]``,
    allocated once; a page number means the same page in each layer.  Requests
    come (:meth:`add`), grow (:meth:`grow`) and go (:meth:`release`) on the host;
    :meth:`page_table` writes their rows for the kernels.  Released pages keep
    what they held: a kernel reads only the slots under the lengths it is given.
    Work that reads a released page and is already on a stream must be ordered
    before the work that writes its next holder's tokens (one stream does)."""

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, *,
                 dtype: torch.dtype, device: torch.device | str):
        if min(num_layers, num_pages, num_kv_heads) < 1:
            raise ValueError("PagedKVCache needs a positive number of layers, pages and heads")
        if page_size < 8 or page_size % 8:
            raise ValueError(f"PagedKVCache: page_size must be a positive multiple of 8 (got {page_size})")
        if dtype not in _DTYPE_CODES or head_dim not in SUPPORTED_HEAD_DIMS:
            raise ValueError(f"PagedKVCache: dtype {dtype}, head_dim {head_dim} are not ones that the kernels take")
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        self.page_size, self.num_pages = page_size, num_pages
        self.keys = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.values = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self._free = list(range(num_pages - 1, -1, -1))  # the lowest page goes out first
        self._held: dict[int, list[int]] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages(self, request: int) -> list[int]:
        """The pages that ``request`` holds, in the order of its tokens."""
        if request not in self._held:
            raise ValueError(f"request {request} holds no pages in this cache")
        return list(self._held[request])

    def add(self, tokens: int) -> int:
        """A new request with room for ``tokens`` tokens; its number."""
        request = self._next
        self._held[request] = []
        try:
            self.grow(request, tokens)
        except ValueError:
            del self._held[request]
            raise
        self._next += 1
        return request

    def grow(self, request: int, tokens: int) -> None:
        """Gives ``request`` room for ``tokens`` tokens in all (never takes any away).
        ``ValueError``, and nothing taken, where the pool has too few pages left."""
        have = len(self.pages(request))
        need = -(-tokens // self.page_size) - have
        if tokens < 0:
            raise ValueError("tokens must not be negative")
        if need > len(self._free):
            raise ValueError(f"paged cache is full: {need} pages needed, {len(self._free)} of {self.num_pages} free")
        for _ in range(need):
            self._held[request].append(self._free.pop())

    def release(self, request: int) -> None:
        """Takes all pages of ``request`` back."""
        self.pages(request)
        self._free.extend(reversed(self._held.pop(request)))

    def page_table(self, requests: Sequence[int], max_pages: int | None = None) -> torch.Tensor:
        """int32 ``[len(requests), max_pages]`` on the pools' device (``max_pages``
        defaults to the longest row's); -1, a page outside the pool, past a row's end."""
        rows = [self.pages(r) for r in requests]
        width = max([len(r) for r in rows], default=0) if max_pages is None else max_pages
        if any(len(r) > width for r in rows):
            raise ValueError(f"page_table: a request holds more than max_pages = {width} pages")
        width = max(width, 1)
        table = torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32).view(len(rows), width)
        return table.to(self.keys[0].device)

    def store(self, layer: int, request: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """Copies rotated keys and values ``[Hkv, S, D]`` (a prompt's, from another
        cache) to the first S slots of ``request``: a set-up step, in plain copies."""
        S, held = key.shape[1], self.pages(request)
        if S > len(held) * self.page_size:
            raise ValueError(f"store: {S} tokens do not fit the {len(held)} pages of request {request}")
        for pool, rows in ((self.keys[layer], key), (self.values[layer], value)):
            if rows.shape != (pool.shape[1], S, pool.shape[3]) or rows.dtype != pool.dtype:
                raise ValueError(f"store: keys and values must be [{pool.shape[1]}, {S}, {pool.shape[3]}] {pool.dtype}")
            full, rest = divmod(S, self.page_size)
            if full:
                where = torch.tensor(held[:full], device=pool.device)
                pool[where] = rows[:, :S - rest].reshape(pool.shape[1], full, self.page_size, -1).transpose(0, 1)
            if rest:
                pool[held[full], :, :rest] = rows[:, S - rest:]
