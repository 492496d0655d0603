"""Decode-side products with 4-bit weights: the weight's format, its
quantisation, and the product itself, :func:`decode_linear_int4`.

A weight ``[N, K]`` is kept as whole numbers 0..15 in groups of 32, 64 or 128
along K, each with a scale and (optionally) a zero point:
``W[n, k] = scales[n, k // g] * (q[n, k] - zeros[n, k // g])``, a quarter of the
bytes that :func:`aicas_b200.decode_linear` streams for each token.
"""
from __future__ import annotations

from typing import NamedTuple, Sequence

import torch

from . import _native as nat
from ._hostpath import fast_int4, launch, plain, pointer
from .ops import _LINEAR_DTYPES, _overlaps, _reject_grad

INT4_GROUP_SIZES = (32, 64, 128)


class Int4Weight(NamedTuple):
    """``qweight`` uint8 ``[N, K / 2]`` (even k in the low half of a byte),
    ``scales`` fp16/bf16 ``[N, K / g]``, ``zeros`` uint8 ``[N, K / g]`` of 0..15 or
    None (8 everywhere).  The kernels read it as it is: nothing is laid out anew."""

    qweight: torch.Tensor
    scales: torch.Tensor
    zeros: torch.Tensor | None = None

    def dequantize(self) -> torch.Tensor:
        """The fp32 weight ``[N, K]`` that the numbers stand for (any device)."""
        n, groups = self.scales.shape
        q = torch.stack([self.qweight & 15, self.qweight >> 4], -1).view(n, groups, -1).float()
        z = 8.0 if self.zeros is None else self.zeros.float()[..., None]
        return ((q - z) * self.scales.float()[..., None]).view(n, -1)


def quantize_int4(weight: torch.Tensor, group_size: int = 128, *, symmetric: bool = False) -> Int4Weight:
    """Rounds an fp16/bf16 (or fp32, then with bf16 scales) ``[N, K]`` weight to
    4 bits: per group the 16 levels are spread over ``[min, max]`` (with a zero
    point; 0 is always a level) or, ``symmetric``, over ``[-a, 7a / 8]`` around 8.
    A set-up step in plain torch operations, on any device."""
    if weight.ndim != 2 or not weight.is_floating_point():
        raise ValueError("quantize_int4 needs a floating-point [N, K] weight")
    n, k = weight.shape
    if group_size not in INT4_GROUP_SIZES or k % group_size or not n or not k:
        raise ValueError(f"quantize_int4: K = {k} must be a multiple of group_size, one of {INT4_GROUP_SIZES}")
    dtype = weight.dtype if weight.dtype in _LINEAR_DTYPES else torch.bfloat16
    w = weight.detach().float().view(n, k // group_size, group_size)
    if symmetric:
        scales = (w.abs().amax(-1) / 8).to(dtype)
        zeros = None
        z = 8.0
    else:
        lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        scales = ((hi - lo) / 15).to(dtype)
        step = torch.where(scales.float() > 0, scales.float(), 1.0)
        zeros = (-lo / step).round().clamp(0, 15).to(torch.uint8)
        z = zeros.float()[..., None]
    step = torch.where(scales.float() > 0, scales.float(), 1.0)[..., None]
    q = ((w / step).round() + z).clamp(0, 15).to(torch.uint8).view(n, k)
    return Int4Weight(q[:, 0::2] | (q[:, 1::2] << 4), scales.contiguous(), zeros)


def _check_weight(w, dtype: torch.dtype, index: int, k: int):
    """(qweight, its row stride, scales, zeros, N, groups) of one weight, checked against x."""
    q, scales, zeros = w
    _reject_grad(scales)
    if q.get_device() != index or scales.get_device() != index:
        raise ValueError("decode_linear_int4 needs CUDA tensors on one device")
    q_shape = q.shape
    if q.dtype is not torch.uint8 or len(q_shape) != 2 or q_shape[1] * 2 != k:
        raise ValueError(f"decode_linear_int4: qweight must be uint8 [N, {k // 2}]")
    n, shape = q_shape[0], scales.shape
    if len(shape) != 2 or shape[0] != n or scales.dtype is not dtype or not scales.is_contiguous():
        raise ValueError(f"decode_linear_int4: scales must be contiguous [{n}, K / g] of the dtype of x")
    s = q.stride()
    if s[1] != 1 or (s[0] | q.data_ptr()) & 15 or s[0] * 2 < k:
        q = plain(q)
        s = q.stride()
    if zeros is not None and (zeros.shape != shape or zeros.dtype is not torch.uint8
                              or zeros.get_device() != index or not zeros.is_contiguous()):
        raise ValueError("decode_linear_int4: zeros must be contiguous uint8 of the shape of the scales")
    return q, s[0], scales, zeros, n, shape[1]


def decode_linear_int4(
    x: torch.Tensor,
    weight: Int4Weight | Sequence[Int4Weight],
    *,
    norm_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    residual: torch.Tensor | None = None,
    swiglu: bool = False,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``x' W^T`` for the few rows of a decode step with a 4-bit ``W``:

    * ``x`` ``[R, K]`` fp16 or bf16, R <= 32; ``weight`` an :class:`Int4Weight` of
      ``[N, K]`` with scales of the dtype of x -> ``[R, N]``.  Several weights of
      one x (q, k and v) are one weight with their rows one after the other.
    * ``norm_weight`` ``[K]``: x' = RMSNorm(x) with that weight and ``eps`` in
      fp32; it enters the products as two fp16 parts, but with fp16's 11 bits for
      a bf16 result of more than 4 rows.
    * ``residual`` ``[R, N]``: returns ``residual + x' W^T``; ``out=residual`` updates
      it in place.
    * ``swiglu=True`` with ``weight=(gate, up)``: ``silu(x' Wg^T) * (x' Wu^T)``.

    Sums are held in fp32 and the result is rounded once.  ``ValueError`` for
    what the kernel cannot take, and for tensors that autograd would have to follow."""
    done = fast_int4(x, weight, norm_weight, eps, residual, swiglu, out)
    if done is not None:
        return done
    if swiglu:
        if len(weight) != 2 or isinstance(weight, Int4Weight):
            raise ValueError("swiglu needs weight=(gate, up)")
        first = weight[0]
    else:
        first = weight
        if len(weight) != 3 or not isinstance(weight[0], torch.Tensor):
            raise ValueError("decode_linear_int4 takes one Int4Weight, or with swiglu=True a (gate, up) pair")
    _reject_grad(x, *(t for t in (norm_weight, residual) if t is not None))
    dtype, device = x.dtype, x.device
    if device.type != "cuda":
        raise ValueError("decode_linear_int4 needs CUDA tensors")
    if dtype not in _LINEAR_DTYPES:
        raise ValueError("decode_linear_int4 needs fp16 or bf16 x")
    if x.ndim != 2:
        raise ValueError("x must be 2-D")
    R, K = x.shape
    index = x.get_device()
    xs = x.stride()
    if xs[1] != 1 or (xs[0] * 2 | x.data_ptr()) & 15 or xs[0] < K:  # unaligned, or rows that overlap
        x = plain(x)
        xs = x.stride()
    if R > nat.LINEAR_MAX_ROWS:
        raise ValueError(f"decode_linear_int4 takes at most {nat.LINEAR_MAX_ROWS} rows (got {R})")
    q, q_stride, scales, zeros, N, groups = _check_weight(first, dtype, index, K)
    if not groups or K % groups or K // groups not in INT4_GROUP_SIZES:
        raise ValueError(f"decode_linear_int4: {groups} scales a row of {K}: groups must be of {INT4_GROUP_SIZES}")
    second = (0, 0, 0, 0)
    if swiglu:
        if residual is not None:
            raise ValueError("decode_linear_int4: residual and swiglu exclude each other")
        q2, q2_stride, scales2, zeros2, *sizes = _check_weight(weight[1], dtype, index, K)
        if sizes != [N, groups] or (zeros2 is None) != (zeros is None):
            raise ValueError("decode_linear_int4: gate and up must be of one shape and kind")
        second = (q2.data_ptr(), scales2.data_ptr(), pointer(zeros2), q2_stride)
    mode, res, res_stride = nat.LINEAR_SWIGLU if swiglu else nat.LINEAR_STORE, 0, 0
    if residual is not None:
        mode, res, res_stride = nat.LINEAR_RESIDUAL, residual.data_ptr(), residual.stride(0)
        if residual.shape != (R, N) or residual.dtype is not dtype or residual.get_device() != index or residual.stride(1) != 1:
            raise ValueError(f"residual must be [{R}, {N}] of the dtype of x with unit stride on the last dimension")
    if norm_weight is not None:
        if norm_weight.shape != (K,) or norm_weight.dtype is not dtype or norm_weight.get_device() != index:
            raise ValueError(f"norm_weight must be a [{K}] tensor of the dtype of x")
        if not norm_weight.is_contiguous() or norm_weight.data_ptr() & 15:
            norm_weight = plain(norm_weight)
    if out is None:
        out, out_stride = torch.empty_strided((R, N), (N, 1), dtype=dtype, device=device), N
    else:
        if out.shape != (R, N) or out.dtype != dtype or out.device != device or out.stride(1) != 1 \
                or (R > 1 and out.stride(0) < N):
            raise ValueError(f"out must be [{R}, {N}] of the dtype of x with rows apart and unit stride within")
        out_stride = out.stride(0)
        # every CTA reads all of x while others already write their outputs
        if _overlaps(out, x) or (norm_weight is not None and _shares(out, norm_weight)):
            raise ValueError("decode_linear_int4: out must not overlap x or norm_weight")
        # a residual is read where its sum is written: the same elements, or others altogether
        if residual is not None and _overlaps(out, residual) and (res != out.data_ptr() or (R > 1 and res_stride != out_stride)):
            raise ValueError("decode_linear_int4: out must be the residual or not overlap it")
    if R and N:
        launch(device, "aicas_linear_int4", nat.PACK_LINEAR_INT4.pack(
            x.data_ptr(), xs[0], pointer(norm_weight), res, res_stride, out.data_ptr(), out_stride,
            q.data_ptr(), scales.data_ptr(), pointer(zeros), q_stride, *second,
            R, K, N, K // groups, mode, _LINEAR_DTYPES[dtype], eps))
    return out


def _shares(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.untyped_storage().data_ptr() == b.untyped_storage().data_ptr()
