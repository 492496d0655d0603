"""Restatement of the 4-bit products on CPU (test infrastructure only):
``aicas_linear_int4`` in float64 from the weight's definition."""
from __future__ import annotations

import numpy as np


def widen(qweight: np.ndarray, scales: np.ndarray, zeros: np.ndarray | None) -> np.ndarray:
    """W[n, k] = scales[n, k // g] * (q[n, k] - zeros[n, k // g])."""
    n, half = qweight.shape
    q = np.empty((n, 2 * half))
    q[:, 0::2], q[:, 1::2] = qweight & 15, qweight >> 4
    g = 2 * half // scales.shape[1]
    z = 8.0 if zeros is None else np.repeat(zeros.astype(np.float64), g, axis=1)
    return (q - z) * np.repeat(scales.astype(np.float64), g, axis=1)


def norm_rows(x: np.ndarray, weight: np.ndarray, eps: float) -> np.ndarray:
    y = x.astype(np.float64)
    return y / np.sqrt((y * y).mean(axis=-1, keepdims=True) + eps) * weight.astype(np.float64)


def linear(x, weights, *, norm_weight=None, eps=1e-6, residual=None, swiglu=False, dtype="bf16"):
    """(y, bound): the product before its one rounding, and a bound of what it may
    be off before that.  fp32 sums of K terms, in whatever order: within 2^-15 of
    the sum of the terms' magnitudes (chains of up to 512 additions of relative
    error 2^-24, of terms up to 16 times larger while the zero point is still in).
    A normalised x of more than 4 rows for a bf16 result is rounded to 11 bits:
    within 2^-11 of itself; any other has two such parts, within 2^-22."""
    xd = norm_rows(x, norm_weight, eps) if norm_weight is not None else np.asarray(x, np.float64)
    ys = [xd @ w.T for w in weights]
    rel = 2.0 ** -15 + (2.0 ** -11 if norm_weight is not None and dtype == "bf16" and xd.shape[0] > 4 else 0.0)
    offs = [rel * (np.abs(xd) @ np.abs(w).T) for w in weights]
    if swiglu:
        s = ys[0] / (1.0 + np.exp(-ys[0]))
        # |silu'| <= 1.1
        return s * ys[1], 1.1 * offs[0] * np.abs(ys[1]) + (np.abs(s) + 1.1 * offs[0]) * offs[1] + 2.0 ** -20 * np.abs(s * ys[1])
    if residual is not None:
        return np.asarray(residual, np.float64) + ys[0], offs[0]
    return ys[0], offs[0]
