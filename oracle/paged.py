"""Restatement of the paged cache's operators on CPU (test infrastructure only).

* ``gather`` - the slots ``[0, n)`` of one request as a contiguous ``[Hkv, n, D]``
* ``append`` - the cache write of ``aicas_paged_rope_append`` (rotation: ``rope``)
* ``decode`` - ``aicas_paged_decode_gqa`` in float64: softmax attention over the
               slots ``[start, len)`` and its base-2 log-sum-exp
* ``rotate`` - per-head RMSNorm and rotate-half rotation in float64
"""
from __future__ import annotations

import numpy as np

from . import attention as oa
from .rope import rotate_half


def gather(pages: np.ndarray, row: np.ndarray, n: int) -> np.ndarray:
    size = pages.shape[2]
    cols = [pages[int(row[t // size]), :, t % size] for t in range(n)]
    return np.stack(cols, axis=1) if n else np.zeros((pages.shape[1], 0, pages.shape[3]))


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, weight=None, eps: float = 1e-6) -> np.ndarray:
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(axis=-1, keepdims=True) + eps) * weight.astype(np.float64)
    return y * cos.astype(np.float64)[:, None] + rotate_half(y) * sin.astype(np.float64)[:, None]


def append(pages: np.ndarray, new: np.ndarray, table: np.ndarray, positions, counts) -> np.ndarray:
    """A copy of ``pages`` with the first ``counts[b]`` tokens of ``new [B, Hkv, S, D]`` written."""
    pages = pages.copy()
    num, _, size, _ = pages.shape
    for b in range(new.shape[0]):
        for s in range(max(0, min(int(counts[b]), new.shape[2]))):
            t = int(positions[b]) + s
            if 0 <= t < table.shape[1] * size and 0 <= table[b, t // size] < num:
                pages[table[b, t // size], :, t % size] = new[b, :, s]
    return pages


def decode(q, k_pages, v_pages, table, lens, starts, scale: float, groups: int):
    """(out [B, Hq, 1, D], lse [B, Hq]) in float64."""
    B, Hq, _, D = q.shape
    out, lse = np.zeros((B, Hq, 1, D)), np.full((B, Hq), -np.inf)
    cap = table.shape[1] * k_pages.shape[2]
    for b in range(B):
        n = min(max(int(lens[b]), 0), cap)
        s = min(max(int(starts[b]), 0), n)
        if s == n:
            continue
        k, v = (gather(p, table[b], n)[None, :, s:].astype(np.float64) for p in (k_pages, v_pages))
        out[b:b + 1] = oa.sdpa(q[b:b + 1], k, v, scale, False, groups)
        lse[b:b + 1] = oa.lse_base2(q[b:b + 1], k, scale, groups)
    return out, lse
