"""Restatement of the 4-bit cache's and the eviction's operators on CPU (test infrastructure only).

* ``levels``   - the (scale, least) pairs and unrounded codes of rows in groups
* ``values``   - what codes and pairs stand for, in float64
* ``unpack`` / ``pack`` - codes [..., D / 2] bytes to [..., D] numbers and back
* ``weights``  - what attention gives to each slot, in float64
* ``evict``    - the kept slots of one (request, head), and a compaction of rows
"""
from __future__ import annotations

import numpy as np

from .rope import round_to


def unpack(codes: np.ndarray) -> np.ndarray:
    out = np.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=np.uint8)
    out[..., 0::2], out[..., 1::2] = codes & 15, codes >> 4
    return out


def pack(q: np.ndarray) -> np.ndarray:
    return (q[..., 0::2] | (q[..., 1::2] << 4)).astype(np.uint8)


def levels(x: np.ndarray, group: int, dtype: str):
    """(scale, least, code before it is rounded) of rows [..., D]: pairs [..., D / g],
    rounded to ``dtype``, the scale after an fp32 difference and an fp32 product with 1 / 15;
    codes [..., D] in float64."""
    y = x.astype(np.float64).reshape(*x.shape[:-1], -1, group)
    least = round_to(y.min(-1), dtype)
    with np.errstate(over="ignore", invalid="ignore"):
        scale = round_to((y.max(-1).astype(np.float32) - least.astype(np.float32)) * np.float32(1 / 15), dtype)
    bad = ~np.isfinite(scale)
    scale[bad] = least[bad] = np.nan
    s, lo = scale[..., None].astype(np.float64), least[..., None].astype(np.float64)
    code = np.where(s > 0, (y - lo) / np.where(s > 0, s, 1.0), 0.0)
    return scale, least, np.clip(code, 0, 15).reshape(x.shape)


def values(q: np.ndarray, scale: np.ndarray, least: np.ndarray) -> np.ndarray:
    g = q.reshape(*q.shape[:-1], scale.shape[-1], -1).astype(np.float64)
    return (g * scale[..., None].astype(np.float64) + least[..., None].astype(np.float64)).reshape(q.shape)


def weights(q: np.ndarray, k: np.ndarray, lse: np.ndarray, length: int, start: int, scale: float) -> np.ndarray:
    """q [G, S, D] of one head's group, k [slots, D], lse [G, S] -> [slots]."""
    out = np.zeros(k.shape[0])
    S = q.shape[1]
    for s in range(S):
        end = length - S + 1 + s
        if end <= start:
            continue
        for j in range(q.shape[0]):
            if np.isneginf(lse[j, s]):
                continue
            score = k[start:end].astype(np.float64) @ q[j, s].astype(np.float64) * scale / np.log(2.0)
            out[start:end] += np.exp2(score - np.float64(lse[j, s]))
    return out


def kept_slots(w: np.ndarray, n: int, keep: int, first: int, last: int, longer_than: int) -> list[int]:
    if n <= longer_than:
        return list(range(n))
    key = [(-np.inf if np.isnan(v) else float(v)) for v in w[:n]]
    nan = [bool(np.isnan(v)) for v in w[:n]]
    middle = sorted(range(first, n - last), key=lambda t: (nan[t], -key[t], t))
    return sorted([*range(first), *middle[: keep - first - last], *range(n - last, n)])


def compact(pages: np.ndarray, row: np.ndarray, head: int, kept: list[int]) -> None:
    """Moves rows of one request and head to the front, in place; pages outside the
    pool read as zeros and take nothing."""
    size, num = pages.shape[2], pages.shape[0]
    inside = lambda t: 0 <= row[t // size] < num  # noqa: E731
    rows = [pages[row[t // size], head, t % size].copy() if inside(t) else np.zeros_like(pages[0, 0, 0]) for t in kept]
    for i, (t, r) in enumerate(zip(kept, rows)):
        if t != i and inside(i):
            pages[row[i // size], head, i % size] = r
