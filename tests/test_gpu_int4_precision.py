"""How near the 4-bit products come to their definition, beyond a bound of the
largest error: shares of results, extreme magnitudes and infinities."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aicas_b200 as ab
from oracle import int4 as oi

pytestmark = pytest.mark.gpu


def _np(t):
    return None if t is None else t.detach().float().cpu().numpy()


def _weight(g, n, k, group, dtype, zeros, device):
    q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.int32).to(torch.uint8)
    s = ((0.5 + torch.rand(n, k // group, generator=g)) / (4 * k ** 0.5)).to(dtype)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.int32).to(torch.uint8) if zeros else None
    return ab.Int4Weight(q.to(device), s.to(device), None if z is None else z.to(device))


def _wide(w):
    return oi.widen(w.qweight.cpu().numpy(), _np(w.scales), None if w.zeros is None else w.zeros.cpu().numpy())


@pytest.mark.parametrize("rows", [1, 2, 3, 4])
@pytest.mark.parametrize("k,zeros,swiglu", [(2048, False, False), (1024, True, False), (640, True, True)])
def test_normalised_rows_give_the_rounded_definition(cuda_device, rows, k, zeros, swiglu):
    """Nearly every bf16 result is the definition's, rounded once.  Errors of the fp32
    sums of 2^-18 of the results' size (twice as much after SiLU * up) move a result
    over a rounding boundary, 2^-8 of it apart, in E[2 * 2^-18 / (2^-8 |y|)] of the
    cases, about 2^-9 * 5.5 = 1.1 % for normal y: 1 in 32 is allowed (an x' of 11 bits
    has errors of 2^-12.8 and moves one in ten)."""
    g = torch.Generator().manual_seed(10 * k + rows)
    x = torch.randn(rows, k, generator=g).to(torch.bfloat16).to(cuda_device)
    nw = (1 + 0.2 * torch.randn(k, generator=g)).to(torch.bfloat16).to(cuda_device)
    w = [_weight(g, 4096, k, 128 if k % 128 == 0 else 64, torch.bfloat16, zeros, cuda_device) for _ in range(1 + swiglu)]
    y = ab.decode_linear_int4(x, w if swiglu else w[0], norm_weight=nw, swiglu=swiglu)
    ref, _ = oi.linear(_np(x), [_wide(v) for v in w], norm_weight=_np(nw), swiglu=swiglu)
    rounded = torch.from_numpy(ref).to(torch.bfloat16).float().numpy()
    assert np.mean(_np(y) != rounded) <= 1 / 32


@pytest.mark.parametrize("size", [1e-30, 1e-34, 1e-36, 1e-37, 2e-38, 3e-39])
@pytest.mark.parametrize("rows", [1, 9])
def test_rows_near_the_smallest_numbers(cuda_device, size, rows):
    """bf16 rows down to subnormal ones.  An element may be off by 2^-30 of its row's
    largest or by 2^-147, whichever is more, before fp32 sums and one rounding (to
    2^-8 of the result, or half of the smallest bf16, 2^-134)."""
    k, n = 512, 200
    g = torch.Generator().manual_seed(int(-np.log10(size) * 10))
    x = (size * torch.randn(rows, k, generator=g)).to(torch.bfloat16).to(cuda_device)
    w = _weight(g, n, k, 64, torch.bfloat16, True, cuda_device)
    w = w._replace(scales=w.scales * 16)
    y = ab.decode_linear_int4(x, w)
    ref, off = oi.linear(_np(x), [_wide(w)])
    each = np.maximum(2.0 ** -30 * np.abs(_np(x)).max(1, keepdims=True).astype(np.float64), 2.0 ** -147)
    off = off + each * np.abs(_wide(w)).sum(1)
    over = np.abs(_np(y).astype(np.float64) - ref) - (2.0 ** -8 * (np.abs(ref) + off) + off + 2.0 ** -134)
    assert over.max() <= 0 and np.abs(ref).max() > 0


@pytest.mark.parametrize("rows", [1, 9])
def test_small_rows_under_large_norm_weights(cuda_device, rows):
    """Rows of zeros, and rows whose large norm weights meet zeros, beside tiny ones:
    no factor on the way is infinite.  x' is fp32: what is normalised to less than its
    smallest normal number, 2^-126, may be lost."""
    k, n = 256, 64
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, k, generator=g) * 1e-30
    nw = torch.full((k,), 1e-20)
    x[:, ::5], nw[::5] = 0.0, 3e38
    x[-1] = 0.0
    x, nw = x.to(torch.bfloat16).to(cuda_device), nw.to(torch.bfloat16).to(cuda_device)
    w = _weight(g, n, k, 64, torch.bfloat16, True, cuda_device)
    w = w._replace(scales=w.scales * 2.0 ** 60)
    y = ab.decode_linear_int4(x, w, norm_weight=nw)
    ref, off = oi.linear(_np(x), [_wide(w)], norm_weight=_np(nw))
    off = off + 2.0 ** -126 * np.abs(_wide(w)).sum(1)
    assert (y[-1] == 0).all() and bool(y.isfinite().all())
    assert np.all(np.abs(_np(y).astype(np.float64) - ref) <= 2.0 ** -8 * (np.abs(ref) + off) + off + 2.0 ** -134)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k,n", [(1, 256, 200), (3, 640, 100), (9, 2048, 130), (32, 6144, 70)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("kind", ["store", "residual", "swiglu"])
def test_infinite_elements_of_x(cuda_device, dtype, rows, k, n, zeros, kind):
    """An infinite x comes out as the definition has it: an infinity, or NaN where it
    meets its zero point or an opposite one.  Rows with NaN are NaN, the others are what
    they are without either."""
    g = torch.Generator().manual_seed(rows + k)
    clean = torch.randn(rows, k, generator=g)
    x = clean.clone()
    inf = float("inf")
    x[0, k // 3] = -inf
    if rows > 2:
        x[1, 5], x[1, k - 1] = inf, inf
        x[2, 0], x[2, k - 2] = inf, float("nan")
    if rows > 8:
        x[4, 1::2] = inf
        x[7, 3], x[7, k - 9] = inf, -inf
        x[rows - 1, k // 2:] = -inf
    w = [_weight(g, n, k, 64, dtype, zeros, cuda_device) for _ in range(1 + (kind == "swiglu"))]
    res = torch.randn(rows, n, generator=g).to(dtype).to(cuda_device) if kind == "residual" else None
    run = lambda t: ab.decode_linear_int4(t.to(dtype).to(cuda_device), w if kind == "swiglu" else w[0],  # noqa: E731
                                          residual=res, swiglu=kind == "swiglu")
    got, base = run(x), run(clean)
    with np.errstate(all="ignore"):
        ref, _ = oi.linear(_np(x.to(dtype)), [_wide(v) for v in w], residual=_np(res), swiglu=kind == "swiglu")
    hit = ~x.isfinite().all(1).numpy()
    assert np.array_equal(_np(got)[hit], ref[hit].astype(np.float32), equal_nan=True)
    assert torch.equal(got[torch.from_numpy(~hit)], base[torch.from_numpy(~hit)]) and bool(base.isfinite().all())
