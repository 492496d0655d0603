"""The 4-bit products on the GPU against their float64 restatement.

Tolerance: half a unit in the last place of the result (it is rounded once) plus
the bound of the fp32 sums that ``oracle.int4.linear`` returns with the value."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _native as nat
from oracle import int4 as oi

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _np(t):
    return None if t is None else t.detach().float().cpu().numpy()


def _weight(g, n, k, group, dtype, zeros, device):
    q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.int32).to(torch.uint8)
    s = ((0.5 + torch.rand(n, k // group, generator=g)) / (4 * k ** 0.5)).to(DT[dtype])
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.int32).to(torch.uint8) if zeros else None
    return ab.Int4Weight(q.to(device), s.to(device), None if z is None else z.to(device))


def _wide(w):
    return oi.widen(w.qweight.cpu().numpy(), _np(w.scales), None if w.zeros is None else w.zeros.cpu().numpy())


def _case(device, rows, k, n, group=128, dtype="bf16", zeros=False, norm=False, residual=False, swiglu=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g).to(DT[dtype]).to(device)
    w = [_weight(g, n, k, group, dtype, zeros, device) for _ in range(2 if swiglu else 1)]
    nw = (1 + 0.2 * torch.randn(k, generator=g)).to(DT[dtype]).to(device) if norm else None
    res = torch.randn(rows, n, generator=g).to(DT[dtype]).to(device) if residual else None
    y = ab.decode_linear_int4(x, w if swiglu else w[0], norm_weight=nw, residual=res, swiglu=swiglu)
    assert y.shape == (rows, n) and y.dtype == x.dtype
    ref, off = oi.linear(_np(x), [_wide(v) for v in w], norm_weight=_np(nw), residual=_np(res), swiglu=swiglu,
                         dtype=dtype)
    over = np.abs(_np(y).astype(np.float64) - ref) - (HALF_ULP[dtype] * (np.abs(ref) + off) + off)
    assert over.max() <= 2.0 ** -24, f"{over.max():.3e} over the bound at {np.unravel_index(over.argmax(), over.shape)}"
    assert nat.device_error_flags() == 0
    return x, w, nw, res, y


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 24, 25, 32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_rows_groups_and_types(cuda_device, rows, group, dtype):
    _case(cuda_device, rows, 640, 200, group, dtype, zeros=rows % 2 == 0, seed=rows)


@pytest.mark.parametrize("k,group", [(32, 32), (64, 32), (64, 64), (96, 32), (128, 128), (160, 32), (192, 64),
                                     (384, 128), (1056, 32), (2048, 128), (6144, 64), (8192, 128)])
@pytest.mark.parametrize("n", [1, 7, 16, 17, 130])
def test_odd_sizes(cuda_device, k, group, n):
    _case(cuda_device, 3, k, n, group, zeros=True, seed=k + n)


@pytest.mark.parametrize("rows", [1, 8, 20])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("kind", ["norm", "residual", "swiglu", "norm+residual", "norm+swiglu"])
def test_prologue_and_epilogues(cuda_device, rows, zeros, kind):
    _case(cuda_device, rows, 512, 333, 64, zeros=zeros, norm="norm" in kind, residual="residual" in kind,
          swiglu="swiglu" in kind, seed=rows)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_norm_of_many_rows(cuda_device, dtype):
    _case(cuda_device, 32, 1536, 90, 64, dtype, zeros=True, norm=True, residual=True)
    _case(cuda_device, 27, 8192, 40, 128, dtype, norm=True)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("norm", [False, True])
def test_rows_of_every_size(cuda_device, dtype, norm):
    """Rows of any magnitude the type has, zeros and single large elements, in one batch."""
    g = torch.Generator().manual_seed(12)
    k, top = 512, 1e36 if dtype == "bf16" else 2e3
    size = torch.tensor([1.0, top / 30, 1e-3 if dtype == "fp16" else 1e-30, 0.0, 37.0, 1e-2, 1.0, 5.0])
    x = (torch.randn(8, k, generator=g) * size[:, None]).to(DT[dtype])
    x[6, 100] = top  # one element far above the others
    x = x.to(cuda_device)
    w = _weight(g, 64, k, 64, dtype, True, cuda_device)
    nw = torch.ones(k, dtype=DT[dtype], device=cuda_device) if norm else None
    y = ab.decode_linear_int4(x, w, norm_weight=nw, eps=1e-6 if norm else 0.0)
    ref, off = oi.linear(_np(x), [_wide(w)], norm_weight=_np(nw), dtype=dtype)
    # elements 2^30 below their row's largest may lose bits: 2^-34 of the largest, K times
    xd = oi.norm_rows(_np(x), _np(nw), 1e-6) if norm else _np(x).astype(np.float64)
    off = off + 2.0 ** -34 * k * np.abs(xd).max(1, keepdims=True) * np.abs(_wide(w)).max()
    off = off + (2.0 ** -25 if dtype == "fp16" else 0.0)
    assert np.all(np.abs(_np(y).astype(np.float64) - ref) <= HALF_ULP[dtype] * (np.abs(ref) + off) + off)
    assert (y[3] == 0).all()


@pytest.mark.parametrize("rows,k,n", [(1, 2048, 4096), (8, 2048, 6144), (32, 6144, 2048), (1, 2048, 40000),
                                      (32, 2048, 9001), (5, 14336, 300), (32, 16384, 64), (1, 32768, 50)])
def test_model_sizes(cuda_device, rows, k, n):
    _case(cuda_device, rows, k, n, seed=n)


def test_every_level_and_zero_point(cuda_device):
    """x picks single columns: each level 0..15 and zero point 0..15 comes back exactly."""
    k, n = 64, 256
    q = torch.arange(n)[:, None] % 16  # row n: level n % 16 in every column
    z = (torch.arange(n) // 16)[:, None].to(torch.uint8).repeat(1, 2)
    w = ab.Int4Weight((q | (q << 4)).to(torch.uint8).repeat(1, k // 2).to(cuda_device),
                      torch.full((n, 2), 0.5, dtype=torch.bfloat16, device=cuda_device), z.to(cuda_device))
    x = torch.zeros(4, k, dtype=torch.bfloat16, device=cuda_device)
    for r, col in enumerate([0, 1, 31, 63]):
        x[r, col] = 1
    y = ab.decode_linear_int4(x, w)
    want = 0.5 * (q[:, 0] - (torch.arange(n) // 16)).float()
    for r in range(4):
        assert torch.equal(y[r].float().cpu(), want)


def test_each_column_meets_its_weight(cuda_device):
    """One-hot rows return the weight's columns: no column is swapped or missed."""
    g = torch.Generator().manual_seed(4)
    for k, group in [(256, 128), (192, 64), (96, 32)]:
        w = _weight(g, 48, k, group, "fp16", True, cuda_device)
        wide = torch.from_numpy(_wide(w)).half()
        for c0 in range(0, k, 32):
            x = torch.zeros(32, k, dtype=torch.float16, device=cuda_device)
            x[torch.arange(32), c0 + torch.arange(32)] = 1
            assert torch.equal(ab.decode_linear_int4(x, w).cpu(), wide[:, c0:c0 + 32].t().contiguous())


def test_in_place_residual_strides_and_views(cuda_device):
    g = torch.Generator().manual_seed(6)
    wide_x = torch.randn(9, 1024, generator=g).to(torch.bfloat16).to(cuda_device)
    x = wide_x[:, 256:768]
    w = _weight(g, 130, 512, 64, "bf16", False, cuda_device)
    base = ab.decode_linear_int4(x.contiguous(), w)
    assert torch.equal(ab.decode_linear_int4(x, w), base)
    assert torch.equal(ab.decode_linear_int4(wide_x[:, 3:515], w),
                       ab.decode_linear_int4(wide_x[:, 3:515].contiguous(), w))
    out = torch.full((9, 140), 7.0, dtype=torch.bfloat16, device=cuda_device)
    ab.decode_linear_int4(x, w, out=out[:, 5:135])
    assert torch.equal(out[:, 5:135], base) and (out[:, :5] == 7).all() and (out[:, 135:] == 7).all()
    res = torch.randn(9, 130, generator=g).to(torch.bfloat16).to(cuda_device)
    want = ab.decode_linear_int4(x, w, residual=res)
    got = ab.decode_linear_int4(x, w, residual=res, out=res)
    assert got is res and torch.equal(res, want)
    one = torch.randn(1, 130, generator=g).to(torch.bfloat16).to(cuda_device)
    assert torch.equal(ab.decode_linear_int4(x, w, residual=one.expand(9, 130)),
                       ab.decode_linear_int4(x, w, residual=one.repeat(9, 1)))
    assert torch.equal(ab.decode_linear_int4(x[:1].expand(4, 512), w), base[:1].expand(4, 130))
    # rows of a larger quantised weight
    part = ab.Int4Weight(w.qweight[64:], w.scales[64:], None)
    assert torch.equal(ab.decode_linear_int4(x, part), base[:, 64:])


def test_rows_do_not_depend_on_the_batch_within_a_tile(cuda_device):
    """A row's result is the same whatever the other rows hold, NaN among it."""
    g = torch.Generator().manual_seed(8)
    w = _weight(g, 100, 256, 32, "bf16", True, cuda_device)
    x = torch.randn(8, 256, generator=g).to(torch.bfloat16).to(cuda_device)
    a = ab.decode_linear_int4(x, w)
    x2 = x.clone()
    x2[1::2] = float("nan")
    b = ab.decode_linear_int4(x2, w)
    assert torch.equal(a[0::2], b[0::2]) and torch.isnan(b[1::2]).all()


def test_repeats_to_the_bit_and_in_a_graph(cuda_device):
    x, w, nw, res, y = _case(cuda_device, 8, 2048, 1000, norm=True, residual=True)
    call = lambda: ab.decode_linear_int4(x, w[0], norm_weight=nw, residual=res)  # noqa: E731
    for _ in range(4):
        assert torch.equal(call(), y)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = call()
    x.mul_(0.5)
    res.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, call())


def test_quantized_layer_is_near_the_dense_one(cuda_device):
    """quantize_int4 and the product together: the error of a 4-bit weight, not more."""
    g = torch.Generator().manual_seed(10)
    w = (torch.randn(512, 1024, generator=g) / 32).to(torch.bfloat16).to(cuda_device)
    x = torch.randn(4, 1024, generator=g).to(torch.bfloat16).to(cuda_device)
    dense = x.float() @ w.float().t()
    for symmetric in (False, True):
        q = ab.quantize_int4(w, 64, symmetric=symmetric)
        y = ab.decode_linear_int4(x, q).float()
        want = x.float() @ q.dequantize().t()
        assert (y - want).abs().max().item() <= 2 ** -8 * want.abs().max().item() + 1e-3
        # a level's spacing is about 5 sigma / 15 and its rounding error spacing / sqrt(12): a tenth of sigma
        assert (y - dense).norm().item() <= 0.15 * dense.norm().item()


def test_empty(cuda_device):
    g = torch.Generator().manual_seed(1)
    w = _weight(g, 16, 64, 32, "bf16", False, cuda_device)
    assert ab.decode_linear_int4(torch.zeros(0, 64, dtype=torch.bfloat16, device=cuda_device), w).shape == (0, 16)


def test_refusals(cuda_device):
    g = torch.Generator().manual_seed(1)
    w = _weight(g, 16, 128, 32, "bf16", True, cuda_device)
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device=cuda_device)
    ok = ab.decode_linear_int4(x, w)
    for text, call in [
        ("CUDA", lambda: ab.decode_linear_int4(x.cpu(), w)),
        ("fp16 or bf16", lambda: ab.decode_linear_int4(x.float(), w)),
        ("at most 32 rows", lambda: ab.decode_linear_int4(x[:1].repeat(33, 1), w)),
        ("qweight", lambda: ab.decode_linear_int4(x[:, :64], w)),
        ("qweight", lambda: ab.decode_linear_int4(x, w._replace(qweight=w.qweight.to(torch.int32)))),
        ("scales", lambda: ab.decode_linear_int4(x, w._replace(scales=w.scales.half()))),
        ("zeros", lambda: ab.decode_linear_int4(x, w._replace(zeros=w.zeros[:, :2]))),
        ("groups", lambda: ab.decode_linear_int4(x, ab.Int4Weight(w.qweight, w.scales[:, :3].contiguous()))),
        ("groups", lambda: ab.decode_linear_int4(x, ab.Int4Weight(w.qweight, w.scales.repeat(1, 2)))),
        ("residual", lambda: ab.decode_linear_int4(x, w, residual=x)),
        ("norm_weight", lambda: ab.decode_linear_int4(x, w, norm_weight=x[0, :64])),
        ("gate, up", lambda: ab.decode_linear_int4(x, w, swiglu=True)),
        ("gate, up", lambda: ab.decode_linear_int4(x, [w, w])),
        ("one shape and kind", lambda: ab.decode_linear_int4(x, [w, w._replace(zeros=None)], swiglu=True)),
        ("exclude", lambda: ab.decode_linear_int4(x, [w, w], swiglu=True, residual=ok)),
        ("out must be", lambda: ab.decode_linear_int4(x, w, out=ok[:, :8])),
        ("overlap", lambda: ab.decode_linear_int4(x, w, out=x[:, :16])),
        ("inference", lambda: ab.decode_linear_int4(x.clone().requires_grad_(), w)),
    ]:
        with pytest.raises(ValueError, match=text):
            call()


@pytest.mark.parametrize("rows,k,dtype", [(32, 2304, "bf16"), (32, 2816, "bf16"), (20, 1280, "fp16"), (32, 6400, "fp16")])
def test_scales_past_the_end_of_k_are_not_read(cuda_device, rows, k, dtype):
    """K in an odd number of 256s, many rows: the last CTA of a cluster has less of
    K than the others.  What follows the scales and zero points counts for nothing."""
    n, group = 96, 128
    g = torch.Generator().manual_seed(k)
    w = _weight(g, n, k, group, dtype, True, cuda_device)
    count = n * (k // group)
    scales = torch.full((count + 64,), float("nan"), dtype=DT[dtype], device=cuda_device)
    zeros = torch.full((count + 64,), 255, dtype=torch.uint8, device=cuda_device)
    scales[:count], zeros[:count] = w.scales.flatten(), w.zeros.flatten()
    inside = ab.Int4Weight(w.qweight, scales[:count].view(n, -1), zeros[:count].view(n, -1))
    x = torch.randn(rows, k, generator=g).to(DT[dtype]).to(cuda_device)
    nw = torch.ones(k, dtype=DT[dtype], device=cuda_device)
    for norm in (None, nw):
        y = ab.decode_linear_int4(x, inside, norm_weight=norm)
        assert torch.equal(y, ab.decode_linear_int4(x, w, norm_weight=norm)) and bool(y.isfinite().all())


@pytest.mark.parametrize("rows,k,n,group,swiglu", [(32, 256, 60000, 128, False), (16, 512, 120000, 128, False),
                                                   (1, 256, 100000, 32, True), (25, 128, 50001, 64, False),
                                                   (32, 256, 30001, 64, True)])
def test_rounds_with_fewer_jobs_than_the_ring_has_stages(cuda_device, rows, k, n, group, swiglu):
    """Short K, many output features: a warp has one or two jobs in each of several rounds."""
    _case(cuda_device, rows, k, n, group, zeros=True, swiglu=swiglu, seed=rows)
