"""The paged attention on values where 16-bit operands could show: far weights,
infinities."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _native as nat

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("groups", [2, 16])
@pytest.mark.parametrize("below", [16, 26, 32])
def test_many_slots_far_below_one(cuda_device, dtype, groups, below):
    """One slot ``below`` (in powers of two) above 40000 equal ones.  The others' share
    of the weight is theirs in the result as in the log-sum-exp: weights are held to
    2^-16 (bf16, two parts of 8 bits) of themselves or 2^-39 (fp16) of the largest, at
    2^-32 that is 2^-7 of themselves; the result is rounded to 2^-8 or 2^-11 of itself."""
    n, D, size = 40000, 64, 16
    q = torch.zeros(1, groups, 1, D, dtype=DT[dtype], device=cuda_device)
    q[..., 0] = 1
    k = torch.zeros(1, 1, n, D, dtype=DT[dtype], device=cuda_device)
    v = torch.full((1, 1, n, D), 96.0, dtype=DT[dtype], device=cuda_device)
    k[:, :, 777, 0], v[:, :, 777] = below, 0.0
    pages = [t.view(n // size, size, 1, D).transpose(1, 2) for t in (k, v)]
    table = torch.arange(n // size, dtype=torch.int32, device=cuda_device).view(1, -1)
    out, lse = ab.paged_gqa_decode_attention(q, *pages, table, sm_scale=float(np.log(2.0)), num_key_value_groups=groups,
                                             return_lse=True)
    tail = (n - 1) * 2.0 ** -below
    want = 96.0 * tail / (1 + tail)
    rel = {"bf16": 2.0 ** -8 + 2.0 ** -14, "fp16": 2.0 ** -11 + 2.0 ** (below - 38) + 2.0 ** -14}[dtype]
    assert (out.double() / want - 1).abs().max().item() <= rel
    assert (lse.double() - (below + np.log2(1 + tail))).abs().max().item() <= 1e-4
    assert nat.device_error_flags() == 0


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("groups", [2, 16])
@pytest.mark.parametrize("n", [1, 2, 40, 3000])
def test_infinite_values_in_live_slots(cuda_device, dtype, groups, n):
    """An infinity of V comes out as itself, opposite ones and NaN as NaN, and every
    other element is what it is without them.  Equal scores among the others: weights
    of one and of exact powers of two."""
    D, size, dt = 64, 16, DT.get(dtype, torch.float32)
    g = torch.Generator().manual_seed(n)
    for equal in (False, True):
        k = torch.zeros(n, D) if equal else torch.randn(n, D, generator=g)
        v = torch.randn(n, D, generator=g)
        clean = v.clone()
        inf = float("inf")
        for d, (t, value) in enumerate([(0, inf), (n // 2, -inf), (n - 1, inf), (n // 3, float("nan"))]):
            v[t, d] = value
        v[0, 4], v[n - 1, 4] = inf, -inf if n > 1 else inf
        v[0, 5] = v[n - 1, 5] = -inf
        q = torch.randn(1, groups, 1, D, generator=g).to(dt).to(cuda_device)
        rows = -(-n // size) * size
        table = torch.arange(rows // size, dtype=torch.int32, device=cuda_device).view(1, -1)

        def run(v):
            pool = torch.full((2, rows, D), float("nan"))
            pool[0, :n], pool[1, :n] = k, v
            kp, vp = (t.to(dt).to(cuda_device).view(-1, 1, size, D) for t in pool)
            return ab.paged_gqa_decode_attention(q, kp, vp, table, sm_scale=0.125, num_key_value_groups=groups, kv_lens=[n])

        got, base = run(v)[0, :, 0], run(clean)[0, :, 0]
        assert (got[:, [0, 2]] == inf).all() and (got[:, [1, 5]] == -inf).all() and got[:, 3].isnan().all()
        assert (got[:, 4].isnan() if n > 1 else got[:, 4] == inf).all()
        assert torch.equal(got[:, 6:], base[:, 6:]) and base.isfinite().all()
    assert nat.device_error_flags() == 0
