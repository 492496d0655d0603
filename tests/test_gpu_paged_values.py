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
