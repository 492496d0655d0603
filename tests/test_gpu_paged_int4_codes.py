"""Codes and pairs of the 4-bit append, to the bit: groups whose scale lies at a border."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aicas_b200 as ab
from oracle import paged_int4 as o4
from tests.test_paged_int4_scales_cpu import DT, border_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64), (128, 128)])
@pytest.mark.parametrize("prompt", [False, True])
def test_scales_at_the_border(cuda_device, dtype, dim, group, prompt):
    """The append writes what quantize_kv_int4 gives on the CPU and on the GPU."""
    rows = border_rows(dtype, dim, group)
    want = ab.quantize_kv_int4(rows, group)
    on_gpu = ab.quantize_kv_int4(rows.to(cuda_device), group)
    assert all(torch.equal(a, b.cpu()) for a, b in zip(want, on_gpu))
    n = len(rows)
    S = max(n, 700) if prompt else 1  # one prompt, or a token a request
    if prompt:
        rows = torch.cat([rows] * -(-S // n))[:S]
        new = rows.view(1, 1, S, dim).to(cuda_device)
    else:
        new = rows.view(n, 1, 1, dim).to(cuda_device)
    B, per = new.shape[0], -(-S // 16)
    kp, vp = (ab.int4_pages(B * per, 1, 16, dim, group, dtype=DT[dtype], device=cuda_device) for _ in range(2))
    table = torch.arange(B * per, dtype=torch.int32, device=cuda_device).view(B, per)
    cos, sin = torch.ones(1, S, dim, device=cuda_device), torch.zeros(1, S, dim, device=cuda_device)
    ab.paged_rope_kv_append_int4(new, new, new, cos, sin, kp, vp, table, torch.zeros(B, dtype=torch.int32, device=cuda_device))
    for pool in (kp, vp):
        for part, w in zip(pool, want):
            got = part.view(B, per, *part.shape[1:]).transpose(1, 2).flatten(2, 3)[:, 0, :S].flatten(0, 1).cpu()
            assert torch.equal(got[:n], w)
    scale, least, _ = o4.levels(rows[:n].float().numpy(), group, dtype)
    np.testing.assert_array_equal(want.scales.float().numpy(), np.stack([scale, least], -1))
