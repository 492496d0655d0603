"""Codes and pairs of the 4-bit append, to the bit: groups whose scale lies at a border, and
keys with tables of the tensors' own type."""
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


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64), (128, 128)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("batch,seq", [(7, 1), (3, 61), (2, 701)])
def test_keys_with_tables_of_their_own_type(cuda_device, dtype, dim, group, norm, batch, seq):
    """Every operation of such keys is rounded, as a 16-bit cache holds them: the codes and pairs
    are those of the rows that paged_rope_kv_append writes."""
    g = torch.Generator().manual_seed(dim + seq)
    dt, hq, hkv, per = DT[dtype], 6, 3, -(-seq // 16)
    q, k, v = (torch.randn(batch, seq, h, dim, generator=g).to(dt).to(cuda_device).transpose(1, 2) for h in (hq, hkv, hkv))
    ang = 3 * torch.randn(batch, seq, dim, generator=g)
    cos, sin = ang.cos().to(dt).to(cuda_device), ang.sin().to(dt).to(cuda_device)
    w = (1 + 0.3 * torch.randn(dim, generator=g)).to(dt).to(cuda_device) if norm else None
    table = torch.randperm(batch * per, generator=g).view(batch, per).int().to(cuda_device)
    pos = torch.zeros(batch, dtype=torch.int32, device=cuda_device)
    wide = [torch.zeros(batch * per, hkv, 16, dim, dtype=dt, device=cuda_device) for _ in range(2)]
    small = [ab.int4_pages(batch * per, hkv, 16, dim, group, dtype=dt, device=cuda_device) for _ in range(2)]
    ab.paged_rope_kv_append(q, k, v, cos, sin, *wide, table, pos, q_norm_weight=w, k_norm_weight=w)
    ab.paged_rope_kv_append_int4(q, k, v, cos, sin, *small, table, pos, q_norm_weight=w, k_norm_weight=w)
    for pages, pool in zip(wide, small):
        rows = pages[table.long()].transpose(1, 2).flatten(2, 3)[:, :, :seq]
        for part, want in zip(pool, ab.quantize_kv_int4(rows, group)):
            assert torch.equal(part[table.long()].transpose(1, 2).flatten(2, 3)[:, :, :seq], want)
