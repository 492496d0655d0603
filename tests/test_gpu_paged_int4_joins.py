"""Joins of 4-bit decode attention: pairs that several teams share, for teams of every
size that a launch may choose.

Tolerances are those of test_gpu_paged_int4.py; repeated calls give the same bits, since
partial results are joined in the order of their ranges, whichever team arrives last."""
from __future__ import annotations

import pytest
import torch

import aicas_b200 as ab
from tests.test_gpu_paged_int4 import DT, _attend_case, _pool, _table

pytestmark = pytest.mark.gpu


# Pairs (request, KV head): many make teams of one warp, which join by themselves; few make larger ones.
@pytest.mark.parametrize("batch,hkv,lens", [(90, 8, (1, 700)), (80, 8, (300, 301)), (40, 8, (1, 900)), (12, 8, (1, 1500)),
                                            (3, 8, (2000, 6000))])
@pytest.mark.parametrize("dtype,dim,group,groups", [("bf16", 128, 128, 2), ("fp16", 64, 64, 6)])
def test_joins_of_every_team(cuda_device, batch, hkv, lens, dtype, dim, group, groups):
    g = torch.Generator().manual_seed(batch)
    n = torch.randint(*lens, (batch,), generator=g).tolist()
    _attend_case(cuda_device, dtype, dim, group, hkv * groups, hkv, n, 16, seed=batch)


@pytest.mark.parametrize("batch,hkv,hi", [(90, 8, 700), (40, 8, 900), (3, 8, 6000)])
def test_joins_repeat_to_the_bit(cuda_device, batch, hkv, hi):
    g = torch.Generator().manual_seed(hi)
    per = -(-hi // 16)
    kp, vp = (_pool(g, batch * per, hkv, 16, 128, 64, "bf16", "hnd", cuda_device) for _ in range(2))
    table = _table(g, batch, per, batch * per, cuda_device)
    q = torch.randn(batch, 2 * hkv, 1, 128, generator=g).to(DT["bf16"]).to(cuda_device)
    lens = torch.randint(1, hi + 1, (batch,), generator=g).int().to(cuda_device)
    run = lambda: ab.paged_gqa_decode_attention_int4(q, kp, vp, table, sm_scale=0.09, num_key_value_groups=2,  # noqa: E731
                                                     kv_lens=lens, return_lse=True)
    first = run()
    again = [run() for _ in range(200)]
    assert all(torch.equal(a, b) for other in again for a, b in zip(first, other))
