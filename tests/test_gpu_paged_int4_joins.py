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


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group,groups", [(128, 128, 2), (128, 64, 2), (64, 64, 2), (128, 128, 8), (128, 64, 8)])
def test_long_sums_do_not_drift(cuda_device, dtype, dim, group, groups):
    """A large batch over long caches of values around 0: a warp adds up hundreds of tiles, and
    what scales times codes come to cancels with the least values.

    Tolerance: products are added up in chains of 16 steps, each of which may cut off 2^-23 of the
    largest number in it, at most what all codes at 15 come to: 16 x 2^-23 x 15 scale, 1.3e-5 for the
    values here; the mean over all outputs within that, each output within twice that (the
    chains' sums are rounded, 2^-24 each) and half a unit of its own rounding."""
    g = torch.Generator(device=cuda_device).manual_seed(dim + group + groups)
    B, hkv, n, size, dt = 128, 4, 65536, 64, DT[dtype]
    hq = hkv * groups
    rows = [torch.randn(n // size, hkv, size, dim, generator=g, device=cuda_device).to(dt) for _ in range(2)]
    kp, vp = (ab.quantize_kv_int4(r, group) for r in rows)
    table = torch.randperm(n // size, generator=g, device=cuda_device).int().expand(B, -1)  # all requests read the same pages
    q = torch.randn(B, hq, 1, dim, generator=g, device=cuda_device).to(dt)
    out = ab.paged_gqa_decode_attention_int4(q, kp, vp, table, sm_scale=dim ** -0.5, num_key_value_groups=groups)
    total, count = 0.0, 0
    bound = 16 * 2.0 ** -23 * 15 * float(vp.scales[..., 0].float().max())
    half = torch.finfo(dt).eps / 2
    for h in range(hkv):
        k, v = (p.dequantize()[:, h].flatten(0, 1).double() for p in (kp, vp))
        for b in range(0, B, 32):
            mine = q[b:b + 32, h * groups:(h + 1) * groups, 0].double()
            ref = torch.softmax(mine @ k.t() * dim ** -0.5, -1) @ v
            off = out[b:b + 32, h * groups:(h + 1) * groups, 0].double() - ref
            assert (off.abs() <= half * ref.abs() + 2 * bound).all()
            total, count = total + float(off.sum()), count + off.numel()
    assert abs(total / count) <= bound


def _late_case(device, dtype, dim, group, groups, edit):
    """Many pairs of some 70 tiles, about 28 a warp, whose first and later halves `edit` sets apart; against
    64 bits on the device, with the tolerances of test_gpu_paged_far_scores.py."""
    g = torch.Generator(device=device).manual_seed(group + groups)
    B, hkv, n, size, dt = 90, 8, 2400, 16, DT[dtype]
    per = n // size
    rows = [torch.randn(B * per, hkv, size, dim, generator=g, device=device) for _ in range(2)]
    q = torch.randn(B, hkv * groups, 1, dim, generator=g, device=device)
    edit(q, *(r.view(B, 2, per // 2, hkv, size, dim) for r in rows))  # [request, half of its pages]
    kp, vp = (ab.quantize_kv_int4(r.to(dt), group) for r in rows)
    q, table = q.to(dt), torch.arange(B * per, dtype=torch.int32, device=device).view(B, per)
    lens = [n - 7 * b for b in range(B)]
    out, lse = ab.paged_gqa_decode_attention_int4(q, kp, vp, table, sm_scale=dim ** -0.5, num_key_value_groups=groups,
                                                  kv_lens=lens, return_lse=True)
    scale, log2 = dim ** -0.5, 0.6931471805599453
    k_all, v_all = (p.dequantize().view(B, per, hkv, size, dim).transpose(1, 2).flatten(2, 3) for p in (kp, vp))
    for b, length in enumerate(lens):
        k, v = (x[b, :, :length].double() for x in (k_all, v_all))
        mine = q[b, :, 0].double().view(hkv, groups, dim)
        s = mine @ k.transpose(1, 2) * scale
        # scale code + |least| is at most three times a row's largest |k|
        e = 40 * 2.0 ** -24 * 3 * (mine.abs().sum(-1) * k.abs().amax((1, 2))[:, None]).flatten() * scale / log2
        ref = (torch.softmax(s, -1) @ v).view(-1, dim)
        ref_lse = torch.logsumexp(s, -1).flatten() / log2
        top = v.abs().max()
        bound = torch.finfo(dt).eps / 2 * ref.abs() + 2e-4 * top + 2 * torch.expm1(e * log2)[:, None] * top
        assert ((out[b, :, 0].double() - ref).abs() <= bound).all()
        assert ((lse[b].double() - ref_lse).abs() <= e + 1e-4 + 2.0 ** -22 * ref_lse.abs()).all()


LATE = pytest.mark.parametrize("dtype,dim,group,groups", [("bf16", 128, 128, 2), ("bf16", 128, 64, 8), ("fp16", 64, 64, 6)])


@LATE
@pytest.mark.parametrize("far", [-100.0, -6.0, 6.0])
def test_references_that_move_late(cuda_device, dtype, dim, group, groups, far):
    """The first half of each cache scores far below or above the second: sums that are held by then are
    scaled with the rest."""

    def edit(q, k, v):
        k[:, 0, :, 0] += 3.0
        q[:, :groups] = 0.1 * q[:, :groups] + far / (dim ** -0.5 * 3.0 * dim)

    _late_case(cuda_device, dtype, dim, group, groups, edit)


@LATE
@pytest.mark.parametrize("early,late", [(2.0 ** -7, 1.0), (2.0 ** -12, 1.0), (1.0, 2.0 ** -7)])
def test_scales_that_grow_late(cuda_device, dtype, dim, group, groups, early, late):
    """Values of another size from the middle of each cache on."""

    def edit(q, k, v):
        v[:, 0] *= early
        v[:, 1] *= late

    _late_case(cuda_device, dtype, dim, group, groups, edit)


@pytest.mark.parametrize("to", [1e-35, 1e-20, 1e20, 1e34, 4e36])
@pytest.mark.parametrize("group", [64, 128])
@pytest.mark.parametrize("groups", [2, 8])
def test_values_over_the_range_of_bf16(cuda_device, to, group, groups):
    """Values of any size that their sums leave room for, against the same in 64 bits."""
    g = torch.Generator().manual_seed(groups)
    B, hkv, per, dim = 3, 2, 8, 128
    rows = [torch.randn(B * per, hkv, 16, dim, generator=g).to(DT["bf16"]) for _ in range(2)]
    rows[1] = (rows[1].double() * to).to(DT["bf16"])
    kp, vp = (ab.Int4Pages(*(t.to(cuda_device) for t in ab.quantize_kv_int4(r, group))) for r in rows)
    table = torch.randperm(B * per, generator=g).view(B, per).int().to(cuda_device)
    q = torch.randn(B, hkv * groups, 1, dim, generator=g).to(DT["bf16"]).to(cuda_device)
    lens = [1, 33, 128]
    out = ab.paged_gqa_decode_attention_int4(q, kp, vp, table, sm_scale=dim ** -0.5, num_key_value_groups=groups, kv_lens=lens)
    for b, n in enumerate(lens):
        k, v = (p.dequantize()[table[b].long()].transpose(0, 1).flatten(1, 2)[:, :n].double() for p in (kp, vp))
        mine = q[b, :, 0].double().view(hkv, groups, dim)
        ref = (torch.softmax(mine @ k.transpose(1, 2) * dim ** -0.5, -1) @ v).view(-1, dim)
        # 2e-4 of values around 1, as at the top; below fp32's normal numbers sums keep fewer bits (a scale is 0.3 to)
        assert ((out[b, :, 0].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2e-4 * to + 2.0 ** -133).all()
