"""The paged cache's append and decode attention on the GPU against their
float64 restatement, at the sizes and masks where they can go wrong.

Tolerances.  A result is rounded once, so it may be off by half a unit in the
last place of its type, 2^-8 (bf16), 2^-11 (fp16) or 2^-24 (fp32) of its value,
on top of what fp32 arithmetic may be off: for the rotation a few additions of
terms below 16 (8 x 2^-24 x 16 < 1e-5); for the attention the score's sum of D
products (standard normal q and k: below 1e-4) and the weights' sums, 1e-3 of
values of order one in 16 bits (probabilities rounded to two 16-bit parts), 2e-5
in fp32."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _native as nat
from oracle import paged as op
from oracle import rope as orope

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _np(t: torch.Tensor) -> np.ndarray:
    return t.detach().float().cpu().numpy()


def _near(got, ref, dtype, atol):
    got = _np(got).astype(np.float64)
    assert got.shape == ref.shape
    assert np.array_equal(np.isfinite(got), np.isfinite(ref))
    fin = np.isfinite(ref)
    off = np.abs(got[fin] - ref[fin]) - (HALF_ULP[dtype] * np.abs(ref[fin]) + atol)
    assert off.size == 0 or off.max() <= 0, f"{off.max():.3e} over the bound"


def _pool(g, pages, hkv, size, dim, dtype, layout, device):
    """k and v pools [P, Hkv, size, D]; 'nhd': stored [P, size, Hkv, D]; 'both': k and
    v interleaved in one tensor [P, 2, Hkv, size, D]."""
    if layout == "nhd":
        return tuple(torch.randn(pages, size, hkv, dim, generator=g).to(DT[dtype]).to(device).transpose(1, 2)
                     for _ in range(2))
    if layout == "both":
        t = torch.randn(pages, 2, hkv, size, dim, generator=g).to(DT[dtype]).to(device)
        return t[:, 0], t[:, 1]
    return tuple(torch.randn(pages, hkv, size, dim, generator=g).to(DT[dtype]).to(device) for _ in range(2))


def _table(g, batch, per, pages, device):
    return torch.randperm(pages, generator=g)[: batch * per].view(batch, per).to(torch.int32).to(device)


# ------------------------------------------------------------------ append


def _append_case(device, dtype, dim, hq, hkv, batch, seq, size, per, layout="hnd", tables="fp32", norm=False, seed=0,
                 positions=None, counts=None, one_table=False):
    g = torch.Generator().manual_seed(seed)
    pages = batch * per + 2
    kp, vp = _pool(g, pages, hkv, size, dim, dtype, layout, device)
    table = _table(g, batch, per, pages, device)
    q, k, v = (torch.randn(batch, seq, h, dim, generator=g).to(DT[dtype]).to(device).transpose(1, 2)
               for h in (hq, hkv, hkv))
    ang = torch.randn(1 if one_table else batch, seq, dim, generator=g) * 3
    cos, sin = ang.cos().to(DT[tables]).to(device), ang.sin().to(DT[tables]).to(device)
    w = [(1 + 0.3 * torch.randn(dim, generator=g)).to(DT[dtype]).to(device) for _ in range(2)] if norm else [None] * 2
    if positions is None:
        positions = torch.randint(0, per * size - seq + 1, (batch,), generator=g).tolist()
    pos = torch.tensor(positions, dtype=torch.int32, device=device)
    lens = torch.full((batch,), -7, dtype=torch.int32, device=device)
    k0, v0 = _np(kp), _np(vp)
    new = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=device)
    out = ab.paged_rope_kv_append(q, k, v, cos, sin, kp, vp, table, pos, num_new=new, kv_lens_out=lens,
                                  q_norm_weight=w[0], k_norm_weight=w[1])
    cnt = [seq] * batch if counts is None else counts
    c, s = (np.broadcast_to(_np(t), (batch, seq, dim)) for t in (cos, sin))
    cap = per * size
    assert lens.tolist() == [min(max(p, 0) + max(0, min(n, seq)), cap) for p, n in zip(positions, cnt)]
    # values are copied; unwritten rows keep their bits
    np.testing.assert_array_equal(_np(vp), op.append(v0, _np(v), table.cpu().numpy(), positions, cnt))
    if tables == dtype and dtype != "fp32":
        rot = lambda t, x: orope.apply_rope(_np(t) if x is None else orope.rms_norm_heads(_np(t), _np(x), 1e-6, dtype),  # noqa: E731
                                            c, s, dtype)
        ref_q, ref_k = rot(q, w[0]), rot(k, w[1])
        ref_kp = op.append(k0, ref_k, table.cpu().numpy(), positions, cnt)
        if not norm:
            np.testing.assert_array_equal(_np(out), ref_q)
            np.testing.assert_array_equal(_np(kp), ref_kp)
        else:
            # the sum of squares' order and rsqrt may move a rounding by one unit
            for got, ref in ((_np(out), ref_q), (_np(kp), ref_kp)):
                assert (got == ref).mean() > 0.98
                assert np.abs(got - ref).max() <= 4 * HALF_ULP[dtype] * max(1.0, np.abs(ref).max())
    else:
        ref_q = op.rotate(_np(q), c, s, None if w[0] is None else _np(w[0]))
        ref_k = op.rotate(_np(k), c, s, None if w[1] is None else _np(w[1]))
        _near(out, ref_q, dtype, 1e-5)
        ref_kp = op.append(k0.astype(np.float64), ref_k, table.cpu().numpy(), positions, cnt)
        untouched = op.append(np.zeros_like(k0), np.ones_like(ref_k), table.cpu().numpy(), positions, cnt) == 0
        assert np.array_equal(_np(kp)[untouched], k0[untouched])
        _near(kp, ref_kp, dtype, 1e-5)
    assert nat.device_error_flags() == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("norm", [False, True])
def test_append_types_and_head_dims(cuda_device, dtype, dim, norm):
    _append_case(cuda_device, dtype, dim, 6, 2, 3, 5, 16, 3, norm=norm, seed=dim)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("norm", [False, True])
def test_append_rounds_as_hf_with_16_bit_tables(cuda_device, dtype, norm):
    _append_case(cuda_device, dtype, 128, 16, 8, 2, 9, 24, 2, tables=dtype, norm=norm, seed=3)


@pytest.mark.parametrize("layout", ["hnd", "nhd", "both"])
@pytest.mark.parametrize("size", [8, 16, 24, 128])
@pytest.mark.parametrize("heads", [(1, 1), (40, 1), (7, 7), (16, 8)])
def test_append_layouts(cuda_device, layout, size, heads):
    per = -(-70 // size)
    _append_case(cuda_device, "bf16", 64, *heads, 2, 67, size, per, layout=layout, one_table=True, seed=size)


def test_append_single_tokens_at_page_edges(cuda_device):
    _append_case(cuda_device, "bf16", 128, 16, 8, 6, 1, 16, 4, positions=[0, 15, 16, 31, 62, 63], norm=True)


def test_append_drops_what_has_no_place(cuda_device):
    """Padding, slots past the table's end and negative slots."""
    _append_case(cuda_device, "fp16", 64, 4, 2, 7, 6, 8, 2, positions=[0, 12, 16, 40, -3, -9, 2147483647],
                 counts=[0, 6, 6, 6, 6, 6, 6])
    _append_case(cuda_device, "fp16", 64, 4, 2, 4, 6, 8, 2, positions=[1, 2, 3, 4], counts=[-2, 99, 1, 5])


def test_append_skips_pages_outside_the_pool(cuda_device):
    g = torch.Generator().manual_seed(1)
    kp, vp = _pool(g, 4, 2, 8, 32, "bf16", "hnd", cuda_device)
    k0, v0 = kp.clone(), vp.clone()
    table = torch.tensor([[-1, 4], [1 << 30, -(1 << 31)]], dtype=torch.int32, device=cuda_device)
    q, k = torch.randn(2, 4, 16, 32, dtype=torch.bfloat16, device=cuda_device), torch.randn(
        2, 2, 16, 32, dtype=torch.bfloat16, device=cuda_device)
    cos = torch.ones(2, 16, 32, device=cuda_device)
    out = ab.paged_rope_kv_append(q, k, k, cos, cos * 0, kp, vp, table, [0, 0])
    assert torch.equal(out, q) and torch.equal(kp, k0) and torch.equal(vp, v0)


def test_append_many_tokens_equals_one_at_a_time(cuda_device):
    """A chunk of a prompt and single tokens leave the same pages, with q rotated in place."""
    g = torch.Generator().manual_seed(5)
    B, S, Hq, Hkv, D, size = 3, 37, 8, 4, 128, 16
    q, k, v = (torch.randn(B, h, S, D, generator=g).to(torch.bfloat16).to(cuda_device) for h in (Hq, Hkv, Hkv))
    ang = torch.randn(B, S, D, generator=g).to(cuda_device)
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(torch.bfloat16).to(cuda_device)
    table = _table(g, B, 4, 13, cuda_device)
    pools = [torch.zeros(13, Hkv, size, D, dtype=torch.bfloat16, device=cuda_device) for _ in range(4)]
    pos = torch.tensor([3, 0, 27], dtype=torch.int32, device=cuda_device)
    kw = dict(q_norm_weight=w, k_norm_weight=w)
    whole = ab.paged_rope_kv_append(q, k, v, ang.cos(), ang.sin(), pools[0], pools[1], table, pos, **kw)
    for s in range(S):
        one = slice(s, s + 1)
        qs = q[:, :, one].clone()
        got = ab.paged_rope_kv_append(qs, k[:, :, one], v[:, :, one], ang.cos()[:, one], ang.sin()[:, one], pools[2],
                                      pools[3], table, pos + s, q_out=qs, **kw)
        assert got is qs and torch.equal(qs, whole[:, :, one])
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


def test_append_and_read_past_two_to_the_31_elements(cuda_device):
    """Pages whose elements start past 2^31 (and bytes past 2^32)."""
    Hkv, size, D = 8, 16, 128
    pages = (1 << 31) // (Hkv * size * D) + 40
    kp = torch.empty(pages, Hkv, size, D, dtype=torch.bfloat16, device=cuda_device)
    vp = torch.empty_like(kp)
    g = torch.Generator().manual_seed(2)
    table = torch.tensor([[pages - 1, 0, pages - 2], [pages - 30, pages - 31, 1]], dtype=torch.int32,
                         device=cuda_device)
    k, v = (torch.randn(2, Hkv, 41, D, generator=g).to(torch.bfloat16).to(cuda_device) for _ in range(2))
    q = torch.randn(2, 16, 41, D, generator=g).to(torch.bfloat16).to(cuda_device)
    cos = torch.ones(1, 41, D, device=cuda_device)
    ab.paged_rope_kv_append(q, k, v, cos, cos * 0, kp, vp, table, [0, 0])
    assert torch.equal(kp[pages - 1], k[0, :, :16]) and torch.equal(vp[pages - 31], v[1, :, 16:32])
    out = ab.paged_gqa_decode_attention(q[:, :, :1], kp, vp, table, sm_scale=0.1, num_key_value_groups=2,
                                        kv_lens=[41, 40])
    ref = ab.gqa_decode_attention(q[:, :, :1], k, v, sm_scale=0.1, num_key_value_groups=2, kv_lens=[41, 40])
    assert (out.float() - ref.float()).abs().max().item() <= 2e-2


# ------------------------------------------------------------------ attention


def _decode_case(device, dtype, dim, hq, hkv, size, lens, starts=None, layout="hnd", seed=0, spoil=True, per=None,
                 scale=None, atol=None):
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    per = per or max(1, -(-max(lens) // size))
    pages = B * per + 1
    kp, vp = _pool(g, pages, hkv, size, dim, dtype, layout, device)
    table = _table(g, B, per, pages, device)
    q = torch.randn(B, 1, hq, dim, generator=g).to(DT[dtype]).to(device).transpose(1, 2)
    begin = starts if starts is not None else [0] * B
    scale = dim ** -0.5 if scale is None else scale
    ref, ref_lse = op.decode(_np(q), _np(kp), _np(vp), table.cpu().numpy(), lens, begin, scale, hq // hkv)
    if spoil:
        # slots out of range hold NaN and infinities, table entries past the end anything
        bad = [float("nan"), float("inf"), float("-inf")]
        for b in range(B):
            n = min(max(lens[b], 0), per * size)
            for t in [*range(min(max(begin[b], 0), n)), *range(n, per * size)]:
                page = int(table[b, t // size])
                kp[page, :, t % size], vp[page, :, t % size] = bad[t % 3], bad[(t + 1) % 3]
            table[b, -(-n // size):] = [-5, 1 << 30][b % 2]
    out, lse = ab.paged_gqa_decode_attention(
        q, kp, vp, table, sm_scale=scale, num_key_value_groups=hq // hkv,
        kv_lens=torch.tensor(lens, dtype=torch.int32, device=device),
        kv_starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device=device), return_lse=True)
    assert out.shape == q.shape and out.dtype == q.dtype
    atol = atol if atol is not None else 2e-5 if dtype == "fp32" else 1e-3
    _near(out, ref, dtype, atol)
    _near(lse, ref_lse, "fp32", 1e-4)
    assert nat.device_error_flags() == 0
    return q, kp, vp, table, out


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("groups", [1, 2, 5, 8, 9, 16, 20, 33])
def test_decode_types_dims_and_groups(cuda_device, dtype, dim, groups):
    _decode_case(cuda_device, dtype, dim, 2 * groups, 2, 16, [77, 0, 1, 260], seed=groups)


@pytest.mark.parametrize("layout", ["hnd", "nhd", "both"])
@pytest.mark.parametrize("size", [8, 16, 24, 32, 40, 64, 256])
def test_decode_pages_and_lengths(cuda_device, layout, size):
    lens = [0, 1, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 500]
    _decode_case(cuda_device, "bf16", 64, 4, 2, size, lens, layout=layout, seed=size)


@pytest.mark.parametrize("dtype,dim", [("bf16", 16), ("fp16", 32), ("bf16", 128), ("fp32", 16), ("fp32", 32), ("fp32", 64),
                                       ("fp32", 128)])
@pytest.mark.parametrize("size", [8, 24, 48])
def test_decode_page_sizes_at_every_row_width(cuda_device, dtype, dim, size):
    _decode_case(cuda_device, dtype, dim, 4, 2, size, [1, 8, 9, 23, 24, 25, 100, 256, 333], seed=dim)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("size", [8, 16, 24])
def test_decode_skips_the_first_slots(cuda_device, dtype, size):
    lens = [300, 300, 300, 300, 300, 17, 16, 5, 0, 300]
    starts = [0, 1, 15, 16, 299, 16, 16, 9, 3, -4]
    _decode_case(cuda_device, dtype, 128, 8, 4, size, lens, starts)


def test_decode_lengths_are_clamped_to_the_table(cuda_device):
    _decode_case(cuda_device, "bf16", 64, 4, 2, 16, [1000, -5, 48], [2000, -1, 47], per=3, spoil=True)


@pytest.mark.parametrize("dtype,size,lens", [
    ("bf16", 16, [20011]), ("fp16", 64, [30000, 3]), ("bf16", 8, [4097, 1, 9000]), ("fp32", 16, [12345])])
def test_decode_long_caches(cuda_device, dtype, size, lens):
    """One long cache spread over every SM and joined again."""
    _decode_case(cuda_device, dtype, 128, 16, 8, size, lens, spoil=False)


def test_decode_many_short_requests(cuda_device):
    rng = np.random.RandomState(0)
    _decode_case(cuda_device, "bf16", 32, 4, 2, 8, rng.randint(0, 60, 700).tolist(), spoil=False)


@pytest.mark.parametrize("lens", [
    [1] * 2500,                                    # one tile a request: most warps have nothing to copy
    [20, 1, 0, 33] * 500 + [3000],                 # and a long cache after them
    [9000] + [0] * 300 + [17] * 1500 + [6000, 2],
    [16] * 40 + [30000] + [16] * 40 + [1] * 2000 + [15000],
])
@pytest.mark.parametrize("dim,dtype", [(16, "fp16"), (64, "bf16"), (32, "fp32")])
def test_decode_ranges_over_mixed_requests(cuda_device, lens, dim, dtype):
    """More requests than CTAs, short and long ones mixed: ranges that hold many, or a part of one."""
    g = torch.Generator().manual_seed(len(lens))
    B, hkv, size = len(lens), 8, 16
    pages = 400
    kp, vp = _pool(g, pages, hkv, size, dim, dtype, "hnd", cuda_device)
    per = -(-max(lens) // size)
    table = torch.randint(0, pages, (B, per), generator=g, dtype=torch.int32).to(cuda_device)
    q = torch.randn(B, 16, 1, dim, generator=g).to(DT[dtype]).to(cuda_device)
    kw = dict(sm_scale=dim ** -0.5, num_key_value_groups=2, kv_lens=torch.tensor(lens, dtype=torch.int32))
    out, lse = ab.paged_gqa_decode_attention(q, kp, vp, table, return_lse=True, **kw)
    for _ in range(3):
        again = ab.paged_gqa_decode_attention(q, kp, vp, table, **kw)
        assert torch.equal(again, out)
    assert nat.device_error_flags() == 0
    pick = sorted(set([0, 1, 2, 3, 40, 41, 300, 301, B // 2, B - 3, B - 2, B - 1]))
    ref, ref_lse = op.decode(_np(q[pick]), _np(kp), _np(vp), table[pick].cpu().numpy(), [lens[b] for b in pick],
                             [0] * len(pick), dim ** -0.5, 2)
    _near(out[pick], ref, dtype, 2e-5 if dtype == "fp32" else 1e-3)
    _near(lse[pick], ref_lse, "fp32", 1e-4)
    # every request, cut differently: in batches of 250
    for b0 in range(0, B, 250):
        part = ab.paged_gqa_decode_attention(q[b0:b0 + 250], kp, vp, table[b0:b0 + 250],
                                             **(kw | {"kv_lens": torch.tensor(lens[b0:b0 + 250], dtype=torch.int32)}))
        assert (part.float() - out[b0:b0 + 250].float()).abs().max().item() <= 2e-2


def test_decode_large_scores(cuda_device):
    """Scores of several hundred: one slot takes all the weight, the others vanish."""
    _decode_case(cuda_device, "bf16", 128, 16, 8, 16, [700, 513], scale=4.0, atol=2e-2)


def test_decode_infinite_and_nan_slots_in_range(cuda_device):
    """A slot in range whose score is -inf has no weight; NaN reaches the output."""
    B, Hkv, D, size = 3, 2, 64, 16
    kp = torch.ones(B, Hkv, size, D, dtype=torch.bfloat16, device=cuda_device)
    vp = torch.randn(B, Hkv, size, D, device=cuda_device).to(torch.bfloat16)
    table = torch.arange(B, dtype=torch.int32, device=cuda_device).view(B, 1)
    q = torch.ones(B, 4, 1, D, dtype=torch.bfloat16, device=cuda_device)
    kp[0, :, 3] = float("-inf")
    kp[1, :, 5] = float("nan")
    vp[2, 0, 2] = float("nan")
    out = ab.paged_gqa_decode_attention(q, kp, vp, table, sm_scale=0.125, num_key_value_groups=2)
    keep = [t for t in range(size) if t != 3]
    ref = vp[0, :, keep].float().mean(1).repeat_interleave(2, 0)
    assert (out[0, :, 0].float() - ref).abs().max().item() <= 4e-3
    assert torch.isnan(out[1]).all()
    assert torch.isnan(out[2, :2]).all() and torch.isfinite(out[2, 2:]).all()


def test_decode_page_numbers_outside_the_pool_read_as_zeros(cuda_device):
    kp = torch.randn(3, 2, 8, 64, dtype=torch.bfloat16, device=cuda_device)
    vp = torch.randn_like(kp)
    q = torch.randn(1, 4, 1, 64, dtype=torch.bfloat16, device=cuda_device)
    table = torch.tensor([[1, -1, 3, 2]], dtype=torch.int32, device=cuda_device)
    out = ab.paged_gqa_decode_attention(q, kp, vp, table, sm_scale=0.1, num_key_value_groups=2, kv_lens=[30])
    z = torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16, device=cuda_device)
    k, v = (torch.cat([p[1:2], z, p[2:3]], 2)[:, :, :30].contiguous() for p in (kp, vp))
    ref = ab.gqa_decode_attention(q, k, v, sm_scale=0.1, num_key_value_groups=2)
    assert (out.float() - ref.float()).abs().max().item() <= 2 ** -7


def test_decode_strided_query_and_shared_pages(cuda_device):
    """A sliced query, a sliced page table, and requests that share a prefix's pages."""
    g = torch.Generator().manual_seed(7)
    kp, vp = _pool(g, 9, 4, 16, 128, "bf16", "hnd", cuda_device)
    wide = torch.tensor([[9, 4, 2, 1, 9], [9, 4, 2, 7, 9]], dtype=torch.int32, device=cuda_device)
    table = wide[:, 1:4]
    q = torch.randn(2, 1, 3, 8, 128, generator=g).to(torch.bfloat16).to(cuda_device)[:, :, 1].transpose(1, 2)
    out = ab.paged_gqa_decode_attention(q, kp, vp, table, sm_scale=0.09, num_key_value_groups=2, kv_lens=[45, 33])
    ref, _ = op.decode(_np(q), _np(kp), _np(vp), table.cpu().numpy(), [45, 33], [0, 0], 0.09, 2)
    _near(out, ref, "bf16", 1e-3)


def test_decode_repeats_to_the_bit_and_on_other_streams(cuda_device):
    q, kp, vp, table, out = _decode_case(cuda_device, "bf16", 128, 16, 8, 16, [5000, 1, 0, 777], spoil=False)
    kw = dict(sm_scale=128 ** -0.5, num_key_value_groups=2, kv_lens=[5000, 1, 0, 777])
    for _ in range(5):
        assert torch.equal(ab.paged_gqa_decode_attention(q, kp, vp, table, **kw), out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ab.paged_gqa_decode_attention(q, kp, vp, table, **kw)
    side.synchronize()
    assert torch.equal(again, out)


def test_decode_shares_the_workspace_with_the_contiguous_decode(cuda_device):
    """Both operators, in turn, at changing shapes, leave the counters at zero."""
    g = torch.Generator().manual_seed(9)
    for batch, length in [(2, 4000), (30, 300), (1, 9000), (2, 4000)]:
        per = length // 16 + 1
        kp, vp = _pool(g, batch * per, 8, 16, 128, "bf16", "hnd", cuda_device)
        table = _table(g, batch, per, batch * per, cuda_device)
        q = torch.randn(batch, 16, 1, 128, generator=g).to(torch.bfloat16).to(cuda_device)
        lens = torch.randint(1, length + 1, (batch,), generator=g).tolist()
        k, v = (p[table.long()].transpose(1, 2).reshape(batch, 8, per * 16, 128).contiguous() for p in (kp, vp))
        a = ab.paged_gqa_decode_attention(q, kp, vp, table, sm_scale=0.09, num_key_value_groups=2, kv_lens=lens)
        b = ab.gqa_decode_attention(q, k, v, sm_scale=0.09, num_key_value_groups=2, kv_lens=lens)
        assert (a.float() - b.float()).abs().max().item() <= 1e-2


def test_append_and_decode_in_a_graph(cuda_device):
    """The step of a growing cache, replayed: each replay appends one token and attends to it."""
    g = torch.Generator().manual_seed(11)
    B, Hq, Hkv, D, size, per = 3, 4, 2, 64, 8, 4
    kp, vp = _pool(g, B * per, Hkv, size, D, "bf16", "hnd", cuda_device)
    table = _table(g, B, per, B * per, cuda_device)
    q, k, v = (torch.randn(B, h, 1, D, generator=g).to(torch.bfloat16).to(cuda_device) for h in (Hq, Hkv, Hkv))
    ang = torch.randn(B, 1, D, generator=g).to(cuda_device)
    lens = torch.tensor([0, 7, 20], dtype=torch.int32, device=cuda_device)
    nxt = torch.empty_like(lens)

    def step():
        r = ab.paged_rope_kv_append(q, k, v, ang.cos(), ang.sin(), kp, vp, table, lens, kv_lens_out=nxt)
        o = ab.paged_gqa_decode_attention(r, kp, vp, table, sm_scale=0.125, num_key_value_groups=2, kv_lens=nxt)
        lens.copy_(nxt)
        return r, o

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        r, o = step()
    for n in range(2, 10):
        graph.replay()
        torch.cuda.synchronize()
        assert lens.tolist() == [n, 7 + n, 20 + n]
        ref, _ = op.decode(_np(r), _np(kp), _np(vp), table.cpu().numpy(), lens.tolist(), [0] * 3, 0.125, 2)
        _near(o, ref, "bf16", 1e-3)


def test_empty_batches(cuda_device):
    kp = torch.zeros(2, 2, 8, 64, dtype=torch.bfloat16, device=cuda_device)
    q = torch.zeros(0, 4, 1, 64, dtype=torch.bfloat16, device=cuda_device)
    table = torch.zeros(0, 3, dtype=torch.int32, device=cuda_device)
    out, lse = ab.paged_gqa_decode_attention(q, kp, kp, table, sm_scale=1.0, num_key_value_groups=2, return_lse=True)
    assert out.shape == q.shape and lse.shape == (0, 4)
    k = torch.zeros(1, 2, 0, 64, dtype=torch.bfloat16, device=cuda_device)
    cos = torch.zeros(1, 0, 64, device=cuda_device)
    lens = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    r = ab.paged_rope_kv_append(torch.zeros(1, 4, 0, 64, dtype=torch.bfloat16, device=cuda_device), k, k, cos, cos, kp,
                                kp.clone(), torch.zeros(1, 3, dtype=torch.int32, device=cuda_device), [5],
                                kv_lens_out=lens)
    assert r.shape == (1, 4, 0, 64) and lens.tolist() == [5]


# ------------------------------------------------------------------ refusals


def _good(device):
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=device)  # noqa: E731
    return {"query": z(2, 4, 1, 64), "key": z(2, 2, 1, 64), "value": z(2, 2, 1, 64),
            "cos": torch.zeros(2, 1, 64, device=device), "sin": torch.zeros(2, 1, 64, device=device),
            "k_pages": z(5, 2, 16, 64), "v_pages": z(5, 2, 16, 64),
            "page_table": torch.zeros(2, 2, dtype=torch.int32, device=device), "positions": [0, 0]}


REFUSED = [
    ("page_size", lambda a, z: a | {"k_pages": z(5, 2, 12, 64), "v_pages": z(5, 2, 12, 64)}),
    ("head_dim", lambda a, z: a | {"k_pages": z(5, 2, 16, 32), "v_pages": z(5, 2, 16, 32)}),
    ("one shape", lambda a, z: a | {"v_pages": z(4, 2, 16, 64)}),
    ("unit-stride", lambda a, z: a | {"k_pages": torch.as_strided(z(40960), (5, 2, 16, 64), (8192, 4096, 256, 2))}),
    ("16 bytes", lambda a, z: a | {"k_pages": torch.as_strided(z(20000), (5, 2, 16, 64), (2076, 1028, 64, 1))}),
    ("aligned", lambda a, z: a | {"k_pages": z(10248)[4:-4].view(5, 2, 16, 64)}),
    ("share a dtype", lambda a, z: a | {"k_pages": z(5, 2, 16, 64).half()}),
    ("page_table", lambda a, z: a | {"page_table": a["page_table"].long()}),
    ("page_table", lambda a, z: a | {"page_table": a["page_table"][:1]}),
    ("CUDA", lambda a, z: a | {"page_table": a["page_table"].cpu()}),
]


@pytest.mark.parametrize("text,change", REFUSED)
@pytest.mark.parametrize("which", ["append", "decode"])
def test_pool_refusals(cuda_device, text, change, which):
    a = change(_good(cuda_device), lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=cuda_device))
    with pytest.raises(ValueError, match=text):
        if which == "append":
            ab.paged_rope_kv_append(**a)
        else:
            ab.paged_gqa_decode_attention(a["query"], a["k_pages"], a["v_pages"], a["page_table"], sm_scale=0.1,
                                          num_key_value_groups=2)


def test_append_refusals(cuda_device):
    ok = _good(cuda_device)
    ab.paged_rope_kv_append(**ok)
    for text, more in [
        ("key and value", {"key": ok["key"][:, :1]}),
        ("dtype", {"value": ok["value"].half()}),
        ("cos/sin", {"cos": ok["cos"][:, :, :32]}),
        ("cos/sin", {"cos": ok["cos"].half(), "sin": ok["sin"].half()}),
        ("kv_lens", {"positions": [0, 0, 0]}),
        ("kv_lens_out", {"kv_lens_out": torch.zeros(2, dtype=torch.int64, device=cuda_device)}),
        ("norm weights", {"q_norm_weight": torch.ones(64, device=cuda_device)}),
        ("q_out", {"q_out": ok["query"][:, :, :, :32]}),
        ("must not be positions", dict.fromkeys(["positions", "kv_lens_out"],
                                                torch.zeros(2, dtype=torch.int32, device=cuda_device))),
        ("not a multiple", {"query": torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16, device=cuda_device)}),
    ]:
        with pytest.raises(ValueError, match=text):
            ab.paged_rope_kv_append(**(ok | more))


def test_decode_refusals(cuda_device):
    ok = _good(cuda_device)
    call = lambda q=ok["query"], g=2, **kw: ab.paged_gqa_decode_attention(  # noqa: E731
        q, ok["k_pages"], ok["v_pages"], ok["page_table"], **({"sm_scale": 0.1, "num_key_value_groups": g} | kw))
    call()
    with pytest.raises(ValueError, match="q_len"):
        call(torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device=cuda_device))
    with pytest.raises(ValueError, match="num_key_value_groups"):
        call(g=3)
    with pytest.raises(ValueError, match="finite"):
        call(sm_scale=float("inf"))
    with pytest.raises(ValueError, match="kv_lens"):
        call(kv_lens=[1])
    with pytest.raises(ValueError, match="inference"):
        call(torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device=cuda_device, requires_grad=True))
