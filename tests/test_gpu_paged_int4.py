"""The 4-bit cache's append, read and decode attention on the GPU against their
float64 restatement, at the sizes and masks where they can go wrong.

Tolerances.  Pairs (scale, least) of values that the kernel holds exactly are exact, and
so are codes, but for elements whose code lies within 2^-15 of a rounding border: the
kernel's (x - least) / scale in fp32 is off by at most 4 roundings of numbers below 16,
4 x 16 x 2^-24 < 2^-17.  Keys that are rotated in fp32 are off by a few roundings
of terms below 16 (8 x 16 x 2^-24 < 1e-5), so a pair may be rounded to the neighbour and a
code be off by 1e-5 of a scale of 0.1 or more: borders are 2^-10 wide there, and keys
are compared by their values, each to a unit of the pair and the code's border.
Attention: a score is a sum of D exact products and a group's term, of absolute values
below 10 in all after scaling, in at most 16 fp32 additions a part (16 x 10 x 2^-24 < 1e-5,
twice for the two parts of q): weights are off by 2e-5 of themselves, outputs by
twice that of values below 5, 2e-4, and by the half unit of their rounding."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _native as nat
from oracle import paged as op
from oracle import paged_int4 as o4
from oracle import rope as orope

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _np(t: torch.Tensor) -> np.ndarray:
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.detach().cpu().numpy()


def _pool(g, pages, hkv, size, dim, group, dtype, layout, device):
    """A pool of rounded random rows; 'nhd': stored [P, size, Hkv, ...]; 'wide': rows with
    room between them."""
    rows = torch.randn(pages, hkv, size, dim, generator=g).to(DT[dtype])
    codes, scales = ab.quantize_kv_int4(rows, group)
    if layout == "nhd":
        codes, scales = (t.transpose(1, 2).contiguous().to(device).transpose(1, 2) for t in (codes, scales))
    elif layout == "wide":
        wide = torch.full((pages, hkv, size, dim // 2 + 16), 255, dtype=torch.uint8, device=device)
        wide[..., : dim // 2] = codes.to(device)
        spread = torch.full((pages, hkv, size, 3 * (dim // group), 2), float("nan"), dtype=DT[dtype], device=device)
        spread[..., : dim // group, :] = scales.to(device)
        codes, scales = wide[..., : dim // 2], spread[..., : dim // group, :]
    else:
        codes, scales = codes.to(device), scales.to(device)
    return ab.Int4Pages(codes, scales)


def _values(pool) -> np.ndarray:
    s = _np(pool.scales)
    return o4.values(o4.unpack(_np(pool.codes)), s[..., 0], s[..., 1])


def _table(g, batch, per, pages, device):
    return torch.randperm(pages, generator=g)[: batch * per].view(batch, per).to(torch.int32).to(device)


# ------------------------------------------------------------------ append


def _append_case(device, dtype, dim, group, hq, hkv, batch, seq, size, per, layout="hnd", tables="fp32", norm=False,
                 seed=0, positions=None, counts=None, one_table=False, edit=None):
    g = torch.Generator().manual_seed(seed)
    pages = batch * per + 2
    kp, vp = (_pool(g, pages, hkv, size, dim, group, dtype, layout, device) for _ in range(2))
    table = _table(g, batch, per, pages, device)
    q, k, v = (torch.randn(batch, seq, h, dim, generator=g).to(DT[dtype]) for h in (hq, hkv, hkv))
    if edit is not None:
        edit(k, v)
    q, k, v = (t.to(device).transpose(1, 2) for t in (q, k, v))
    ang = torch.randn(1 if one_table else batch, seq, dim, generator=g) * 3
    tdt = torch.float32 if tables == "fp32" else DT[tables]
    cos, sin = ang.cos().to(tdt).to(device), ang.sin().to(tdt).to(device)
    w = [(1 + 0.3 * torch.randn(dim, generator=g)).to(DT[dtype]).to(device) for _ in range(2)] if norm else [None] * 2
    if positions is None:
        positions = torch.randint(0, per * size - seq + 1, (batch,), generator=g).tolist()
    pos = torch.tensor(positions, dtype=torch.int32, device=device)
    lens = torch.full((batch,), -7, dtype=torch.int32, device=device)
    new = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=device)
    before = [_np(t) for t in (*kp, *vp)]
    out = ab.paged_rope_kv_append_int4(q, k, v, cos, sin, kp, vp, table, pos, num_new=new, kv_lens_out=lens,
                                       q_norm_weight=w[0], k_norm_weight=w[1])
    cnt = [seq] * batch if counts is None else counts
    c, s = (np.broadcast_to(_np(t), (batch, seq, dim)) for t in (cos, sin))
    cap = per * size
    assert lens.tolist() == [min(max(p, 0) + max(0, min(n, seq)), cap) for p, n in zip(positions, cnt)]
    # q as paged_rope_kv_append returns it, bit for bit
    like = ab.PagedKVCache(1, pages, size, hkv, dim, dtype=DT[dtype], device=device)
    assert torch.equal(out, ab.paged_rope_kv_append(q, k, v, cos, sin, like.keys[0], like.values[0], table, pos, num_new=new,
                                                    q_norm_weight=w[0], k_norm_weight=w[1]))
    tab = table.cpu().numpy()
    for side, (pool, rows) in enumerate(((kp, k), (vp, v))):
        exact = side == 1 or tables != "fp32"
        if side == 0 and tables != "fp32":
            x = orope.apply_rope(_np(rows) if w[1] is None else orope.rms_norm_heads(_np(rows), _np(w[1]), 1e-6, dtype),
                                 c, s, dtype)
            exact = w[1] is None  # the sum of squares' order may move a key by a unit
        elif side == 0:
            x = op.rotate(_np(rows), c, s, None if w[1] is None else _np(w[1]))
        else:
            x = _np(rows)
        scale, least, code = o4.levels(x, group, dtype)
        old_c, old_s = before[2 * side:2 * side + 2]
        wrote = op.append(np.zeros((*old_c.shape[:3], 1)), np.ones((*x.shape[:3], 1)), tab, positions, cnt)[..., 0] == 1
        got_c, got_s = _np(pool.codes), _np(pool.scales)
        np.testing.assert_array_equal(got_c[~wrote], old_c[~wrote])
        np.testing.assert_array_equal(got_s[~wrote], old_s[~wrote])
        flat = lambda a: op.append(np.zeros((*old_c.shape[:3], a.shape[-1])), a.astype(np.float64), tab, positions, cnt)[wrote]  # noqa: E731
        want_code, want_scale, want_least = flat(code), flat(scale), flat(least)
        q4 = o4.unpack(got_c)[wrote].astype(np.float64)
        sc, lo = got_s[wrote][..., 0].astype(np.float64), got_s[wrote][..., 1].astype(np.float64)
        if exact:
            np.testing.assert_array_equal(sc, want_scale)
            np.testing.assert_array_equal(lo, want_least)
            ok = np.isfinite(want_scale).repeat(group, -1)
            assert (np.abs(q4 - want_code)[ok] <= 0.5 + 2.0 ** -15).all()
            assert (q4[~ok] == 0).all()
        else:
            unit = 2 * HALF_ULP[dtype]
            near = 4 if norm and tables != "fp32" else 0  # a key's own unit
            assert (np.abs(sc - want_scale) <= unit * np.abs(want_scale) * (1 + near)).all()
            assert (np.abs(lo - want_least) <= (unit * (1 + near)) * np.abs(want_least) + 1e-5).all()
            val = flat(x)
            each = sc.repeat(group, -1)
            off = np.abs(q4 * each + lo.repeat(group, -1) - val)
            # half a step, what the ends of the range lose to the pair's rounding, and the key's own error
            slack = 15 * each * unit + unit * np.abs(lo).repeat(group, -1) + 1e-5 + near * HALF_ULP[dtype] * np.abs(x).max()
            assert (off <= (0.5 + 2.0 ** -10) * each + slack).all()
    assert nat.device_error_flags() == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64), (128, 128)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("tables", ["fp32", "own"])
def test_append_types_and_groups(cuda_device, dtype, dim, group, norm, tables):
    _append_case(cuda_device, dtype, dim, group, 6, 2, 3, 5, 16, 3, norm=norm, tables=dtype if tables == "own" else "fp32",
                 seed=dim + group)


@pytest.mark.parametrize("layout", ["hnd", "nhd", "wide"])
@pytest.mark.parametrize("size", [8, 24, 128])
@pytest.mark.parametrize("heads", [(1, 1), (20, 1), (7, 7)])
def test_append_layouts(cuda_device, layout, size, heads):
    per = -(-70 // size)
    _append_case(cuda_device, "bf16", 128, 64, *heads, 2, 67, size, per, layout=layout, one_table=True, seed=size)


def test_append_many_tokens(cuda_device):
    _append_case(cuda_device, "bf16", 128, 128, 16, 8, 3, 200, 16, 14, norm=True, counts=[200, 0, 77])


@pytest.mark.parametrize("dtype,dim,group,tables", [("bf16", 128, 128, "fp32"), ("fp16", 128, 64, "fp32"), ("bf16", 64, 64, "fp32"),
                                                    ("fp16", 128, 128, "own"), ("bf16", 64, 64, "own")])
@pytest.mark.parametrize("heads", [(6, 2), (20, 1), (7, 7), (34, 17)])
def test_append_long_prompts(cuda_device, dtype, dim, group, tables, heads):
    """More tokens than warps, heads that do not fill a unit of rows, requests with fewer and no new tokens."""
    _append_case(cuda_device, dtype, dim, group, *heads, 5, 523, 16, 34, norm=True, tables=dtype if tables == "own" else "fp32",
                 counts=[523, 0, 77, 523, 522], one_table=heads[0] == 7, seed=heads[0] + dim)


@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64), (128, 128)])
@pytest.mark.parametrize("dtype,norm", [("bf16", True), ("bf16", False), ("fp16", True), ("fp16", False)])
@pytest.mark.parametrize("batch,seq", [(8, 2048), (500, 1)])
def test_append_keys_get_the_codes_of_torchs_keys(cuda_device, dim, group, dtype, norm, batch, seq):
    """Codes and pairs to the bit: those of the keys that torch's operations give on the GPU."""
    g = torch.Generator(device=cuda_device).manual_seed(dim + seq)
    dt, hq, hkv, per = DT[dtype], 8, 8, -(-seq // 16)
    q, k, v = (torch.randn(batch, seq, h, dim, generator=g, device=cuda_device).to(dt).transpose(1, 2) for h in (hq, hkv, hkv))
    ang = 3 * torch.randn(batch, seq, dim, generator=g, device=cuda_device)
    cos, sin = ang.cos(), ang.sin()
    w = (1 + 0.3 * torch.randn(dim, generator=g, device=cuda_device)).to(dt) if norm else None
    kp, vp = (ab.int4_pages(batch * per, hkv, 16, dim, group, dtype=dt, device=cuda_device) for _ in range(2))
    table = torch.arange(batch * per, dtype=torch.int32, device=cuda_device).view(batch, per)
    ab.paged_rope_kv_append_int4(q, k, v, cos, sin, kp, vp, table, torch.zeros(batch, dtype=torch.int32, device=cuda_device),
                                 q_norm_weight=w, k_norm_weight=w)
    x = k.float()
    if norm:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    x = x * cos[:, None] + torch.cat([-x[..., dim // 2:], x[..., : dim // 2]], -1) * sin[:, None]
    for pool, rows in ((kp, x), (vp, v.float())):
        y = rows.unflatten(-1, (-1, group))
        least = y.amin(-1).to(dt)
        scale = ((y.amax(-1) - least.float()) / 15).to(dt)
        code = ((y - least.float()[..., None]) / scale.float()[..., None]).round().clamp(0, 15).to(torch.uint8).flatten(-2)
        for part, want in zip(pool, (code[..., 0::2] | (code[..., 1::2] << 4), torch.stack([scale, least], -1))):
            got = part.view(batch, per, *part.shape[1:]).transpose(1, 2).flatten(2, 3)[:, :, :seq]
            assert torch.equal(got, want)


@pytest.mark.parametrize("layout", ["hnd", "nhd", "wide"])
def test_append_long_prompts_layouts(cuda_device, layout):
    _append_case(cuda_device, "bf16", 128, 64, 4, 2, 3, 331, 24, 14, layout=layout, positions=[0, 5, 300], seed=9)
    _append_case(cuda_device, "bf16", 64, 64, 1, 1, 1, 3001, 8, 376, layout=layout, norm=True, seed=10)


def test_append_single_tokens_at_page_edges(cuda_device):
    _append_case(cuda_device, "fp16", 64, 64, 16, 8, 6, 1, 16, 4, positions=[0, 15, 16, 31, 62, 63], norm=True)


def test_append_drops_what_has_no_place(cuda_device):
    _append_case(cuda_device, "fp16", 64, 64, 4, 2, 7, 6, 8, 2, positions=[0, 12, 16, 40, -3, -9, 2147483647],
                 counts=[0, 6, 6, 6, 6, 6, 6])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_append_constant_rows_and_far_scales(cuda_device, dtype):
    """All one value, one outlier, tiny and huge ranges."""

    def edit(k, v):
        v[:, 0], v[:, 1] = 1.75, 0.0
        v[:, 2, :, 7] = 900.0
        v[:, 3] *= 1e-4
        v[:, 4] *= 500.0
        if dtype == "bf16":
            v[:, 5] *= 1e-36
            v[:, 6] *= 1e36

    _append_case(cuda_device, dtype, 128, 64, 4, 2, 2, 7, 16, 1, edit=edit, seed=4)


def test_append_rows_that_are_not_finite(cuda_device):
    """Their group reads back as NaN; the row's other group and its neighbours do not."""

    def edit(k, v):
        v[0, 0, 0, 3], v[0, 1, 0, 100], v[0, 2, 1, 64] = float("nan"), float("inf"), float("-inf")

    _append_case(cuda_device, "bf16", 128, 64, 4, 2, 2, 5, 16, 1, edit=edit, seed=5)
    _append_case(cuda_device, "fp16", 128, 128, 4, 2, 2, 5, 16, 1, edit=edit, seed=5)


# ------------------------------------------------------------------ read


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64), (128, 128)])
@pytest.mark.parametrize("layout", ["hnd", "nhd", "wide"])
def test_read(cuda_device, dtype, dim, group, layout):
    g = torch.Generator().manual_seed(dim)
    B, hkv, size, per, S = 6, 3, 24, 3, 61
    kp, vp = (_pool(g, B * per + 2, hkv, size, dim, group, dtype, layout, cuda_device) for _ in range(2))
    table = _table(g, B, per, B * per + 2, cuda_device)
    table[3, 1], table[4, 0] = -1, 10 ** 9
    positions, counts = [0, 5, 40, 3, 0, -4], [61, 20, 61, 61, 30, 61]
    k, v = ab.paged_kv_read_int4(kp, vp, table, positions, S, num_tokens=torch.tensor(counts, dtype=torch.int32,
                                                                                       device=cuda_device))
    tab = table.cpu().numpy()
    for got, pool in ((k, kp), (v, vp)):
        assert got.shape == (B, hkv, S, dim) and got.dtype is DT[dtype]
        val, ref = _values(pool), np.zeros((B, hkv, S, dim))
        for b in range(B):
            for s in range(counts[b]):
                t = positions[b] + s
                if 0 <= t < per * size and 0 <= tab[b, t // size] < val.shape[0]:
                    ref[b, :, s] = val[tab[b, t // size], :, t % size]
        np.testing.assert_array_equal(_np(got), orope.round_to(ref.astype(np.float32), dtype))
    whole, _ = ab.paged_kv_read_int4(kp, vp, table, positions, S)
    np.testing.assert_array_equal(_np(whole[0]), _np(k[0]))
    assert ab.paged_kv_read_int4(kp, vp, table, positions, 0)[0].shape == (B, hkv, 0, dim)


# ------------------------------------------------------------------ attention


def _attend_case(device, dtype, dim, group, hq, hkv, lens, size, layout="hnd", starts=None, seed=0, per=None, edit=None,
                 scale=None, capacity=False, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    per = max(1, -(-max(lens) // size)) if per is None else per
    pages = B * per + 2
    kp, vp = (_pool(g, pages, hkv, size, dim, group, dtype, layout, device) for _ in range(2))
    table = _table(g, B, per, pages, device)
    q = (spread * torch.randn(B, hq, 1, dim, generator=g)).to(DT[dtype]).to(device)
    if edit is not None:
        edit(q, kp, vp, table)
    scale = dim ** -0.5 if scale is None else scale
    t32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    out, lse = ab.paged_gqa_decode_attention_int4(
        q, kp, vp, table, sm_scale=scale, num_key_value_groups=hq // hkv, kv_lens=None if capacity else t32(lens),
        kv_starts=t32(starts), return_lse=True)
    k, v = (np.nan_to_num(_values(p)) for p in (kp, vp))
    tab = table.cpu().numpy().copy()
    outside = (tab < 0) | (tab >= pages)
    if outside.any():  # pages of zeros
        k, v = (np.concatenate([p, np.zeros_like(p[:1])]) for p in (k, v))
        tab[outside] = pages
    ref, ref_lse = op.decode(_np(q), k, v, tab, [per * size] * B if capacity else lens, starts or [0] * B, scale, hq // hkv)
    got, got_lse = _np(out).astype(np.float64), _np(lse).astype(np.float64)
    assert np.isfinite(got).all()
    off = np.abs(got - ref) - (HALF_ULP[dtype] * np.abs(ref) + 2e-4)
    assert off.max() <= 0, f"{off.max():.3e} over the bound"
    dead = np.isneginf(ref_lse)
    assert np.array_equal(np.isneginf(got_lse), dead)
    assert (np.abs(got_lse[~dead] - ref_lse[~dead]) <= 1e-4 + 2.0 ** -22 * np.abs(ref_lse[~dead])).all()
    assert nat.device_error_flags() == 0
    return out, lse


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64), (128, 128)])
@pytest.mark.parametrize("heads", [(1, 1), (4, 2), (6, 2), (10, 2), (16, 2), (16, 1), (20, 1), (36, 1)])
def test_attend_types_and_groups(cuda_device, dtype, dim, group, heads):
    _attend_case(cuda_device, dtype, dim, group, *heads, [0, 1, 7, 16, 33, 300], 16, seed=dim + heads[0])


@pytest.mark.parametrize("layout", ["hnd", "nhd", "wide"])
@pytest.mark.parametrize("size", [8, 16, 24, 40, 128])
def test_attend_layouts(cuda_device, layout, size):
    _attend_case(cuda_device, "bf16", 128, 64, 4, 2, [1, 31, 32, 33, 200, 517], size, layout=layout, seed=size)


@pytest.mark.parametrize("batch,hi", [(1, 1024), (1, 9000), (3, 2500), (40, 700), (200, 40)])
def test_attend_batches(cuda_device, batch, hi):
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, hi + 1, (batch,), generator=g).tolist()
    lens[0] = hi
    starts = [int(n * f) for n, f in zip(lens, torch.rand(batch, generator=g).tolist())]
    _attend_case(cuda_device, "bf16", 128, 128, 8, 4, lens, 16, starts=starts, seed=batch)
    _attend_case(cuda_device, "fp16", 64, 64, 6, 2, lens, 24, seed=batch)


def test_attend_starts_and_empty_rows(cuda_device):
    _attend_case(cuda_device, "bf16", 128, 64, 4, 2, [0, 5, 5, 40, 100, 100], 16, starts=[0, 5, 9, 39, 17, -3])
    _attend_case(cuda_device, "bf16", 64, 64, 4, 2, [64, 64], 16, capacity=True, starts=[0, 63])


def test_attend_pages_outside_the_pool_and_dead_slots(cuda_device):
    """Pages outside the pool read as zeros; NaN in slots out of range is not seen."""

    def edit(q, kp, vp, table):
        table[0, 1], table[1, 0] = -1, 2 ** 30
        for b, (lo, hi) in enumerate(((3, 61), (0, 50))):  # behind the length and before the start
            for t in [*range(lo), *range(hi, 64)]:
                page = int(table[b, t // 16])
                if 0 <= page < kp.codes.shape[0]:
                    for p in (kp, vp):
                        p.scales[page, :, t % 16] = float("nan")

    _attend_case(cuda_device, "bf16", 128, 64, 4, 2, [61, 50], 16, starts=[3, 0], edit=edit, per=4)


def test_attend_far_values(cuda_device):
    """Peaked softmaxes, scales far apart between slots, and large and tiny queries."""

    def edit(q, kp, vp, table):
        vp.scales[:, :, ::3] *= 1e-3
        kp.scales[:, :, 5::7] *= 0.01
        q[0] *= 1e-4

    for dtype in ("bf16", "fp16"):
        _attend_case(cuda_device, dtype, 128, 64, 4, 2, [400, 900], 16, edit=edit, spread=3.0)
        _attend_case(cuda_device, dtype, 64, 64, 4, 2, [400, 900], 16, edit=edit, scale=-0.3)


def test_attend_values_that_are_not_finite(cuda_device):
    """A live slot with NaN makes its head's result NaN, and no other's."""
    g = torch.Generator().manual_seed(1)
    kp, vp = (_pool(g, 8, 2, 16, 128, 64, "bf16", "hnd", cuda_device) for _ in range(2))
    table = torch.arange(8, dtype=torch.int32, device=cuda_device).view(2, 4)
    q = torch.randn(2, 4, 1, 128, generator=g).to(torch.bfloat16).to(cuda_device)
    clean = ab.paged_gqa_decode_attention_int4(q, kp, vp, table, sm_scale=0.09, num_key_value_groups=2)
    vp.scales[1, 0, 3, 1] = float("nan")  # request 0, head 0, the second group
    out = ab.paged_gqa_decode_attention_int4(q, kp, vp, table, sm_scale=0.09, num_key_value_groups=2)
    assert out[0, :2, 0, 64:].isnan().all()
    assert torch.equal(out[0, :2, 0, :64], clean[0, :2, 0, :64])
    assert torch.equal(out[0, 2:], clean[0, 2:]) and torch.equal(out[1], clean[1])
    kp.scales[5, 1, 0, 0] = float("nan")  # request 1, head 1
    out = ab.paged_gqa_decode_attention_int4(q, kp, vp, table, sm_scale=0.09, num_key_value_groups=2)
    assert out[1, 2:].isnan().all() and torch.equal(out[1, :2], clean[1, :2])


def test_attend_repeats_to_the_bit_and_replays(cuda_device):
    g = torch.Generator().manual_seed(2)
    B, per = 5, 60
    kp, vp = (_pool(g, B * per, 4, 16, 128, 128, "bf16", "hnd", cuda_device) for _ in range(2))
    table = _table(g, B, per, B * per, cuda_device)
    q = torch.randn(B, 8, 1, 128, generator=g).to(torch.bfloat16).to(cuda_device)
    lens = torch.tensor([960, 3, 0, 500, 961 - 5], dtype=torch.int32, device=cuda_device)
    run = lambda: ab.paged_gqa_decode_attention_int4(q, kp, vp, table, sm_scale=0.09, num_key_value_groups=2,  # noqa: E731
                                                     kv_lens=lens, return_lse=True)
    first = run()
    for _ in range(3):
        again = run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first[0], other[0])
    lens.copy_(torch.tensor([10, 959, 400, 1, 0], dtype=torch.int32))
    graph.replay()
    fresh = run()
    torch.cuda.synchronize()
    assert torch.equal(captured[0], fresh[0]) and torch.equal(captured[1], fresh[1])


# ------------------------------------------------------------------ refusals


def test_refusals(cuda_device):
    pool = ab.int4_pages(4, 2, 16, 128, 64, dtype=torch.bfloat16, device=cuda_device)
    table = torch.zeros(1, 2, dtype=torch.int32, device=cuda_device)
    q = torch.zeros(1, 4, 1, 128, dtype=torch.bfloat16, device=cuda_device)
    kv = torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16, device=cuda_device)
    cs = torch.zeros(1, 1, 128, device=cuda_device)
    pos = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    attend = lambda q=q, k=pool, v=pool, t=table, g=2: ab.paged_gqa_decode_attention_int4(  # noqa: E731
        q, k, v, t, sm_scale=0.1, num_key_value_groups=g)
    append = lambda k=pool, v=pool, **kw: ab.paged_rope_kv_append_int4(q, kv, kv, cs, cs, k, v, table, pos, **kw)  # noqa: E731
    attend()
    append()
    half = ab.Int4Pages(pool.codes, pool.scales.half())
    cases = [
        lambda: attend(q=q.float()), lambda: attend(q=q[..., :64]), lambda: attend(q=q.repeat(1, 1, 2, 1)),
        lambda: attend(g=1), lambda: attend(g=0), lambda: attend(t=table.long()), lambda: attend(t=table[0]),
        lambda: attend(k=half, v=half), lambda: attend(v=half), lambda: attend(k=pool.codes),
        lambda: attend(k=ab.Int4Pages(pool.codes[:, :, :12], pool.scales[:, :, :12])),
        lambda: attend(k=ab.Int4Pages(pool.codes, pool.scales[..., :1, :])),
        lambda: attend(k=ab.Int4Pages(pool.codes[..., ::2], pool.scales)),
        lambda: attend(k=ab.Int4Pages(pool.codes.int(), pool.scales)),
        lambda: attend(k=ab.Int4Pages(pool.codes.cpu(), pool.scales.cpu())),
        lambda: attend(q=q.clone().requires_grad_()),
        lambda: append(k=half, v=half), lambda: append(kv_lens_out=pos), lambda: append(kv_lens_out=table[0, :1]),
        lambda: append(q_norm_weight=torch.ones(64, dtype=torch.bfloat16, device=cuda_device)),
        lambda: ab.paged_rope_kv_append_int4(q, kv[:, :1], kv, cs, cs, pool, pool, table, pos),
        lambda: ab.paged_kv_read_int4(pool, pool, table, pos, -1), lambda: ab.paged_kv_read_int4(pool, pool, table, None, 1),
        lambda: ab.paged_kv_read_int4(pool.codes, pool, table, pos, 1),
    ]
    for i, case in enumerate(cases):
        with pytest.raises(ValueError):
            case()
            pytest.fail(f"case {i} was taken")
    # codes whose rows do not lie on 16 bytes
    odd = torch.zeros(4, 2, 16, 72, dtype=torch.uint8, device=cuda_device)[..., :64]
    with pytest.raises(ValueError, match="16"):
        attend(k=ab.Int4Pages(odd, pool.scales))
