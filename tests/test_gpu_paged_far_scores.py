"""Attention over 4-bit caches, the weights that it gives and a cut by them where scores lie far
from zero, as keys with a common offset make them: against float64.

Tolerances.  A score in base-2 units is a sum of D products in at most 8 fp32 accumulations that
may cut off (2^-23 each), the sum of q's elements (18 additions a lane and across lanes, 2^-24
each) and 4 further roundings: below 40 x 2^-24 of A, the sum of the absolute values of
q's elements times what a key is made of (scale times code, and |least|).  e = 40 x 2^-24 A is 1e-2 for
the scores of 1000 here.  A probability is off by 2^e - 1 of itself, and so is
their sum: an output by twice that of the largest |value|, and by half a unit of its rounding (2^-8
of bf16, 2^-11 of fp16) and 2e-4 as at ordinary scores (test_gpu_paged_int4.py); a log-sum-exp by e,
1e-4 and 2^-22 of itself; a weight by 2^(2 e + 2e-4) - 1 of itself, since score and
log-sum-exp enter, and 2^-22 of the sum."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _native as nat
from oracle import paged_int4 as o4
from tests.test_gpu_paged_int4 import DT, HALF_ULP, _np, _table, _values

pytestmark = pytest.mark.gpu

OFFSET = 3.0  # of a far head's keys


def _case(device, dtype, dim, group, hkv, groups, lens, far, seed, near=None, size=16):
    """Head 0 of each request has scores of about ``far`` (all its slots, or, with ``near``, all but the
    slots [near, ...), which score around 0); the other heads ordinary ones."""
    g = torch.Generator().manual_seed(seed)
    B, per = len(lens), -(-max(lens) // size)
    table = _table(g, B, per, B * per, device)
    rows = torch.randn(B * per, hkv, size, dim, generator=g)
    rows[:, 0] += OFFSET
    if near is not None:
        for b in range(B):
            for t in range(near, per * size):
                rows[int(table[b, t // size]), 0, t % size] -= OFFSET
    values = torch.randn(B * per, hkv, size, dim, generator=g)
    kp, vp = (ab.Int4Pages(*(t.to(device) for t in ab.quantize_kv_int4(r.to(DT[dtype]), group))) for r in (rows, values))
    q = torch.randn(B, hkv * groups, 1, dim, generator=g)
    scale = dim ** -0.5
    # sum_d q_d k_d scale = far for q_d = far / (scale OFFSET dim)
    q[:, :groups] = 0.1 * q[:, :groups] + far / (scale * OFFSET * dim)
    q = q.to(DT[dtype]).to(device)
    n = torch.tensor(lens, dtype=torch.int32, device=device)
    seen = dict(sm_scale=scale, num_key_value_groups=groups, kv_lens=n)
    out, lse = ab.paged_gqa_decode_attention_int4(q, kp, vp, table, return_lse=True, **seen)
    w = torch.zeros(B, hkv, per * size, device=device)
    ab.paged_attention_weights(q, kp, table, lse, w, **seen)
    got, got_lse, got_w = _np(out).astype(np.float64), _np(lse).astype(np.float64), _np(w).astype(np.float64)
    assert np.isfinite(got).all() and np.isfinite(got_lse).all() and np.isfinite(got_w).all()
    k64, v64, tab = _values(kp), _values(vp), table.cpu().numpy()
    codes, pairs = o4.unpack(_np(kp.codes)).astype(np.float64), _np(kp.scales).astype(np.float64)
    parts = codes * np.abs(pairs[..., 0]).repeat(group, -1) + np.abs(pairs[..., 1]).repeat(group, -1)
    log2e = 1.0 / np.log(2.0)
    for b, length in enumerate(lens):
        rows_of = lambda x: x[tab[b]].transpose(1, 0, 2, 3).reshape(hkv, -1, dim)[:, :length]  # noqa: E731
        q64 = _np(q)[b, :, 0].astype(np.float64).reshape(hkv, groups, dim)
        s = np.einsum("hgd,htd->hgt", q64, rows_of(k64)) * scale * log2e
        e = 40 * 2.0 ** -24 * (np.einsum("hgd,htd->hgt", np.abs(q64), rows_of(parts)).max(-1) * scale * log2e)
        m = s.max(-1, keepdims=True)
        p = np.exp2(s - m)
        want_lse = (m[..., 0] + np.log2(p.sum(-1))).reshape(-1)
        p /= p.sum(-1, keepdims=True)
        want = np.einsum("hgt,htd->hgd", p, rows_of(v64))
        top = np.abs(rows_of(v64)).max()
        bound = HALF_ULP[dtype] * np.abs(want) + 2e-4 + 2 * np.expm1(e * np.log(2.0))[..., None] * top
        off = np.abs(got[b, :, 0].reshape(want.shape) - want)
        assert (off <= bound).all(), f"request {b}: {(off - bound).max():.3e} over the bound"
        assert (np.abs(got_lse[b] - want_lse) <= e.reshape(-1) + 1e-4 + 2.0 ** -22 * np.abs(want_lse)).all()
        each = np.expm1((2 * e + 2e-4) * np.log(2.0))[..., None]
        total = p.sum(1)
        assert (np.abs(got_w[b, :, :length] - total) <= (each * p).sum(1) + 2.0 ** -22 * total + 1e-30).all()
        assert not got_w[b, :, length:].any()
    # a cut by these weights
    keep, first, last = 40, 2, 9
    before = [x.clone() for x in (*kp, *vp)]
    after = torch.empty_like(n)
    kept = ab.paged_kv_evict(kp, vp, table, w.clone(), n, keep=keep, keep_first=first, keep_last=last, kv_lens_out=after)
    for b, length in enumerate(lens):
        for h in range(hkv):
            mine = o4.kept_slots(got_w[b, h], length, keep, first, last, keep)
            assert kept[b, h, : len(mine)].tolist() == mine
            for now, was in zip((*kp, *vp), before):
                new, old = (t[table[b].long(), h].flatten(0, 1) for t in (now, was))
                assert torch.equal(new[: len(mine)], old[torch.tensor(mine, device=device)])
    again = ab.paged_gqa_decode_attention_int4(q, kp, vp, table, **{**seen, "kv_lens": after})
    assert torch.isfinite(again.float()).all()
    assert nat.device_error_flags() == 0


@pytest.mark.parametrize("far", [-1000.0, -200.0, -100.0, 100.0, 1000.0])
@pytest.mark.parametrize("groups", [1, 4, 8])
@pytest.mark.parametrize("dtype,dim,group", [("bf16", 128, 128), ("bf16", 128, 64), ("fp16", 64, 64)])
def test_heads_of_far_scores(cuda_device, far, groups, dtype, dim, group):
    """One slot, less than a tile, several hundred slots."""
    _case(cuda_device, dtype, dim, group, 2, groups, [1, 1, 20, 33, 400, 700], far, seed=groups)


@pytest.mark.parametrize("far", [-1000.0, -100.0, 100.0])
@pytest.mark.parametrize("batch,hkv,length", [(90, 8, 150), (2, 4, 6000)])
def test_far_scores_in_small_and_large_teams(cuda_device, far, batch, hkv, length):
    """Teams of one warp (many pairs) and of sixteen."""
    lens = [1 + (length - 1) * (b + 1) // batch for b in range(batch)]
    _case(cuda_device, "bf16", 128, 128, hkv, 2, lens, far, seed=batch)


@pytest.mark.parametrize("far", [-1000.0, -100.0, 100.0])
@pytest.mark.parametrize("near", [5, 32, 300])
def test_far_scores_before_ordinary_ones(cuda_device, far, near):
    """A reference that has to move by hundreds, or that later scores do not reach."""
    _case(cuda_device, "bf16", 128, 64, 2, 4, [6, 40, 333, 700], far, seed=near, near=near)
    _case(cuda_device, "fp16", 64, 64, 1, 8, [310, 1500], far, seed=near, near=near)
