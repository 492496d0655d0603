"""Attention weights added up and evictions by them on the GPU against their float64
restatement.

Tolerances.  A weight is 2^(score - lse) with a score that is off by less than 2e-5 (a sum
of D products of 16-bit numbers, below 10 in absolute values after scaling, in fp32; 4e-5
in base 2 units with the rounding of lse): 1e-4 of the weight, and the sum's fp32
additions, 2^-22 of it.  Evictions move bits: they are exact."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _native as nat
from oracle import paged as op
from oracle import paged_int4 as o4
from tests.test_gpu_paged_int4 import _np, _pool, _table, _values

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _pages(g, pages, hkv, size, dim, group, dtype, device, layout="hnd"):
    if group:
        return _pool(g, pages, hkv, size, dim, group, dtype, layout, device)
    if layout == "nhd":
        return torch.randn(pages, size, hkv, dim, generator=g).to(DT[dtype]).to(device).transpose(1, 2)
    return torch.randn(pages, hkv, size, dim, generator=g).to(DT[dtype]).to(device)


def _wide(pool) -> np.ndarray:
    return _values(pool) if isinstance(pool, ab.Int4Pages) else _np(pool).astype(np.float64)


def _lse(q, k, tab, lens, starts, scale, groups):
    """[B, Hq, S] of each window query over the slots that it sees."""
    B, Hq, S, _ = q.shape
    out = np.full((B, Hq, S), -np.inf)
    for s in range(S):
        out[:, :, s] = op.decode(q[:, :, s:s + 1], k, k, tab, [n - S + 1 + s for n in lens], starts, scale, groups)[1]
    return out


# ------------------------------------------------------------------ weights


def _weigh_case(device, dtype, dim, group, hq, hkv, seq, lens, size, starts=None, layout="hnd", seed=0, per=None,
                edit=None, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    B, per = len(lens), max(1, -(-max(lens) // size)) if per is None else per
    pages = B * per + 2
    kp = _pages(g, pages, hkv, size, dim, group, dtype, device, layout)
    table = _table(g, B, per, pages, device)
    if edit is not None:
        edit(kp, table)
    q = (spread * torch.randn(B, seq, hq, dim, generator=g)).to(DT[dtype]).to(device).transpose(1, 2)
    scale = dim ** -0.5
    k, tab = np.nan_to_num(_wide(kp)), table.cpu().numpy().copy()
    outside = (tab < 0) | (tab >= pages)
    k = np.concatenate([k, np.zeros_like(k[:1])])
    tab[outside] = pages
    starts = starts or [0] * B
    lse = _lse(_np(q), k, tab, lens, starts, scale, hq // hkv).astype(np.float32)
    C = per * size + 5
    before = torch.rand(B, hkv, C, generator=g)
    w = before.to(device)
    t32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    got = ab.paged_attention_weights(q, kp, table, torch.from_numpy(lse).to(device), w, sm_scale=scale,
                                     num_key_value_groups=hq // hkv, kv_lens=t32(lens), kv_starts=t32(starts))
    assert got is w
    for b in range(B):
        rows = op.gather(k, tab[b], min(lens[b], per * size))
        s0 = min(max(starts[b], 0), len(rows[0]))
        for h in range(hkv):
            add = o4.weights(_np(q)[b, h * (hq // hkv):(h + 1) * (hq // hkv)], rows[h], lse[b, h * (hq // hkv):(h + 1) * (hq // hkv)],
                             lens[b], s0, scale)
            ref = before[b, h].numpy().astype(np.float64)
            seen = np.zeros(C, bool)
            seen[s0:len(add)] = True
            assert np.array_equal(_np(w)[b, h][~seen], before[b, h].numpy()[~seen])
            off = np.abs(_np(w)[b, h][: len(add)] - (ref[: len(add)] + add)) - (1e-4 * add + 2.0 ** -22 * (ref[: len(add)] + add))
            assert off.size == 0 or off.max() <= 0, f"{off.max():.3e} over the bound"
    assert nat.device_error_flags() == 0
    return w


@pytest.mark.parametrize("dtype,dim,group", [("bf16", 128, 0), ("fp16", 64, 0), ("bf16", 16, 0), ("fp16", 32, 0),
                                             ("fp32", 128, 0), ("fp32", 16, 0), ("fp32", 64, 0), ("bf16", 128, 64),
                                             ("fp16", 128, 128), ("bf16", 64, 64)])
@pytest.mark.parametrize("heads", [(1, 1), (4, 2), (10, 2), (20, 1)])
@pytest.mark.parametrize("seq", [1, 5])
def test_weights_types_and_heads(cuda_device, dtype, dim, group, heads, seq):
    _weigh_case(cuda_device, dtype, dim, group, *heads, seq, [0, 1, 4, 17, 200], 16, seed=dim + seq)


@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("size,layout", [(8, "hnd"), (24, "nhd"), (128, "hnd"), (40, "nhd")])
def test_weights_layouts_and_starts(cuda_device, group, size, layout):
    _weigh_case(cuda_device, "bf16", 128, group, 4, 2, 3, [1, 2, 3, 130, 131, 257], size, starts=[0, 1, 3, 64, -5, 256],
                layout=layout, seed=size)


@pytest.mark.parametrize("group", [0, 128])
def test_weights_long_windows(cuda_device, group):
    """More queries than slots, windows of an odd size, many columns."""
    _weigh_case(cuda_device, "bf16", 128, group, 4, 2, 33, [10, 32, 33, 700], 16, seed=3)
    _weigh_case(cuda_device, "fp16", 128, group, 24, 1, 13, [100, 600], 32, seed=4)


@pytest.mark.parametrize("group", [0, 64])
def test_weights_dead_slots_and_pages(cuda_device, group):
    def edit(kp, table):
        table[0, 1], table[1, 0] = -1, 2 ** 30
        for b, hi in ((0, 61), (1, 50)):
            for t in range(hi, 64):
                part = kp.scales if group else kp
                part[int(table[b, t // 16]), :, t % 16] = float("nan")

    _weigh_case(cuda_device, "bf16", 128, group, 4, 2, 1, [61, 50], 16, edit=edit, per=4)


def test_weights_add_up_to_the_queries(cuda_device):
    """With the attention's own log-sum-exp, a step adds one a query head; and steps repeat to the bit."""
    g = torch.Generator().manual_seed(9)
    B, hq, hkv, per = 3, 8, 4, 30
    for group in (0, 128):
        kp, vp = (_pages(g, B * per, hkv, 16, 128, group, "bf16", cuda_device) for _ in range(2))
        table = _table(g, B, per, B * per, cuda_device)
        q = torch.randn(B, hq, 1, 128, generator=g).to(torch.bfloat16).to(cuda_device)
        lens = torch.tensor([480, 1, 333], dtype=torch.int32, device=cuda_device)
        attend = ab.paged_gqa_decode_attention_int4 if group else ab.paged_gqa_decode_attention
        kw = dict(sm_scale=128 ** -0.5, num_key_value_groups=hq // hkv, kv_lens=lens)
        _, lse = attend(q, kp, vp, table, return_lse=True, **kw)
        w = [ab.paged_attention_weights(q, kp, table, lse, torch.zeros(B, hkv, per * 16, device=cuda_device), **kw)
             for _ in range(2)]
        assert torch.equal(w[0], w[1])
        assert (w[0].double().sum(-1) - hq / hkv).abs().max() < 1e-4 * hq / hkv


def test_weights_refusals(cuda_device):
    kp = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device=cuda_device)
    table = torch.zeros(1, 2, dtype=torch.int32, device=cuda_device)
    q = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16, device=cuda_device)
    lse, w = torch.zeros(1, 4, 1, device=cuda_device), torch.zeros(1, 2, 32, device=cuda_device)
    call = lambda q=q, k=kp, t=table, lse=lse, w=w, g=2: ab.paged_attention_weights(  # noqa: E731
        q, k, t, lse, w, sm_scale=0.1, num_key_value_groups=g)
    call()
    call(lse=lse[..., 0])
    pool = ab.int4_pages(4, 2, 16, 64, dtype=torch.float16, device=cuda_device)
    for case in (lambda: call(q=q.half()), lambda: call(q=q[..., :32]), lambda: call(g=4), lambda: call(t=table.long()),
                 lambda: call(lse=lse.double()), lambda: call(lse=lse[:, :2]), lambda: call(w=w[..., :31]),
                 lambda: call(w=w.half()), lambda: call(w=w.cpu()), lambda: call(w=w[:, :1].expand(1, 2, 32)),
                 lambda: call(k=kp[..., ::2]), lambda: call(k=pool), lambda: call(k=kp.int()),
                 lambda: call(q=q.clone().requires_grad_()), lambda: call(w=w.clone().requires_grad_())):
        with pytest.raises(ValueError):
            case()


# ------------------------------------------------------------------ eviction


def _parts(pool):
    return list(pool) if isinstance(pool, tuple) else [pool]


def _bits(t: torch.Tensor) -> np.ndarray:
    return t.contiguous().view(torch.uint8).cpu().numpy()


def _evict_case(device, dtype, dim, group, hkv, lens, size, keep, first=0, last=0, longer=None, layout="hnd", seed=0,
                edit=None, per=None, alias=False, out=False, tables=None):
    g = torch.Generator().manual_seed(seed)
    B, per = len(lens), max(1, -(-max(lens) // size)) if per is None else per
    pages = B * per + 2
    kp, vp = (_pages(g, pages, hkv, size, dim, group, dtype, device, layout) for _ in range(2))
    table = _table(g, B, per, pages, device)
    if tables is not None:
        tables(table)
    w = (torch.rand(B, hkv, per * size + 3, generator=g) ** 4).float()
    if edit is not None:
        edit(w)
    before = [_bits(t) for p in (kp, vp) for t in _parts(p)]
    dw = w.to(device)
    wo = torch.full_like(dw, -5.0) if out else None
    dl = torch.tensor(lens, dtype=torch.int32, device=device)
    new = dl if alias else torch.full((B,), -7, dtype=torch.int32, device=device)
    kept = ab.paged_kv_evict(kp, vp, table, dw, dl, keep=keep, keep_first=first, keep_last=last, longer_than=longer,
                             kv_lens_out=new, weights_out=wo)
    longer = keep if longer is None else longer
    cap, tab = per * size, table.cpu().numpy()
    clamped = [min(max(n, 0), cap) for n in lens]
    assert new.tolist() == [keep if n > longer else n for n in clamped]
    if out:
        assert torch.equal(dw.cpu().nan_to_num(-1), w.nan_to_num(-1))
    ref = [x.copy() for x in before]
    for b, n in enumerate(clamped):
        for h in range(hkv):
            mine = o4.kept_slots(w[b, h].numpy(), n, keep, first, last, longer)
            row = kept[b, h].tolist()
            cut = n > longer
            assert row == (mine + [-1] * keep)[:keep], (b, h)
            want = (torch.full_like(w[b, h], -5.0) if out else w[b, h]).clone()
            want[: len(mine)] = w[b, h][mine]
            want[len(mine):n] = 0
            assert torch.equal((wo if out else dw)[b, h].cpu().nan_to_num(-1), want.nan_to_num(-1)), (b, h)
            if cut:
                for pool in ref:
                    o4.compact(pool, tab[b], h, mine)
    for x, t in zip(ref, [t for p in (kp, vp) for t in _parts(p)]):
        np.testing.assert_array_equal(_bits(t), x)
    assert nat.device_error_flags() == 0


@pytest.mark.parametrize("dtype,dim,group", [("bf16", 128, 0), ("fp16", 64, 0), ("fp32", 128, 0), ("bf16", 16, 0),
                                             ("fp32", 16, 0), ("bf16", 32, 0), ("bf16", 128, 64), ("fp16", 128, 128),
                                             ("bf16", 64, 64)])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_evict_types(cuda_device, dtype, dim, group, layout):
    _evict_case(cuda_device, dtype, dim, group, 3, [0, 1, 50, 51, 200, 333], 24, 50, 4, 10, layout=layout, seed=dim)


@pytest.mark.parametrize("keep,first,last", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (40, 20, 20), (40, 0, 40), (40, 40, 0),
                                             (255, 3, 7), (256, 0, 0), (513, 4, 100)])
def test_evict_counts(cuda_device, keep, first, last):
    _evict_case(cuda_device, "bf16", 64, 0, 2, [keep, keep + 1, 2 * keep, 1025], 16, keep, first, last, seed=keep)


@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("alias", [False, True])
def test_evict_longer_than(cuda_device, out, alias):
    _evict_case(cuda_device, "bf16", 64, 64, 2, [10, 100, 120, 121, 300, -4, 5000], 16, 80, 2, 20, longer=120, out=out,
                alias=alias, per=20)


def test_evict_weights_of_every_kind(cuda_device):
    """Equal weights, zeros of both signs, negative ones, infinities, NaN, subnormals."""

    def equal(w):
        w[:] = 0.25

    def odd(w):
        w -= 0.3
        w[..., 3::7] = float("nan")
        w[..., 5::11] = -0.0
        w[..., 6::11] = 0.0
        w[..., 8::13] = float("inf")
        w[..., 9::17] = float("-inf")
        w[..., 10::19] = 1e-42

    def nan(w):
        w[:] = float("nan")

    for edit in (equal, odd, nan):
        _evict_case(cuda_device, "bf16", 64, 0, 2, [400, 1000], 16, 150, 3, 11, edit=edit)
        _evict_case(cuda_device, "bf16", 64, 0, 2, [400, 1000], 16, 390, 0, 0, edit=edit)


def test_evict_pages_outside_the_pool(cuda_device):
    def tables(t):
        t[0, 1], t[1, 5], t[1, 0] = -1, 2 ** 30, -7

    _evict_case(cuda_device, "bf16", 128, 64, 2, [150, 160], 16, 70, 4, 10, tables=tables)


def test_evict_long_caches(cuda_device):
    _evict_case(cuda_device, "bf16", 16, 0, 1, [20000, 9999], 128, 8000, 4, 500, seed=1)
    _evict_case(cuda_device, "fp16", 64, 64, 2, [40001], 64, 1500, 4, 500, seed=2)


@pytest.mark.parametrize("n,keep", [(4097, 4000), (16384, 9000), (16400, 3), (33000, 32999), (70000, 35000), (131073, 70000)])
def test_evict_caches_of_many_slots(cuda_device, n, keep):
    """A thread's slots, clusters of CTAs and the way for still longer caches; many equal weights."""

    def coarse(w):
        w[:] = (w * 16).floor() / 16

    _evict_case(cuda_device, "bf16", 16, 0, 1, [n, n - 1, 5], 64, keep, 1, 2, edit=coarse, seed=n)
    _evict_case(cuda_device, "bf16", 16, 0, 1, [n], 64, keep, 0, 0, seed=n, out=True)


def test_evict_refusals(cuda_device):
    kp = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device=cuda_device)
    pool = ab.int4_pages(4, 2, 16, 64, dtype=torch.float16, device=cuda_device)
    table = torch.zeros(1, 2, dtype=torch.int32, device=cuda_device)
    w, lens = torch.zeros(1, 2, 32, device=cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device)
    call = lambda k=kp, v=kp, t=table, w=w, n=lens, keep=8, **kw: ab.paged_kv_evict(k, v, t, w, n, keep=keep, **kw)  # noqa: E731
    call()
    shared = torch.zeros(2, 2, 32, device=cuda_device)
    for case in (lambda: call(keep=0), lambda: call(keep_first=5, keep_last=4), lambda: call(keep_first=-1),
                 lambda: call(longer_than=7), lambda: call(v=pool), lambda: call(k=pool), lambda: call(v=kp[:3]),
                 lambda: call(w=w[..., :31]), lambda: call(w=w.double()), lambda: call(n=None),
                 lambda: call(kv_lens_out=torch.zeros(2, dtype=torch.int32, device=cuda_device)),
                 lambda: call(kv_lens_out=table[0, :1]), lambda: call(t=table.long()),
                 lambda: call(w=shared[:1], weights_out=shared.view(-1)[16:80].view(1, 2, 32)),
                 lambda: call(k=kp.cpu()), lambda: call(k=kp.int(), v=kp.int())):
        with pytest.raises(ValueError):
            case()


@pytest.mark.parametrize("group,batch", [(0, 2), (128, 2), (64, 40)])
def test_evict_of_one_pool_as_keys_and_values(cuda_device, group, batch):
    """Rows that are both move once (batches of the one launch, and of the two)."""
    g = torch.Generator().manual_seed(5)
    per, hkv = 20, 2
    pool = _pages(g, batch * per, hkv, 16, 128, group, "bf16", cuda_device)
    copy = ab.Int4Pages(*(t.clone() for t in pool)) if group else pool.clone()
    table = _table(g, batch, per, batch * per, cuda_device)
    w = torch.rand(batch, hkv, per * 16, generator=g).to(cuda_device)
    lens = torch.full((batch,), per * 16, dtype=torch.int32, device=cuda_device)
    kept = ab.paged_kv_evict(pool, pool, table, w, lens, keep=100, keep_first=4, keep_last=20)
    for now, was in zip(pool, copy) if group else [(pool, copy)]:
        for b in range(batch):
            new, old = (t[table[b].long()].transpose(0, 1).flatten(1, 2) for t in (now, was))
            for h in range(hkv):
                assert torch.equal(new[h, :100], old[h, kept[b, h].long()])
                assert torch.equal(new[h, 100:], old[h, 100:])


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("group", [0, 128])
def test_steps_with_evictions(cuda_device, group):
    """Decode steps on a cache that is cut again and again, against a float64 cache that
    is cut to the slots that the eviction named."""
    g = torch.Generator().manual_seed(11)
    B, hq, hkv, D, size, keep, slack = 2, 4, 2, 128, 16, 40, 9
    cache = ab.PagedKVCache(1, 12, size, hkv, D, dtype=torch.bfloat16, device=cuda_device, int4_group_size=group or None)
    held = [cache.add(n) for n in (keep + slack + 1,) * B]
    table = cache.page_table(held)
    kp, vp = cache.keys[0], cache.values[0]
    append = ab.paged_rope_kv_append_int4 if group else ab.paged_rope_kv_append
    attend = ab.paged_gqa_decode_attention_int4 if group else ab.paged_gqa_decode_attention
    lens = torch.tensor([30, 5], dtype=torch.int32, device=cuda_device)
    rows = torch.randn(2, B, hkv, 30, D, generator=g).to(torch.bfloat16).to(cuda_device)
    for b, n in enumerate(lens.tolist()):
        cache.store(0, held[b], rows[0, b, :, :n], rows[1, b, :, :n])
    w = torch.zeros(B, hkv, table.shape[1] * size, device=cuda_device)
    mirror = None
    cuts = 0
    for step in range(60):
        q, k, v = (torch.randn(B, 1, h, D, generator=g).to(torch.bfloat16).to(cuda_device).transpose(1, 2) for h in (hq, hkv, hkv))
        ang = torch.full((B, 1, D), 0.1 * step, device=cuda_device)
        now = torch.empty_like(lens)
        q = append(q, k, v, ang.cos(), ang.sin(), kp, vp, table, lens, kv_lens_out=now)
        kw = dict(sm_scale=D ** -0.5, num_key_value_groups=hq // hkv, kv_lens=now)
        out, lse = attend(q, kp, vp, table, return_lse=True, **kw)
        wide = [_wide(p) for p in (kp, vp)]
        tab = table.cpu().numpy()
        if mirror is None:
            mirror = [[op.gather(p, tab[b], int(now[b])) for p in wide] for b in range(B)]
        else:
            for b in range(B):
                t = int(now[b]) - 1
                mirror[b] = [np.concatenate([m, p[tab[b, t // size], :, t % size][:, None]], 1) for m, p in zip(mirror[b], wide)]
        for b in range(B):
            k64, v64 = mirror[b]
            assert k64.shape[1] == int(now[b])
            s = np.einsum("hgd,htd->hgt", _np(q)[b].reshape(hkv, -1, D).astype(np.float64), k64) * D ** -0.5
            p = np.exp(s - s.max(-1, keepdims=True))
            ref = np.einsum("hgt,htd->hgd", p / p.sum(-1, keepdims=True), v64).reshape(hq, D)
            assert (np.abs(_np(out)[b, :, 0] - ref) <= 2.0 ** -8 * np.abs(ref) + 1e-3).all()
        ab.paged_attention_weights(q, kp, table, lse, w, **kw)
        kept = ab.paged_kv_evict(kp, vp, table, w, now, keep=keep, keep_first=2, keep_last=8, longer_than=keep + slack,
                                 kv_lens_out=lens)
        for b in range(B):
            if int(now[b]) > keep + slack:
                cuts += 1
                mine = kept[b].cpu().numpy()
                mirror[b] = [np.stack([m[h, mine[h]] for h in range(hkv)]) for m in mirror[b]]
                assert int(lens[b]) == keep
            else:
                assert int(lens[b]) == int(now[b])
    assert cuts >= 5
    assert nat.device_error_flags() == 0


@pytest.mark.parametrize("group", [0, 128])
def test_two_streams_at_once(cuda_device, group):
    """Attention, weights and eviction on two streams, eager and from two graphs, many times over: the
    same bits as alone."""
    g = torch.Generator().manual_seed(21)
    B, hq, hkv, D, per = 3, 8, 4, 128, 40
    attend = ab.paged_gqa_decode_attention_int4 if group else ab.paged_gqa_decode_attention
    sets = []
    for _ in range(2):
        kp, vp = (_pages(g, B * per, hkv, 16, D, group, "bf16", cuda_device) for _ in range(2))
        table = _table(g, B, per, B * per, cuda_device)
        q = torch.randn(B, hq, 1, D, generator=g).to(torch.bfloat16).to(cuda_device)
        lens = torch.tensor([640, 17, 500], dtype=torch.int32, device=cuda_device)
        held = [t.clone() for p in (kp, vp) for t in (p if group else (p,))]
        w0 = torch.rand(B, hkv, per * 16, generator=g).to(cuda_device)
        sets.append((kp, vp, table, q, lens, held, w0))

    def run(kp, vp, table, q, lens, held, w0):
        for t, was in zip([t for p in (kp, vp) for t in (p if group else (p,))], held):
            t.copy_(was)
        w = w0.clone()
        kw = dict(sm_scale=0.09, num_key_value_groups=hq // hkv, kv_lens=lens)
        out, lse = attend(q, kp, vp, table, return_lse=True, **kw)
        ab.paged_attention_weights(q, kp, table, lse, w, **kw)
        now = torch.empty_like(lens)
        kept = ab.paged_kv_evict(kp, vp, table, w, lens, keep=200, keep_first=4, keep_last=30, kv_lens_out=now)
        after = attend(q, kp, vp, table, sm_scale=0.09, num_key_value_groups=hq // hkv, kv_lens=now)
        return out, lse, w, kept, now, after

    alone = [[t.clone() for t in run(*s)] for s in sets]
    torch.cuda.synchronize()
    streams, graphs, results = [torch.cuda.Stream() for _ in sets], [], []
    for s, stream in zip(sets, streams):
        with torch.cuda.stream(stream):
            run(*s)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                results.append(run(*s))
            graphs.append(graph)
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(results, alone):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for _ in range(5):
        eager = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                eager.append(run(*s))
        torch.cuda.synchronize()
        for got, want in zip(eager, alone):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert nat.device_error_flags() == 0
