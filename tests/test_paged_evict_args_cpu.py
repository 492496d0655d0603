"""What the eviction's operators refuse before they look at a device: weights whose memory
is not what their shape says."""
from __future__ import annotations

import ctypes

import pytest
import torch

from aicas_b200 import _native as nat
from aicas_b200.eviction import _check_weights


def _check(w, slots):
    return _check_weights("op", "weights", w, w.shape[0], w.shape[1], slots, -1)  # -1: the "device" of CPU tensors


@pytest.mark.parametrize("shape", [(1, 1), (1, 3), (2, 1), (2, 3)])
def test_weights_expanded_over_slots_are_refused(shape):
    """One number behind every slot: a kernel that takes slots as neighbours would write past it."""
    for w in (torch.zeros(*shape, 1).expand(*shape, 32), torch.zeros(*shape, 64)[..., ::2],
              torch.zeros(1).expand(*shape, 32)):
        with pytest.raises(ValueError, match="contiguous slots"):
            _check(w, 32)


@pytest.mark.parametrize("shape", [(1, 1), (1, 3), (2, 1), (2, 3)])
def test_weights_of_contiguous_slots_are_taken(shape):
    b, h = shape
    step = lambda n, s: s if n > 1 else 0  # noqa: E731
    assert _check(torch.zeros(b, h, 32), 32) == (step(b, 32 * h), step(h, 32))
    assert _check(torch.zeros(b, h, 40)[..., 4:37], 32) == (step(b, 40 * h), step(h, 40))
    assert _check(torch.zeros(h, b, 32).transpose(0, 1), 32) == (step(b, 32), step(h, 32 * b))
    odd = torch.zeros(32).as_strided((1, 1, 32), (7, 5, 1))
    assert _check(odd, 32) == (0, 0)


@pytest.mark.parametrize("at,strides,taken", [
    (0, (4096, 512), True), (2 * 4096, (4096, 512), True), (-2 * 4096, (4096, 512), True),  # in place, behind, before
    (64, (4096, 512), False), (2 * 4096 - 1, (4096, 512), False), (1 - 2 * 4096, (4096, 512), False), (0, (4096, 256), False),
    (256, (4096, 512), False)])
def test_weights_out_of_the_c_entry(native_lib, at, strides, taken):
    """The entry's checks come before any launch: what passes this one fails at the lengths' own."""
    p = nat.PagedEvictParams()
    base = 1 << 20  # fake addresses, never dereferenced
    pl = p.plane[0]
    pl.data, pl.stride_p, pl.stride_h, pl.stride_t, pl.row_bytes = base * 8, 8 * 16 * 256, 16 * 256, 256, 256
    p.num_planes, p.weights, p.weights_out, p.kept, p.page_table = 1, base * 2, base * 2 + 4 * at, base * 3, base * 5
    p.kv_lens, p.kv_lens_out = base * 6, base * 6 + 4  # refused, last of all
    p.w_stride_b, p.w_stride_h, p.wo_stride_b, p.wo_stride_h, p.table_stride = 4096, 512, *strides, 64
    p.batch, p.num_kv_heads, p.num_pages, p.page_size, p.max_pages = 2, 8, 100, 16, 32
    p.keep, p.longer_than = 100, 100
    assert native_lib.aicas_paged_evict(ctypes.byref(p), None) == nat.ERR_INVALID
    assert ("kv_lens_out" if taken else "weights_out") in nat.last_error()


@pytest.mark.parametrize("batch,heads,max_pages,taken", [(1 << 24, 8, 1, False), (14_000_000, 8, 1, False), (12_000_000, 8, 1, True), (1 << 16, 8, 128, True),
                                                         (1 << 16, 8, 4096, False)])
def test_pairs_whose_units_exceed_32_bits_are_refused(native_lib, batch, heads, max_pages, taken):
    """Pairs of few tiles count by what beginning and ending them costs (8 tiles of a block of warps)."""
    p = nat.PagedWeightsParams()
    base = 1 << 20  # fake addresses, never dereferenced
    p.q, p.k_pages, p.lse, p.weights, p.page_table, p.table_stride = base, base * 2, base * 3, base * 4, base * 5, 0
    p.q_stride_b, p.q_stride_h, p.q_stride_s = 2048, 128, 128
    p.kp_stride_p, p.kp_stride_h, p.kp_stride_t = 8 * 8 * 128, 8 * 128, 128
    p.batch, p.num_q_heads, p.num_kv_heads, p.seq_len, p.head_dim = batch, 2 * heads, heads, 9, 128
    p.num_pages, p.page_size, p.max_pages, p.dtype = 100, 8, max_pages, nat.DTYPE_BF16
    p.sm_scale = float("inf")  # refused, last of all
    assert native_lib.aicas_paged_weights(ctypes.byref(p), None) == (nat.ERR_INVALID if taken else nat.ERR_UNSUPPORTED)
    assert ("finite" if taken else "2^30") in nat.last_error()
