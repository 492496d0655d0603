"""Calls of the paged operators that must be refused, or answered the same way
however they are made."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aicas_b200 as ab

pytestmark = pytest.mark.gpu


def _append_args(device, batch=3, seq=2):
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=device)  # noqa: E731
    return {"query": z(batch, 4, seq, 64), "key": z(batch, 2, seq, 64), "value": z(batch, 2, seq, 64),
            "cos": torch.zeros(batch, seq, 64, device=device), "sin": torch.zeros(batch, seq, 64, device=device),
            "k_pages": z(7, 2, 16, 64), "v_pages": z(7, 2, 16, 64),
            "page_table": torch.arange(6, dtype=torch.int32, device=device).view(3, 2)[:batch],
            "positions": torch.tensor([0, 3, 9], dtype=torch.int32, device=device)[:batch]}


def test_append_refuses_lengths_over_what_it_reads(cuda_device):
    """The first token's CTA writes kv_lens_out[b] while the others' still read
    positions, num_new and the page table: no shared memory, shifted views included."""
    ok = _append_args(cuda_device)
    buf = torch.zeros(16, dtype=torch.int32, device=cuda_device)
    ab.paged_rope_kv_append(**ok, num_new=buf[:3], kv_lens_out=buf[3:6])
    assert buf[3:6].tolist() == [0, 3, 9]
    ab.paged_rope_kv_append(**(ok | {"positions": buf[6:9]}), num_new=buf[:3], kv_lens_out=buf[3:6])
    table = buf[:6].view(3, 2)
    for more in (dict(num_new=buf[:3], kv_lens_out=buf[:3]), dict(num_new=buf[:3], kv_lens_out=buf[2:5]),
                 dict(num_new=buf[2:5], kv_lens_out=buf[:3]), dict(positions=buf[:3], kv_lens_out=buf[:3]),
                 dict(positions=buf[1:4], kv_lens_out=buf[:3]), dict(positions=buf[:3], kv_lens_out=buf[2:5]),
                 dict(page_table=table, kv_lens_out=buf[5:8])):
        with pytest.raises(ValueError, match="nor share memory"):
            ab.paged_rope_kv_append(**(ok | more))
    ab.paged_rope_kv_append(**(ok | dict(page_table=table, kv_lens_out=buf[6:9])))


@pytest.mark.parametrize("batch", [1, 2])
def test_decode_returns_the_lse_for_any_true_value(cuda_device, batch):
    """Values that are true without being True, on a stream's first call and later ones."""
    ok = _append_args(cuda_device, batch, 1)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(batch, 4, 1, 64, generator=g).to(torch.bfloat16).to(cuda_device)
    kp, vp = (torch.randn(7, 2, 16, 64, generator=g).to(torch.bfloat16).to(cuda_device) for _ in range(2))
    call = lambda flag: ab.paged_gqa_decode_attention(q, kp, vp, ok["page_table"], sm_scale=0.125,  # noqa: E731
                                                      num_key_value_groups=2, return_lse=flag)
    out, lse = call(True)
    for flag in (1, np.bool_(True), "yes", torch.tensor(True)):
        for _ in range(2):
            got = call(flag)
            assert isinstance(got, tuple) and torch.equal(got[0], out) and torch.equal(got[1], lse)
    for flag in (0, np.bool_(False), None, ""):
        assert torch.equal(call(flag), out)


def test_strides_of_single_entries_mean_nothing(cuda_device):
    """A dimension of one entry may carry any stride (views, slices and transposes leave
    odd ones): batch, heads, tokens, pages and the tables of the rotation."""
    g = torch.Generator().manual_seed(3)
    mk = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(cuda_device)  # noqa: E731
    odd = lambda t, *s: torch.as_strided(t, t.shape, s)  # noqa: E731
    q, k, v = mk(1, 4, 1, 64), mk(1, 1, 1, 64), mk(1, 1, 1, 64)
    cos, sin = (torch.randn(1, 1, 64, generator=g).to(cuda_device) for _ in range(2))
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda_device)
    pos = torch.tensor([2], dtype=torch.int32, device=cuda_device)
    out = []
    for strange in (False, True):
        kp, vp = torch.zeros(2, 1, 1, 16, 64, dtype=torch.bfloat16, device=cuda_device)
        a, to = [q, k, v, cos, sin, kp, vp, table], torch.zeros_like(q)
        if strange:
            a = [odd(q, 7, 64, 1, 1), odd(k, 3, 5, 1, 1), odd(v, 1, 1, 1, 1), odd(cos, 3, 1, 1), odd(sin, 5, 7, 1),
                 odd(kp, 9, 1, 64, 1), odd(vp, 1, 3, 64, 1), odd(table, 11, 3)]
            to = odd(to, 5, 64, 3, 1)
        r = ab.paged_rope_kv_append(*a, pos, q_out=to)
        o = ab.paged_gqa_decode_attention(a[0], *a[5:], sm_scale=0.125, num_key_value_groups=4, kv_lens=[3])
        out.append([r, kp, vp, o])
    for x, y in zip(*out):
        assert torch.equal(x, y) and bool((x != 0).any())
