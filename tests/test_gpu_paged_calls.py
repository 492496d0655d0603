"""Calls of the paged operators that must be refused, or answered the same way
however they are made."""
from __future__ import annotations

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
