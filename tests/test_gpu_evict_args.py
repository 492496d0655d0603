"""Arguments of the eviction's operators at their edges: refused, or taken as they are meant, on the compiled way
and in Python."""
from __future__ import annotations

import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _hostpath as hp
from aicas_b200 import eviction

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["compiled", "python"])
def way(request, monkeypatch):
    hp.library()
    if request.param == "python":
        monkeypatch.setattr(eviction, "fast", lambda *args: None)


def _state(device, B=2, hkv=2, per=4):
    g = torch.Generator().manual_seed(0)
    kp, vp = (torch.randn(B * per, hkv, 16, 64, generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    table = torch.arange(B * per, dtype=torch.int32, device=device).view(B, per)
    w = torch.rand(B, hkv, per * 16, generator=g).to(device)
    lens = torch.full((B,), per * 16, dtype=torch.int32, device=device)
    return kp, vp, table, w, lens


@pytest.mark.parametrize("first,last", [(2 ** 62, 2 ** 62), (2 ** 63 - 1, 2 ** 63 - 1), (2 ** 63 - 1, 1), (2 ** 62, 0), (0, 2 ** 63 - 1),
                                        (2 ** 32, 0), (2 ** 70, 0)])
def test_counts_whose_sum_overflows_are_refused(cuda_device, way, first, last):
    kp, vp, table, w, lens = _state(cuda_device)
    before = [t.clone() for t in (kp, vp, w)]
    with pytest.raises(ValueError, match="keep"):
        ab.paged_kv_evict(kp, vp, table, w, lens, keep=20, keep_first=first, keep_last=last)
    assert all(torch.equal(a, b) for a, b in zip((kp, vp, w), before))


@pytest.mark.parametrize("B,hkv", [(2, 2), (1, 1), (1, 3)])
def test_weights_of_one_buffer_in_turn(cuda_device, way, B, hkv):
    """Two halves of one buffer share no element: one may receive what the other becomes."""
    kp, vp, table, w, lens = _state(cuda_device, B, hkv)
    both = torch.full((2, B, hkv, 64), -5.0, device=cuda_device)
    both[0] = w
    pools = [(kp.clone(), vp.clone()) for _ in range(3)]
    apart = torch.full_like(w, -5.0)
    want = ab.paged_kv_evict(*pools[0], table, w, lens, keep=20, keep_last=3, weights_out=apart)
    got = ab.paged_kv_evict(*pools[1], table, both[0], lens, keep=20, keep_last=3, weights_out=both[1])
    assert torch.equal(got, want) and torch.equal(both[1], apart) and torch.equal(both[0], w)
    both[1], both[0] = w, -5.0
    got = ab.paged_kv_evict(*pools[2], table, both[1], lens, keep=20, keep_last=3, weights_out=both[0])
    assert torch.equal(got, want) and torch.equal(both[0], apart)
    for other in pools[1:]:
        assert all(torch.equal(a, b) for a, b in zip(other, pools[0]))
    flat = both.view(-1)
    n = B * hkv * 64
    for shift in (1, 16, n - 1):
        with pytest.raises(ValueError, match="weights_out"):
            ab.paged_kv_evict(kp, vp, table, both[0], lens, keep=20, weights_out=flat[shift:shift + n].view(B, hkv, 64))


def test_weights_out_that_needs_a_gradient_is_refused(cuda_device, way):
    kp, vp, table, w, lens = _state(cuda_device)
    out = torch.zeros_like(w).requires_grad_()
    with pytest.raises(ValueError):
        ab.paged_kv_evict(kp, vp, table, w, lens, keep=20, weights_out=out)
    assert not out.any()
    with torch.no_grad():
        ab.paged_kv_evict(kp, vp, table, w, lens, keep=20, weights_out=out)
    assert out[..., :20].all() and not out[..., 20:].any()
