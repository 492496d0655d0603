"""What the eviction's operators refuse before they look at a device: weights whose memory
is not what their shape says."""
from __future__ import annotations

import pytest
import torch

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
