"""Calls of the 4-bit products that must be refused, or answered the same way
however they are made."""
from __future__ import annotations

import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _hostpath as hp

pytestmark = pytest.mark.gpu


def _call_args(device, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(device)  # noqa: E731
    return mk(2, 256), [ab.quantize_int4(mk(96, 256), 64) for _ in range(2)], mk(256), mk(2, 96)


def test_every_tensor_that_needs_a_gradient_is_refused(cuda_device):
    """With grad enabled; under no_grad the same tensors go the compiled way."""
    x, w, nw, res = _call_args(cuda_device)
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    lw = w[0]._replace(scales=leaf(w[0].scales))
    first = ab.decode_linear_int4(x, w[0])  # the compiled calls are bound after this
    calls = [(leaf(x), w[0], {}), (x, w[0], {"norm_weight": leaf(nw)}), (x, w[0], {"residual": leaf(res)}), (x, lw, {}),
             (x, (w[0], lw), {"swiglu": True}), (x, (lw, w[0]), {"swiglu": True})]
    for xx, ww, kw in calls:
        with pytest.raises(ValueError, match="inference"):
            ab.decode_linear_int4(xx, ww, **kw)
    for xx, ww, kw in calls:
        plain = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
        pw = tuple(w[0] for _ in ww) if "swiglu" in kw else w[0]
        want = ab.decode_linear_int4(x, pw, **plain)
        with torch.no_grad():
            assert torch.equal(ab.decode_linear_int4(xx, ww, **kw), want)
            assert hp._calls is None or hp.fast_int4(xx, ww, kw.get("norm_weight"), 1e-6, kw.get("residual"),
                                                     kw.get("swiglu", False), None) is not None
    assert torch.equal(ab.decode_linear_int4(x, w[0]), first)


def test_strides_of_single_entries_mean_nothing(cuda_device):
    """One row of x, one output feature: whatever the stride of that dimension."""
    x, w, nw, res = _call_args(cuda_device)
    want = ab.decode_linear_int4(x[:1], w[0], norm_weight=nw, residual=res[:1])
    for stride in (1, 3, 256, 999):
        row = torch.as_strided(x, (1, 256), (stride, 1))
        got = ab.decode_linear_int4(row, w[0], norm_weight=nw, residual=torch.as_strided(res, (1, 96), (stride, 1)),
                                    out=torch.as_strided(torch.empty_like(want), (1, 96), (stride, 1)))
        assert torch.equal(got, want)
    first = ab.Int4Weight(w[0].qweight[:1], w[0].scales[:1], w[0].zeros[:1])
    one = ab.decode_linear_int4(x, first)
    for stride in (1, 5, 48):
        odd = first._replace(qweight=torch.as_strided(first.qweight, (1, 128), (stride, 1)))
        assert torch.equal(ab.decode_linear_int4(x, odd), one)
