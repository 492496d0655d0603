"""The compiled calls of the short operators without a GPU: they build with the
package, and leave tensors that are not on a GPU, and calls of another form, to Python."""
from __future__ import annotations

import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import build


@pytest.fixture(scope="module")
def calls():
    build.build_hostcalls()
    from aicas_b200 import _hostcalls

    return _hostcalls


def test_cpu_tensors_and_odd_calls_are_left_to_python(calls):
    calls.bind(0, 0, 0)
    x, w = torch.zeros(1, 64, dtype=torch.bfloat16), ab.quantize_int4(torch.randn(8, 64), 32)
    for bound in (0, 4096):  # an address that is never called: the arguments are refused first
        calls.bind(bound, bound, bound)
        assert calls.int4(x, w, None, 1e-6, None, False, None) is None
        assert calls.int4(x, (w, w), None, 1e-6, None, True, None) is None
        assert calls.int4("x", w, None, 1e-6, None, False, None) is None
        assert calls.int4() is None and calls.append() is None and calls.decode() is None
        q = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
        pages, table = torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32)
        assert calls.decode(q, pages, pages, table, 0.1, 2, None, None, False, {}) is None
        cs, pos = torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int32)
        k = q[:, :1]
        assert calls.append(q, k, k, cs, cs, pages, pages, table, pos, None, None, None, None, None, 1e-6) is None
    calls.bind(0, 0, 0)


def test_bind_refuses_what_is_not_three_addresses(calls):
    with pytest.raises(TypeError):
        calls.bind(1, 2)
    with pytest.raises(TypeError):
        calls.bind("a", "b", "c")


def test_the_operators_still_refuse_cpu_tensors():
    w = ab.quantize_int4(torch.randn(8, 64), 32)
    with pytest.raises(ValueError, match="CUDA"):
        ab.decode_linear_int4(torch.zeros(1, 64, dtype=torch.bfloat16), w)
