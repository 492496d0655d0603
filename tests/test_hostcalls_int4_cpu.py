"""The compiled calls of 4-bit pages and eviction without a GPU: what is not on a GPU, and
calls of another form, are left to Python."""
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
    pool = ab.int4_pages(2, 1, 8, 64, dtype=torch.bfloat16, device="cpu")
    wide = torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16)
    table, one = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q, cs, w = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 1, 64), torch.zeros(1, 1, 16)
    k = q[:, :1]
    for bound in (0, 4096):  # an address that is never called: the arguments are refused first
        calls.bind_int4(*[bound] * 5)
        assert calls.append_int4(q, k, k, cs, cs, pool, pool, table, one, None, None, None, None, None, 1e-6) is None
        assert calls.read_int4(pool, pool, table, one, 1, None) is None
        assert calls.decode_int4(q, pool, pool, table, 0.1, 2, None, None, False, {}) is None
        for pages in (pool, wide, None, (pool.codes,), "x"):
            assert calls.weigh(q, pages, table, torch.zeros(1, 2), w, 0.1, 2, None, None) is None
            assert calls.evict(pages, pages, table, w, one, 4, 0, 0, None, None, None) is None
        assert calls.evict(wide, wide, table, w, one, "a", 0, 0, None, None, None) is None
        assert calls.read_int4(pool, pool, table, one, 1.5, None) is None
        for name in ("append_int4", "read_int4", "decode_int4", "weigh", "evict"):
            assert getattr(calls, name)() is None
    calls.bind_int4(*[0] * 5)


def test_bind_refuses_what_is_not_five_addresses(calls):
    for args in ((1, 2, 3), ("a",) * 5, ()):
        with pytest.raises(TypeError):
            calls.bind_int4(*args)
