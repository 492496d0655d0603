"""The compiled calls launch without the interpreter's lock."""
from __future__ import annotations

import ctypes

import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _hostpath as hp
from aicas_b200 import _native as nat

pytestmark = pytest.mark.gpu


def test_launches_release_the_interpreter_lock(cuda_device):
    """In the place of an entry point PyGILState_Check: its 1, the lock is held, is
    an error, for which a compiled call returns None; its 0 is success."""
    from aicas_b200 import _hostcalls as calls

    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=cuda_device)  # noqa: E731
    q, kv, pages = z(1, 4, 1, 64), z(1, 2, 1, 64), z(3, 2, 16, 64)
    cs = torch.zeros(1, 1, 64, device=cuda_device)
    table, pos = (torch.zeros(*s, dtype=torch.int32, device=cuda_device) for s in ((1, 2), (1,)))
    w = ab.quantize_int4(torch.ones(8, 64, dtype=torch.bfloat16, device=cuda_device), 32)
    stream = torch.cuda.current_stream().cuda_stream
    spaces = {(cuda_device.index, stream): torch.zeros(1 << 23, dtype=torch.uint8, device=cuda_device)}
    hp.library()
    real = [ctypes.cast(f, ctypes.c_void_p).value for f in (
        nat.lib().aicas_paged_rope_append, nat.lib().aicas_paged_decode_gqa, nat.lib().aicas_linear_int4)]
    held = ctypes.cast(ctypes.pythonapi.PyGILState_Check, ctypes.c_void_p).value
    try:
        calls.bind(held, held, held)
        done = [calls.append(q, kv, kv, cs, cs, pages, pages, table, pos, None, None, None, None, None, 1e-6),
                calls.decode(q, pages, pages, table, 0.1, 2, None, None, False, spaces),
                calls.int4(z(1, 64), w, None, 1e-6, None, False, None)]
    finally:
        calls.bind(*real)
    assert all(isinstance(t, torch.Tensor) for t in done), [type(t) for t in done]
