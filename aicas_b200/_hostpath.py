"""The host side of a launch for operators that run a few microseconds: what they
check and look up on every call, at the least cost torch allows.  A tensor
attribute is 40-100 ns, ``torch.cuda.current_stream`` 1.2 us and a strided view
1 us, against kernels of 2-10 us.  Calls whose arguments need nothing done to
them take the compiled ``fast_*`` way; the others the Python operators' own."""
from __future__ import annotations

import ctypes

import torch

from . import _native as nat
from .ops import _WORKSPACES, _as_lens, _workspace

try:  # the handle alone, without a Stream object around it (58 ns against 1.2 us)
    from torch._C import _cuda_getCurrentRawStream as raw_stream
except ImportError:  # pragma: no cover - torch without the binding

    def raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


# The common calls' checks and packing, compiled.  Loaded and bound with the native
# library (importing the package maps neither); until then, or where it was not
# built or was built for another torch, the Python operators do it all.
_calls = None


def fast_append(*args):
    """The compiled ``paged_rope_kv_append``; None where it leaves a call to Python."""
    return None if _calls is None else _calls.append(*args)


def fast_decode(*args):
    return None if _calls is None else _calls.decode(*args)


def fast_int4(*args):
    return None if _calls is None else _calls.int4(*args)


def fast(name: str, *args):
    """The compiled call ``name`` of 4-bit pages and eviction; None as above."""
    return None if _calls is None else getattr(_calls, name)(*args)


_bound = False


def library():
    """The native library, its entry points known to the compiled calls too."""
    global _bound, _calls
    lib = nat.lib()
    if not _bound:
        _bound = True
        try:
            from . import _hostcalls
        except ImportError:
            return lib
        _hostcalls.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
            lib.aicas_paged_rope_append, lib.aicas_paged_decode_gqa, lib.aicas_linear_int4)))
        _hostcalls.bind_int4(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
            lib.aicas_paged_append_int4, lib.aicas_paged_read_int4, lib.aicas_paged_decode_int4, lib.aicas_paged_weights,
            lib.aicas_paged_evict)))
        _calls = _hostcalls
    return lib


def steps(t: torch.Tensor) -> tuple[int, ...]:
    """The strides of a tensor, 0 for a dimension of one entry, whose stride may be
    any number and means nothing."""
    return tuple([0 if n == 1 else s for n, s in zip(t.shape, t.stride())])


def plain(t: torch.Tensor) -> torch.Tensor:
    """A copy with the strides of its shape (``contiguous`` and ``clone`` keep odd
    strides of dimensions of one entry)."""
    return t.clone(memory_format=torch.contiguous_format)


def rows_ready(t: torch.Tensor, item: int):
    """(t, its steps) for a 4-D tensor of ``item``-byte elements whose rows lie
    on 16 bytes, copying it where they do not."""
    s = steps(t)
    if s[3] != 1 or ((s[0] | s[1] | s[2]) * item | t.data_ptr()) & 15:
        t = plain(t)
        s = t.stride()
    return t, s


def heads_out(batch: int, heads: int, seq: int, dim: int, dtype: torch.dtype, device: torch.device):
    """(an uninitialised [B, H, S, D] output stored as [B, S, H, D], its strides)."""
    strides = (seq * heads * dim, dim, heads * dim, 1)
    return torch.empty_strided((batch, heads, seq, dim), strides, dtype=dtype, device=device), strides


def lengths(t, batch: int, device: torch.device) -> torch.Tensor | None:
    """An int32 [B] vector on the device, as it is or brought there."""
    if t.__class__ is torch.Tensor and t.dtype is torch.int32 and t.get_device() == device.index and t.shape == (batch,) \
            and t.is_contiguous():
        return t
    return _as_lens(t, batch, device)


def pointer(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def launch(device: torch.device, name: str, args: bytes) -> None:
    """Calls ``name(args, stream)`` on the device's current stream."""
    index = device.index
    if torch.cuda.current_device() != index:
        with torch.cuda.device(device):
            return launch(device, name, args)
    rc = getattr(library(), name)(args, raw_stream(index))
    if rc:
        nat.check(rc, name)


def launch_with_workspace(device: torch.device, name: str, bytes_name: str, args: bytes) -> None:
    """The same with the stream's zero-initialised decode workspace, enlarged when
    the call says that it is too small (so a call that fits asks nothing first)."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return launch_with_workspace(device, name, bytes_name, args)
    lib = library()
    stream = raw_stream(device.index)
    ws = _WORKSPACES.get((device.index, stream))
    if ws is not None:
        rc = getattr(lib, name)(args, ws.data_ptr(), ws.numel(), stream)
        if rc == 0:
            return
        if rc != nat.ERR_WORKSPACE:
            nat.check(rc, name)
    need = getattr(lib, bytes_name)(args)
    if need == 0:
        nat.check(nat.ERR_INVALID, name)
    ws = _workspace(device, stream, need)
    nat.check(getattr(lib, name)(args, ws.data_ptr(), ws.numel(), stream), name)
