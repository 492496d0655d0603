"""Workspaces that a captured graph holds: later, larger calls on the same stream
and captures without a call before them."""
from __future__ import annotations

import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _native as nat
from aicas_b200 import ops

pytestmark = pytest.mark.gpu


def _contiguous(device, batch, length, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(batch, 16, 1, 128, generator=g).to(torch.bfloat16).to(device)
    k, v = (torch.randn(batch, 8, length, 128, generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    return lambda: ab.gqa_decode_attention(q, k, v, sm_scale=0.09, num_key_value_groups=2)


def _paged(device, batch, length, seed):
    g = torch.Generator().manual_seed(seed)
    per = length // 16
    q = torch.randn(batch, 16, 1, 128, generator=g).to(torch.bfloat16).to(device)
    kp, vp = (torch.randn(batch * per, 8, 16, 128, generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    table = torch.arange(batch * per, dtype=torch.int32, device=device).view(batch, per)
    return lambda: ab.paged_gqa_decode_attention(q, kp, vp, table, sm_scale=0.09, num_key_value_groups=2)


@pytest.fixture
def stream(cuda_device):
    """A stream with no workspace yet."""
    s = torch.cuda.Stream(cuda_device)
    for table in (ops._WORKSPACES, ops._LINEAR_WORKSPACES):
        table.pop((cuda_device.index, s.cuda_stream), None)
    return s


def _captured(call, stream, warm):
    stream.wait_stream(torch.cuda.current_stream())
    if warm:
        with torch.cuda.stream(stream):
            call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = call()
    return graph, out


@pytest.mark.parametrize("small", [_contiguous, _paged])
def test_a_larger_call_leaves_a_captured_workspace_alone(cuda_device, stream, small):
    """Capture a small decode, then run larger ones of both kinds on the stream and
    fill new memory: the replay still finds its workspace zeroed and its own."""
    call = small(cuda_device, 1, 4096, 1)
    want = call()
    graph, out = _captured(call, stream, True)
    with torch.cuda.stream(stream):
        for larger in (_paged(cuda_device, 8, 2048, 2), _contiguous(cuda_device, 64, 4096, 3)):
            larger()
        filled = [torch.full((1 << 20,), 255, dtype=torch.uint8, device=cuda_device) for _ in range(16)]
    torch.cuda.synchronize()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert all(bool((t == 255).all()) for t in filled) and nat.device_error_flags() == 0


@pytest.mark.parametrize("make", [_contiguous, _paged])
def test_a_capture_without_a_call_before_it(cuda_device, stream, make):
    """Its workspace is the graph's: replays and eager calls on the stream agree."""
    call = make(cuda_device, 2, 4096, 4)
    want = call()
    graph, out = _captured(call, stream, False)
    with torch.cuda.stream(stream):
        eager = call()  # before any replay has zeroed the graph's
    torch.cuda.synchronize()
    assert torch.equal(eager, want)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
