"""The compiled calls of 4-bit pages and eviction: they take the common call, leave
everything else to the Python operators, and either way gives the same bits."""
from __future__ import annotations

import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _hostpath as hp
from aicas_b200 import eviction, paged_int4

pytestmark = pytest.mark.gpu


@pytest.fixture
def ways(monkeypatch):
    """(calls taken by the compiled way so far, a switch to Python and back)."""
    hp.library()
    seen, state = [], {"on": True}

    def fast(name, *args):
        done = hp.fast(name, *args) if state["on"] else None
        seen.append(done is not None)
        return done

    for module in (paged_int4, eviction):
        monkeypatch.setattr(module, "fast", fast)
    return seen, state


def _state(device, int4, dtype=torch.bfloat16, seq=5):
    g = torch.Generator().manual_seed(3)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    rows = [torch.randn(12, 2, 8, 128, generator=g).to(dtype) for _ in range(2)]
    pools = [ab.Int4Pages(*(t.to(device) for t in ab.quantize_kv_int4(r, 64))) if int4 else r.to(device) for r in rows]
    return dict(q=mk(3, seq, 4, 128).transpose(1, 2), k=mk(3, seq, 2, 128).transpose(1, 2),
                v=mk(3, seq, 2, 128).transpose(1, 2), cos=mk(3, seq, 128).float(), sin=mk(3, seq, 128).float(), pools=pools,
                table=torch.randperm(12, generator=g).view(3, 4).int().to(device),
                pos=torch.tensor([0, 7, 20], dtype=torch.int32, device=device),
                new=torch.tensor([5, 2, 4], dtype=torch.int32, device=device), nw=mk(128),
                lens=torch.tensor([32, 9, 0], dtype=torch.int32, device=device),
                w=torch.rand(3, 2, 40, generator=g).to(device), lse=torch.rand(3, 4, seq, generator=g).to(device))


def _append(st, **kw):
    lens = torch.zeros_like(st["pos"])
    q = ab.paged_rope_kv_append_int4(st["q"], st["k"], st["v"], st["cos"], st["sin"], *st["pools"], st["table"], st["pos"],
                                     num_new=st["new"], kv_lens_out=lens, q_norm_weight=st["nw"], **kw)
    return [q, lens, *st["pools"][0], *st["pools"][1]]


def _read(st, count=None):
    return list(ab.paged_kv_read_int4(*st["pools"], st["table"], st["pos"], 6, num_tokens=count))


def _decode(st, lens=None):
    return list(ab.paged_gqa_decode_attention_int4(st["q"][:, :, :1], *st["pools"], st["table"], sm_scale=0.1,
                                                   num_key_value_groups=2, kv_lens=st["lens"] if lens is None else lens,
                                                   kv_starts=st["new"], return_lse=True))


def _weigh(st, **kw):
    return [ab.paged_attention_weights(st["q"], st["pools"][0], st["table"], st["lse"], st["w"], sm_scale=0.1,
                                       num_key_value_groups=2, kv_lens=st["lens"], **kw)]


def _evict(st, **kw):
    out, wo = torch.zeros_like(st["lens"]), torch.zeros_like(st["w"])
    kept = ab.paged_kv_evict(*st["pools"], st["table"], st["w"], st["lens"], keep=6, keep_first=1, keep_last=2,
                             kv_lens_out=out, weights_out=wo, **kw)
    return [kept, out, wo, *(t for p in st["pools"] for t in (p if isinstance(p, tuple) else (p,)))]


CALLS = [(_append, True), (_read, True), (_decode, True), (_weigh, True), (_weigh, False), (_evict, True), (_evict, False)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("call,int4", CALLS)
def test_either_way(cuda_device, ways, call, int4, dtype):
    seen, state = ways
    got = []
    for on in (True, False):
        state["on"] = on
        st = _state(cuda_device, int4, dtype)
        if call is _decode:
            call(st)  # the first call makes the workspace
        seen.clear()
        got.append(call(st))
        assert seen == [on]
    for a, b in zip(*got):
        assert a.dtype is b.dtype and a.shape == b.shape and a.stride() == b.stride()
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_odd_arguments_are_left_to_python(cuda_device, ways):
    seen, _ = ways
    st = _state(cuda_device, True)
    want = _read(st)
    seen.clear()
    wide = torch.stack([st["table"], st["table"]], -1)
    st["table"] = wide[..., 0]  # not of unit stride
    for a, b in zip(_read(st, count=[6, 6, 6]), want):
        assert torch.equal(a, b)
    _decode(st, lens=[32, 9, 0])
    _append(st, q_out=torch.empty_like(st["q"].transpose(1, 2).contiguous()).transpose(1, 2))
    _weigh(st, kv_starts=[0, 0, 0])
    _evict(st, longer_than=10 ** 12)
    assert seen == [False] * 5
    for bad in (lambda: _evict(st, longer_than=2), lambda: _append(st, eps=-1.0)):
        with pytest.raises(ValueError):
            bad()
    st["lse"].requires_grad_()
    with pytest.raises(ValueError):
        _weigh(st)


def test_weights_that_share_memory_are_refused(cuda_device, ways):
    st = _state(cuda_device, False)
    base = torch.zeros(400, device=cuda_device)
    for strides in ((40, 40, 1), (80, 20, 1), (0, 40, 1)):
        st["w"] = base.as_strided((3, 2, 40), strides)
        with pytest.raises(ValueError):
            _weigh(st)
    for strides in ((80, 40, 1), (40, 120, 1)):
        st["w"] = base.as_strided((3, 2, 40), strides)
        _weigh(st)
