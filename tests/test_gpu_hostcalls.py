"""The compiled calls of the short operators: they take the common call, leave
everything else to the Python operators, and either way gives the same bits."""
from __future__ import annotations

import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _hostpath as hp
from aicas_b200 import int4, paged

pytestmark = pytest.mark.gpu


@pytest.fixture
def taken(monkeypatch):
    """Counts which calls the compiled way took; ``off()`` leaves all to Python."""
    seen = []

    def watch(module, name):
        real = getattr(hp, name)

        def call(*args):
            r = real(*args)
            seen.append(r is not None)
            return r

        monkeypatch.setattr(module, name, call)

    def off():
        for module, name in ((paged, "fast_append"), (paged, "fast_decode"), (int4, "fast_int4")):
            monkeypatch.setattr(module, name, lambda *args: None)

    hp.library()
    for module, name in ((paged, "fast_append"), (paged, "fast_decode"), (int4, "fast_int4")):
        watch(module, name)
    seen_off = seen
    return seen_off, off


def _paged_state(device, batch=3, seq=5, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    st = dict(q=mk(batch, seq, 4, 64).transpose(1, 2), k=mk(batch, seq, 2, 64).transpose(1, 2),
              v=mk(batch, seq, 2, 64).transpose(1, 2), cos=mk(batch, seq, 64), sin=mk(batch, seq, 64),
              table=torch.randperm(12, generator=g).view(3, 4)[:batch].int().to(device),
              pos=torch.tensor([0, 7, 20], dtype=torch.int32)[:batch].to(device))
    st["pools"] = [torch.zeros(12, 2, 8, 64, dtype=dtype, device=device) for _ in range(2)]
    return st


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("extras", [False, True])
def test_append_and_decode_either_way(cuda_device, taken, dtype, extras):
    seen, off = taken
    out = []
    for way in range(2):
        st = _paged_state(cuda_device, dtype=dtype)
        kp, vp = st["pools"]
        kw = {}
        if extras:
            w = torch.linspace(0.5, 1.5, 64).to(dtype).to(cuda_device)
            kw = dict(num_new=torch.tensor([5, 0, 3], dtype=torch.int32, device=cuda_device), q_norm_weight=w,
                      k_norm_weight=w, eps=1e-5, q_out=torch.empty_like(st["q"]),
                      kv_lens_out=torch.empty(3, dtype=torch.int32, device=cuda_device))
        q = ab.paged_rope_kv_append(st["q"], st["k"], st["v"], st["cos"], st["sin"], kp, vp, st["table"], st["pos"], **kw)
        assert not extras or q is kw["q_out"]
        lens = torch.tensor([5, 12, 25], dtype=torch.int32, device=cuda_device)
        starts = torch.tensor([0, 3, 30], dtype=torch.int32, device=cuda_device) if extras else None
        call = dict(sm_scale=0.125, num_key_value_groups=2, kv_lens=lens, kv_starts=starts, return_lse=True)
        ab.paged_gqa_decode_attention(q[:, :, :1], kp, vp, st["table"], **call)  # the stream has its workspace after this
        o, lse = ab.paged_gqa_decode_attention(q[:, :, :1], kp, vp, st["table"], **call)
        only = ab.paged_gqa_decode_attention(q[:, :, :1], kp, vp, st["table"], **(call | {"return_lse": False}))
        out.append([q, kp, vp, o, lse, only, kw.get("kv_lens_out", lens)])
        assert q.stride() == st["q"].stride() or extras
        if way == 0:
            assert seen[0] and seen[-1] and seen[-2]
            off()
    for a, b in zip(*out):
        assert torch.equal(a, b) and a.stride() == b.stride()


@pytest.mark.parametrize("kind", ["store", "norm", "residual", "in place", "swiglu", "out"])
def test_products_either_way(cuda_device, taken, kind):
    seen, off = taken
    g = torch.Generator().manual_seed(3)
    mk = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(cuda_device)  # noqa: E731
    x, res, nw = mk(3, 256), mk(3, 96), mk(256)
    w = [ab.quantize_int4(mk(96, 256), 64, symmetric=i == 2) for i in range(3)]
    out = []
    for way in range(2):
        kw = {"norm": dict(norm_weight=nw), "residual": dict(residual=res), "swiglu": dict(swiglu=True),
              "out": dict(out=torch.empty(3, 96, dtype=torch.bfloat16, device=cuda_device))}.get(kind, {})
        if kind == "in place":
            kw["residual"] = kw["out"] = res.clone()
        y = ab.decode_linear_int4(x, w[:2] if kind == "swiglu" else w[2] if kind == "store" else w[0], **kw)
        assert "out" not in kw or y is kw["out"]
        out.append(y)
        if way == 0:
            assert seen[-1]
            off()
    assert torch.equal(*out)


def test_what_the_compiled_way_leaves_to_python(cuda_device, taken):
    seen, _ = taken
    st = _paged_state(cuda_device)
    kp, vp = st["pools"]
    base = [st[n] for n in ("q", "k", "v", "cos", "sin")]
    args = [kp, vp, st["table"], st["pos"]]
    ref = ab.paged_rope_kv_append(*base, *args)
    assert seen[-1]
    pad = torch.empty(3, 4, 5, 65, dtype=torch.bfloat16, device=cuda_device)
    pad[..., 1:] = st["q"]
    wide = torch.zeros(3, 8, dtype=torch.int32, device=cuda_device)
    wide[:, ::2] = st["table"]
    for i, other in ((0, pad[..., 1:]), (7, wide[:, ::2]), (8, [0, 7, 20])):
        changed = [*base, *args]
        changed[i] = other
        assert torch.equal(ab.paged_rope_kv_append(*changed), ref) and not seen[-1]
    with pytest.raises(ValueError):
        ab.paged_rope_kv_append(*base, kp, vp, st["table"].long(), st["pos"])
    with pytest.raises(ValueError):
        ab.paged_rope_kv_append(base[0].clone().requires_grad_(), *base[1:], *args)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 128, generator=g).to(torch.bfloat16).to(cuda_device)
    w = ab.quantize_int4(torch.randn(128, 128, generator=g).to(torch.bfloat16).to(cuda_device), 128)
    with pytest.raises(ValueError, match="overlap"):
        ab.decode_linear_int4(x, w, out=x)
    with pytest.raises(ValueError, match="at most"):
        ab.decode_linear_int4(x.repeat(20, 1), w)
    y = ab.decode_linear_int4(x, w)
    assert seen[-1]
    both = torch.empty(2, 129, dtype=torch.bfloat16, device=cuda_device)
    both[:, 1:] = x
    assert torch.equal(ab.decode_linear_int4(both[:, 1:], w), y) and not seen[-1]


def test_another_stream_and_a_graph(cuda_device, taken):
    seen, _ = taken
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, 128, generator=g).to(torch.bfloat16).to(cuda_device)
    w = ab.quantize_int4(torch.randn(64, 128, generator=g).to(torch.bfloat16).to(cuda_device), 128)
    ref = ab.decode_linear_int4(x, w)
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = ab.decode_linear_int4(x, w)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        z = ab.decode_linear_int4(x, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ref) and torch.equal(z, ref) and all(seen[1:])
