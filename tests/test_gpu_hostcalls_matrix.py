"""The compiled calls against the Python operators over odd arguments of every
kind: the same result, or the same refusal, whichever way a call goes."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _hostpath as hp

pytestmark = pytest.mark.gpu

ODD = [None, True, False, 0, 1, 2, -1, 2.0, 0.5, float("nan"), float("inf"), "2", np.float32(0.25), np.int64(2),
       np.bool_(True), [1, 2], (3, 4), []]


def _tensors(device):
    """Tensors that are wrong somewhere for most arguments, and right for a few."""
    g = torch.Generator().manual_seed(0)
    mk = lambda *s, dt=torch.bfloat16: torch.randn(*s, generator=g).to(dt).to(device)  # noqa: E731
    full = mk(2, 4, 2, 64)
    return [full, full.cpu(), full.float(), full.half(), full[:1], full[:, :2], full[..., :32], full.transpose(1, 2),
            mk(2, 2, 4, 64).transpose(1, 2), mk(2, 4, 2, 128)[..., ::2], mk(2, 4, 2, 72)[..., 4:68], full.clone().requires_grad_(),
            torch.nn.Parameter(full.clone()), mk(2, 2, 2, 64), mk(2, 2, 64), mk(2, 2, 64, dt=torch.float32), mk(1, 2, 64),
            mk(64), mk(64, dt=torch.float32), mk(65)[1:], mk(128)[::2], mk(5, 2, 16, 64), mk(5, 2, 24, 64), mk(5, 2, 12, 64),
            mk(5, 16, 2, 64).transpose(1, 2), torch.zeros(2, dtype=torch.int32, device=device),
            torch.tensor([3, 40], dtype=torch.int32, device=device), torch.tensor([3, 9], dtype=torch.int64, device=device),
            torch.tensor([1, 2], dtype=torch.int32), torch.zeros(3, dtype=torch.int32, device=device),
            torch.zeros(4, dtype=torch.int32, device=device)[::2], torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=device),
            torch.tensor([[0, 1], [2, 3]], dtype=torch.int64, device=device), torch.zeros(2, 0, dtype=torch.int32, device=device),
            mk(2, 64), mk(2, 96), mk(2, 72)[:, :64], mk(2, 72)[:, 4:68], mk(64, 2).t(), mk(1, 64).expand(2, 64), mk(33, 64),
            mk(0, 64), mk(2, 64, dt=torch.float16), mk(1, 96).expand(2, 96), mk(96, 2).t()]


def _outcome(call, args, kwargs, written):
    """What a call returns or raises, and what it leaves in ``written``."""
    kept = [t.clone() for t in written]
    try:
        made = call(*args, **kwargs)
    except Exception as e:  # noqa: BLE001 - every kind is compared
        return type(e), str(e)
    finally:
        for t, k in zip(written, kept):
            now, _ = t.clone(), t.copy_(k)
            k.copy_(now)
    tensors = [*(made if isinstance(made, tuple) else (made,)), *kept]
    return type(made), [(tuple(t.shape), t.stride() if i == 0 else None, t.dtype, t.detach().float().cpu()) for i, t in
                        enumerate(tensors)]


def _same(a, b):
    if a[0] is not b[0] or not isinstance(a[1], list):
        return a == b
    return len(a[1]) == len(b[1]) and all(x[:3] == y[:3] and torch.equal(x[3].nan_to_num(7.0), y[3].nan_to_num(7.0))
                                          for x, y in zip(a[1], b[1]))


def _both_ways(monkeypatch, call, args, kwargs, written=()):
    first = _outcome(call, args, kwargs, written)
    with monkeypatch.context() as m:
        m.setattr(hp, "_calls", None)
        second = _outcome(call, args, kwargs, written)
    assert _same(first, second), (first, second)
    return isinstance(first[1], list)


def _sweep(monkeypatch, call, good, written, device, names):
    assert _both_ways(monkeypatch, call, (), good, written)
    taken = 0
    for name in names:
        for value in ODD + _tensors(device):
            taken += _both_ways(monkeypatch, call, (), good | {name: value}, written)
    return taken


def test_append(cuda_device, monkeypatch):
    hp.library()
    t = _tensors(cuda_device)
    pools = [torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16, device=cuda_device) for _ in range(2)]
    good = dict(query=t[0], key=t[13], value=t[13].clone(), cos=t[14], sin=t[14].clone(), k_pages=pools[0], v_pages=pools[1],
                page_table=t[31], positions=t[26])
    with torch.no_grad():
        assert _sweep(monkeypatch, ab.paged_rope_kv_append, good, pools, cuda_device, [
            *good, "num_new", "q_norm_weight", "k_norm_weight", "eps", "q_out", "kv_lens_out"]) > 0
    assert _sweep(monkeypatch, ab.paged_rope_kv_append, good, pools, cuda_device, ["query", "key", "value", "cos"]) > 0


def test_decode(cuda_device, monkeypatch):
    t = _tensors(cuda_device)
    good = dict(query=t[0][:, :, :1], k_pages=t[21], v_pages=t[21].clone(), page_table=t[31], sm_scale=0.125,
                num_key_value_groups=2)
    ab.paged_gqa_decode_attention(**good)  # the stream has its workspace after this
    assert _sweep(monkeypatch, ab.paged_gqa_decode_attention, good, (), cuda_device,
                  [*good, "kv_lens", "kv_starts", "return_lse"]) > 0


def test_products(cuda_device, monkeypatch):
    hp.library()
    t = _tensors(cuda_device)
    w = [ab.quantize_int4(torch.randn(96, 64).to(torch.bfloat16).to(cuda_device), 32) for _ in range(2)]
    x = t[34]
    names = ["x", "norm_weight", "eps", "residual", "swiglu", "out"]
    assert _sweep(monkeypatch, ab.decode_linear_int4, dict(x=x, weight=w[0]), (), cuda_device, names) > 0
    assert _sweep(monkeypatch, ab.decode_linear_int4, dict(x=x, weight=w[0], norm_weight=t[17], residual=t[35]), (),
                  cuda_device, names) > 0
    assert _sweep(monkeypatch, ab.decode_linear_int4, dict(x=x, weight=w, swiglu=True), (), cuda_device, names) > 0
    for field in ("qweight", "scales", "zeros"):
        of = getattr(w[0], field)
        for value in [None, of.cpu(), of.int(), of.half(), of[:90], of[:, :1], of.t(), of.t().contiguous().t(), of.clone(),
                      torch.cat([of, of], 1)[:, :of.shape[1]], torch.cat([of, of], 1)[:, 1:1 + of.shape[1]], of.flatten()]:
            odd = w[0]._replace(**{field: value})
            _both_ways(monkeypatch, ab.decode_linear_int4, (x, odd), {})
            for pair in ((odd, w[1]), [w[1], odd], (odd, odd)):
                _both_ways(monkeypatch, ab.decode_linear_int4, (x, pair), {"swiglu": True})
