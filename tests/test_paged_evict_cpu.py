"""The 4-bit cache and the eviction without a GPU: the rounding of rows, the pools of
PagedKVCache, what the operators refuse, and the C ABI's own checks, which come before
anything is launched."""
from __future__ import annotations

import ctypes
import subprocess

import numpy as np
import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _native as nat
from oracle import paged_int4 as o4
from tests.conftest import REPO

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64), (128, 128)])
def test_rounding_of_rows(dtype, dim, group):
    g = torch.Generator().manual_seed(dim)
    x = torch.randn(3, 5, dim, generator=g).to(DT[dtype])
    x[0, 0], x[0, 1, 3], x[0, 2, 5], x[0, 3, dim - 1] = 2.5, 700.0, float("nan"), float("inf")
    codes, scales = ab.quantize_kv_int4(x, group)
    scale, least, code = o4.levels(x.float().numpy(), group, dtype)
    np.testing.assert_array_equal(scales[..., 0].float().numpy(), scale)
    np.testing.assert_array_equal(scales[..., 1].float().numpy(), least)
    q = o4.unpack(codes.numpy()).astype(np.float64)
    assert (np.abs(q - np.nan_to_num(code)) <= 0.5 + 2.0 ** -15).all()
    back = ab.Int4Pages(codes, scales).dequantize().numpy()
    np.testing.assert_allclose(back, o4.values(o4.unpack(codes.numpy()), scale, least), rtol=2.0 ** -22, atol=1e-6)
    fin = np.isfinite(back)
    # half a step, and what the rounding of the pair moves at the ends of the range
    step = scale.repeat(group, -1)
    unit = 2.0 ** -7 if dtype == "bf16" else 2.0 ** -10
    assert (np.abs(back - x.float().numpy())[fin] <= (step * (0.5 + 15 * unit) + unit * np.abs(least.repeat(group, -1)) + 1e-5)[fin]).all()


def test_pools_store_and_shrink():
    cache = ab.PagedKVCache(2, 6, 16, 3, 128, dtype=torch.bfloat16, device="cpu", int4_group_size=64)
    assert isinstance(cache.keys[1], ab.Int4Pages) and cache.keys[1].scales.shape == (6, 3, 16, 2, 2)
    request = cache.add(40)
    k, v = torch.randn(2, 3, 37, 128).to(torch.bfloat16)
    cache.store(1, request, k, v)
    table = cache.page_table([request])
    for pool, rows in ((cache.keys[1], k), (cache.values[1], v)):
        want = ab.quantize_kv_int4(rows, 64)
        for part, w in zip(pool, want):
            got = part[table[0].long()].transpose(0, 1).flatten(1, 2)
            assert torch.equal(got[:, :37], w)
            assert not got[:, 37:].any()
    assert not cache.keys[0].codes.any()
    with pytest.raises(ValueError):
        cache.store(1, request, k.half(), v.half())
    held = cache.pages(request)
    cache.shrink(request, 17)
    assert cache.pages(request) == held[:2] and cache.free_pages == 4
    cache.shrink(request, 60)
    assert cache.pages(request) == held[:2]
    cache.grow(request, 40)
    assert cache.pages(request) == held
    cache.shrink(request, 0)
    assert cache.pages(request) == [] and cache.free_pages == 6
    for bad in (lambda: cache.shrink(request, -1), lambda: cache.shrink(99, 1)):
        with pytest.raises(ValueError):
            bad()


def test_pools_refuse_other_groups():
    for dim, group, dtype in ((128, 32, torch.bfloat16), (64, 128, torch.bfloat16), (32, 32, torch.bfloat16),
                              (128, 64, torch.float32)):
        with pytest.raises(ValueError):
            ab.int4_pages(2, 1, 16, dim, group, dtype=dtype, device="cpu")
        with pytest.raises(ValueError):
            ab.quantize_kv_int4(torch.zeros(2, dim, dtype=dtype), group)


def test_operators_refuse_cpu_tensors():
    pool = ab.int4_pages(2, 1, 16, 64, dtype=torch.bfloat16, device="cpu")
    wide = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    table, one = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q, w = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 1, 32)
    cs = torch.zeros(1, 1, 64)
    for case in (
        lambda: ab.paged_rope_kv_append_int4(q, q[:, :1], q[:, :1], cs, cs, pool, pool, table, one),
        lambda: ab.paged_kv_read_int4(pool, pool, table, one, 1),
        lambda: ab.paged_gqa_decode_attention_int4(q, pool, pool, table, sm_scale=0.1, num_key_value_groups=2),
        lambda: ab.paged_attention_weights(q, wide, table, torch.zeros(1, 2), w, sm_scale=0.1, num_key_value_groups=2),
        lambda: ab.paged_kv_evict(wide, wide, table, w, one, keep=1),
        lambda: ab.paged_kv_evict(pool, pool, table, w, one, keep=1),
    ):
        with pytest.raises(ValueError, match="CUDA"):
            case()


# ------------------------------------------------------------------ the C ABI

STRUCTS = {
    "aicas_int4_pages": nat.Int4PagesRef,
    "aicas_paged_append_int4_params": nat.PagedAppendInt4Params,
    "aicas_paged_read_int4_params": nat.PagedReadInt4Params,
    "aicas_paged_decode_int4_params": nat.PagedDecodeInt4Params,
    "aicas_paged_weights_params": nat.PagedWeightsParams,
    "aicas_evict_plane": nat.EvictPlane,
    "aicas_paged_evict_params": nat.PagedEvictParams,
}


def test_struct_layouts_match_the_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{REPO / "include" / "aicas_b200.h"}"', "int main(void) {"]
    for name, py in STRUCTS.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    (tmp_path / "layout.c").write_text("\n".join([*lines, "  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    for line in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.splitlines():
        name, field, value = line.split()
        py = STRUCTS[name]
        assert int(value) == (ctypes.sizeof(py) if field == "size" else getattr(py, field).offset), line


BASE = 1 << 20  # fake addresses, never dereferenced: validation fails first


def _kv(p):
    for i in range(2):
        r = p.kv[i]
        r.codes, r.scales = BASE * (10 + i), BASE * (12 + i)
        r.cs_p, r.cs_h, r.cs_t, r.ss_p, r.ss_h, r.ss_t = 8 * 16 * 64, 16 * 64, 64, 8 * 16 * 4, 16 * 4, 4
    p.page_table, p.table_stride = BASE, 64
    p.batch, p.num_kv_heads, p.head_dim, p.group_size = 2, 8, 128, 64
    p.num_pages, p.page_size, p.max_pages, p.dtype = 100, 16, 64, nat.DTYPE_BF16
    return p


def _set(p, over):
    for k, v in over.items():
        obj = p
        *path, last = k.split(".")
        for part in path:
            obj = obj[int(part)] if part.isdigit() else getattr(obj, part)
        setattr(obj, last, v)
    return p


SHARED = [
    ({"kv.0.codes": None}, nat.ERR_INVALID, "codes and scales"), ({"kv.1.scales": None}, nat.ERR_INVALID, "codes and scales"),
    ({"kv.0.codes": BASE + 8}, nat.ERR_INVALID, "16-byte"), ({"kv.0.scales": BASE + 4}, nat.ERR_INVALID, "pairs"),
    ({"kv.1.cs_t": 72}, nat.ERR_INVALID, "16 bytes"), ({"kv.1.ss_t": 6}, nat.ERR_INVALID, "pairs"),
    ({"kv.0.cs_p": -16}, nat.ERR_INVALID, "non-negative"), ({"head_dim": 32, "group_size": 32}, nat.ERR_UNSUPPORTED, "head_dim"),
    ({"group_size": 32}, nat.ERR_UNSUPPORTED, "group_size"), ({"dtype": nat.DTYPE_F32}, nat.ERR_UNSUPPORTED, "fp16 or bf16"),
    ({"page_size": 12}, nat.ERR_UNSUPPORTED, "page_size"), ({"max_pages": 1 << 28}, nat.ERR_UNSUPPORTED, "2^31"),
    ({"page_table": None}, nat.ERR_INVALID, "page_table"), ({"batch": 0}, nat.ERR_INVALID, "batch=0"),
]


def _refused(rc, code, text):
    assert rc == code and text in nat.last_error(), (rc, nat.last_error())


@pytest.mark.parametrize("over, code, text", SHARED + [
    ({"num_q_heads": 12}, nat.ERR_INVALID, "not a multiple"), ({"q": BASE + 2}, nat.ERR_INVALID, "aligned"),
    ({"sm_scale": float("nan")}, nat.ERR_INVALID, "finite"), ({"q_stride_h": 4}, nat.ERR_INVALID, "16 bytes"),
    ({"batch": 1 << 20, "max_pages": 1 << 15}, nat.ERR_UNSUPPORTED, "2^30"), ({}, nat.ERR_WORKSPACE, "workspace"),
])
def test_decode_validation(native_lib, over, code, text):
    p = _kv(nat.PagedDecodeInt4Params())
    p.q, p.out, p.num_q_heads, p.sm_scale = BASE, BASE * 2, 16, 0.1
    p.q_stride_b, p.q_stride_h, p.o_stride_b, p.o_stride_h = 2048, 128, 2048, 128
    _refused(native_lib.aicas_paged_decode_int4(ctypes.byref(_set(p, over)), None, 0, None), code, text)


@pytest.mark.parametrize("over, code, text", SHARED + [
    ({"q_in": None}, nat.ERR_INVALID, "must be set"), ({"positions": None}, nat.ERR_INVALID, "must be set"),
    ({"kv_lens_out": BASE * 5}, nat.ERR_INVALID, "kv_lens_out"), ({"kv_lens_out": BASE + 64}, nat.ERR_INVALID, "kv_lens_out"),
    ({"cs_dtype": nat.DTYPE_F16}, nat.ERR_UNSUPPORTED, "cos/sin"), ({"seq_len": 0}, nat.ERR_INVALID, "seq_len"),
    ({"num_q_heads": 0}, nat.ERR_INVALID, "num_q_heads"), ({"k_stride_s": 4}, nat.ERR_INVALID, "16 bytes"),
    ({"q_norm_weight": BASE * 7, "norm_eps": -1.0}, nat.ERR_INVALID, "eps"),
])
def test_append_validation(native_lib, over, code, text):
    p = _kv(nat.PagedAppendInt4Params())
    p.q_in = p.q_out = p.k_in = p.v_in = p.cos = p.sin = BASE * 4
    p.positions, p.num_q_heads, p.seq_len, p.cs_dtype = BASE * 5, 16, 1, nat.DTYPE_F32
    for f, _ in p._fields_:
        if "_stride_" in f:
            setattr(p, f, 128)
    _refused(native_lib.aicas_paged_append_int4(ctypes.byref(_set(p, over)), None), code, text)


@pytest.mark.parametrize("over, code, text", SHARED + [
    ({"positions": None}, nat.ERR_INVALID, "positions"), ({"seq_len": 0}, nat.ERR_INVALID, "seq_len"),
    ({"out_stride_h": 4}, nat.ERR_INVALID, "16 bytes"),
])
def test_read_validation(native_lib, over, code, text):
    p = _kv(nat.PagedReadInt4Params())
    p.out[0] = p.out[1] = BASE * 2
    p.positions, p.seq_len, p.out_stride_b, p.out_stride_h, p.out_stride_s = BASE * 3, 4, 4096, 512, 128
    _refused(native_lib.aicas_paged_read_int4(ctypes.byref(_set(p, over)), None), code, text)


@pytest.mark.parametrize("over, code, text", [
    ({"lse": None}, nat.ERR_INVALID, "must be set"), ({"k_scales": None, "group_size": 64}, nat.ERR_INVALID, "codes and scales"),
    ({"dtype": 9}, nat.ERR_UNSUPPORTED, "dtype"), ({"head_dim": 96}, nat.ERR_UNSUPPORTED, "head_dim"),
    ({"head_dim": 32, "group_size": 32}, nat.ERR_UNSUPPORTED, "head_dim"), ({"kp_stride_t": 4}, nat.ERR_INVALID, "page strides"),
    ({"k_pages": BASE + 8}, nat.ERR_INVALID, "16-byte"), ({"seq_len": 0}, nat.ERR_INVALID, "seq_len"),
    ({"w_stride_b": -1}, nat.ERR_INVALID, "negative"), ({"weights": BASE + 2}, nat.ERR_INVALID, "4-byte"),
    ({"sm_scale": float("inf")}, nat.ERR_INVALID, "finite"), ({"num_q_heads": 9}, nat.ERR_INVALID, "not a multiple"),
    ({"batch": 1 << 20, "max_pages": 1 << 15}, nat.ERR_UNSUPPORTED, "2^30"),
])
def test_weights_validation(native_lib, over, code, text):
    p = nat.PagedWeightsParams()
    p.q, p.k_pages, p.lse, p.weights, p.page_table, p.table_stride = BASE, BASE * 2, BASE * 3, BASE * 4, BASE * 5, 64
    p.q_stride_b, p.q_stride_h, p.q_stride_s = 2048, 128, 128
    p.kp_stride_p, p.kp_stride_h, p.kp_stride_t = 8 * 16 * 128, 16 * 128, 128
    p.batch, p.num_q_heads, p.num_kv_heads, p.seq_len, p.head_dim = 2, 16, 8, 1, 128
    p.num_pages, p.page_size, p.max_pages, p.dtype, p.sm_scale = 100, 16, 64, nat.DTYPE_BF16, 0.1
    _refused(native_lib.aicas_paged_weights(ctypes.byref(_set(p, over)), None), code, text)


@pytest.mark.parametrize("over, code, text", [
    ({"weights": None}, nat.ERR_INVALID, "must be set"), ({"kept": None}, nat.ERR_INVALID, "must be set"),
    ({"num_planes": 0}, nat.ERR_INVALID, "num_planes"), ({"num_planes": 5}, nat.ERR_INVALID, "num_planes"),
    ({"plane.1.data": None}, nat.ERR_INVALID, "plane"), ({"plane.0.row_bytes": 12}, nat.ERR_INVALID, "rows"),
    ({"plane.0.row_bytes": 144}, nat.ERR_INVALID, "rows"), ({"plane.0.row_bytes": 1024}, nat.ERR_INVALID, "rows"),
    ({"plane.0.data": BASE + 4}, nat.ERR_INVALID, "aligned"), ({"plane.1.stride_t": 8}, nat.ERR_INVALID, "strides"),
    ({"keep": 0}, nat.ERR_INVALID, "keep"), ({"keep_first": 60, "keep_last": 50}, nat.ERR_INVALID, "keep"),
    ({"longer_than": 99}, nat.ERR_INVALID, "longer_than"), ({"keep_last": -1}, nat.ERR_INVALID, "keep"),
    ({"kv_lens_out": BASE * 6 + 4}, nat.ERR_INVALID, "kv_lens_out"), ({"kv_lens_out": BASE * 5}, nat.ERR_INVALID, "kv_lens_out"),
    ({"wo_stride_h": -4}, nat.ERR_INVALID, "negative"), ({"page_size": 20}, nat.ERR_UNSUPPORTED, "page_size"),
])
def test_evict_validation(native_lib, over, code, text):
    p = nat.PagedEvictParams()
    for i in range(2):
        pl = p.plane[i]
        pl.data, pl.stride_p, pl.stride_h, pl.stride_t, pl.row_bytes = BASE * (8 + i), 8 * 16 * 256, 16 * 256, 256, 256
    p.num_planes, p.weights, p.weights_out, p.kept, p.page_table, p.kv_lens = 2, BASE, BASE * 2, BASE * 3, BASE * 5, BASE * 6
    p.w_stride_b, p.w_stride_h, p.wo_stride_b, p.wo_stride_h, p.table_stride = 8192, 1024, 8192, 1024, 64
    p.batch, p.num_kv_heads, p.num_pages, p.page_size, p.max_pages = 2, 8, 100, 16, 64
    p.keep, p.keep_first, p.keep_last, p.longer_than = 100, 4, 20, 100
    _refused(native_lib.aicas_paged_evict(ctypes.byref(_set(p, over)), None), code, text)
