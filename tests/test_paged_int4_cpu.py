"""The paged cache's and the 4-bit products' host side, without a GPU: struct
layouts against the header, argument checks of the C entry points, the weight
format, and the refusal of CPU tensors."""
from __future__ import annotations

import ctypes
import subprocess

import numpy as np
import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _native as nat
from oracle import int4 as oi
from tests.conftest import REPO

STRUCTS = {
    "aicas_paged_append_params": (nat.PagedAppendParams, nat.PACK_PAGED_APPEND),
    "aicas_paged_decode_params": (nat.PagedDecodeParams, nat.PACK_PAGED_DECODE),
    "aicas_int4_weight": (nat.Int4WeightRef, None),
    "aicas_linear_int4_params": (nat.LinearInt4Params, nat.PACK_LINEAR_INT4),
}


def test_struct_layouts_match_the_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{REPO}/include/aicas_b200.h"', "int main(void) {"]
    for cname, (py, _) in STRUCTS.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join([*lines, "  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}
    for cname, (py, pack) in STRUCTS.items():
        assert got[(cname, "size")] == ctypes.sizeof(py)
        assert pack is None or pack.size == ctypes.sizeof(py)
        for f, _ in py._fields_:
            assert got[(cname, f)] == getattr(py, f).offset, (cname, f)


@pytest.mark.parametrize("cname", [n for n, (_, p) in STRUCTS.items() if p is not None])
def test_packed_fields_land_where_the_struct_has_them(cname):
    py, pack = STRUCTS[cname]

    def flat(cls):
        for name, kind in cls._fields_:
            if isinstance(kind, type) and issubclass(kind, ctypes.Array):
                for i in range(kind._length_):
                    yield from ((f"{name}[{i}].{n}", k) for n, k in flat(kind._type_))
            else:
                yield name, kind

    fields = list(flat(py))
    values = [i + 1 for i in range(len(fields))]
    p = py.from_buffer_copy(pack.pack(*values))
    for (name, _), v in zip(fields, values):
        assert eval(f"p.{name}", {"p": p}) == v, name


def _decode(**over):
    p = nat.PagedDecodeParams()
    base = 1 << 20  # fake, aligned; never dereferenced: validation fails first or only sizes are computed
    p.q, p.k_pages, p.v_pages, p.out, p.page_table = base, 2 * base, 3 * base, 4 * base, 5 * base
    p.batch, p.num_q_heads, p.num_kv_heads, p.head_dim = 4, 16, 8, 128
    p.num_pages, p.page_size, p.max_pages, p.table_stride = 100, 16, 20, 20
    p.dtype, p.sm_scale = nat.DTYPE_BF16, 0.1
    p.q_stride_b, p.q_stride_h, p.o_stride_b, p.o_stride_h = 2048, 128, 2048, 128
    p.kp_stride_p, p.kp_stride_h, p.kp_stride_t = 8 * 16 * 128, 16 * 128, 128
    p.vp_stride_p, p.vp_stride_h, p.vp_stride_t = 8 * 16 * 128, 16 * 128, 128
    for k, v in over.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,code,text", [
    ({"q": None}, nat.ERR_INVALID, "q and out"),
    ({"k_pages": None}, nat.ERR_INVALID, "must be set"),
    ({"page_size": 12}, nat.ERR_UNSUPPORTED, "multiple of 8"),
    ({"page_size": 0}, nat.ERR_UNSUPPORTED, "multiple of 8"),
    ({"head_dim": 96}, nat.ERR_UNSUPPORTED, "head_dim"),
    ({"num_q_heads": 12}, nat.ERR_INVALID, "not a multiple"),
    ({"dtype": 9}, nat.ERR_UNSUPPORTED, "dtype"),
    ({"max_pages": 1 << 28}, nat.ERR_UNSUPPORTED, "2^31"),
    ({"max_pages": 1 << 26, "batch": 1 << 10}, nat.ERR_UNSUPPORTED, "2^30"),
    ({"kp_stride_h": 2044}, nat.ERR_INVALID, "16 bytes"),
    ({"vp_stride_p": -128}, nat.ERR_INVALID, "16 bytes"),
    ({"k_pages": (1 << 20) + 8}, nat.ERR_INVALID, "aligned"),
    ({"o_stride_h": 4}, nat.ERR_INVALID, "q/out strides"),
    ({"sm_scale": float("nan")}, nat.ERR_INVALID, "finite"),
])
def test_paged_decode_validation(native_lib, over, code, text):
    p = _decode(**over)
    assert native_lib.aicas_paged_decode_gqa(ctypes.byref(p), None, 0, None) == code
    assert text in nat.last_error()
    assert native_lib.aicas_paged_decode_workspace_bytes(ctypes.byref(p)) == 0


def test_paged_append_validation(native_lib):
    assert native_lib.aicas_paged_rope_append(None, None) == nat.ERR_INVALID
    p = nat.PagedAppendParams()
    assert native_lib.aicas_paged_rope_append(ctypes.byref(p), None) == nat.ERR_INVALID
    base = 1 << 20
    for f in ("q_in", "q_out", "k_in", "v_in", "cos", "sin", "k_pages", "v_pages", "page_table", "positions"):
        setattr(p, f, base)
    p.batch, p.num_q_heads, p.num_kv_heads, p.seq_len, p.head_dim = 1, 4, 2, 1, 64
    p.num_pages, p.page_size, p.max_pages = 4, 16, 2
    p.dtype, p.cs_dtype = nat.DTYPE_BF16, nat.DTYPE_F16
    assert native_lib.aicas_paged_rope_append(ctypes.byref(p), None) == nat.ERR_UNSUPPORTED
    assert "cos/sin" in nat.last_error()
    p.cs_dtype, p.k_stride_s = nat.DTYPE_F32, 4
    assert native_lib.aicas_paged_rope_append(ctypes.byref(p), None) == nat.ERR_INVALID
    assert "q/k/v strides" in nat.last_error()
    p.k_stride_s, p.cs_stride_s = 64, 2
    assert native_lib.aicas_paged_rope_append(ctypes.byref(p), None) == nat.ERR_INVALID
    assert "cos/sin strides" in nat.last_error()


@pytest.mark.parametrize("over,code,text", [
    ({"rows": 33}, nat.ERR_UNSUPPORTED, "0..32 rows"),
    ({"group_size": 48}, nat.ERR_UNSUPPORTED, "group_size"),
    ({"in_features": 320}, nat.ERR_UNSUPPORTED, "multiple of group_size"),
    ({"dtype": nat.DTYPE_F32}, nat.ERR_UNSUPPORTED, "fp16 or bf16"),
    ({"mode": 7}, nat.ERR_INVALID, "mode"),
    ({"mode": nat.LINEAR_RESIDUAL}, nat.ERR_INVALID, "residual"),
    ({"mode": nat.LINEAR_SWIGLU}, nat.ERR_INVALID, "weight 1"),
    ({"x": 8}, nat.ERR_INVALID, "x must be"),
    ({"out": None}, nat.ERR_INVALID, "out must be"),
    ({"out_stride": 99}, nat.ERR_INVALID, "out_stride"),
])
def test_linear_int4_validation(native_lib, over, code, text):
    p = nat.LinearInt4Params()
    base = 1 << 20
    p.x, p.x_stride, p.out, p.out_stride = base, 512, 2 * base, 100
    p.w[0].q, p.w[0].scales, p.w[0].q_stride = 3 * base, 4 * base, 256
    p.rows, p.in_features, p.out_features, p.group_size = 2, 512, 100, 128
    p.dtype = nat.DTYPE_BF16
    for k, v in over.items():
        setattr(p, k, v)
    assert native_lib.aicas_linear_int4(ctypes.byref(p), None) == code
    assert text in nat.last_error()


def test_capability_bits(native_lib):
    assert nat.capabilities() & nat.CAP_PAGED and nat.capabilities() & nat.CAP_LINEAR_INT4


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_int4(symmetric, group, dtype):
    torch.manual_seed(group)
    w = (torch.randn(24, 256) * 0.3).to(dtype)
    w[3] = 0
    w[4] = w[4].abs()
    q = ab.quantize_int4(w, group, symmetric=symmetric)
    assert q.qweight.shape == (24, 128) and q.scales.shape == (24, 256 // group)
    assert (q.zeros is None) == symmetric and q.scales.dtype == (torch.bfloat16 if dtype == torch.float32 else dtype)
    wide = q.dequantize()
    np.testing.assert_array_equal(wide.double().numpy(),
                                  oi.widen(q.qweight.numpy(), q.scales.float().numpy(),
                                           None if symmetric else q.zeros.numpy()).astype(np.float32))
    # half a level, a whole one at the ends of the range (its top in the symmetric kind, and where
    # the 16-bit scale rounds down), and the rounding of the scale (2^-8) over 15 levels
    step = q.scales.float().repeat_interleave(group, 1)
    assert ((wide - w.float()).abs() <= 1.07 * step + 1e-12).all()
    inner = w.float().abs() < 0.5 * step * 7
    assert ((wide - w.float()).abs()[inner] <= 0.501 * step[inner] + 1e-12).all()
    assert (wide[3] == 0).all()


def test_quantize_int4_refusals():
    for bad in (torch.zeros(4), torch.zeros(4, 100), torch.zeros(4, 64, dtype=torch.int32), torch.zeros(0, 128)):
        with pytest.raises(ValueError, match="quantize_int4"):
            ab.quantize_int4(bad, 64)
    with pytest.raises(ValueError, match="group_size"):
        ab.quantize_int4(torch.zeros(4, 256), 256)


def test_operators_refuse_cpu_tensors():
    z = torch.zeros
    table = z(1, 1, dtype=torch.int32)
    pool = z(2, 2, 16, 64, dtype=torch.bfloat16)
    q = z(1, 4, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ab.paged_gqa_decode_attention(q, pool, pool, table, sm_scale=1.0, num_key_value_groups=2)
    with pytest.raises(ValueError, match="CUDA"):
        ab.paged_rope_kv_append(q, q[:, :2], q[:, :2], z(1, 1, 64), z(1, 1, 64), pool, pool, table, [0])
    w = ab.quantize_int4(torch.randn(8, 64), 32)
    with pytest.raises(ValueError, match="CUDA"):
        ab.decode_linear_int4(z(1, 64, dtype=torch.bfloat16), w)
