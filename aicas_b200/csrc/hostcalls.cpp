// The host side of the short operators' launches: what paged.py and int4.py check
// and pack, for arguments that need nothing done to them.  Each function returns
// the result, or None where anything is other than the kernels take it as it is
// (a copy to make, a workspace to enlarge, an error to report): the Python
// operator then does the whole of its own checks.  So this file decides nothing
// by itself; it only makes the common call cheap.  A tensor attribute read from
// Python is 40-100 ns and a call reads 40 to 90 of them, against kernels of 2-10 us:
// an append of one token 17 us a call through Python, an attention 15, a product 12.
#include <Python.h>

#include <cstring>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty_strided.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include "aicas_b200.h"

namespace {

using at::Tensor;

decltype(&aicas_paged_rope_append) g_append = nullptr;
decltype(&aicas_paged_decode_gqa) g_decode = nullptr;
decltype(&aicas_linear_int4) g_int4 = nullptr;

PyObject* none() { Py_RETURN_NONE; }

// A launch without the GIL: one into a full queue waits for the GPU.
template <typename F, typename... Args>
int launch(F* entry, Args... args) {
  PyThreadState* const thread = PyEval_SaveThread();
  const int rc = entry(args...);
  PyEval_RestoreThread(thread);
  return rc;
}

// A plain tensor (or parameter), else null.
const Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

// An optional one: false where it is neither None nor a plain tensor.
bool optional(PyObject* o, const Tensor** t) {
  *t = o == Py_None ? nullptr : tensor(o);
  return o == Py_None || *t != nullptr;
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return AICAS_DTYPE_F32;
    case at::kHalf: return AICAS_DTYPE_F16;
    case at::kBFloat16: return AICAS_DTYPE_BF16;
    default: return -1;
  }
}

bool same(const Tensor& t, const Tensor& like) {
  return t.is_cuda() && t.get_device() == like.get_device() && t.scalar_type() == like.scalar_type();
}

// Autograd would have to follow one of them: the operators refuse that.
template <typename... Ts>
bool recorded(const Ts*... t) {
  return c10::GradMode::is_enabled() && ((t != nullptr && t->requires_grad()) || ...);
}

bool shaped(const Tensor& t, at::IntArrayRef shape) { return t.sizes() == shape; }

// [B, H, S, D] (or fewer dimensions) of unit-stride rows that lie on 16 bytes.
bool rows_ready(const Tensor& t) {
  const auto s = t.strides();
  int64_t bits = 0;
  for (size_t i = 0; i + 1 < s.size(); ++i) bits |= s[i] * (int64_t)t.element_size();
  return s.back() == 1 && ((bits | (int64_t)reinterpret_cast<uintptr_t>(t.data_ptr())) & 15) == 0;
}

// A contiguous int32 [n] vector on the device of `like`.
bool vector32(const Tensor& t, int64_t n, const Tensor& like) {
  return t.is_cuda() && t.get_device() == like.get_device() && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n &&
         t.is_contiguous();
}

template <typename P>
P pointer(const Tensor* t) {
  return t == nullptr ? nullptr : static_cast<P>(t->data_ptr());
}

// The pools and the page table as paged.py's _check_pool takes them.
bool pool_ok(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table) {
  if (!q.is_cuda() || q.dim() != 4 || k.dim() != 4 || dtype_code(q) < 0 || !same(k, q) || !same(v, q)) return false;
  const int64_t d = q.size(3);
  return v.sizes() == k.sizes() && k.size(3) == d && (d == 16 || d == 32 || d == 64 || d == 128) && k.size(2) >= 8 &&
         k.size(2) % 8 == 0 && k.stride(3) == 1 && v.stride(3) == 1 && k.size(0) <= INT32_MAX && k.size(2) <= INT32_MAX &&
         table.is_cuda() && table.get_device() == q.get_device() && table.scalar_type() == at::kInt && table.dim() == 2 &&
         table.size(0) == q.size(0) && table.stride(1) == 1 && table.size(1) <= INT32_MAX;
}

bool sizes_ok(const Tensor& q) {
  for (const int64_t s : q.sizes())
    if (s < 1 || s > INT32_MAX) return false;
  return true;
}

bool here(const Tensor& q) { return c10::cuda::current_device() == q.get_device(); }
void* stream(const Tensor& q) { return c10::cuda::getCurrentCUDAStream(q.get_device()).stream(); }

Tensor heads_out(const Tensor& q) {  // [B, H, S, D] stored as [B, S, H, D]
  const int64_t h = q.size(1), s = q.size(2), d = q.size(3);
  return at::empty_strided(q.sizes(), {s * h * d, d, h * d, 1}, q.options());
}

// append(query, key, value, cos, sin, k_pages, v_pages, page_table, positions, num_new, q_out, kv_lens_out,
//        q_norm_weight, k_norm_weight, eps)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 15 || g_append == nullptr) return none();
  const Tensor* t[9];
  for (int i = 0; i < 9; ++i)
    if ((t[i] = tensor(args[i])) == nullptr) return none();
  const Tensor *fresh, *q_out, *lens_out, *qw, *kw;
  if (!optional(args[9], &fresh) || !optional(args[10], &q_out) || !optional(args[11], &lens_out) || !optional(args[12], &qw) ||
      !optional(args[13], &kw))
    return none();
  const Tensor &q = *t[0], &k = *t[1], &v = *t[2], &cos = *t[3], &sin = *t[4], &kp = *t[5], &vp = *t[6], &table = *t[7],
               &pos = *t[8];
  if (recorded(&q, &k, &v) || !pool_ok(q, kp, vp, table) || !sizes_ok(q)) return none();
  const int64_t B = q.size(0), Hq = q.size(1), S = q.size(2), D = q.size(3), Hkv = kp.size(1);
  if (Hkv < 1 || Hq % Hkv != 0 || !shaped(k, {B, Hkv, S, D}) || !shaped(v, {B, Hkv, S, D}) || !same(k, q) || !same(v, q) ||
      !rows_ready(q) || !rows_ready(k) || !rows_ready(v))
    return none();
  if (cos.dim() != 3 || cos.size(1) != S || cos.size(2) != D || (cos.size(0) != B && cos.size(0) != 1) || !cos.is_cuda() ||
      cos.get_device() != q.get_device() || (cos.scalar_type() != at::kFloat && cos.scalar_type() != q.scalar_type()) ||
      sin.sizes() != cos.sizes() || !same(sin, cos) || sin.strides() != cos.strides() || !rows_ready(cos) || !rows_ready(sin))
    return none();
  if (!vector32(pos, B, q) || (fresh != nullptr && !vector32(*fresh, B, q))) return none();
  if (lens_out != nullptr && !vector32(*lens_out, B, q)) return none();
  for (const Tensor* w : {qw, kw})
    if (w != nullptr && (!same(*w, q) || !shaped(*w, {D}) || !w->is_contiguous())) return none();
  if (q_out != nullptr && (!same(*q_out, q) || q_out->sizes() != q.sizes() || q_out->stride(3) != 1)) return none();
  if (!here(q)) return none();
  const Tensor out = q_out != nullptr ? *q_out : heads_out(q);
  aicas_paged_append_params p;
  memset(&p, 0, sizeof(p));
  p.q_in = q.data_ptr(), p.q_out = out.data_ptr(), p.k_in = k.data_ptr(), p.v_in = v.data_ptr();
  p.cos = cos.data_ptr(), p.sin = sin.data_ptr(), p.k_pages = kp.data_ptr(), p.v_pages = vp.data_ptr();
  p.page_table = static_cast<const int32_t*>(table.data_ptr()), p.positions = static_cast<const int32_t*>(pos.data_ptr());
  p.num_new = pointer<const int32_t*>(fresh), p.kv_lens_out = pointer<int32_t*>(lens_out);
  p.q_norm_weight = pointer<const void*>(qw), p.k_norm_weight = pointer<const void*>(kw);
  p.qi_stride_b = q.stride(0), p.qi_stride_h = q.stride(1), p.qi_stride_s = q.stride(2);
  p.qo_stride_b = out.stride(0), p.qo_stride_h = out.stride(1), p.qo_stride_s = out.stride(2);
  p.k_stride_b = k.stride(0), p.k_stride_h = k.stride(1), p.k_stride_s = k.stride(2);
  p.v_stride_b = v.stride(0), p.v_stride_h = v.stride(1), p.v_stride_s = v.stride(2);
  p.cs_stride_b = cos.size(0) == B ? cos.stride(0) : 0, p.cs_stride_s = cos.stride(1);
  p.kp_stride_p = kp.stride(0), p.kp_stride_h = kp.stride(1), p.kp_stride_t = kp.stride(2);
  p.vp_stride_p = vp.stride(0), p.vp_stride_h = vp.stride(1), p.vp_stride_t = vp.stride(2);
  p.table_stride = table.stride(0);
  p.batch = (int32_t)B, p.num_q_heads = (int32_t)Hq, p.num_kv_heads = (int32_t)Hkv, p.seq_len = (int32_t)S;
  p.head_dim = (int32_t)D, p.num_pages = (int32_t)kp.size(0), p.page_size = (int32_t)kp.size(2);
  p.max_pages = (int32_t)table.size(1), p.dtype = dtype_code(q), p.cs_dtype = dtype_code(cos);
  p.norm_eps = (float)PyFloat_AsDouble(args[14]);
  if (PyErr_Occurred() != nullptr) return PyErr_Clear(), none();
  if (launch(g_append, &p, stream(q)) != AICAS_OK) return none();
  return q_out != nullptr ? Py_NewRef(args[10]) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// decode(query, k_pages, v_pages, page_table, sm_scale, groups, kv_lens, kv_starts, return_lse, workspaces)
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 10 || g_decode == nullptr) return none();
  const Tensor* t[4];
  for (int i = 0; i < 4; ++i)
    if ((t[i] = tensor(args[i])) == nullptr) return none();
  const Tensor *lens, *starts;
  const bool want_lse = args[8] == Py_True;
  if ((!want_lse && args[8] != Py_False) || !optional(args[6], &lens) || !optional(args[7], &starts)) return none();
  const Tensor &q = *t[0], &kp = *t[1], &vp = *t[2], &table = *t[3];
  if (recorded(&q, &kp, &vp) || !pool_ok(q, kp, vp, table) || !sizes_ok(q)) return none();
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(3), Hkv = kp.size(1);
  const double scale = PyFloat_AsDouble(args[4]);
  const long long groups = PyLong_AsLongLong(args[5]);
  if (PyErr_Occurred() != nullptr) return PyErr_Clear(), none();
  if (q.size(2) != 1 || groups < 1 || Hkv < 1 || Hq % Hkv != 0 || Hq / Hkv != groups || !rows_ready(q)) return none();
  if ((lens != nullptr && !vector32(*lens, B, q)) || (starts != nullptr && !vector32(*starts, B, q))) return none();
  if (!here(q)) return none();
  void* const st = stream(q);
  THPObjectPtr key(Py_BuildValue("(iK)", (int)q.get_device(), (unsigned long long)reinterpret_cast<uintptr_t>(st)));
  PyObject* found = key ? PyDict_GetItemWithError(args[9], key.get()) : nullptr;
  if (found == nullptr) return PyErr_Clear(), none();
  if (tensor(found) == nullptr) return none();
  const Tensor ws = *tensor(found);  // held: another thread may enlarge the stream's workspace during the launch
  const Tensor out = heads_out(q);
  Tensor lse;
  if (want_lse) lse = at::empty_strided({B, Hq}, {Hq, 1}, q.options().dtype(at::kFloat));
  aicas_paged_decode_params p;
  memset(&p, 0, sizeof(p));
  p.q = q.data_ptr(), p.k_pages = kp.data_ptr(), p.v_pages = vp.data_ptr(), p.out = out.data_ptr();
  p.lse = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  p.page_table = static_cast<const int32_t*>(table.data_ptr());
  p.kv_lens = pointer<const int32_t*>(lens), p.kv_starts = pointer<const int32_t*>(starts);
  p.q_stride_b = q.stride(0), p.q_stride_h = q.stride(1), p.o_stride_b = out.stride(0), p.o_stride_h = out.stride(1);
  p.kp_stride_p = kp.stride(0), p.kp_stride_h = kp.stride(1), p.kp_stride_t = kp.stride(2);
  p.vp_stride_p = vp.stride(0), p.vp_stride_h = vp.stride(1), p.vp_stride_t = vp.stride(2);
  p.table_stride = table.stride(0);
  p.batch = (int32_t)B, p.num_q_heads = (int32_t)Hq, p.num_kv_heads = (int32_t)Hkv, p.head_dim = (int32_t)D;
  p.num_pages = (int32_t)kp.size(0), p.page_size = (int32_t)kp.size(2), p.max_pages = (int32_t)table.size(1);
  p.dtype = dtype_code(q), p.sm_scale = (float)scale;
  if (launch(g_decode, &p, ws.data_ptr(), (size_t)ws.numel(), st) != AICAS_OK) return none();
  if (!want_lse) return THPVariable_Wrap(out);
  THPObjectPtr a(THPVariable_Wrap(out)), b(THPVariable_Wrap(lse));
  return a && b ? PyTuple_Pack(2, a.get(), b.get()) : nullptr;
  END_HANDLE_TH_ERRORS
}

// One weight as int4.py's _check_weight takes it; n and groups are compared where already set.
bool weight_ok(PyObject* o, const Tensor& x, int64_t* n, int64_t* groups, aicas_int4_weight* w) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 3) return false;
  const Tensor *q = tensor(PyTuple_GET_ITEM(o, 0)), *s = tensor(PyTuple_GET_ITEM(o, 1)), *z;
  if (q == nullptr || s == nullptr || !optional(PyTuple_GET_ITEM(o, 2), &z)) return false;
  if (!q->is_cuda() || q->get_device() != x.get_device() || q->scalar_type() != at::kByte || q->dim() != 2 ||
      q->size(1) * 2 != x.size(1) || !rows_ready(*q) || q->stride(0) * 2 < x.size(1))
    return false;
  if (recorded(s) || !same(*s, x) || s->dim() != 2 || s->size(0) != q->size(0) || !s->is_contiguous()) return false;
  if (z != nullptr && (!z->is_cuda() || z->get_device() != x.get_device() || z->scalar_type() != at::kByte ||
                       z->sizes() != s->sizes() || !z->is_contiguous()))
    return false;
  if (*n >= 0 && (*n != q->size(0) || *groups != s->size(1))) return false;
  *n = q->size(0), *groups = s->size(1);
  w->q = q->data_ptr(), w->scales = s->data_ptr(), w->zeros = pointer<const void*>(z), w->q_stride = q->stride(0);
  return true;
}

// int4(x, weight, norm_weight, eps, residual, swiglu, out)
PyObject* int4(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 7 || g_int4 == nullptr) return none();
  const Tensor *xp = tensor(args[0]), *nw, *res, *outp;
  if (xp == nullptr || !optional(args[2], &nw) || !optional(args[4], &res) || !optional(args[6], &outp)) return none();
  const Tensor& x = *xp;
  const bool pair = args[5] == Py_True;
  if ((!pair && args[5] != Py_False) || recorded(&x, nw, res) || !x.is_cuda() || x.dim() != 2) return none();
  const int code = dtype_code(x);
  const int64_t R = x.size(0), K = x.size(1);
  if ((code != AICAS_DTYPE_F16 && code != AICAS_DTYPE_BF16) || R < 1 || R > AICAS_LINEAR_MAX_ROWS || K < 1 || K > INT32_MAX ||
      !rows_ready(x) || x.stride(0) < K)
    return none();
  aicas_linear_int4_params p;
  memset(&p, 0, sizeof(p));
  int64_t N = -1, groups = -1;
  if (pair) {
    const bool list = PyList_Check(args[1]);
    if (res != nullptr || (!list && !PyTuple_Check(args[1])) || PySequence_Fast_GET_SIZE(args[1]) != 2) return none();
    for (int i = 0; i < 2; ++i)
      if (!weight_ok(PySequence_Fast_GET_ITEM(args[1], i), x, &N, &groups, &p.w[i])) return none();
    if ((p.w[0].zeros == nullptr) != (p.w[1].zeros == nullptr)) return none();
  } else if (!weight_ok(args[1], x, &N, &groups, &p.w[0])) {
    return none();
  }
  if (N < 1 || N > INT32_MAX || groups < 1 || K % groups != 0) return none();
  const int64_t g = K / groups;
  if (g != 32 && g != 64 && g != 128) return none();
  if (res != nullptr && (!same(*res, x) || !shaped(*res, {R, N}) || res->stride(1) != 1)) return none();
  if (nw != nullptr && (!same(*nw, x) || !shaped(*nw, {K}) || !rows_ready(*nw))) return none();
  if (outp != nullptr) {
    const Tensor& o = *outp;
    if (!same(o, x) || !shaped(o, {R, N}) || o.stride(1) != 1 || (R > 1 && o.stride(0) < N)) return none();
    // memory shared in any other way than out == residual is for the operator's own checks
    if (o.storage().data() == x.storage().data() || (nw != nullptr && o.storage().data() == nw->storage().data())) return none();
    if (res != nullptr && o.storage().data() == res->storage().data() &&
        (o.data_ptr() != res->data_ptr() || (R > 1 && o.stride(0) != res->stride(0))))
      return none();
  }
  if (!here(x)) return none();
  p.eps = (float)PyFloat_AsDouble(args[3]);
  if (PyErr_Occurred() != nullptr) return PyErr_Clear(), none();
  const Tensor out = outp != nullptr ? *outp : at::empty_strided({R, N}, {N, 1}, x.options());
  p.x = x.data_ptr(), p.x_stride = x.stride(0), p.norm_weight = pointer<const void*>(nw);
  p.residual = pointer<const void*>(res), p.residual_stride = res != nullptr ? res->stride(0) : 0;
  p.out = out.data_ptr(), p.out_stride = out.stride(0);
  p.rows = (int32_t)R, p.in_features = (int32_t)K, p.out_features = (int32_t)N, p.group_size = (int32_t)g;
  p.mode = pair ? AICAS_LINEAR_SWIGLU : res != nullptr ? AICAS_LINEAR_RESIDUAL : AICAS_LINEAR_STORE;
  p.dtype = code;
  if (launch(g_int4, &p, stream(x)) != AICAS_OK) return none();
  return outp != nullptr ? Py_NewRef(args[6]) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// bind(append, decode, int4): addresses of the library's entry points.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != 3) return PyErr_SetString(PyExc_TypeError, "bind takes three addresses"), nullptr;
  void* at[3];
  for (int i = 0; i < 3; ++i) at[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  g_append = reinterpret_cast<decltype(g_append)>(at[0]);
  g_decode = reinterpret_cast<decltype(g_decode)>(at[1]);
  g_int4 = reinterpret_cast<decltype(g_int4)>(at[2]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, "paged_rope_kv_append, or None"},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(decode)), METH_FASTCALL, "paged_gqa_decode_attention, or None"},
    {"int4", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(int4)), METH_FASTCALL, "decode_linear_int4, or None"},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, "sets the entry points' addresses"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hostcalls", "Cheap calls of the short operators.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hostcalls(void) { return PyModule_Create(&module); }
