// The host side of the short operators' launches: what paged.py, int4.py, paged_int4.py
// and eviction.py check and pack, for arguments that need nothing done to them.  Each function returns
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
decltype(&aicas_paged_append_int4) g_append4 = nullptr;
decltype(&aicas_paged_read_int4) g_read4 = nullptr;
decltype(&aicas_paged_decode_int4) g_decode4 = nullptr;
decltype(&aicas_paged_weights) g_weigh = nullptr;
decltype(&aicas_paged_evict) g_evict = nullptr;

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

// What the two appends take beside the pages: query, key, value, cos, sin, and behind
// the page table positions, num_new, q_out, kv_lens_out, q_norm_weight, k_norm_weight, eps.
struct NewRows {
  const Tensor *q, *k, *v, *cos, *sin, *pos, *fresh, *q_out, *lens_out, *qw, *kw;

  bool unpack(PyObject* const* rows, PyObject* const* rest) {
    const Tensor** const t[] = {&q, &k, &v, &cos, &sin};
    for (int i = 0; i < 5; ++i)
      if ((*t[i] = tensor(rows[i])) == nullptr) return false;
    return (pos = tensor(rest[0])) != nullptr && optional(rest[1], &fresh) && optional(rest[2], &q_out) &&
           optional(rest[3], &lens_out) && optional(rest[4], &qw) && optional(rest[5], &kw) && !recorded(q, k, v);
  }

  bool ok(int64_t Hkv) const {
    const int64_t B = q->size(0), Hq = q->size(1), S = q->size(2), D = q->size(3);
    if (Hkv < 1 || Hq % Hkv != 0 || !shaped(*k, {B, Hkv, S, D}) || !shaped(*v, {B, Hkv, S, D}) || !same(*k, *q) ||
        !same(*v, *q) || !rows_ready(*q) || !rows_ready(*k) || !rows_ready(*v))
      return false;
    if (cos->dim() != 3 || cos->size(1) != S || cos->size(2) != D || (cos->size(0) != B && cos->size(0) != 1) || !cos->is_cuda() ||
        cos->get_device() != q->get_device() || (cos->scalar_type() != at::kFloat && cos->scalar_type() != q->scalar_type()) ||
        sin->sizes() != cos->sizes() || !same(*sin, *cos) || sin->strides() != cos->strides() || !rows_ready(*cos) || !rows_ready(*sin))
      return false;
    if (!vector32(*pos, B, *q) || (fresh != nullptr && !vector32(*fresh, B, *q))) return false;
    if (lens_out != nullptr && !vector32(*lens_out, B, *q)) return false;
    for (const Tensor* w : {qw, kw})
      if (w != nullptr && (!same(*w, *q) || !shaped(*w, {D}) || !w->is_contiguous())) return false;
    return q_out == nullptr || (same(*q_out, *q) && q_out->sizes() == q->sizes() && q_out->stride(3) == 1);
  }

  // P: the parameters of either append.
  template <typename P>
  bool fill(P& p, const Tensor& out, const Tensor& table, PyObject* eps) const {
    p.q_in = q->data_ptr(), p.q_out = out.data_ptr(), p.k_in = k->data_ptr(), p.v_in = v->data_ptr();
    p.cos = cos->data_ptr(), p.sin = sin->data_ptr();
    p.page_table = static_cast<const int32_t*>(table.data_ptr()), p.positions = static_cast<const int32_t*>(pos->data_ptr());
    p.num_new = pointer<const int32_t*>(fresh), p.kv_lens_out = pointer<int32_t*>(lens_out);
    p.q_norm_weight = pointer<const void*>(qw), p.k_norm_weight = pointer<const void*>(kw);
    p.qi_stride_b = q->stride(0), p.qi_stride_h = q->stride(1), p.qi_stride_s = q->stride(2);
    p.qo_stride_b = out.stride(0), p.qo_stride_h = out.stride(1), p.qo_stride_s = out.stride(2);
    p.k_stride_b = k->stride(0), p.k_stride_h = k->stride(1), p.k_stride_s = k->stride(2);
    p.v_stride_b = v->stride(0), p.v_stride_h = v->stride(1), p.v_stride_s = v->stride(2);
    p.cs_stride_b = cos->size(0) == q->size(0) ? cos->stride(0) : 0, p.cs_stride_s = cos->stride(1);
    p.table_stride = table.stride(0);
    p.batch = (int32_t)q->size(0), p.num_q_heads = (int32_t)q->size(1), p.num_kv_heads = (int32_t)k->size(1);
    p.seq_len = (int32_t)q->size(2), p.head_dim = (int32_t)q->size(3);
    p.max_pages = (int32_t)table.size(1), p.dtype = dtype_code(*q), p.cs_dtype = dtype_code(*cos);
    p.norm_eps = (float)PyFloat_AsDouble(eps);
    if (PyErr_Occurred() != nullptr) return PyErr_Clear(), false;
    return true;
  }
};

// append(query, key, value, cos, sin, k_pages, v_pages, page_table, positions, num_new, q_out, kv_lens_out,
//        q_norm_weight, k_norm_weight, eps)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 15 || g_append == nullptr) return none();
  NewRows n;
  const Tensor *kpp = tensor(args[5]), *vpp = tensor(args[6]), *tp = tensor(args[7]);
  if (kpp == nullptr || vpp == nullptr || tp == nullptr || !n.unpack(args, args + 8)) return none();
  const Tensor &q = *n.q, &kp = *kpp, &vp = *vpp, &table = *tp;
  if (!pool_ok(q, kp, vp, table) || !sizes_ok(q) || !n.ok(kp.size(1)) || !here(q)) return none();
  const Tensor out = n.q_out != nullptr ? *n.q_out : heads_out(q);
  aicas_paged_append_params p;
  memset(&p, 0, sizeof(p));
  if (!n.fill(p, out, table, args[14])) return none();
  p.k_pages = kp.data_ptr(), p.v_pages = vp.data_ptr();
  p.kp_stride_p = kp.stride(0), p.kp_stride_h = kp.stride(1), p.kp_stride_t = kp.stride(2);
  p.vp_stride_p = vp.stride(0), p.vp_stride_h = vp.stride(1), p.vp_stride_t = vp.stride(2);
  p.num_pages = (int32_t)kp.size(0), p.page_size = (int32_t)kp.size(2);
  if (launch(g_append, &p, stream(q)) != AICAS_OK) return none();
  return n.q_out != nullptr ? Py_NewRef(args[10]) : THPVariable_Wrap(out);
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

// ------------------------------------------------------------------ 4-bit pages and eviction

struct Pool4 {
  int64_t pages = -1, heads, size, dim, group;
  bool operator==(const Pool4& o) const {
    return pages == o.pages && heads == o.heads && size == o.size && dim == o.dim && group == o.group;
  }
};

// One side as paged_int4.py's _side takes it, with scales of type `type` on device `index`.
bool side_ok(PyObject* o, int64_t index, at::ScalarType type, Pool4* s, aicas_int4_pages* r) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) return false;
  const Tensor *c = tensor(PyTuple_GET_ITEM(o, 0)), *p = tensor(PyTuple_GET_ITEM(o, 1));
  if (c == nullptr || p == nullptr || !c->is_cuda() || !p->is_cuda() || c->get_device() != index || p->get_device() != index ||
      c->scalar_type() != at::kByte || p->scalar_type() != type || (type != at::kHalf && type != at::kBFloat16) || c->dim() != 4 ||
      p->dim() != 5 || recorded(p))
    return false;
  const int64_t dim = 2 * c->size(3), groups = p->size(3);
  if ((dim != 64 && dim != 128) || p->size(0) != c->size(0) || p->size(1) != c->size(1) || p->size(2) != c->size(2) ||
      p->size(4) != 2 || groups < 1 || (dim / groups != 64 && groups != 1) || dim % groups != 0 || c->size(2) < 8 ||
      c->size(2) % 8 != 0 || c->size(0) > INT32_MAX || c->size(2) > INT32_MAX || c->stride(3) != 1 || p->stride(4) != 1 ||
      (groups > 1 && p->stride(3) != 2))
    return false;
  s->pages = c->size(0), s->heads = c->size(1), s->size = c->size(2), s->dim = dim, s->group = dim / groups;
  r->codes = c->data_ptr(), r->scales = p->data_ptr();
  r->cs_p = c->stride(0), r->cs_h = c->stride(1), r->cs_t = c->stride(2);
  r->ss_p = p->stride(0), r->ss_h = p->stride(1), r->ss_t = p->stride(2);
  return true;
}

bool table_ok(const Tensor& t, int64_t batch, int64_t index) {
  return t.is_cuda() && t.get_device() == index && t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == batch &&
         t.stride(1) == 1 && t.size(1) >= 1 && t.size(1) <= INT32_MAX;
}

bool number(PyObject* o, int64_t* v) {
  *v = PyLong_AsLongLong(o);
  return PyErr_Occurred() == nullptr || (PyErr_Clear(), false);
}

// append_int4: the arguments of append, with Int4Pages
PyObject* append_int4(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 15 || g_append4 == nullptr) return none();
  NewRows n;
  const Tensor* tp = tensor(args[7]);
  if (tp == nullptr || !n.unpack(args, args + 8)) return none();
  const Tensor &q = *n.q, &table = *tp;
  if (!q.is_cuda() || q.dim() != 4 || !sizes_ok(q) || !table_ok(table, q.size(0), q.get_device())) return none();
  aicas_paged_append_int4_params p;
  memset(&p, 0, sizeof(p));
  Pool4 k, v;
  if (!side_ok(args[5], q.get_device(), q.scalar_type(), &k, &p.kv[0]) ||
      !side_ok(args[6], q.get_device(), q.scalar_type(), &v, &p.kv[1]) || !(k == v) || k.dim != q.size(3) || !n.ok(k.heads) || !here(q))
    return none();
  const Tensor out = n.q_out != nullptr ? *n.q_out : heads_out(q);
  if (!n.fill(p, out, table, args[14])) return none();
  p.group_size = (int32_t)k.group, p.num_pages = (int32_t)k.pages, p.page_size = (int32_t)k.size;
  if (launch(g_append4, &p, stream(q)) != AICAS_OK) return none();
  return n.q_out != nullptr ? Py_NewRef(args[10]) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// read_int4(k_pages, v_pages, page_table, positions, seq_len, num_tokens)
PyObject* read_int4(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 6 || g_read4 == nullptr) return none();
  const Tensor *tp = tensor(args[2]), *pos = tensor(args[3]), *fresh;
  int64_t S;
  if (tp == nullptr || pos == nullptr || !optional(args[5], &fresh) || !number(args[4], &S) || S < 1 || S > INT32_MAX) return none();
  const Tensor& table = *tp;
  if (!PyTuple_Check(args[0]) || PyTuple_GET_SIZE(args[0]) != 2 || tensor(PyTuple_GET_ITEM(args[0], 1)) == nullptr) return none();
  const Tensor& scales = *tensor(PyTuple_GET_ITEM(args[0], 1));
  if (!table.is_cuda() || table.dim() != 2 || table.size(0) < 1 || table.size(0) > INT32_MAX ||
      !table_ok(table, table.size(0), table.get_device()))
    return none();
  const int64_t B = table.size(0);
  aicas_paged_read_int4_params p;
  memset(&p, 0, sizeof(p));
  Pool4 k, v;
  if (!side_ok(args[0], table.get_device(), scales.scalar_type(), &k, &p.kv[0]) ||
      !side_ok(args[1], table.get_device(), scales.scalar_type(), &v, &p.kv[1]) || !(k == v) || k.heads < 1 || k.heads > INT32_MAX ||
      k.pages < 1 || !vector32(*pos, B, table) || (fresh != nullptr && !vector32(*fresh, B, table)) || !here(table))
    return none();
  const int64_t sb = k.heads * S * k.dim, sh = S * k.dim;
  Tensor out[2];
  for (int i = 0; i < 2; ++i) {
    out[i] = at::empty_strided({B, k.heads, S, k.dim}, {sb, sh, k.dim, 1}, scales.options());
    p.out[i] = out[i].data_ptr();
  }
  p.page_table = static_cast<const int32_t*>(table.data_ptr()), p.positions = static_cast<const int32_t*>(pos->data_ptr());
  p.num_tokens = pointer<const int32_t*>(fresh);
  p.out_stride_b = sb, p.out_stride_h = sh, p.out_stride_s = k.dim, p.table_stride = table.stride(0);
  p.batch = (int32_t)B, p.num_kv_heads = (int32_t)k.heads, p.seq_len = (int32_t)S, p.head_dim = (int32_t)k.dim;
  p.group_size = (int32_t)k.group, p.num_pages = (int32_t)k.pages, p.page_size = (int32_t)k.size;
  p.max_pages = (int32_t)table.size(1), p.dtype = dtype_code(scales);
  if (launch(g_read4, &p, stream(table)) != AICAS_OK) return none();
  THPObjectPtr a(THPVariable_Wrap(out[0])), b(THPVariable_Wrap(out[1]));
  return a && b ? PyTuple_Pack(2, a.get(), b.get()) : nullptr;
  END_HANDLE_TH_ERRORS
}

// decode_int4: the arguments of decode, with Int4Pages
PyObject* decode_int4(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 10 || g_decode4 == nullptr) return none();
  const Tensor *qp = tensor(args[0]), *tp = tensor(args[3]), *lens, *starts;
  const bool want_lse = args[8] == Py_True;
  if (qp == nullptr || tp == nullptr || (!want_lse && args[8] != Py_False) || !optional(args[6], &lens) || !optional(args[7], &starts))
    return none();
  const Tensor &q = *qp, &table = *tp;
  if (recorded(&q) || !q.is_cuda() || q.dim() != 4 || !sizes_ok(q) || !table_ok(table, q.size(0), q.get_device())) return none();
  const int64_t B = q.size(0), Hq = q.size(1);
  const double scale = PyFloat_AsDouble(args[4]);
  const long long groups = PyLong_AsLongLong(args[5]);
  if (PyErr_Occurred() != nullptr) return PyErr_Clear(), none();
  aicas_paged_decode_int4_params p;
  memset(&p, 0, sizeof(p));
  Pool4 k, v;
  if (!side_ok(args[1], q.get_device(), q.scalar_type(), &k, &p.kv[0]) ||
      !side_ok(args[2], q.get_device(), q.scalar_type(), &v, &p.kv[1]) || !(k == v) || k.dim != q.size(3) || q.size(2) != 1 ||
      groups < 1 || k.heads < 1 || Hq % k.heads != 0 || Hq / k.heads != groups || !rows_ready(q))
    return none();
  if ((lens != nullptr && !vector32(*lens, B, q)) || (starts != nullptr && !vector32(*starts, B, q)) || !here(q)) return none();
  void* const st = stream(q);
  THPObjectPtr key(Py_BuildValue("(iK)", (int)q.get_device(), (unsigned long long)reinterpret_cast<uintptr_t>(st)));
  PyObject* found = key ? PyDict_GetItemWithError(args[9], key.get()) : nullptr;
  if (found == nullptr) return PyErr_Clear(), none();
  if (tensor(found) == nullptr) return none();
  const Tensor ws = *tensor(found);  // held: another thread may enlarge the stream's workspace during the launch
  const Tensor out = heads_out(q);
  Tensor lse;
  if (want_lse) lse = at::empty_strided({B, Hq}, {Hq, 1}, q.options().dtype(at::kFloat));
  p.q = q.data_ptr(), p.out = out.data_ptr(), p.lse = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  p.page_table = static_cast<const int32_t*>(table.data_ptr());
  p.kv_lens = pointer<const int32_t*>(lens), p.kv_starts = pointer<const int32_t*>(starts);
  p.q_stride_b = q.stride(0), p.q_stride_h = q.stride(1), p.o_stride_b = out.stride(0), p.o_stride_h = out.stride(1);
  p.table_stride = table.stride(0);
  p.batch = (int32_t)B, p.num_q_heads = (int32_t)Hq, p.num_kv_heads = (int32_t)k.heads, p.head_dim = (int32_t)k.dim;
  p.group_size = (int32_t)k.group, p.num_pages = (int32_t)k.pages, p.page_size = (int32_t)k.size;
  p.max_pages = (int32_t)table.size(1), p.dtype = dtype_code(q), p.sm_scale = (float)scale;
  if (launch(g_decode4, &p, ws.data_ptr(), (size_t)ws.numel(), st) != AICAS_OK) return none();
  if (!want_lse) return THPVariable_Wrap(out);
  THPObjectPtr a(THPVariable_Wrap(out)), b(THPVariable_Wrap(lse));
  return a && b ? PyTuple_Pack(2, a.get(), b.get()) : nullptr;
  END_HANDLE_TH_ERRORS
}

// fp32 [B, Hkv, C] of contiguous rows that share no memory, C at least `slots`.
bool weights_ok(const Tensor& w, int64_t B, int64_t H, int64_t slots, int64_t index) {
  if (!w.is_cuda() || w.get_device() != index || w.scalar_type() != at::kFloat || w.dim() != 3 || w.size(0) != B || w.size(1) != H ||
      w.size(2) < slots || w.stride(2) != 1 || recorded(&w))
    return false;
  const int64_t sb = w.stride(0), sh = w.stride(1), C = w.size(2);
  return sh >= C && sb >= C && (sb >= sh * H || sh >= sb * B);
}

// weigh(query, k_pages, page_table, lse, weights, sm_scale, groups, kv_lens, kv_starts)
PyObject* weigh(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 9 || g_weigh == nullptr) return none();
  const Tensor *qp = tensor(args[0]), *tp = tensor(args[2]), *lp = tensor(args[3]), *wp = tensor(args[4]), *lens, *starts;
  if (qp == nullptr || tp == nullptr || lp == nullptr || wp == nullptr || !optional(args[7], &lens) || !optional(args[8], &starts))
    return none();
  const Tensor &q = *qp, &table = *tp, &lse = *lp, &w = *wp;
  if (recorded(&q, &lse) || !q.is_cuda() || q.dim() != 4 || !sizes_ok(q) || dtype_code(q) < 0 || !rows_ready(q)) return none();
  const int64_t B = q.size(0), Hq = q.size(1), S = q.size(2), D = q.size(3), index = q.get_device();
  const double scale = PyFloat_AsDouble(args[5]);
  const long long groups = PyLong_AsLongLong(args[6]);
  if (PyErr_Occurred() != nullptr) return PyErr_Clear(), none();
  aicas_paged_weights_params p;
  memset(&p, 0, sizeof(p));
  Pool4 k;
  if (const Tensor* pages = tensor(args[1])) {
    if (!same(*pages, q) || pages->dim() != 4 || pages->size(2) < 8 || pages->size(2) % 8 != 0 || pages->stride(3) != 1 ||
        pages->size(0) > INT32_MAX || pages->size(2) > INT32_MAX || recorded(pages))
      return none();
    k.pages = pages->size(0), k.heads = pages->size(1), k.size = pages->size(2), k.dim = pages->size(3), k.group = 0;
    if (k.dim != 16 && k.dim != 32 && k.dim != 64 && k.dim != 128) return none();
    p.k_pages = pages->data_ptr();
    p.kp_stride_p = pages->stride(0), p.kp_stride_h = pages->stride(1), p.kp_stride_t = pages->stride(2);
  } else {
    aicas_int4_pages r;
    if (!side_ok(args[1], index, q.scalar_type(), &k, &r)) return none();
    p.k_pages = r.codes, p.k_scales = r.scales;
    p.kp_stride_p = r.cs_p, p.kp_stride_h = r.cs_h, p.kp_stride_t = r.cs_t;
    p.ks_stride_p = r.ss_p, p.ks_stride_h = r.ss_h, p.ks_stride_t = r.ss_t;
  }
  if (k.dim != D || groups < 1 || k.heads < 1 || Hq % k.heads != 0 || Hq / k.heads != groups || !table_ok(table, B, index) ||
      !weights_ok(w, B, k.heads, table.size(1) * k.size, index))
    return none();
  const bool flat = lse.dim() == 2 && S == 1;
  if (!lse.is_cuda() || lse.get_device() != index || lse.scalar_type() != at::kFloat ||
      !(flat ? shaped(lse, {B, Hq}) : shaped(lse, {B, Hq, S})))
    return none();
  if ((lens != nullptr && !vector32(*lens, B, q)) || (starts != nullptr && !vector32(*starts, B, q)) || !here(q)) return none();
  p.q = q.data_ptr(), p.lse = static_cast<const float*>(lse.data_ptr()), p.weights = static_cast<float*>(w.data_ptr());
  p.page_table = static_cast<const int32_t*>(table.data_ptr());
  p.kv_lens = pointer<const int32_t*>(lens), p.kv_starts = pointer<const int32_t*>(starts);
  p.q_stride_b = q.stride(0), p.q_stride_h = q.stride(1), p.q_stride_s = q.stride(2);
  p.lse_stride_b = lse.stride(0), p.lse_stride_h = lse.stride(1), p.lse_stride_s = flat ? 0 : lse.stride(2);
  p.w_stride_b = w.stride(0), p.w_stride_h = w.stride(1), p.table_stride = table.stride(0);
  p.batch = (int32_t)B, p.num_q_heads = (int32_t)Hq, p.num_kv_heads = (int32_t)k.heads, p.seq_len = (int32_t)S;
  p.head_dim = (int32_t)D, p.group_size = (int32_t)k.group, p.num_pages = (int32_t)k.pages, p.page_size = (int32_t)k.size;
  p.max_pages = (int32_t)table.size(1), p.dtype = dtype_code(q), p.sm_scale = (float)scale;
  if (launch(g_weigh, &p, stream(q)) != AICAS_OK) return none();
  return Py_NewRef(args[4]);
  END_HANDLE_TH_ERRORS
}

// evict(k_pages, v_pages, page_table, weights, kv_lens, keep, keep_first, keep_last, longer_than, kv_lens_out, weights_out)
PyObject* evict(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 11 || g_evict == nullptr) return none();
  const Tensor *tp = tensor(args[2]), *wp = tensor(args[3]), *np = tensor(args[4]), *lens_out, *wo;
  int64_t keep, first, last, longer;
  if (tp == nullptr || wp == nullptr || np == nullptr || !number(args[5], &keep) || !number(args[6], &first) || !number(args[7], &last) ||
      !optional(args[9], &lens_out) || !optional(args[10], &wo))
    return none();
  if (args[8] == Py_None)
    longer = keep;
  else if (!number(args[8], &longer))
    return none();
  const Tensor &table = *tp, &w = *wp;
  if (!table.is_cuda() || table.dim() != 2 || table.size(0) < 1 || table.size(0) > INT32_MAX ||
      !table_ok(table, table.size(0), table.get_device()))
    return none();
  const int64_t B = table.size(0), index = table.get_device();
  if (keep < 1 || keep > INT32_MAX || first < 0 || last < 0 || first > keep || last > keep - first || longer < keep || longer > INT32_MAX)
    return none();
  aicas_paged_evict_params p;
  memset(&p, 0, sizeof(p));
  Pool4 shapes[2];
  for (int i = 0; i < 2; ++i) {
    Pool4& s = shapes[i];
    if (const Tensor* pages = tensor(args[i])) {
      const int64_t item = pages->element_size();
      if (!pages->is_cuda() || pages->get_device() != index || pages->dim() != 4 || dtype_code(*pages) < 0 || pages->size(2) < 8 ||
          pages->size(2) % 8 != 0 || pages->stride(3) != 1 || pages->size(0) > INT32_MAX || pages->size(2) > INT32_MAX || recorded(pages))
        return none();
      s.pages = pages->size(0), s.heads = pages->size(1), s.size = pages->size(2), s.dim = pages->size(3), s.group = 0;
      if (s.dim != 16 && s.dim != 32 && s.dim != 64 && s.dim != 128) return none();
      p.plane[p.num_planes++] = {pages->data_ptr(), item * pages->stride(0), item * pages->stride(1), item * pages->stride(2), item * s.dim};
    } else {
      aicas_int4_pages r;
      PyObject* o = args[i];
      if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2 || tensor(PyTuple_GET_ITEM(o, 1)) == nullptr ||
          !side_ok(o, index, tensor(PyTuple_GET_ITEM(o, 1))->scalar_type(), &s, &r))
        return none();
      p.plane[p.num_planes++] = {r.codes, r.cs_p, r.cs_h, r.cs_t, s.dim / 2};
      p.plane[p.num_planes++] = {r.scales, 2 * r.ss_p, 2 * r.ss_h, 2 * r.ss_t, 4 * (s.dim / s.group)};
    }
  }
  const Pool4& k = shapes[0];
  if (!(k == shapes[1]) || k.heads < 1 || k.heads > INT32_MAX || k.pages < 1) return none();
  const int64_t slots = table.size(1) * k.size;
  if (!weights_ok(w, B, k.heads, slots, index) || !vector32(*np, B, table) || (lens_out != nullptr && !vector32(*lens_out, B, table)))
    return none();
  // memory shared in any other way than weights_out is weights is for the operator's own checks
  if (wo != nullptr && (!weights_ok(*wo, B, k.heads, slots, index) || (args[10] != args[3] && wo->storage().data() == w.storage().data())))
    return none();
  if (!here(table)) return none();
  const Tensor& into = wo != nullptr ? *wo : w;
  const Tensor kept = at::empty_strided({B, k.heads, keep}, {k.heads * keep, keep, 1}, table.options());
  p.weights = static_cast<const float*>(w.data_ptr()), p.weights_out = static_cast<float*>(into.data_ptr());
  p.kept = static_cast<int32_t*>(kept.data_ptr()), p.page_table = static_cast<const int32_t*>(table.data_ptr());
  p.kv_lens = static_cast<const int32_t*>(np->data_ptr()), p.kv_lens_out = pointer<int32_t*>(lens_out);
  p.w_stride_b = w.stride(0), p.w_stride_h = w.stride(1), p.wo_stride_b = into.stride(0), p.wo_stride_h = into.stride(1);
  p.table_stride = table.stride(0);
  p.batch = (int32_t)B, p.num_kv_heads = (int32_t)k.heads, p.num_pages = (int32_t)k.pages, p.page_size = (int32_t)k.size;
  p.max_pages = (int32_t)table.size(1), p.keep = (int32_t)keep, p.keep_first = (int32_t)first, p.keep_last = (int32_t)last;
  p.longer_than = (int32_t)longer;
  if (launch(g_evict, &p, stream(table)) != AICAS_OK) return none();
  return THPVariable_Wrap(kept);
  END_HANDLE_TH_ERRORS
}

// Addresses of the library's entry points.
bool addresses(PyObject* const* args, Py_ssize_t count, Py_ssize_t wanted, void** at) {
  if (count != wanted) return PyErr_Format(PyExc_TypeError, "%zd addresses are taken", wanted), false;
  for (Py_ssize_t i = 0; i < count; ++i) at[i] = PyLong_AsVoidPtr(args[i]);
  return PyErr_Occurred() == nullptr;
}

// bind(append, decode, int4)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t count) {
  void* at[3];
  if (!addresses(args, count, 3, at)) return nullptr;
  g_append = reinterpret_cast<decltype(g_append)>(at[0]);
  g_decode = reinterpret_cast<decltype(g_decode)>(at[1]);
  g_int4 = reinterpret_cast<decltype(g_int4)>(at[2]);
  Py_RETURN_NONE;
}

// bind_int4(append_int4, read_int4, decode_int4, weigh, evict)
PyObject* bind_int4(PyObject*, PyObject* const* args, Py_ssize_t count) {
  void* at[5];
  if (!addresses(args, count, 5, at)) return nullptr;
  g_append4 = reinterpret_cast<decltype(g_append4)>(at[0]);
  g_read4 = reinterpret_cast<decltype(g_read4)>(at[1]);
  g_decode4 = reinterpret_cast<decltype(g_decode4)>(at[2]);
  g_weigh = reinterpret_cast<decltype(g_weigh)>(at[3]);
  g_evict = reinterpret_cast<decltype(g_evict)>(at[4]);
  Py_RETURN_NONE;
}

template <typename F>
PyMethodDef method(const char* name, F* f, const char* doc) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL, doc};
}

PyMethodDef methods[] = {
    method("append", append, "paged_rope_kv_append, or None"),
    method("decode", decode, "paged_gqa_decode_attention, or None"),
    method("int4", int4, "decode_linear_int4, or None"),
    method("append_int4", append_int4, "paged_rope_kv_append_int4, or None"),
    method("read_int4", read_int4, "paged_kv_read_int4, or None"),
    method("decode_int4", decode_int4, "paged_gqa_decode_attention_int4, or None"),
    method("weigh", weigh, "paged_attention_weights, or None"),
    method("evict", evict, "paged_kv_evict, or None"),
    method("bind", bind, "sets the entry points' addresses"),
    method("bind_int4", bind_int4, "sets the entry points' addresses of 4-bit pages and eviction"),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hostcalls", "Cheap calls of the short operators.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hostcalls(void) { return PyModule_Create(&module); }
