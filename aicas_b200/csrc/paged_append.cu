// Fused (optional per-head RMSNorm) + rotate-half RoPE + append to a paged KV
// cache: rope_append.cu's operator with the cache rows found through a page
// table.
//
//   y = x * rsqrt(mean x^2 + eps) * w        (with a norm weight, else y = x)
//   r = y * cos + rotate_half(y) * sin,      rotate_half(y) = cat(-y[D/2:], y[:D/2])
//   slot t = positions[b] + s  ->  row t % page_size of page table[b, t / page_size]
//
// Rounding: with fp32 tables norm and rotation stay in fp32 and a result is
// rounded once; with 16-bit tables every operation is rounded to that type, as
// Hugging Face's modules and rope_append.cu do, so a model whose tables are
// 16-bit gets the same keys in a paged as in a contiguous cache.
#include <cstdio>
#include <type_traits>

#include "common.cuh"
#include "paged.cuh"

namespace aicas {
namespace {

template <typename T>
__device__ __forceinline__ float rounded(float x) {
  return Elem<T>::to_float(Elem<T>::from_float(x));
}

template <typename T>
__device__ __forceinline__ uint4 pack_vec(const float* f) {
  constexpr int kV = Elem<T>::kPerVec;
  union {
    uint4 u;
    T t[kV];
  } r;
#pragma unroll
  for (int i = 0; i < kV; ++i) r.t[i] = Elem<T>::from_float(f[i]);
  return r.u;
}

// N floats of a cos/sin row.
template <typename CS, int N>
__device__ __forceinline__ void load_table(const CS* p, float* f) {
  constexpr int kV = Elem<CS>::kPerVec;
  if constexpr (N >= kV) {
#pragma unroll
    for (int i = 0; i < N / kV; ++i) Elem<CS>::unpack(reinterpret_cast<const uint4*>(p)[i], f + i * kV);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = Elem<CS>::to_float(p[i]);
  }
}

constexpr int kAppendThreads = 256;

// One CTA a token.  A row (one head of q, k or v) belongs to D / (2 * kV)
// threads; each holds one 16-byte vector of the row's first half and the
// matching one of its second half, so a rotation needs no exchange.
template <typename T, typename CS, int D>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const aicas_paged_append_params a) {
  constexpr bool kRoundEach = std::is_same<T, CS>::value;
  constexpr int kV = Elem<T>::kPerVec;
  constexpr int kTpr = D / (2 * kV);                 // threads a row
  constexpr int kRows = kAppendThreads / kTpr;       // rows a pass
  const int b = blockIdx.x / a.seq_len, s = blockIdx.x % a.seq_len;
  const int c = threadIdx.x % kTpr * kV;
  grid_launch_dependents();
  grid_dependency_wait();
  const int cap = a.max_pages * a.page_size;
  const int pos = a.positions[b];
  const int fresh = a.num_new != nullptr ? min(max(a.num_new[b], 0), a.seq_len) : a.seq_len;
  if (a.kv_lens_out != nullptr && s == 0 && threadIdx.x == 0)
    a.kv_lens_out[b] = (int)min((long long)max(pos, 0) + fresh, (long long)cap);
  // where this token goes; -1: nowhere
  const long long slot = (long long)pos + s;
  int page = -1, row = 0;
  if (s < fresh && slot >= 0 && slot < cap) {
    page = a.page_table[b * a.table_stride + slot / a.page_size];
    row = (int)(slot % a.page_size);
    if (page >= a.num_pages) page = -1;
  }
  float c1[kV], c2[kV], s1[kV], s2[kV];
  const CS* cp = static_cast<const CS*>(a.cos) + b * a.cs_stride_b + s * a.cs_stride_s + c;
  const CS* sp = static_cast<const CS*>(a.sin) + b * a.cs_stride_b + s * a.cs_stride_s + c;
  load_table<CS, kV>(cp, c1);
  load_table<CS, kV>(cp + D / 2, c2);
  load_table<CS, kV>(sp, s1);
  load_table<CS, kV>(sp + D / 2, s2);

  const int hq = a.num_q_heads, hkv = a.num_kv_heads, rows = hq + 2 * hkv;
  // every lane stays for the row sums' shuffles
  for (int r0 = 0; r0 < rows; r0 += kRows) {
    const int r = r0 + threadIdx.x / kTpr;
    const T* src = nullptr;
    T* dst = nullptr;
    const T* w = nullptr;
    if (r < hq) {
      src = static_cast<const T*>(a.q_in) + b * a.qi_stride_b + r * a.qi_stride_h + s * a.qi_stride_s;
      dst = static_cast<T*>(a.q_out) + b * a.qo_stride_b + r * a.qo_stride_h + s * a.qo_stride_s;
      w = static_cast<const T*>(a.q_norm_weight);
    } else if (r < hq + hkv) {
      const int h = r - hq;
      src = static_cast<const T*>(a.k_in) + b * a.k_stride_b + h * a.k_stride_h + s * a.k_stride_s;
      if (page >= 0) dst = static_cast<T*>(a.k_pages) + page * a.kp_stride_p + h * a.kp_stride_h + row * a.kp_stride_t;
      w = static_cast<const T*>(a.k_norm_weight);
    } else if (r < rows) {
      const int h = r - hq - hkv;
      src = static_cast<const T*>(a.v_in) + b * a.v_stride_b + h * a.v_stride_h + s * a.v_stride_s;
      if (page >= 0) dst = static_cast<T*>(a.v_pages) + page * a.vp_stride_p + h * a.vp_stride_h + row * a.vp_stride_t;
    }
    const bool live = dst != nullptr;
    uint4 u1 = make_uint4(0, 0, 0, 0), u2 = u1;
    if (live) {
      u1 = *reinterpret_cast<const uint4*>(src + c);
      u2 = *reinterpret_cast<const uint4*>(src + c + D / 2);
    }
    float x1[kV], x2[kV];
    Elem<T>::unpack(u1, x1);
    Elem<T>::unpack(u2, x2);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kV; ++i) ss += x1[i] * x1[i] + x2[i] * x2[i];
#pragma unroll
    for (int off = kTpr / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    if (!live) continue;
    if (r < hq + hkv) {
      if (w != nullptr) {
        const float inv = rsqrtf(ss / (float)D + a.norm_eps);
        float w1[kV], w2[kV];
        load_table<T, kV>(w + c, w1);
        load_table<T, kV>(w + c + D / 2, w2);
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          if (kRoundEach) {
            x1[i] = rounded<T>(__fmul_rn(w1[i], rounded<T>(__fmul_rn(x1[i], inv))));
            x2[i] = rounded<T>(__fmul_rn(w2[i], rounded<T>(__fmul_rn(x2[i], inv))));
          } else {
            x1[i] *= inv * w1[i];
            x2[i] *= inv * w2[i];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const float p1 = x1[i], p2 = x2[i];
        if (kRoundEach) {
          x1[i] = __fadd_rn(rounded<T>(__fmul_rn(p1, c1[i])), rounded<T>(__fmul_rn(-p2, s1[i])));
          x2[i] = __fadd_rn(rounded<T>(__fmul_rn(p2, c2[i])), rounded<T>(__fmul_rn(p1, s2[i])));
        } else {
          x1[i] = p1 * c1[i] - p2 * s1[i];
          x2[i] = p2 * c2[i] + p1 * s2[i];
        }
      }
      u1 = pack_vec<T>(x1);
      u2 = pack_vec<T>(x2);
    }
    *reinterpret_cast<uint4*>(dst + c) = u1;
    *reinterpret_cast<uint4*>(dst + c + D / 2) = u2;
  }
}

template <typename T, typename CS>
cudaError_t launch_append(const aicas_paged_append_params& p, cudaStream_t st) {
  const dim3 grid((unsigned)(p.batch * p.seq_len)), block(kAppendThreads);
  switch (p.head_dim) {
    case 16: return launch_pdl(paged_append_kernel<T, CS, 16>, grid, block, 0, st, p);
    case 32: return launch_pdl(paged_append_kernel<T, CS, 32>, grid, block, 0, st, p);
    case 64: return launch_pdl(paged_append_kernel<T, CS, 64>, grid, block, 0, st, p);
    case 128: return launch_pdl(paged_append_kernel<T, CS, 128>, grid, block, 0, st, p);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

int run_paged_append(const aicas_paged_append_params* p, cudaStream_t stream, char* err, size_t errlen) {
  const bool f32cs = p->cs_dtype == AICAS_DTYPE_F32;
  cudaError_t e = cudaErrorInvalidValue;
  switch (p->dtype) {
    case AICAS_DTYPE_F32: e = launch_append<float, float>(*p, stream); break;
    case AICAS_DTYPE_F16:
      e = f32cs ? launch_append<__half, float>(*p, stream) : launch_append<__half, __half>(*p, stream);
      break;
    case AICAS_DTYPE_BF16:
      e = f32cs ? launch_append<__nv_bfloat16, float>(*p, stream)
                : launch_append<__nv_bfloat16, __nv_bfloat16>(*p, stream);
      break;
  }
  if (e != cudaSuccess) {
    snprintf(err, errlen, "paged append launch: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
    return AICAS_ERR_CUDA;
  }
  return AICAS_OK;
}

}  // namespace aicas
