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

// 16 bytes of T from floats, two a conversion.
template <typename T>
__device__ __forceinline__ uint4 pack_vec(const float* f) {
  union {
    uint4 u;
    __nv_bfloat162 b[4];
    __half2 h[4];
    float f[4];
  } r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      r.b[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    else if constexpr (std::is_same<T, __half>::value)
      r.h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    else
      r.f[i] = f[i];
  }
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


// HBM bound: every row is read and written once (8 prompts of 2048 tokens, 16 + 2 * 8
// heads of 128: 285 MB in 50 us, 5700 GB/s, 88 % of the measured copy rate).  One CTA
// a token, so that cos, sin and the slot are looked up once for all its heads.  A row
// (one head of q, k or v) belongs to D / (2 * kV) threads; each holds one 16-byte
// vector of the row's first half and the matching one of its second half, so a
// rotation needs no exchange, and has kAppendRows rows in flight against one set of
// table values.
template <typename T, typename CS, int D, int kAppendThreads, int kAppendRows>
__global__ void __launch_bounds__(kAppendThreads, kAppendThreads == 32 ? 18 : 1) paged_append_kernel(const __grid_constant__ aicas_paged_append_params a) {
  constexpr bool kRoundEach = std::is_same<T, CS>::value;
  constexpr int kV = Elem<T>::kPerVec;
  constexpr int kTpr = D / (2 * kV);                 // threads a row
  constexpr int kSlots = kAppendThreads / kTpr;      // rows side by side
  const int b = blockIdx.x / a.seq_len, s = blockIdx.x - b * a.seq_len;
  const int c = threadIdx.x % kTpr * kV;
  const uint32_t row_lanes = ((1u << kTpr) - 1u) << (threadIdx.x % 32 / kTpr * kTpr);
  const int hq = a.num_q_heads, hkv = a.num_kv_heads, rows = hq + 2 * hkv;
  grid_launch_dependents();
  grid_dependency_wait();
  // the token's slot; asked for first, needed last
  const int pos = a.positions[b];
  const int fresh = a.num_new != nullptr ? min(max(a.num_new[b], 0), a.seq_len) : a.seq_len;
  const int cap = a.max_pages * a.page_size;
  const long long slot = (long long)pos + s;
  int page = -1, row = 0;  // -1: nowhere
  if (s < fresh && slot >= 0 && slot < cap) {
    const int i = (int)slot / a.page_size;
    row = (int)slot - i * a.page_size;
    page = a.page_table[b * a.table_stride + i];
    if (page >= a.num_pages) page = -1;
  }
  if (a.kv_lens_out != nullptr && s == 0 && threadIdx.x == 0)
    a.kv_lens_out[b] = (int)min((long long)max(pos, 0) + fresh, (long long)cap);

  float c1[kV], c2[kV], s1[kV], s2[kV];
  bool tables = false;
  for (int r0 = threadIdx.x / kTpr; r0 - (int)threadIdx.x / kTpr < rows; r0 += kSlots * kAppendRows) {
    uint4 u1[kAppendRows], u2[kAppendRows];
#pragma unroll
    for (int j = 0; j < kAppendRows; ++j) {
      const int r = r0 + j * kSlots;
      u1[j] = u2[j] = make_uint4(0, 0, 0, 0);
      if (r >= rows) continue;
      const T* src = r < hq ? static_cast<const T*>(a.q_in) + b * a.qi_stride_b + r * a.qi_stride_h + s * a.qi_stride_s
                     : r < hq + hkv
                         ? static_cast<const T*>(a.k_in) + b * a.k_stride_b + (r - hq) * a.k_stride_h + s * a.k_stride_s
                         : static_cast<const T*>(a.v_in) + b * a.v_stride_b + (r - hq - hkv) * a.v_stride_h + s * a.v_stride_s;
      u1[j] = *reinterpret_cast<const uint4*>(src + c);
      u2[j] = *reinterpret_cast<const uint4*>(src + c + D / 2);
    }
    if (!tables) {
      const CS* cp = static_cast<const CS*>(a.cos) + b * a.cs_stride_b + s * a.cs_stride_s + c;
      const CS* sp = static_cast<const CS*>(a.sin) + b * a.cs_stride_b + s * a.cs_stride_s + c;
      load_table<CS, kV>(cp, c1);
      load_table<CS, kV>(cp + D / 2, c2);
      load_table<CS, kV>(sp, s1);
      load_table<CS, kV>(sp + D / 2, s2);
      tables = true;
    }
#pragma unroll
    for (int j = 0; j < kAppendRows; ++j) {
      const int r = r0 + j * kSlots;
      if (r >= rows || (r >= hq && page < 0)) continue;  // the lanes of a row stay together
      T* dst;
      if (r >= hq + hkv) {
        dst = static_cast<T*>(a.v_pages) + page * a.vp_stride_p + (r - hq - hkv) * a.vp_stride_h + row * a.vp_stride_t;
      } else {
        const T* w;
        if (r < hq) {
          dst = static_cast<T*>(a.q_out) + b * a.qo_stride_b + r * a.qo_stride_h + s * a.qo_stride_s;
          w = static_cast<const T*>(a.q_norm_weight);
        } else {
          dst = static_cast<T*>(a.k_pages) + page * a.kp_stride_p + (r - hq) * a.kp_stride_h + row * a.kp_stride_t;
          w = static_cast<const T*>(a.k_norm_weight);
        }
        float x1[kV], x2[kV];
        Elem<T>::unpack(u1[j], x1);
        Elem<T>::unpack(u2[j], x2);
        if (w != nullptr) {
          float w1[kV], w2[kV];
          load_table<T, kV>(w + c, w1);
          load_table<T, kV>(w + c + D / 2, w2);
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < kV; ++i) ss += x1[i] * x1[i] + x2[i] * x2[i];
#pragma unroll
          for (int off = kTpr / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(row_lanes, ss, off);
          const float inv = rsqrtf(ss / (float)D + a.norm_eps);
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
        u1[j] = pack_vec<T>(x1);
        u2[j] = pack_vec<T>(x2);
      }
      *reinterpret_cast<uint4*>(dst + c) = u1[j];
      *reinterpret_cast<uint4*>(dst + c + D / 2) = u2[j];
    }
  }
}

template <typename T, typename CS, int THREADS, int ROWS>
cudaError_t launch_append_rows(const aicas_paged_append_params& p, cudaStream_t st) {
  const dim3 grid((unsigned)(p.batch * p.seq_len)), block(THREADS);
  switch (p.head_dim) {
    case 16: return launch_pdl(paged_append_kernel<T, CS, 16, THREADS, ROWS>, grid, block, 0, st, p);
    case 32: return launch_pdl(paged_append_kernel<T, CS, 32, THREADS, ROWS>, grid, block, 0, st, p);
    case 64: return launch_pdl(paged_append_kernel<T, CS, 64, THREADS, ROWS>, grid, block, 0, st, p);
    case 128: return launch_pdl(paged_append_kernel<T, CS, 128, THREADS, ROWS>, grid, block, 0, st, p);
  }
  return cudaErrorInvalidValue;
}

template <typename T, typename CS>
cudaError_t launch_append(const aicas_paged_append_params& p, cudaStream_t st) {
  // Few tokens (a decode step): a row a thread, 256 threads, the shortest way through (64 tokens of 16 + 2 * 8 heads of
  // 128: 2.6 against 5.1 us).  Many: one warp a CTA with four rows in flight each, 18 CTAs an SM (8192 tokens: 28.6
  // against 60.3 us).  Where they cross depends on a token's bytes and the tables' type, and 384 tokens are a middle:
  // 6 + 2 * 2 heads of 64 cross between 256 (2.4, 2.6) and 384 (3.8, 2.7); 16 + 2 * 8 heads of 128 near 1024 (7.7, 7.8;
  // 512: 4.8, 5.8) with fp32 tables and below 2048 (16.7, 14.9; 1024: 9.2, 13.2) with 16-bit ones.
  return p.batch * p.seq_len <= 384 ? launch_append_rows<T, CS, 256, 1>(p, st) : launch_append_rows<T, CS, 32, 4>(p, st);
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
