// Append to and reads from a paged KV cache of 4-bit rows.
//
//   y = x * rsqrt(mean x^2 + eps) * w        (with a norm weight, else y = x)
//   r = y * cos + rotate_half(y) * sin,      rotate_half(y) = cat(-y[D/2:], y[:D/2])
//   of each group of 64 (or D) elements of r (keys) and v:
//     least = T(min r),  scale = T((max r - least) / 15)
//     code  = (r - least) / scale to the nearest of 0..15   (0 where scale is 0)
//   read back as fma(scale, code, least), rounded to T.
//
// Rounding of r: paged_append.cu's (fp32 tables: fp32 to the code; 16-bit tables: every
// operation).  The codes are taken against the rounded least and scale, so that what
// rounding those two moved is not added to a code's own half step.
#include <cstdio>
#include <type_traits>

#include "common.cuh"
#include "paged_int4.cuh"
#include "paged_rows.cuh"

namespace aicas {
namespace {

// Least and largest of a group over its TPR lanes; NaN as least where an element is no finite number.
template <int TPR>
__device__ __forceinline__ void group_range(uint32_t lanes, float& lo, float& hi, bool bad) {
#pragma unroll
  for (int off = TPR / 2; off >= 1; off >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(lanes, lo, off));
    hi = fmaxf(hi, __shfl_xor_sync(lanes, hi, off));
  }
  if (__any_sync(lanes, bad)) lo = __int_as_float(0x7fc00000);
}

// (scale, least) of a group as the cache holds them, and as floats.
template <typename T>
__device__ __forceinline__ uint32_t group_levels(float lo, float hi, float& scale, float& least) {
  const T l = Elem<T>::from_float(lo);
  least = Elem<T>::to_float(l);
  const T s = Elem<T>::from_float((hi - least) / 15.f);
  scale = Elem<T>::to_float(s);
  if (!(fabsf(scale) < INFINITY)) scale = least = __int_as_float(0x7fc00000);  // infinities, NaN
  union {
    T t[2];
    uint32_t u;
  } r;
  r.t[0] = Elem<T>::from_float(scale), r.t[1] = Elem<T>::from_float(least);
  return r.u;
}

__device__ __forceinline__ uint32_t codes_of(const float* x, float scale, float least) {
  // the reciprocal of a scale near the least normal number would be infinite
  const float lift = scale < 1e-30f ? 0x1p64f : 1.f;
  const float inv = scale > 0.f ? 1.f / (scale * lift) : 0.f;
  scale *= lift;
  // 1.5 x 2^23: a sum with it has the number, rounded to a whole one, in its low bits
  constexpr float kWhole = 12582912.f;
  uint32_t u = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // 16-bit values often lie on the border between two codes, where a product with the
    // reciprocal may fall on either side: what the nearest code leaves, which fma gives
    // exactly, brings the quotient back to the border
    const float d = (x[i] - least) * lift, t = d * inv, near = (t + kWhole) - kWhole;
    const float q = fmaf(fmaf(-near, scale, d), inv, near);
    u |= (__float_as_uint(fminf(fmaxf(q, 0.f), 15.f) + kWhole) & 15u) << (4 * i);
  }
  return u;
}

// HBM bound: the token's rows are read once, q written in 16 and k and v in 4 bits.  The
// CTA, its threads and the rows in flight are paged_append.cu's: a row (one head of q, k
// or v) belongs to D / 16 threads, each with one 16-byte vector of the row's first half
// and the matching one of its second half, so that the rotation needs no exchange, and
// with groups of 64 in rows of 128 each half is a group.
template <typename T, typename CS, int D, bool HALVES, int THREADS, int ROWS>
__global__ void __launch_bounds__(THREADS) paged_append_int4_kernel(const __grid_constant__ aicas_paged_append_int4_params a) {
  constexpr bool kRoundEach = std::is_same<T, CS>::value;
  constexpr int kV = 8;
  constexpr int kTpr = D / (2 * kV);
  constexpr int kSlots = THREADS / kTpr;
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
  for (int r0 = threadIdx.x / kTpr; r0 - (int)threadIdx.x / kTpr < rows; r0 += kSlots * ROWS) {
    uint4 u1[ROWS], u2[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
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
      load_floats<CS, kV>(cp, c1);
      load_floats<CS, kV>(cp + D / 2, c2);
      load_floats<CS, kV>(sp, s1);
      load_floats<CS, kV>(sp + D / 2, s2);
      tables = true;
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int r = r0 + j * kSlots;
      if (r >= rows || (r >= hq && page < 0)) continue;  // the lanes of a row stay together
      float x1[kV], x2[kV];
      Elem<T>::unpack(u1[j], x1);
      Elem<T>::unpack(u2[j], x2);
      if (r < hq + hkv) {
        const T* w = static_cast<const T*>(r < hq ? a.q_norm_weight : a.k_norm_weight);
        if (w != nullptr) {
          float w1[kV], w2[kV];
          load_floats<T, kV>(w + c, w1);
          load_floats<T, kV>(w + c + D / 2, w2);
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < kV; ++i) ss += x1[i] * x1[i] + x2[i] * x2[i];
#pragma unroll
          for (int off = kTpr / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(row_lanes, ss, off);
          const float inv = rsqrtf(ss / (float)D + a.norm_eps);
          normed_pair<T, kRoundEach, kV>(x1, x2, w1, w2, inv);
        }
        rotated_pair<T, kRoundEach, kV>(x1, x2, c1, c2, s1, s2);
      }
      if (r < hq) {
        T* dst = static_cast<T*>(a.q_out) + b * a.qo_stride_b + r * a.qo_stride_h + s * a.qo_stride_s;
        *reinterpret_cast<uint4*>(dst + c) = pack_vec<T>(x1);
        *reinterpret_cast<uint4*>(dst + c + D / 2) = pack_vec<T>(x2);
        continue;
      }
      const aicas_int4_pages& to = a.kv[r >= hq + hkv];
      const int h = r >= hq + hkv ? r - hq - hkv : r - hq;
      if (kRoundEach && r < hq + hkv) {
#pragma unroll
        for (int i = 0; i < kV; ++i) x1[i] = rounded<T>(x1[i]), x2[i] = rounded<T>(x2[i]);
      }
      float lo1 = x1[0], hi1 = x1[0], lo2 = x2[0], hi2 = x2[0], bad1 = 0.f, bad2 = 0.f;
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        lo1 = fminf(lo1, x1[i]), hi1 = fmaxf(hi1, x1[i]), bad1 = fmaf(x1[i], 0.f, bad1);
        lo2 = fminf(lo2, x2[i]), hi2 = fmaxf(hi2, x2[i]), bad2 = fmaf(x2[i], 0.f, bad2);
      }
      if constexpr (HALVES) {
        group_range<kTpr>(row_lanes, lo1, hi1, bad1 != 0.f);  // 0 but where an element is no finite number
        group_range<kTpr>(row_lanes, lo2, hi2, bad2 != 0.f);
      } else {
        lo1 = fminf(lo1, lo2), hi1 = fmaxf(hi1, hi2);
        group_range<kTpr>(row_lanes, lo1, hi1, bad1 + bad2 != 0.f);
      }
      float scale1, least1, scale2, least2;
      const uint32_t p1 = group_levels<T>(lo1, hi1, scale1, least1);
      const uint32_t p2 = HALVES ? group_levels<T>(lo2, hi2, scale2, least2) : (scale2 = scale1, least2 = least1, 0u);
      uint8_t* codes = static_cast<uint8_t*>(to.codes) + page * to.cs_p + h * to.cs_h + row * to.cs_t;
      *reinterpret_cast<uint32_t*>(codes + c / 2) = codes_of(x1, scale1, least1);
      *reinterpret_cast<uint32_t*>(codes + c / 2 + D / 4) = codes_of(x2, scale2, least2);
      if (c == 0) {
        T* pair = static_cast<T*>(to.scales) + page * to.ss_p + h * to.ss_h + row * to.ss_t;
        if constexpr (HALVES) {
          *reinterpret_cast<uint2*>(pair) = make_uint2(p1, p2);
        } else {
          *reinterpret_cast<uint32_t*>(pair) = p1;
        }
      }
    }
  }
}

template <typename T, typename CS, int D, bool HALVES>
cudaError_t launch_append_sized(const aicas_paged_append_int4_params& p, cudaStream_t st) {
  const dim3 grid((unsigned)(p.batch * p.seq_len));
  // as paged_append.cu chooses: the shortest way for a decode step, more CTAs and rows in flight for prompts
  return p.batch * p.seq_len <= 384
             ? launch_pdl(paged_append_int4_kernel<T, CS, D, HALVES, 256, 1>, grid, dim3(256), 0, st, p)
             : launch_pdl(paged_append_int4_kernel<T, CS, D, HALVES, 32, 4>, grid, dim3(32), 0, st, p);
}

template <typename T, typename CS>
cudaError_t launch_append(const aicas_paged_append_int4_params& p, cudaStream_t st) {
  if (p.head_dim == 64) return launch_append_sized<T, CS, 64, false>(p, st);
  return p.group_size == 64 ? launch_append_sized<T, CS, 128, true>(p, st) : launch_append_sized<T, CS, 128, false>(p, st);
}

// ------------------------------------------------------------------ reads

// HBM bound: 8 elements a thread, 4 bytes of codes in and 16 bytes out.
template <typename T, int D, bool HALVES>
__global__ void __launch_bounds__(256) paged_read_int4_kernel(const __grid_constant__ aicas_paged_read_int4_params a) {
  constexpr int kTpr = D / 8, kSlots = 256 / kTpr;
  grid_launch_dependents();
  grid_dependency_wait();
  const int64_t total = (int64_t)a.batch * 2 * a.num_kv_heads * a.seq_len;
  for (int64_t r = (int64_t)blockIdx.x * kSlots + threadIdx.x / kTpr; r < total; r += (int64_t)gridDim.x * kSlots) {
    const int s = (int)(r % a.seq_len);
    const int64_t head = r / a.seq_len;
    const int h = (int)(head % a.num_kv_heads), side = (int)(head / a.num_kv_heads) & 1;
    const int b = (int)(head / (2 * a.num_kv_heads));
    const int c = threadIdx.x % kTpr * 8;
    const int fresh = a.num_tokens != nullptr ? a.num_tokens[b] : a.seq_len;
    const long long slot = (long long)a.positions[b] + s;
    float f[8] = {};
    if (s < fresh && slot >= 0 && slot < (long long)a.max_pages * a.page_size) {
      const int i = (int)slot / a.page_size, row = (int)slot - i * a.page_size;
      const int page = a.page_table[b * a.table_stride + i];
      if (page >= 0 && page < a.num_pages) {
        const aicas_int4_pages& from = a.kv[side];
        const uint32_t u = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(from.codes) + page * from.cs_p +
                                                              h * from.cs_h + row * from.cs_t + c / 2);
        const T* pair = static_cast<const T*>(from.scales) + page * from.ss_p + h * from.ss_h + row * from.ss_t +
                        (HALVES && c >= D / 2 ? 2 : 0);
        const float scale = Elem<T>::to_float(pair[0]), least = Elem<T>::to_float(pair[1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = fmaf(scale, (float)(u >> (4 * e) & 15u), least);
      }
    }
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out[side]) + b * a.out_stride_b + h * a.out_stride_h + s * a.out_stride_s + c) =
        pack_vec<T>(f);
  }
}

template <typename T>
cudaError_t launch_read(const aicas_paged_read_int4_params& p, cudaStream_t st) {
  const int64_t rows = (int64_t)p.batch * 2 * p.num_kv_heads * p.seq_len, slots = 256 / (p.head_dim / 8);
  const int64_t ctas = (rows + slots - 1) / slots;
  const dim3 grid((unsigned)(ctas < 1 << 20 ? ctas : 1 << 20)), block(256);
  if (p.head_dim == 64) return launch_pdl(paged_read_int4_kernel<T, 64, false>, grid, block, 0, st, p);
  return p.group_size == 64 ? launch_pdl(paged_read_int4_kernel<T, 128, true>, grid, block, 0, st, p)
                            : launch_pdl(paged_read_int4_kernel<T, 128, false>, grid, block, 0, st, p);
}

int status(cudaError_t e, const char* what, char* err, size_t errlen) {
  if (e == cudaSuccess) return AICAS_OK;
  snprintf(err, errlen, "%s launch: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
  return AICAS_ERR_CUDA;
}

}  // namespace

int run_paged_append_int4(const aicas_paged_append_int4_params* p, cudaStream_t stream, char* err, size_t errlen) {
  const bool f32cs = p->cs_dtype == AICAS_DTYPE_F32;
  cudaError_t e = cudaErrorInvalidValue;
  if (p->dtype == AICAS_DTYPE_F16)
    e = f32cs ? launch_append<__half, float>(*p, stream) : launch_append<__half, __half>(*p, stream);
  else if (p->dtype == AICAS_DTYPE_BF16)
    e = f32cs ? launch_append<__nv_bfloat16, float>(*p, stream) : launch_append<__nv_bfloat16, __nv_bfloat16>(*p, stream);
  return status(e, "paged 4-bit append", err, errlen);
}

int run_paged_read_int4(const aicas_paged_read_int4_params* p, cudaStream_t stream, char* err, size_t errlen) {
  return status(p->dtype == AICAS_DTYPE_F16 ? launch_read<__half>(*p, stream) : launch_read<__nv_bfloat16>(*p, stream),
                "paged 4-bit read", err, errlen);
}

}  // namespace aicas
