// What attention gave to each cached slot, added up for an eviction:
//   w[b, h, t] += sum over queries s and heads j of the group of 2^(c q[b, j, s].k[b, h, t] - lse[b, j, s]),
// c = scale log2(e), for the slots start <= t <= len - S + s that query s sees.
//
// A slot has one writer and its sum one order, so results repeat to the bit.  A thread a
// slot, its row of K read once for each block of 8 queries.
#include <cstdio>
#include <type_traits>

#include "common.cuh"
#include "paged_int4.cuh"

namespace aicas {
namespace {

constexpr int kThreads = 128, kBlock = 8;

// 8 elements d.. of a cached row, as floats.
template <typename T, bool INT4>
__device__ __forceinline__ void load_row8(const aicas_paged_weights_params& a, int page, int h, int row, int d, float* f) {
  if constexpr (INT4) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.k_pages) + page * a.kp_stride_p +
                                                          h * a.kp_stride_h + row * a.kp_stride_t + d / 2);
    const T* pair = static_cast<const T*>(a.k_scales) + page * a.ks_stride_p + h * a.ks_stride_h + row * a.ks_stride_t +
                    d / a.group_size * 2;
    const float s = Elem<T>::to_float(pair[0]), least = Elem<T>::to_float(pair[1]);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fmaf(s, (float)(u >> (4 * e) & 15u), least);
  } else {
    const T* p = static_cast<const T*>(a.k_pages) + page * a.kp_stride_p + h * a.kp_stride_h + row * a.kp_stride_t + d;
#pragma unroll
    for (int e = 0; e < 8; e += Elem<T>::kPerVec) Elem<T>::unpack(*reinterpret_cast<const uint4*>(p + e), f + e);
  }
}

template <typename T, bool INT4>
__global__ void __launch_bounds__(kThreads) paged_weights_kernel(const __grid_constant__ aicas_paged_weights_params a) {
  __shared__ float q_s[kBlock][128], lse_s[kBlock];
  __shared__ int end_s[kBlock];
  const int group = a.num_q_heads / a.num_kv_heads, D = a.head_dim, cap = a.max_pages * a.page_size;
  const int chunks = (cap + kThreads - 1) / kThreads;
  const int kvh = blockIdx.x / chunks % a.num_kv_heads, b = blockIdx.x / chunks / a.num_kv_heads;
  grid_launch_dependents();
  grid_dependency_wait();
  const int len = a.kv_lens != nullptr ? min(max(a.kv_lens[b], 0), cap) : cap;
  const int start = a.kv_starts != nullptr ? max(a.kv_starts[b], 0) : 0;
  const int t0 = blockIdx.x % chunks * kThreads, t = t0 + threadIdx.x;
  if (t0 >= len || t0 + kThreads <= start) return;
  int page = -1, row = 0;
  if (t >= start && t < len) {
    const int i = t / a.page_size;
    row = t - i * a.page_size;
    page = a.page_table[b * a.table_stride + i];
  }
  const float c = a.sm_scale * 1.4426950408889634f;
  float sum = 0.f;
  for (int r0 = 0; r0 < group * a.seq_len; r0 += kBlock) {
    __syncthreads();
    for (int x = threadIdx.x; x < kBlock * D; x += kThreads) {
      const int r = r0 + x / D, j = kvh * group + r / a.seq_len, s = r % a.seq_len;
      if (r < group * a.seq_len) {
        q_s[x / D][x % D] = Elem<T>::to_float(static_cast<const T*>(a.q)[b * a.q_stride_b + j * a.q_stride_h + s * a.q_stride_s + x % D]);
        if (x % D == 0) {
          lse_s[x / D] = a.lse[b * a.lse_stride_b + j * a.lse_stride_h + s * a.lse_stride_s];
          end_s[x / D] = len - a.seq_len + 1 + s;
        }
      } else {
        q_s[x / D][x % D] = 0.f;
        if (x % D == 0) end_s[x / D] = 0;
      }
    }
    __syncthreads();
    if (t >= start && t < len) {
      float s[kBlock] = {};
      if (page >= 0 && page < a.num_pages)
        for (int d = 0; d < D; d += 8) {
          float k[8];
          load_row8<T, INT4>(a, page, kvh, row, d, k);
#pragma unroll
          for (int r = 0; r < kBlock; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[r] = fmaf(q_s[r][d + e], k[e], s[r]);
        }
#pragma unroll
      for (int r = 0; r < kBlock; ++r)
        if (t < end_s[r] && lse_s[r] != -INFINITY) sum += exp2f(fmaf(s[r], c, -lse_s[r]));
    }
  }
  if (t >= start && t < len) a.weights[b * a.w_stride_b + kvh * a.w_stride_h + t] += sum;
}

template <typename T>
cudaError_t launch_weights(const aicas_paged_weights_params& p, cudaStream_t st) {
  const int64_t chunks = ((int64_t)p.max_pages * p.page_size + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)(chunks * p.batch * p.num_kv_heads)), block(kThreads);
  if constexpr (!std::is_same<T, float>::value) {
    if (p.group_size != 0) return launch_pdl(paged_weights_kernel<T, true>, grid, block, 0, st, p);
  }
  return launch_pdl(paged_weights_kernel<T, false>, grid, block, 0, st, p);
}

}  // namespace

int run_paged_weights(const aicas_paged_weights_params* p, int, cudaStream_t stream, char* err, size_t errlen) {
  cudaError_t e = cudaErrorInvalidValue;
  switch (p->dtype) {
    case AICAS_DTYPE_F32: e = launch_weights<float>(*p, stream); break;
    case AICAS_DTYPE_F16: e = launch_weights<__half>(*p, stream); break;
    case AICAS_DTYPE_BF16: e = launch_weights<__nv_bfloat16>(*p, stream); break;
  }
  if (e == cudaSuccess) return AICAS_OK;
  snprintf(err, errlen, "paged weights launch: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
  return AICAS_ERR_CUDA;
}

}  // namespace aicas
