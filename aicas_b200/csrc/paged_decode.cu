// GQA decode attention (one query token per request) over a paged KV cache:
//   o = softmax(scale * q K^T) V over the slots [start, len) of a request, slot
//   t being row t % page_size of page table[b, t / page_size];
//   lse = log2(sum_j 2^(scale log2(e) q.k_j)).
// fp32 online softmax in base 2.  A CTA serves one query head; its warps take
// the slots in turn and their states are merged in shared memory.
#include <cstdio>

#include "common.cuh"
#include "paged.cuh"

namespace aicas {
namespace {

template <typename T, int D>
__global__ void __launch_bounds__(128) paged_decode_kernel(const aicas_paged_decode_params a) {
  constexpr int kPer = (D + 31) / 32;
  __shared__ float sm[4], sl[4], so[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / a.num_q_heads, h = blockIdx.x % a.num_q_heads;
  const int kvh = h / (a.num_q_heads / a.num_kv_heads);
  const int cap = a.max_pages * a.page_size;
  const int len = a.kv_lens != nullptr ? min(max(a.kv_lens[b], 0), cap) : cap;
  const int start = a.kv_starts != nullptr ? min(max(a.kv_starts[b], 0), len) : 0;
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride_b + h * a.q_stride_h;
  const float scale = a.sm_scale * 1.4426950408889634f;
  float qf[kPer], o[kPer] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) qf[i] = lane + 32 * i < D ? Elem<T>::to_float(q[lane + 32 * i]) : 0.f;
  for (int t = start + warp; t < len; t += 4) {
    const int page = a.page_table[b * a.table_stride + t / a.page_size], row = t % a.page_size;
    const bool in = page >= 0 && page < a.num_pages;
    const T* k = static_cast<const T*>(a.k_pages) + page * a.kp_stride_p + kvh * a.kp_stride_h + row * a.kp_stride_t;
    const T* v = static_cast<const T*>(a.v_pages) + page * a.vp_stride_p + kvh * a.vp_stride_h + row * a.vp_stride_t;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (in && lane + 32 * i < D) s += qf[i] * Elem<T>::to_float(k[lane + 32 * i]);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= scale;
    const float mn = fmaxf(m, s), use = mn == -INFINITY ? 0.f : mn;
    const float r = exp2f(m - use), p = exp2f(s - use);
    l = l * r + p;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      o[i] = o[i] * r + (in && lane + 32 * i < D ? p * Elem<T>::to_float(v[lane + 32 * i]) : 0.f);
    m = mn;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + 32 * i < D) so[warp][lane + 32 * i] = o[i];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  __syncthreads();
  float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), L = 0.f;
  const float use = M == -INFINITY ? 0.f : M;
  for (int w = 0; w < 4; ++w) L += sl[w] * exp2f(sm[w] - use);
  for (int d = threadIdx.x; d < D; d += 128) {
    float O = 0.f;
    for (int w = 0; w < 4; ++w) O += so[w][d] * exp2f(sm[w] - use);
    static_cast<T*>(a.out)[b * a.o_stride_b + h * a.o_stride_h + d] = Elem<T>::from_float(len > start ? O / L : 0.f);
  }
  if (a.lse != nullptr && threadIdx.x == 0)
    a.lse[(int64_t)b * a.num_q_heads + h] = len > start ? M + log2f(L) : -INFINITY;
}

template <typename T>
cudaError_t launch_paged(const aicas_paged_decode_params& p, cudaStream_t st) {
  const unsigned grid = (unsigned)(p.batch * p.num_q_heads);
  switch (p.head_dim) {
    case 16: paged_decode_kernel<T, 16><<<grid, 128, 0, st>>>(p); break;
    case 32: paged_decode_kernel<T, 32><<<grid, 128, 0, st>>>(p); break;
    case 64: paged_decode_kernel<T, 64><<<grid, 128, 0, st>>>(p); break;
    case 128: paged_decode_kernel<T, 128><<<grid, 128, 0, st>>>(p); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace

size_t paged_decode_workspace(const aicas_paged_decode_params*, int) { return 0; }

int run_paged_decode(const aicas_paged_decode_params* p, int, void*, cudaStream_t stream, unsigned int*, char* err,
                     size_t errlen) {
  cudaError_t e = cudaErrorInvalidValue;
  switch (p->dtype) {
    case AICAS_DTYPE_F32: e = launch_paged<float>(*p, stream); break;
    case AICAS_DTYPE_F16: e = launch_paged<__half>(*p, stream); break;
    case AICAS_DTYPE_BF16: e = launch_paged<__nv_bfloat16>(*p, stream); break;
  }
  if (e != cudaSuccess) {
    snprintf(err, errlen, "paged decode launch: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
    return AICAS_ERR_CUDA;
  }
  return AICAS_OK;
}

}  // namespace aicas
