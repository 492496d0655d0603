// GQA decode attention (one query token per request) over a paged cache of 4-bit rows:
//   k_t = sk_t * ck_t + lk_t,  v_t = sv_t * cv_t + lv_t  (codes 0..15; scale and least a group)
//   o = softmax(scale * q K^T) V over the slots [start, len) of a request,
//   lse = log2(sum_j 2^(scale log2(e) q.k_j)).
//
// One CTA a (request, KV head, block of up to 8 query heads), a slot a warp at a time.
#include <cstdio>
#include <cstring>

#include "common.cuh"
#include "paged_int4.cuh"

namespace aicas {
namespace {

constexpr int kWarps = 8, kHeads = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) paged_decode_int4_kernel(const __grid_constant__ aicas_paged_decode_int4_params a) {
  constexpr int kE = D / 32;  // elements a lane
  __shared__ float red[kWarps][kHeads][D + 2];
  const int group = a.num_q_heads / a.num_kv_heads, blocks = (group + kHeads - 1) / kHeads;
  const int blk = blockIdx.x % blocks, kvh = blockIdx.x / blocks % a.num_kv_heads, b = blockIdx.x / blocks / a.num_kv_heads;
  const int h0 = kvh * group + blk * kHeads, heads = min(kHeads, group - blk * kHeads);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, d0 = lane * kE;
  grid_launch_dependents();
  grid_dependency_wait();
  const int cap = a.max_pages * a.page_size;
  const int len = a.kv_lens != nullptr ? min(max(a.kv_lens[b], 0), cap) : cap;
  const int start = a.kv_starts != nullptr ? max(a.kv_starts[b], 0) : 0;
  const float c = a.sm_scale * 1.4426950408889634f;
  float q[kHeads][kE], o[kHeads][kE], m[kHeads], l[kHeads];
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      o[h][e] = 0.f;
      q[h][e] = h < heads ? Elem<T>::to_float(static_cast<const T*>(a.q)[b * a.q_stride_b + (h0 + h) * a.q_stride_h + d0 + e]) : 0.f;
    }
  }
  for (int t = start + warp; t < len; t += kWarps) {
    const int i = t / a.page_size, row = t - i * a.page_size, page = a.page_table[b * a.table_stride + i];
    float kv[2][kE] = {};
    if (page >= 0 && page < a.num_pages) {
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const aicas_int4_pages& p = a.kv[side];
        const uint8_t* codes = static_cast<const uint8_t*>(p.codes) + page * p.cs_p + kvh * p.cs_h + row * p.cs_t;
        const T* pair = static_cast<const T*>(p.scales) + page * p.ss_p + kvh * p.ss_h + row * p.ss_t + d0 / a.group_size * 2;
        const float s = Elem<T>::to_float(pair[0]), least = Elem<T>::to_float(pair[1]);
#pragma unroll
        for (int e = 0; e < kE; ++e) kv[side][e] = fmaf(s, (float)(codes[(d0 + e) / 2] >> (4 * ((d0 + e) & 1)) & 15), least);
      }
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < kE; ++e) s = fmaf(q[h][e], kv[0][e], s);
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      s *= c;
      const float mn = fmaxf(m[h], s), use = mn == -INFINITY ? 0.f : mn;
      const float alpha = exp2f(m[h] - use), p = exp2f(s - use);
      m[h] = mn, l[h] = fmaf(l[h], alpha, p);
#pragma unroll
      for (int e = 0; e < kE; ++e) o[h][e] = fmaf(o[h][e], alpha, p * kv[1][e]);
    }
  }
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
#pragma unroll
    for (int e = 0; e < kE; ++e) red[warp][h][d0 + e] = o[h][e];
    if (lane == 0) red[warp][h][D] = m[h], red[warp][h][D + 1] = l[h];
  }
  __syncthreads();
  for (int x = threadIdx.x; x < heads * D; x += kWarps * 32) {
    const int h = x / D, d = x % D;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, red[w][h][D]);
    const float use = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(red[w][h][D] - use);
      L = fmaf(f, red[w][h][D + 1], L), O = fmaf(f, red[w][h][d], O);
    }
    static_cast<T*>(a.out)[b * a.o_stride_b + (h0 + h) * a.o_stride_h + d] = Elem<T>::from_float(L == 0.f ? 0.f : O / L);
    if (a.lse != nullptr && d == 0) a.lse[(int64_t)b * a.num_q_heads + h0 + h] = L == 0.f ? -INFINITY : M + log2f(L);
  }
}

template <typename T>
cudaError_t launch_decode_int4(const aicas_paged_decode_int4_params& p, cudaStream_t st) {
  const int blocks = (p.num_q_heads / p.num_kv_heads + kHeads - 1) / kHeads;
  const dim3 grid((unsigned)(p.batch * p.num_kv_heads * blocks)), block(kWarps * 32);
  return p.head_dim == 64 ? launch_pdl(paged_decode_int4_kernel<T, 64>, grid, block, 0, st, p)
                          : launch_pdl(paged_decode_int4_kernel<T, 128>, grid, block, 0, st, p);
}

}  // namespace

size_t paged_decode_int4_workspace(int) { return 256; }

int run_paged_decode_int4(const aicas_paged_decode_int4_params* p, int, void*, cudaStream_t stream, char* err, size_t errlen) {
  const cudaError_t e = p->dtype == AICAS_DTYPE_F16 ? launch_decode_int4<__half>(*p, stream) : launch_decode_int4<__nv_bfloat16>(*p, stream);
  if (e == cudaSuccess) return AICAS_OK;
  snprintf(err, errlen, "paged 4-bit decode launch: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
  return AICAS_ERR_CUDA;
}

}  // namespace aicas
