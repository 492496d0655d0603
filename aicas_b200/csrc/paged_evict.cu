// Eviction from a paged cache: of each (request, KV head) the first keep_first slots, the
// last keep_last, and of those between the ones of the largest weights, moved to the front
// in their order.
//
// Two launches.  paged_select_kernel finds the weight of the last slot that stays by radix
// selection (exact: equal weights go to the lower slot), lists the kept slots in order and
// moves their weights.  paged_move_kernel moves the rows: slot i of the cut cache was slot
// kept[i] >= i, so a CTA that reads a run of rows before it writes them, run after run,
// never reads what it has overwritten; the columns of a row are independent, so they are
// given to CTAs of their own.
#include <cstdio>

#include "common.cuh"
#include "paged_int4.cuh"

namespace aicas {
namespace {

constexpr int kSelectThreads = 512, kSelectWarps = kSelectThreads / 32;

// A weight as a whole number of the same order; NaN below all numbers, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelectThreads) paged_select_kernel(const __grid_constant__ aicas_paged_evict_params a) {
  __shared__ int hist[256];
  __shared__ uint32_t s_key;
  __shared__ int s_need, s_eq[kSelectWarps], s_kept[kSelectWarps];
  const int b = blockIdx.x / a.num_kv_heads, h = blockIdx.x - b * a.num_kv_heads;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  grid_launch_dependents();
  grid_dependency_wait();
  const int n = min(max(a.kv_lens[b], 0), a.max_pages * a.page_size);
  const float* w = a.weights + b * a.w_stride_b + h * a.w_stride_h;
  float* wo = a.weights_out + b * a.wo_stride_b + h * a.wo_stride_h;
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.keep;
  if (n <= a.longer_than) {
    for (int i = tid; i < a.keep; i += kSelectThreads) kept[i] = i < n ? i : -1;
    if (wo != w)
      for (int i = tid; i < n; i += kSelectThreads) wo[i] = w[i];
    return;
  }
  // the key of the last slot that stays for its weight, a byte at a time
  const int lo = a.keep_first, hi = n - a.keep_last;
  int need = a.keep - a.keep_first - a.keep_last;
  uint32_t key = 0;
  if (need > 0)
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int t = lo + tid; t < hi; t += kSelectThreads) {
        const uint32_t u = order_of(w[t]);
        if (shift == 24 || u >> (shift + 8) == key >> (shift + 8)) atomicAdd(&hist[u >> shift & 255u], 1);
      }
      __syncthreads();
      if (warp == 0) {  // lane: 8 bytes' counts, from the largest down
        int c[8], sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += c[e] = hist[255 - 8 * lane - e];
        int before = sum;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, before, off);
          if (lane >= off) before += v;
        }
        before -= sum;
        if (before < need && need <= before + sum)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (before < need && need <= before + c[e]) {
              s_key = key | (uint32_t)(255 - 8 * lane - e) << shift;
              s_need = need - before;
            }
            before += c[e];
          }
      }
      __syncthreads();
      key = s_key, need = s_need;
      __syncthreads();
    }
  // need: how many of the slots with that key stay, the lower ones first
  int eq_base = 0, kept_base = 0;
  for (int t0 = 0; t0 < n; t0 += kSelectThreads) {
    const int t = t0 + tid;
    const float x = t < n ? w[t] : 0.f;
    const bool forced = t < lo || t >= hi, in = t < n;
    const uint32_t u = order_of(x);
    const bool equal = in && !forced && need > 0 && u == key;
    const uint32_t eq = __ballot_sync(0xffffffffu, equal), below = (1u << lane) - 1u;
    if (lane == 0) s_eq[warp] = __popc(eq);
    __syncthreads();
    int eq_before = eq_base + __popc(eq & below);
    for (int i = 0; i < kSelectWarps; ++i) {
      if (i < warp) eq_before += s_eq[i];
      eq_base += s_eq[i];
    }
    const bool stays = in && (forced || (need > 0 && (u > key || (equal && eq_before < need))));
    const uint32_t st = __ballot_sync(0xffffffffu, stays);
    if (lane == 0) s_kept[warp] = __popc(st);
    __syncthreads();
    int at = kept_base + __popc(st & below);
    for (int i = 0; i < kSelectWarps; ++i) {
      if (i < warp) at += s_kept[i];
      kept_base += s_kept[i];
    }
    if (stays) {  // at <= t, and this run's weights are read
      kept[at] = t;
      wo[at] = x;
    }
  }
  __syncthreads();
  for (int t = a.keep + tid; t < n; t += kSelectThreads) wo[t] = 0.f;
}

constexpr int kMoveThreads = 256, kMoveRows = 4;

struct MoveArgs {
  aicas_paged_evict_params p;
  int parts[AICAS_EVICT_MAX_PLANES + 1];  // the planes' first column parts
  int part_bytes[AICAS_EVICT_MAX_PLANES];
};

template <typename V>
__device__ void move_rows(const aicas_paged_evict_params& a, const aicas_evict_plane& pl, const int32_t* kept, int b, int h,
                          int part_bytes, int part) {
  const int tpr = part_bytes / (int)sizeof(V), rows = kMoveThreads / tpr;
  const int r = threadIdx.x / tpr;
  const int64_t col = (int64_t)part * part_bytes + (threadIdx.x - r * tpr) * (int)sizeof(V);
  char* data = static_cast<char*>(pl.data) + h * pl.stride_h + col;
  const int32_t* table = a.page_table + b * a.table_stride;
  const auto at = [&](int slot) -> char* {
    const int i = slot / a.page_size, page = table[i];
    return page >= 0 && page < a.num_pages ? data + page * pl.stride_p + (slot - i * a.page_size) * pl.stride_t : nullptr;
  };
  for (int i0 = 0; i0 < a.keep; i0 += rows * kMoveRows) {
    V v[kMoveRows] = {};
    char* to[kMoveRows];
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k) {
      const int i = i0 + k * rows + r;
      to[k] = nullptr;
      if (r < rows && i < a.keep) {
        const int from = kept[i];
        if (from > i) {
          const char* src = at(from);
          to[k] = at(i);
          if (src != nullptr) v[k] = *reinterpret_cast<const V*>(src);
        }
      }
    }
    __syncthreads();  // the run is read
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k)
      if (to[k] != nullptr) *reinterpret_cast<V*>(to[k]) = v[k];
  }
}

__global__ void __launch_bounds__(kMoveThreads) paged_move_kernel(const __grid_constant__ MoveArgs m) {
  const aicas_paged_evict_params& a = m.p;
  const int parts = m.parts[a.num_planes];
  const int pair = blockIdx.x / parts, at = blockIdx.x - pair * parts;
  const int b = pair / a.num_kv_heads, h = pair - b * a.num_kv_heads;
  grid_launch_dependents();
  grid_dependency_wait();
  if (a.kv_lens_out != nullptr && at == 0 && h == 0 && threadIdx.x == 0) {
    const int n = min(max(a.kv_lens[b], 0), a.max_pages * a.page_size);
    a.kv_lens_out[b] = n > a.longer_than ? a.keep : n;
  }
  int i = 0;
  while (at >= m.parts[i + 1]) ++i;
  const aicas_evict_plane& pl = a.plane[i];
  const int32_t* kept = a.kept + (int64_t)pair * a.keep;
  const int bytes = m.part_bytes[i], part = at - m.parts[i];
  if (bytes % 16 == 0) move_rows<uint4>(a, pl, kept, b, h, bytes, part);
  else if (bytes == 8) move_rows<uint2>(a, pl, kept, b, h, bytes, part);
  else move_rows<uint32_t>(a, pl, kept, b, h, bytes, part);
}

}  // namespace

int run_paged_evict(const aicas_paged_evict_params* p, cudaStream_t stream, char* err, size_t errlen) {
  const unsigned pairs = (unsigned)(p->batch * p->num_kv_heads);
  cudaError_t e = launch_pdl(paged_select_kernel, dim3(pairs), dim3(kSelectThreads), 0, stream, *p);
  MoveArgs m;
  m.p = *p;
  m.parts[0] = 0;
  for (int i = 0; i < p->num_planes; ++i) {
    const int bytes = (int)p->plane[i].row_bytes;
    m.part_bytes[i] = bytes > 128 ? 128 : bytes;
    m.parts[i + 1] = m.parts[i] + (bytes + m.part_bytes[i] - 1) / m.part_bytes[i];
  }
  if (e == cudaSuccess)
    e = launch_pdl(paged_move_kernel, dim3(pairs * m.parts[p->num_planes]), dim3(kMoveThreads), 0, stream, m);
  if (e == cudaSuccess) return AICAS_OK;
  snprintf(err, errlen, "paged evict launch: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
  return AICAS_ERR_CUDA;
}

}  // namespace aicas
