// Eviction from a paged cache: of each (request, KV head) the first keep_first slots, the
// last keep_last, and of those between the ones of the largest weights, moved to the front
// in their order.
//
// The selection finds the weight of the last slot that stays (exact: equal weights go to the
// lower slot), lists the kept slots in order and moves their weights; then the rows are moved.
// Slot i of the cut cache was slot kept[i] >= i, so a CTA that reads a run of rows before it
// writes them, run after run, never reads what it has overwritten; the columns of a row are
// independent, so where there are few pairs, CTAs share a row by its columns.  Short caches of
// few pairs do both in one launch, a cluster of CTAs a pair; the others in two.
//
// Bound: HBM, for the rows, after a selection of about 14 us.  8 KV heads of 128 in bf16: 32
// caches of up to 4096 slots cut to 1024 62 us (5.3 TB/s while rows move), 4 of 32768 cut to
// 8192 97 us, 64 4-bit ones of 2048 cut to 1024 and read back 118 us.
#include <cstdio>

#include "common.cuh"
#include "paged_int4.cuh"

namespace aicas {
namespace {

// A weight as a whole number of the same order; NaN below all numbers, -0 as 0.  Never 0.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 1u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// A cache that is not cut: its slots, and its weights where they are wanted elsewhere.
__device__ __forceinline__ void keep_all(const aicas_paged_evict_params& a, int n, const float* w, float* wo, int32_t* kept, int from,
                                         int step) {
  for (int i = from; i < a.keep; i += step) kept[i] = i < n ? i : -1;
  if (wo != w)
    for (int i = from; i < n; i += step) wo[i] = w[i];
}

// ------------------------------------------------------------------ rows

constexpr int kMostRows = 512;  // of a run

struct MoveArgs {
  aicas_paged_evict_params p;
  int parts[AICAS_EVICT_MAX_PLANES + 1];  // the planes' first column parts
  int part_bytes[AICAS_EVICT_MAX_PLANES];
  uint32_t octets_mul;                    // n / octets of a page = (umulhi(n, octets_mul) + n) >> octets_shift
  int octets_shift;
};

struct Move {
  int64_t src, dst;  // places in the plane, in bytes; -1: none (zeros; nothing to write)
};

// A row has LANES threads with a V each; ROWS rows a thread and run.  While a run's rows are
// on their way, where the next one's lie is looked up, a row a thread.
template <int THREADS, typename V, int LANES, int ROWS>
__device__ __forceinline__ void move_rows(const MoveArgs& m, const aicas_evict_plane& pl, const int32_t* kept, int b, int h, int part,
                                          Move (*where)[kMostRows]) {
  const aicas_paged_evict_params& a = m.p;
  constexpr int kSlots = THREADS / LANES, kRun = kSlots * ROWS;
  static_assert(kRun <= kMostRows, "a run's places");
  const int r = threadIdx.x / LANES;
  char* data = static_cast<char*>(pl.data) + h * pl.stride_h + (int64_t)part * (LANES * sizeof(V)) + threadIdx.x % LANES * sizeof(V);
  const int32_t* table = a.page_table + b * a.table_stride;
  const auto at = [&](int slot) -> int64_t {
    const uint32_t n = (uint32_t)slot >> 3, i = (__umulhi(n, m.octets_mul) + n) >> m.octets_shift;
    const int page = table[i];
    return page >= 0 && page < a.num_pages ? page * pl.stride_p + (slot - (int)i * a.page_size) * pl.stride_t : -1;
  };
  const auto look = [&](int run) {
    for (int x = threadIdx.x; x < kRun; x += THREADS) {
      const int i = run * kRun + x, from = i < a.keep ? kept[i] : -1;
      Move w = {-1, -1};
      if (from > i) w.src = at(from), w.dst = at(i);
      where[run % 3][x] = w;
    }
  };
  const int runs = (a.keep + kRun - 1) / kRun;
  int run = 0;
  // what stays in place, where it may be worth a look
  while (run < runs && runs > 2 && kept[min(a.keep, (run + 1) * kRun) - 1] <= min(a.keep, (run + 1) * kRun) - 1) ++run;
  if (run == runs) return;
  V v[ROWS], next[ROWS];
  const auto load = [&](int run, V (&x)[ROWS]) {
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int64_t src = where[run % 3][k * kSlots + r].src;
      x[k] = V{};
      if (src >= 0) x[k] = *reinterpret_cast<const V*>(data + src);
    }
  };
  look(run);
  __syncthreads();
  load(run, v);
  for (; run < runs; ++run) {
    if (run + 1 < runs) look(run + 1);
    __syncthreads();  // this run is read; the next one's rows are not among those written now
    if (run + 1 < runs) load(run + 1, next);
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int64_t dst = where[run % 3][k * kSlots + r].dst;
      if (dst >= 0) *reinterpret_cast<V*>(data + dst) = v[k];
      v[k] = next[k];
    }
  }
}

// Part `at` of a pair's parts.  ROWS: vectors a thread has in flight, twice.
template <int THREADS, int ROWS>
__device__ __forceinline__ void move_part(const MoveArgs& m, const int32_t* kept, int b, int h, int at, Move (*where)[kMostRows]) {
  int i = 0;
  while (at >= m.parts[i + 1]) ++i;
  const aicas_evict_plane& pl = m.p.plane[i];
  const int part = at - m.parts[i];
  constexpr int kFew = kMostRows / THREADS;  // rows of a thread that a run has places for
  switch (m.part_bytes[i]) {
    case 256: return move_rows<THREADS, uint4, 16, ROWS>(m, pl, kept, b, h, part, where);
    case 128: return move_rows<THREADS, uint4, 8, ROWS>(m, pl, kept, b, h, part, where);
    case 64: return move_rows<THREADS, uint4, 4, (4 * kFew < ROWS ? 4 * kFew : ROWS)>(m, pl, kept, b, h, part, where);
    case 32: return move_rows<THREADS, uint4, 2, (2 * kFew < ROWS ? 2 * kFew : ROWS)>(m, pl, kept, b, h, part, where);
    case 16: return move_rows<THREADS, uint4, 1, kFew>(m, pl, kept, b, h, part, where);
    case 8: return move_rows<THREADS, uint2, 1, kFew>(m, pl, kept, b, h, part, where);
    default: return move_rows<THREADS, uint32_t, 1, kFew>(m, pl, kept, b, h, part, where);
  }
}

// ------------------------------------------------------------------ caches whose weights fit the registers of a cluster

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Writes to the word at this CTA's shared-memory address `at`, of CTA `rank` of the cluster.
__device__ __forceinline__ void store_peer(uint32_t at, uint32_t rank, uint4 v) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(there), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// KEYS slots a thread in registers; each CTA of a cluster has a run of the slots, or, where the
// kernel MOVES the rows too, has them all and finds by itself what the others find.  The key of
// the last slot that stays is found two bits at a time: how many keys are not below each of
// three candidates, counted in registers, over a warp, through shared memory and, between the
// CTAs that share the slots, distributed shared memory: at most 16 short rounds, whatever the
// weights are (counting them by their bytes meets the same few counters again and again).
template <int THREADS, int KEYS>
struct Select {
  static constexpr int kWarps = THREADS / 32, kCells = KEYS * kWarps;
  static_assert(KEYS <= 16 && kCells % 32 == 0, "a warp's count has 10 bits");
  uint32_t cells[kCells];    // per (key of a thread, warp): flags counted, then those before
  uint32_t packed[2][kWarps];
  uint4 peers[2][8];         // counts of the CTAs that share the slots
};

template <int THREADS, int KEYS, bool MOVES>
__global__ void __launch_bounds__(THREADS) paged_select_kernel(const __grid_constant__ MoveArgs m, int ctas) {
  using S = Select<THREADS, KEYS>;
  __shared__ S sm;
  const aicas_paged_evict_params& a = m.p;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, rank = ctas > 1 ? (int)cluster_rank() : 0;
  const int pair = blockIdx.x / ctas, b = pair / a.num_kv_heads, h = pair - b * a.num_kv_heads;
  grid_launch_dependents();
  grid_dependency_wait();
  const int n = min(max(a.kv_lens[b], 0), a.max_pages * a.page_size);
  const float* w = a.weights + b * a.w_stride_b + h * a.w_stride_h;
  float* wo = a.weights_out + b * a.wo_stride_b + h * a.wo_stride_h;
  int32_t* kept = a.kept + (int64_t)pair * a.keep;
  if (MOVES && a.kv_lens_out != nullptr && h == 0 && rank == 0 && tid == 0) a.kv_lens_out[b] = n > a.longer_than ? a.keep : n;
  if (n <= a.longer_than) return keep_all(a, n, w, wo, kept, rank * THREADS + tid, ctas * THREADS);

  if (!MOVES && ctas > 1) cluster_sync();  // every CTA runs before another writes to its shared memory
  const int run = MOVES ? n : (n + ctas - 1) / ctas, t0 = MOVES ? 0 : rank * run, t1 = min(n, t0 + run);  // this CTA's slots
  const int lo = a.keep_first, hi = n - a.keep_last;
  // The weights stay in registers where these hold them beside the keys.
  constexpr bool kHeld = KEYS <= 8;
  float x[KEYS];
  uint32_t key[KEYS];  // above all weights' for the slots that stay whatever theirs is, 0 past the run's end
#pragma unroll
  for (int j = 0; j < KEYS; ++j) {
    const int t = t0 + j * THREADS + tid;
    x[j] = t < t1 ? w[t] : 0.f;
    key[j] = t >= t1 ? 0u : t < lo || t >= hi ? 0xffffffffu : order_of(x[j]);
  }

  int round = 0;
  // Sums of three numbers over the cluster; a thread's at most KEYS each.  before: over the CTAs of lower rank.
  const auto sums = [&](uint32_t x, uint32_t y, uint32_t z, uint3* before) {
    const int buf = round++ & 1;
    const uint32_t packed = __reduce_add_sync(0xffffffffu, x | y << 10 | z << 20);
    if (lane == 0) sm.packed[buf][warp] = packed;
    __syncthreads();
    const uint32_t p = lane < S::kWarps ? sm.packed[buf][lane] : 0u;
    uint3 s = make_uint3(__reduce_add_sync(0xffffffffu, p & 1023u), __reduce_add_sync(0xffffffffu, p >> 10 & 1023u),
                         __reduce_add_sync(0xffffffffu, p >> 20));
    if (before != nullptr) *before = make_uint3(0u, 0u, 0u);
    if (!MOVES && ctas > 1) {
      if (warp == 0 && lane < ctas) store_peer(smem_u32(&sm.peers[buf][rank]), lane, make_uint4(s.x, s.y, s.z, 0u));
      __syncwarp();
      cluster_sync();
      s = make_uint3(0u, 0u, 0u);
      for (int r = 0; r < ctas; ++r) {
        const uint4 v = sm.peers[buf][r];
        if (before != nullptr && r == rank) *before = s;
        s.x += v.x, s.y += v.y, s.z += v.z;
      }
    }
    return s;
  };
  const auto at_least = [&](uint32_t than) {
    uint32_t c = 0u;
#pragma unroll
    for (int j = 0; j < KEYS; ++j) c += key[j] >= than;
    return c;
  };
  // The places of the flagged keys in the order of slots, from `base` on.
  uint32_t place[KEYS];
  const auto places = [&](uint32_t flags, uint32_t base) {
    __syncthreads();  // the last ones are read
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      const uint32_t bits = __ballot_sync(0xffffffffu, flags >> j & 1u);
      place[j] = __popc(bits & ((1u << lane) - 1u));
      if (lane == 0) sm.cells[j * S::kWarps + warp] = __popc(bits);
    }
    __syncthreads();
    if (warp == 0) {
      constexpr int kEach = S::kCells / 32;
      uint32_t c[kEach], sum = 0u;
#pragma unroll
      for (int e = 0; e < kEach; ++e) sum += c[e] = sm.cells[lane * kEach + e];
      uint32_t before = sum;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, before, off);
        if (lane >= off) before += v;
      }
      before -= sum;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        sm.cells[lane * kEach + e] = before;
        before += c[e];
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < KEYS; ++j) place[j] += base + sm.cells[j * S::kWarps + warp];
  };

  const uint32_t need = (uint32_t)a.keep;
  uint32_t least = 0u;   // the largest key that `need` keys are not below
  uint32_t enough = 0u;  // how many are not below it
  for (int shift = 30; shift >= 0 && enough != need; shift -= 2) {
    const uint3 c = sums(at_least(least | 1u << shift), at_least(least | 2u << shift), at_least(least | 3u << shift), nullptr);
    const uint32_t digit = c.z >= need ? 3u : c.y >= need ? 2u : c.x >= need ? 1u : 0u;
    if (digit != 0u) enough = digit == 3u ? c.z : digit == 2u ? c.y : c.x;
    least |= digit << shift;
  }
  uint32_t stays = 0u;  // bit j: key j's slot stays
#pragma unroll
  for (int j = 0; j < KEYS; ++j) stays |= (uint32_t)(key[j] >= least) << j;
  if (enough > need) {  // of those with the least key the lower slots
    uint32_t equal = 0u;
#pragma unroll
    for (int j = 0; j < KEYS; ++j) equal |= (uint32_t)(key[j] == least) << j;
    uint3 before;
    const uint3 c = sums(__popc(equal), __popc(stays & ~equal), 0u, &before);
    places(equal, before.x);
#pragma unroll
    for (int j = 0; j < KEYS; ++j)
      if ((equal >> j & 1u) && place[j] >= need - c.y) stays &= ~(1u << j);
  }
  if constexpr (!kHeld)
#pragma unroll
    for (int j = 0; j < KEYS; ++j) x[j] = stays >> j & 1u ? w[t0 + j * THREADS + tid] : 0.f;
  uint3 before = make_uint3(0u, 0u, 0u);
  if (!MOVES)
    sums(__popc(stays), 0u, 0u, &before);
  else if (ctas > 1)
    cluster_sync();  // all CTAs have read the weights
  places(stays, before.x);
  __shared__ int32_t list[MOVES ? THREADS * KEYS : 1];
#pragma unroll
  for (int j = 0; j < KEYS; ++j) {
    const int t = t0 + j * THREADS + tid;
    if (stays >> j & 1u) {
      if (MOVES) list[place[j]] = t;
      if (!MOVES || rank == 0) {
        kept[place[j]] = t;
        wo[place[j]] = x[j];  // below keep
      }
    }
    if ((!MOVES || rank == 0) && t >= a.keep && t < t1) wo[t] = 0.f;
  }
  if constexpr (MOVES) {
    __shared__ Move where[3][kMostRows];
    for (int at = rank; at < m.parts[a.num_planes]; at += ctas) {
      __syncthreads();  // the list is written, the places of the part before are done with
      move_part<THREADS, 4>(m, list, b, h, at, where);
    }
  }
}

// ------------------------------------------------------------------ longer caches

// One CTA a (request, KV head); the key of the last slot that stays by its bytes, from
// counts of all weights' bytes, read anew for each.
constexpr int kLongThreads = 1024, kLongWarps = kLongThreads / 32;

__global__ void __launch_bounds__(kLongThreads) paged_select_long_kernel(const __grid_constant__ aicas_paged_evict_params a) {
  __shared__ int hist[256];
  __shared__ uint32_t s_key;
  __shared__ int s_need, s_eq[kLongWarps], s_kept[kLongWarps];
  const int b = blockIdx.x / a.num_kv_heads, h = blockIdx.x - b * a.num_kv_heads;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  grid_launch_dependents();
  grid_dependency_wait();
  const int n = min(max(a.kv_lens[b], 0), a.max_pages * a.page_size);
  const float* w = a.weights + b * a.w_stride_b + h * a.w_stride_h;
  float* wo = a.weights_out + b * a.wo_stride_b + h * a.wo_stride_h;
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.keep;
  if (n <= a.longer_than) return keep_all(a, n, w, wo, kept, tid, kLongThreads);
  const int lo = a.keep_first, hi = n - a.keep_last;
  int need = a.keep - a.keep_first - a.keep_last;
  uint32_t key = 0;
  if (need > 0)
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int t = lo + tid; t < hi; t += kLongThreads) {
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
  for (int t0 = 0; t0 < n; t0 += kLongThreads) {
    const int t = t0 + tid;
    const float x = t < n ? w[t] : 0.f;
    const bool forced = t < lo || t >= hi, in = t < n;
    const uint32_t u = order_of(x);
    const bool equal = in && !forced && need > 0 && u == key;
    const uint32_t eq = __ballot_sync(0xffffffffu, equal), below = (1u << lane) - 1u;
    if (lane == 0) s_eq[warp] = __popc(eq);
    __syncthreads();
    const int e = s_eq[lane];  // as many warps as lanes
    const int eq_before = eq_base + __reduce_add_sync(0xffffffffu, lane < warp ? e : 0) + __popc(eq & below);
    eq_base += __reduce_add_sync(0xffffffffu, e);
    const bool stays = in && (forced || (need > 0 && (u > key || (equal && eq_before < need))));
    const uint32_t st = __ballot_sync(0xffffffffu, stays);
    if (lane == 0) s_kept[warp] = __popc(st);
    __syncthreads();
    const int k = s_kept[lane];
    const int at = kept_base + __reduce_add_sync(0xffffffffu, lane < warp ? k : 0) + __popc(st & below);
    kept_base += __reduce_add_sync(0xffffffffu, k);
    if (stays) {  // at <= t, and this run's weights are read
      kept[at] = t;
      wo[at] = x;
    }
  }
  __syncthreads();
  for (int t = a.keep + tid; t < n; t += kLongThreads) wo[t] = 0.f;
}

constexpr int kMoveThreads = 256;

template <int ROWS>
__global__ void __launch_bounds__(kMoveThreads) paged_move_kernel(const __grid_constant__ MoveArgs m) {
  __shared__ Move where[3][kMostRows];
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
  // kv_lens_out may be kv_lens: the others go by the list of slots alone, whose last says whether any slot moves
  const int32_t* kept = a.kept + (int64_t)pair * a.keep;
  if (kept[a.keep - 1] >= a.keep) move_part<kMoveThreads, ROWS>(m, kept, b, h, at, where);
}

// One launch for as many pairs as have their clusters of 8 at once.  One launch, two:
// 8 pairs cut from 1500 to 1024 slots of 256 bytes 8.5 us, 11.8, from 4096 to 2900 16.4, 24.5;
// 14 from 1501 to 333 11.7, 14.0; 16 from 1500 to 1024 14.8, 12.0, from 4096 to 1024 20.0, 15.5.
constexpr int kOneLaunch = 10;  // SMs a pair

// Columns that the planes' rows are moved by: as wide as leaves `least` parts, at most 256 bytes
// (32 caches cut to 1024 slots: rows of 256 bytes 51 us, in columns of 32 85).
void set_parts(MoveArgs& m, int64_t least) {
  for (int most = 256;; most /= 2) {
    m.parts[0] = 0;
    for (int i = 0; i < m.p.num_planes; ++i) {
      const int bytes = (int)m.p.plane[i].row_bytes;
      int part = 16;
      if (bytes < 16)
        part = bytes;
      else
        while (part < most && bytes % (2 * part) == 0) part *= 2;
      m.part_bytes[i] = part;
      m.parts[i + 1] = m.parts[i] + bytes / part;
    }
    if (most == 32 || m.parts[m.p.num_planes] >= least) return;
  }
}

template <int THREADS, int KEYS, bool MOVES>
cudaError_t launch_select(const MoveArgs& m, int ctas, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(m.p.batch * m.p.num_kv_heads * ctas));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, paged_select_kernel<THREADS, KEYS, MOVES>, m, ctas);
}

// Clusters of CTAs of 512 threads with 4 or 8 keys each, 16 where 8 CTAs need them: 1024 threads,
// or more keys a thread than needed, were slower by a tenth to a third.
cudaError_t launch_select_for(const MoveArgs& m, cudaStream_t st) {
  const int64_t slots = (int64_t)m.p.max_pages * m.p.page_size;
  if (slots <= 512 * 4) return launch_select<512, 4, false>(m, 1, st);
  for (int ctas = 1; ctas <= 8; ctas *= 2)
    if (slots <= (int64_t)512 * 8 * ctas) return launch_select<512, 8, false>(m, ctas, st);
  if (slots <= 512 * 16 * 8) return launch_select<512, 16, false>(m, 8, st);
  if (slots <= 1024 * 16 * 8) return launch_select<1024, 16, false>(m, 8, st);
  return launch_pdl(paged_select_long_kernel, dim3((unsigned)(m.p.batch * m.p.num_kv_heads)), dim3(kLongThreads), 0, st, m.p);
}

}  // namespace

int run_paged_evict(const aicas_paged_evict_params* p, int sms, cudaStream_t stream, char* err, size_t errlen) {
  const int64_t pairs = (int64_t)p->batch * p->num_kv_heads, slots = (int64_t)p->max_pages * p->page_size;
  MoveArgs m;
  m.p = *p;
  // rows that are keys and values at once move once
  m.p.num_planes = 0;
  for (int i = 0; i < p->num_planes; ++i) {
    const aicas_evict_plane& x = p->plane[i];
    bool there = false;
    for (int j = 0; j < m.p.num_planes; ++j) {
      const aicas_evict_plane& y = m.p.plane[j];
      there |= x.data == y.data && x.stride_p == y.stride_p && x.stride_h == y.stride_h && x.stride_t == y.stride_t && x.row_bytes == y.row_bytes;
    }
    if (!there) m.p.plane[m.p.num_planes++] = x;
  }
  // n / d for n < 2^28, as in paged_int4_tiles.cuh
  const int octets = p->page_size / 8;
  m.octets_shift = 0;
  while ((1ll << m.octets_shift) < octets) ++m.octets_shift;
  m.octets_mul = (uint32_t)((((1ull << m.octets_shift) - octets) << 32) / octets + 1);
  cudaError_t e;
  if (slots <= 512 * 8 && pairs * kOneLaunch <= sms && (p->kv_lens_out == nullptr || p->kv_lens_out != p->kv_lens)) {
    set_parts(m, 8);
    const int ctas = m.parts[m.p.num_planes] >= 8 ? 8 : m.parts[m.p.num_planes] >= 4 ? 4 : 2;
    e = slots <= 512 * 4 ? launch_select<512, 4, true>(m, ctas, stream) : launch_select<512, 8, true>(m, ctas, stream);
  } else {
    e = launch_select_for(m, stream);
    // whole rows, or as many parts of them as give each SM a CTA
    set_parts(m, (sms + pairs - 1) / pairs);
    const int64_t ctas = pairs * m.parts[m.p.num_planes];
    if (e == cudaSuccess)
      // 32 caches cut to 1024 slots (512 CTAs) 65.2 us with 8, 62.6 with 4; 4 caches cut to 8192 (256 CTAs) 97, 133
      e = launch_pdl(ctas <= 2 * sms ? paged_move_kernel<8> : paged_move_kernel<4>, dim3((unsigned)ctas), dim3(kMoveThreads), 0, stream, m);
  }
  if (e == cudaSuccess) return AICAS_OK;
  snprintf(err, errlen, "paged evict launch: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
  return AICAS_ERR_CUDA;
}

}  // namespace aicas
