// Decode-side products with 4-bit weights:
//   y[r, n] = sum_k x'[r, k] * scale[n, k / g] * (q[n, k] - zero[n, k / g])
// with x' = x or its RMSNorm, and a residual or SiLU(gate) * up epilogue.
//
// HBM bound: N K / 2 bytes of weights for at most 2 * 32 * N K flops.  What it
// takes is turning 4-bit numbers into tensor-core operands as fast as they come.
//
//   * Operands: mma.sync m16n8k16 in fp16 with the weights as the 16 x 16 side, in
//     registers, and the activations as columns.  A 32-bit word of weights holds
//     k0..k7 of a row.  word & 0x000f000f is the pair (k0, k4) as it stands: a
//     4-bit number in the low bits of an fp16 is that number times 2^-24, a
//     subnormal that the tensor cores take exactly.  word & 0x00f000f0 is (k1, k5)
//     times 2^-20, and the word shifted by 8 gives the other two pairs: 5
//     instructions for 8 weights.  The odd k's activations are held times 2^-4 to
//     match, and the products do not care in what order k goes by, so the weights
//     stay as stored and the activations are laid out in shared memory to suit.
//     tcgen05 would need the widened weights written back to shared or tensor
//     memory: four times the bytes that came from HBM.
//   * Activations: x' of a row times a power of two that brings its largest
//     element to [2^9, 2^10), as fp16.  16-bit x is exact so (an element 2^30
//     times smaller than the row's largest loses its last bits).  A normalised x'
//     is rounded to fp16's 11 bits where the result has bf16's 8, and carried as
//     two fp16 parts in neighbouring columns where the result is fp16.
//   * Sums: a group's sum over the whole numbers q in fp32, less zero point times
//     the group's sum of activations, times the scale in fp32; groups, warps and
//     CTAs are added up in fp32; one rounding at the end.
//   * Work: a cluster of S CTAs takes a run of 16-row tiles (8 gate + 8 up rows
//     for SiLU * up), each CTA one S-th of K, so that its share of x' fits beside
//     the ring (S = 1 wherever all of it does).  Tiles are taken in rounds; a
//     round's (tile, 256 k) jobs are cut evenly over the warps, whatever tile
//     they belong to, and the warps' and CTAs' partial sums are added in a fixed
//     order, so results repeat to the bit.  Each warp streams its own jobs through
//     a private TMA ring that runs on across rounds.
#include <cstdio>
#include <cstring>
#include <type_traits>

#include "common.cuh"
#include "linear_int4.cuh"
#include "tma_host.cuh"

namespace aicas {
namespace {

constexpr int kJobK = 256;              // k of a job: 128 bytes of a row
constexpr int kJobBytes = 16 * 128;     // 16 rows
constexpr int kPitch = 20;              // floats a column of a partial tile (16 rows; 20 keeps stores conflict free)
constexpr int kMaxSmem = 232448;

constexpr int kMaxRound = 80;           // tiles of a round
constexpr int kEntries = 128;           // rows' statistics: (largest element, sum of squares) of 256 k each
constexpr int kVarBytes = 64 + kEntries * 8 + 2 * 32 * 4 + kMaxRound * 4;

// Warps of a CTA: more of them hide the products' latency, fewer leave shared
// memory for the columns of many rows.
constexpr int warps_for(int nt) { return nt <= 4 ? 16 : 8; }

struct Int4Args {
  CUtensorMap tm_w[2];
  const void* x;
  const void* norm_weight;
  const void* residual;
  void* out;
  const void* scales[2];
  const uint8_t* zeros[2];
  int64_t x_stride, res_stride, out_stride;
  int rows, k, n, groups;  // groups along K
  int mode;
  float eps;
  int s;                   // CTAs of a cluster
  int kb;                  // jobs of a tile for each of them
  int tiles, tiles_round;  // 16-row tiles of the launch; tiles of a round
  int tiles_each, tiles_more;  // tiles of a cluster; the first tiles_more clusters take one more
  int stages;
  int off_part, off_x, off_sum, off_bars;
  unsigned int* err;
};

__device__ __forceinline__ void mma_f16(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ float low_half(uint32_t v) {
  union {
    uint16_t u;
    T t;
  } r;
  r.u = (uint16_t)v;
  return Elem<T>::to_float(r.t);
}

__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync_all() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// Row of a tile that lane group g (= lane / 4) holds: g with its bits reversed,
// so that the rows of a shared-memory phase differ where the swizzle looks.
__device__ __forceinline__ int tile_row(int g) { return (g & 1) << 2 | (g & 2) | g >> 2; }

// A warp's jobs: those of each round's (tile, job along K) list that fall to it.
template <int WARPS>
struct Jobs {
  int round;       // first tile of the round
  int left;        // jobs of the round still this warp's
  int tile, jk;    // the next one: tile of the round, job along K

  __device__ __forceinline__ void cut(const Int4Args& a, int tile_end) {
    const int warp = threadIdx.x >> 5;
    const int total = min(a.tiles_round, tile_end - round) * a.kb;
    const int begin = warp * total / WARPS;
    left = (warp + 1) * total / WARPS - begin;
    tile = begin / a.kb;
    jk = begin - tile * a.kb;
  }
  // Finds the next job, over the rounds; false after the last.
  __device__ __forceinline__ bool settle(const Int4Args& a, int tile_end) {
    while (left == 0) {
      round += a.tiles_round;
      if (round >= tile_end) {
        round -= a.tiles_round;
        return false;
      }
      cut(a, tile_end);
    }
    return true;
  }
  __device__ __forceinline__ void step(const Int4Args& a) {
    --left;
    if (++jk == a.kb) jk = 0, ++tile;
  }
};

// Largest |x * w| over the vectors in [lo, hi) of those first, first + 32, .. below
// end, and the sum of squares of x * by over all of them, over the warp.  w: ones where null.
template <typename T>
__device__ __noinline__ float2 row_stats(const T* row, const T* w, int first, int end, int lo, int hi, float by) {
  float top = 0.f, ss = 0.f;
#pragma unroll 4
  for (int v = first; v < end; v += 32) {
    float f[8], g[8];
    Elem<T>::unpack(reinterpret_cast<const uint4*>(row)[v], f);
    if (w != nullptr) Elem<T>::unpack(reinterpret_cast<const uint4*>(w)[v], g);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = f[e] * by;
      ss = fmaf(y, y, ss);
      if (v >= lo && v < hi) top = fmaxf(top, fabsf(w != nullptr ? f[e] * g[e] : f[e]));
    }
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, off);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  }
  return make_float2(top, ss);
}

// W: 32-bit words of weights that a lane takes side by side (4 W lanes' words
// = 32 W of k share a group of g = 32 W).  NT: blocks of 8 columns.
template <typename T, int NT, int W>
__global__ void __launch_bounds__(warps_for(NT) * 32, 1) linear_int4_kernel(const __grid_constant__ Int4Args a) {
  constexpr int kWarps = warps_for(NT), kThreads = kWarps * 32;
  constexpr int kSegs = 8 / W;          // groups of a job
  constexpr int kHold = kSegs / 2;      // (scale, zero) pairs a lane holds of a job: two rows' kSegs over four lanes
  constexpr int kTileFloats = NT * 8 * kPitch;
  constexpr int kFly = NT <= 2 ? 4 : 8; // vectors of x a thread holds at once
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, i = lane & 3;
  const bool pair = a.mode == AICAS_LINEAR_SWIGLU;
  const int tile_n = pair ? 8 : 16;     // output features of a tile
  const uint32_t ring = smem_u32(smem) + warp * a.stages * kJobBytes;
  const uint32_t bars = smem_u32(smem + a.off_bars) + warp * a.stages * 8;
  float* part = reinterpret_cast<float*>(smem + a.off_part);  // [tiles_round][kTileFloats], then [kWarps] heads
  uint8_t* xs = smem + a.off_x;
  float* xsum = reinterpret_cast<float*>(smem + a.off_sum);   // [group of this CTA's K][NT * 8 columns]
  int* s_abort = reinterpret_cast<int*>(smem + a.off_bars + kWarps * a.stages * 8);
  float2* s_stat = reinterpret_cast<float2*>(s_abort + 16);   // [kEntries]
  float* s_scale = reinterpret_cast<float*>(s_stat + kEntries);  // [32]
  float* s_inv = s_scale + 32;                                // [32]
  int* s_heads = reinterpret_cast<int*>(s_inv + 32);          // [tile of the round] the warps after the tile's first
  const int rank = a.s > 1 ? (int)cluster_rank() : 0;
  const int cluster = (int)blockIdx.x / a.s;
  const int kb0 = rank * a.kb;  // this CTA's first job along K
  const T* nw = static_cast<const T*>(a.norm_weight);
  const bool split = nw != nullptr && std::is_same<T, __half>::value;  // two parts a row

  if (tid == 0) *s_abort = 0;
  if (lane < a.stages) mbar_init(bars + 8 * lane, 1);
  grid_launch_dependents();

  const int tile0 = cluster * a.tiles_each + min(cluster, a.tiles_more);
  const int tile_end = tile0 + a.tiles_each + (cluster < a.tiles_more ? 1 : 0);
  Jobs<kWarps> job;
  job.round = tile0;
  job.cut(a, tile_end);
  // the ring's first jobs, a lane each
  Jobs<kWarps> mine = job;
  const bool fill = lane < min(a.stages, job.left);
  mine.jk += lane;
  while (mine.jk >= a.kb) mine.jk -= a.kb, ++mine.tile;
  const int fill_x = (kb0 + mine.jk) * 128, fill_n = (mine.round + mine.tile) * tile_n;
  if (fill) {
    // into L2 (where every earlier write is seen) while the kernel before this one ends
    tma_prefetch_l2_2d(&a.tm_w[0], fill_x, fill_n);
    if (pair) tma_prefetch_l2_2d(&a.tm_w[1], fill_x, fill_n);
  }
  fence_mbar_init();
  __syncwarp();
  grid_dependency_wait();

  // ---- x: this thread's vectors of the CTA's share of K, ahead of the weights
  const T* x = static_cast<const T*>(a.x);
  const int vec0 = kb0 * (kJobK / 8), vecs = a.kb * (kJobK / 8), all_vecs = a.k / 8;
  // at once, where they fit and nothing else of the rows is needed; else in passes
  const bool once = a.rows * vecs <= kFly * kThreads && (nw == nullptr || a.s == 1);
  uint4 xq[kFly], wq[kFly];
  int xr[kFly];
  if (once) {
#pragma unroll
    for (int j = 0; j < kFly; ++j) {
      const int entry = warp + j * kWarps;  // 32 vectors: of one row
      xr[j] = entry / a.kb;
      const int v = vec0 + (entry - xr[j] * a.kb) * 32 + lane;
      xq[j] = wq[j] = make_uint4(0, 0, 0, 0);
      if (xr[j] < a.rows && v < all_vecs) {
        xq[j] = reinterpret_cast<const uint4*>(x + xr[j] * a.x_stride)[v];
        if (nw != nullptr) wq[j] = reinterpret_cast<const uint4*>(nw)[v];
      }
    }
  }

  const uint64_t policy = l2_policy_evict_first();
  if (fill) {
    const uint32_t dst = ring + lane * kJobBytes, bar = bars + 8 * lane;
    mbar_arrive_expect_tx(bar, kJobBytes);
    tma_load_2d_hint(dst, &a.tm_w[0], fill_x, fill_n, bar, policy);
    if (pair) tma_load_2d_hint(dst + 1024, &a.tm_w[1], fill_x, fill_n, bar, policy);
  }
  Jobs<kWarps> ld = job;  // next job to copy
  int flying = min(a.stages, job.left);
  ld.left -= flying;
  ld.jk += flying;
  while (ld.jk >= a.kb) ld.jk -= a.kb, ++ld.tile;
  const auto issue = [&](int stage) -> int {
    if (!ld.settle(a, tile_end)) return 0;
    if (lane == 0) {
      const int n = (ld.round + ld.tile) * tile_n, xk = (kb0 + ld.jk) * 128;
      const uint32_t dst = ring + stage * kJobBytes, bar = bars + 8 * stage;
      mbar_arrive_expect_tx(bar, kJobBytes);
      tma_load_2d_hint(dst, &a.tm_w[0], xk, n, bar, policy);
      if (pair) tma_load_2d_hint(dst + 1024, &a.tm_w[1], xk, n, bar, policy);
    }
    ld.step(a);
    return 1;
  };

  // ---- (scale, zero) of a job: lane i of a row's four holds rows g + 8 (i / 2), groups (i % 2) kHold ..;
  // fetched a job ahead, from L2 where the round before asked for them
  Jobs<kWarps> sj = job;  // next job whose scales are fetched
  const int my_row = tile_row(g), hi_row = i >> 1;
  const uint8_t* const my_zeros = pair && hi_row ? a.zeros[1] : a.zeros[0];
  const uint16_t* const my_scales = static_cast<const uint16_t*>(pair && hi_row ? a.scales[1] : a.scales[0]);
  const int n_off = my_row + (pair ? 0 : 8 * hi_row);
  uint32_t sz[kHold], next_s[kHold], next_z[kHold];
  const auto fetch = [&]() {
    if (!sj.settle(a, tile_end)) return;
    const int t = sj.round + sj.tile, n = t * tile_n + n_off, grp0 = (kb0 + sj.jk) * kSegs + (i & 1) * kHold;
    sj.step(a);
    const int64_t at = (int64_t)n * a.groups + grp0;
    if (t + a.tiles_round < tile_end && n + a.tiles_round * tile_n < a.n && grp0 < a.groups) {
      const int64_t next = at + (int64_t)a.tiles_round * tile_n * a.groups;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(my_scales + next));
      if (my_zeros != nullptr) asm volatile("prefetch.global.L2 [%0];" ::"l"(my_zeros + next));
    }
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      next_s[j] = 0u;
      next_z[j] = 8u;
      if (n >= a.n || grp0 + j >= a.groups) continue;
      next_s[j] = my_scales[at + j];
      if (my_zeros != nullptr) next_z[j] = my_zeros[at + j];
    }
  };
  const auto take = [&]() {  // the fetched ones become the next job's
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      union {
        T t;
        uint16_t u;
      } z;
      z.t = Elem<T>::from_float((float)next_z[j]);  // 0..15: exact
      sz[j] = next_s[j] | (uint32_t)z.u << 16;
    }
  };
  fetch();

  // ---- which warps share a tile of a full round, for the sums at its end
  const auto find_heads = [&](int tiles) {
    const int total = tiles * a.kb;
    if (tid < tiles) {
      // job j is warp ((j + 1) kWarps - 1) / total's
      const int w0 = ((tid * a.kb + 1) * kWarps - 1) / total, w1 = ((tid + 1) * a.kb * kWarps - 1) / total;
      s_heads[tid] = w0 | w1 << 16;
    }
  };
  find_heads(min(a.tiles_round, tile_end - tile0));

  // ---- rows' largest element (of this CTA's K) and sum of squares (of all K)
  const auto row_scale = [&](int r, float top, float ss) {
    float rstd = 1.f;
    if (nw != nullptr) {
      rstd = rsqrtf(ss / (float)a.k + a.eps);
      if (!(ss < INFINITY)) {  // squares past fp32's range: of the elements times 2^-70
        const float by = 8.470329472543003e-22f;
        rstd = rsqrtf(row_stats<T>(x + r * a.x_stride, nw, lane, all_vecs, 0, 0, by).y / (float)a.k) * by;
      }
    }
    // 2^e that brings the largest element to [2^9, 2^10); 1 for a row of zeros or one with inf
    const uint32_t bits = __float_as_uint(top * rstd) >> 23;
    const int e = bits == 0u || bits >= 255u ? 0 : min(136 - (int)bits, 100);
    if (lane == 0) {
      s_scale[r] = rstd * __uint_as_float((uint32_t)(127 + e) << 23);
      s_inv[r] = __uint_as_float((uint32_t)(127 - e) << 23);
    }
  };
  if (once) {
#pragma unroll
    for (int j = 0; j < kFly; ++j) {
      if (xr[j] >= a.rows) break;
      float f[8], w[8], top = 0.f, ss = 0.f;
      Elem<T>::unpack(xq[j], f);
      if (nw != nullptr) {
        Elem<T>::unpack(wq[j], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss), f[e] *= w[e];
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[e]));
      const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(top));  // magnitudes order as their bits
      if (lane == 0) s_stat[warp + j * kWarps] = make_float2(__uint_as_float(most), ss);
    }
    __syncthreads();
    for (int r = warp; r < a.rows; r += kWarps) {
      float top = 0.f, ss = 0.f;
      for (int e = lane; e < a.kb; e += 32) {
        const float2 st = s_stat[r * a.kb + e];
        top = fmaxf(top, st.x);
        ss += st.y;
      }
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, off);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      }
      row_scale(r, top, ss);
    }
  } else {
    for (int r = warp; r < a.rows; r += kWarps) {
      const float2 st = nw != nullptr
                            ? row_stats<T>(x + r * a.x_stride, nw, lane, all_vecs, vec0, vec0 + vecs, 1.f)
                            : row_stats<T>(x + r * a.x_stride, nullptr, vec0 + lane, min(vec0 + vecs, all_vecs), vec0, vec0 + vecs, 1.f);
      row_scale(r, st.x, st.y);
    }
  }
  __syncthreads();

  // ---- x' into shared memory, in the order in which the products take it
  const auto lay_out = [&](const uint4& q, const uint4& wv, int r, int v) {
    float f[8];
    Elem<T>::unpack(q, f);
    const float scale = s_scale[r];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= scale;
    if (nw != nullptr) {
      float w[8];
      Elem<T>::unpack(wv, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= w[e];
    }
    const int wd = v & 31, rem = wd % (4 * W);
    const int step = (v >> 5) * 8 + wd / (4 * W) * W + rem % W, li = rem / W;
    // pairs (k0, k4), (k1, k5) / 16, (k2, k6), (k3, k7) / 16
    const auto put = [&](int col) {
      union {
        __half2 h[4];
        uint4 u;
      } d;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        d.h[e] = e & 1 ? __floats2half2_rn(f[e] * 0.0625f, f[e + 4] * 0.0625f) : __floats2half2_rn(f[e], f[e + 4]);
      *reinterpret_cast<uint4*>(xs + ((step * NT + (col >> 3)) * 32 + (col & 7) * 4 + li) * 16) = d.u;
    };
    if (split) {
      put(2 * r);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] -= __half2float(__float2half_rn(f[e]));
      put(2 * r + 1);
    } else {
      put(r);
    }
  };
  if (once) {
#pragma unroll
    for (int j = 0; j < kFly; ++j)
      if (xr[j] < a.rows) lay_out(xq[j], wq[j], xr[j], (warp + j * kWarps - xr[j] * a.kb) * 32 + lane);
  } else {
#pragma unroll 4
    for (int at = tid; at < a.rows * vecs; at += kThreads) {
      const int r = at / vecs, v = at - r * vecs;
      uint4 q = make_uint4(0, 0, 0, 0), w = q;
      if (vec0 + v < all_vecs) {
        q = reinterpret_cast<const uint4*>(x + r * a.x_stride)[vec0 + v];
        if (nw != nullptr) w = reinterpret_cast<const uint4*>(nw)[vec0 + v];
      }
      lay_out(q, w, r, v);
    }
  }
  __syncthreads();
  // a group's sums of x', times the weights' 2^-24: products with ones in the weights' place
  for (int grp = warp; grp < a.kb * kSegs; grp += kWarps) {
    float acc[NT][4] = {};
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 b = *reinterpret_cast<const uint4*>(xs + (((grp * W + w) * NT + n) * 32 + lane) * 16);
        mma_f16(acc[n], 0x00010001u, 0u, 0x00100010u, 0u, b.x, b.y);
        mma_f16(acc[n], 0x00010001u, 0u, 0x00100010u, 0u, b.z, b.w);
      }
    if (g == 0)
#pragma unroll
      for (int n = 0; n < NT; ++n)
        *reinterpret_cast<float2*>(xsum + (grp * NT + n) * 8 + 2 * i) = make_float2(acc[n][0], acc[n][1]);
  }
  take();
  __syncthreads();

  // ---- rounds
  int stage = 0;
  uint32_t phase = 0;
  bool bad = false;
  for (;;) {
    float tot[NT][4];
    bool head = job.jk != 0;  // a tile begun by an earlier warp is this warp's head; its own tiles have a place each
    bool fresh = true;
#pragma unroll 1
    while (job.left > 0) {
      if (fresh) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) tot[n][e] = 0.f;
      }
      if (!bad && !mbar_wait(bars + 8 * stage, phase, s_abort, a.err)) bad = true;  // computes no more, keeps to the barriers
      if (!bad) {
        fetch();
        const uint32_t wrow = ring + stage * kJobBytes + my_row * 128;
        const uint8_t* xf = xs + (size_t)(job.jk * 8 * NT * 32 + lane) * 16;
        const float* gs = xsum + job.jk * kSegs * NT * 8 + 2 * i;
#pragma unroll
        for (int seg = 0; seg < kSegs; ++seg) {
          const uint32_t s_lo = __shfl_sync(0xffffffffu, sz[seg % kHold], (lane & ~3) | seg / kHold);
          const uint32_t s_hi = __shfl_sync(0xffffffffu, sz[seg % kHold], (lane & ~3) | 2 | seg / kHold);
          // this lane's W words of rows my_row and my_row + 8
          uint32_t w0[4], w1[4];
          {
            const int byte = (seg * 4 + i) * W * 4;
            const uint32_t at = wrow + ((byte & ~15) ^ ((my_row & 7) << 4)) + (byte & 15);
            if constexpr (W == 4) {
              asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                           : "=r"(w0[0]), "=r"(w0[1]), "=r"(w0[2]), "=r"(w0[3]) : "r"(at) : "memory");
              asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                           : "=r"(w1[0]), "=r"(w1[1]), "=r"(w1[2]), "=r"(w1[3]) : "r"(at + 1024) : "memory");
            } else if constexpr (W == 2) {
              asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w0[0]), "=r"(w0[1]) : "r"(at) : "memory");
              asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w1[0]), "=r"(w1[1]) : "r"(at + 1024) : "memory");
            } else {
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w0[0]) : "r"(at) : "memory");
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w1[0]) : "r"(at + 1024) : "memory");
            }
          }
          float acc[NT][4] = {};
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const uint32_t lo8 = w0[w] >> 8, hi8 = w1[w] >> 8;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint4 b = *reinterpret_cast<const uint4*>(xf + ((seg * W + w) * NT + n) * 512);
              mma_f16(acc[n], w0[w] & 0x000f000fu, w1[w] & 0x000f000fu, w0[w] & 0x00f000f0u, w1[w] & 0x00f000f0u, b.x, b.y);
              mma_f16(acc[n], lo8 & 0x000f000fu, hi8 & 0x000f000fu, lo8 & 0x00f000f0u, hi8 & 0x00f000f0u, b.z, b.w);
            }
          }
          const float f_lo = low_half<T>(s_lo) * 16777216.f, f_hi = low_half<T>(s_hi) * 16777216.f;  // the weights' 2^24
          const float z_lo = low_half<T>(s_lo >> 16), z_hi = low_half<T>(s_hi >> 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 xg = *reinterpret_cast<const float2*>(gs + (seg * NT + n) * 8);
            tot[n][0] = fmaf(f_lo, fmaf(-z_lo, xg.x, acc[n][0]), tot[n][0]);
            tot[n][1] = fmaf(f_lo, fmaf(-z_lo, xg.y, acc[n][1]), tot[n][1]);
            tot[n][2] = fmaf(f_hi, fmaf(-z_hi, xg.x, acc[n][2]), tot[n][2]);
            tot[n][3] = fmaf(f_hi, fmaf(-z_hi, xg.y, acc[n][3]), tot[n][3]);
          }
        }
        __syncwarp();  // every lane has read the stage
        flying += issue(stage) - 1;
        if (++stage == a.stages) stage = 0, phase ^= 1;
        take();
      }
      const int tile = job.tile;
      job.step(a);
      fresh = job.jk == 0;
      if (fresh || job.left == 0) {
        float* dst = part + (head ? a.tiles_round + warp : tile) * kTileFloats + my_row;
        head = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          dst[(8 * n + 2 * i) * kPitch] = tot[n][0], dst[(8 * n + 2 * i + 1) * kPitch] = tot[n][1];
          dst[(8 * n + 2 * i) * kPitch + 8] = tot[n][2], dst[(8 * n + 2 * i + 1) * kPitch + 8] = tot[n][3];
        }
      }
    }
    if (a.s > 1) cluster_sync_all(); else __syncthreads();

    // ---- the round's outputs: partial tiles of the warps and CTAs added in their order
    const int total = min(a.tiles_round, tile_end - job.round) * a.kb;
    const int n0 = job.round * tile_n, width = min(min(a.tiles_round, tile_end - job.round) * tile_n, a.n - n0);
    for (int at = rank * kThreads + tid; at < width * a.rows; at += a.s * kThreads) {
      const int r = at / width, c = at - r * width, tile = c / tile_n;
      const int place = (split ? 2 * r : r) * kPitch + c - tile * tile_n;
      const int heads = s_heads[tile], w0 = heads & 0xffff, w1 = heads >> 16;
      float y0 = 0.f, y1 = 0.f;
#pragma unroll 1
      for (int w = w0; w <= w1; ++w) {
        if (w * total / kWarps == (w + 1) * total / kWarps) continue;  // a warp without jobs
        const float* p = part + (w == w0 ? tile : a.tiles_round + w) * kTileFloats + place;
        if (a.s == 1) {
          y0 += split ? p[0] + p[kPitch] : p[0];
          if (pair) y1 += split ? p[8] + p[kPitch + 8] : p[8];
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            if (q >= a.s) break;
            const float inv = ld_cluster(smem_u32(s_inv + r), q);
            float t = ld_cluster(smem_u32(p), q);
            if (split) t += ld_cluster(smem_u32(p + kPitch), q);
            y0 = fmaf(t, inv, y0);
            if (pair) {
              t = ld_cluster(smem_u32(p + 8), q);
              if (split) t += ld_cluster(smem_u32(p + 8 + kPitch), q);
              y1 = fmaf(t, inv, y1);
            }
          }
        }
      }
      if (a.s == 1) y0 *= s_inv[r], y1 *= s_inv[r];
      if (pair) y0 = y0 / (1.f + expf(-y0)) * y1;
      if (a.mode == AICAS_LINEAR_RESIDUAL)
        y0 += Elem<T>::to_float(static_cast<const T*>(a.residual)[r * a.res_stride + n0 + c]);
      static_cast<T*>(a.out)[r * a.out_stride + n0 + c] = Elem<T>::from_float(y0);
    }
    job.round += a.tiles_round;
    if (job.round >= tile_end) break;
    job.cut(a, tile_end);
    if (a.s > 1) cluster_sync_all(); else __syncthreads();  // the partial tiles have been read
    if (tile_end - job.round < a.tiles_round) find_heads(tile_end - job.round);  // read after the next barrier
  }
  if (bad)
    for (; flying > 0; --flying) {  // leave once this warp's copies have landed (bounded again)
      mbar_wait(bars + 8 * stage, phase, nullptr, a.err);
      if (++stage == a.stages) stage = 0, phase ^= 1;
    }
  if (a.s > 1) cluster_sync_all();  // no CTA leaves while its partial tiles are read
}

// ------------------------------------------------------------------ host side

bool weight_map(CUtensorMap* m, const aicas_int4_weight& w, int n, int k, int box_rows, char* err, size_t errlen) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (enc == nullptr) {
    snprintf(err, errlen, "cuTensorMapEncodeTiled is unavailable from the driver");
    return false;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)k / 2, (cuuint64_t)n}, strides[1] = {(cuuint64_t)w.q_stride};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(w.q), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    snprintf(err, errlen, "cuTensorMapEncodeTiled failed (%d) for a 4-bit weight [%d, %d] with row stride %lld", (int)r, n, k,
             (long long)w.q_stride);
    return false;
  }
  return true;
}

int log2_of(int v) { return v <= 1 ? 0 : 1 + log2_of(v / 2); }

template <typename T, int NT, int W>
cudaError_t launch_int4(Int4Args a, int smem, int sms, cudaStream_t st) {
  static bool attr_set[64] = {false};
  static int max_clusters[64][4] = {};  // by device and cluster size
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool known = dev >= 0 && dev < 64;
  if (!known || !attr_set[dev]) {
    e = cudaFuncSetAttribute(linear_int4_kernel<T, NT, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
    if (e != cudaSuccess) return e;
    if (known) attr_set[dev] = true;
  }
  int clusters = sms;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)a.s;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.blockDim = dim3(warps_for(NT) * 32);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = a.s > 1 ? 2 : 1;
  if (a.s > 1) {
    int* cached = known ? &max_clusters[dev][log2_of(a.s)] : nullptr;
    if (cached != nullptr && *cached > 0) {
      clusters = *cached;
    } else {
      cfg.gridDim = dim3((unsigned)a.s);
      cudaLaunchAttribute only = attr[1];
      cfg.attrs = &only;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&clusters, linear_int4_kernel<T, NT, W>, &cfg);
      if (e != cudaSuccess) return e;
      if (clusters < 1) return cudaErrorInvalidConfiguration;
      if (cached != nullptr) *cached = clusters;
      cfg.attrs = attr;
      cfg.numAttrs = 2;
    }
  }
  if (clusters > a.tiles) clusters = a.tiles;
  a.tiles_each = a.tiles / clusters;
  a.tiles_more = a.tiles % clusters;
  cfg.gridDim = dim3((unsigned)(clusters * a.s));
  return cudaLaunchKernelEx(&cfg, linear_int4_kernel<T, NT, W>, a);
}

template <typename T, int NT>
cudaError_t dispatch_group(int group, const Int4Args& a, int smem, int sms, cudaStream_t st) {
  switch (group) {
    case 32: return launch_int4<T, NT, 1>(a, smem, sms, st);
    case 64: return launch_int4<T, NT, 2>(a, smem, sms, st);
    case 128: return launch_int4<T, NT, 4>(a, smem, sms, st);
  }
  return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t dispatch_int4(int nt, int group, const Int4Args& a, int smem, int sms, cudaStream_t st) {
  switch (nt) {
    case 1: return dispatch_group<T, 1>(group, a, smem, sms, st);
    case 2: return dispatch_group<T, 2>(group, a, smem, sms, st);
    case 4: return dispatch_group<T, 4>(group, a, smem, sms, st);
  }
  if constexpr (std::is_same<T, __half>::value)  // 32 rows in two parts
    if (nt == 8) return dispatch_group<T, 8>(group, a, smem, sms, st);
  return cudaErrorInvalidValue;
}

// Shared memory of a launch of nt column blocks with K split s ways; 0: does not fit.
int plan_int4(Int4Args* a, int nt, int s, int sms) {
  const int jobs = (a->k + kJobK - 1) / kJobK;
  a->s = s;
  a->kb = (jobs + s - 1) / s;
  // a round holds a cluster's tiles, if shared memory does
  const int most = nt == 8 ? 8 : kMaxRound / nt, want = (int)((int64_t)a->tiles * s * 4 / (3 * sms)) + 1;
  a->tiles_round = want < most ? want : most;
  const int warps = warps_for(nt);
  const int part = (a->tiles_round + warps) * nt * 8 * kPitch * 4, xs = a->kb * nt * 4096;
  const int sums = a->kb * (kJobK / (a->k / a->groups)) * nt * 32;
  const int tail = warps * 8 * 8 + kVarBytes, rest = part + xs + sums + tail, ring = warps * kJobBytes;
  a->stages = (kMaxSmem - rest) / ring;
  if (a->stages < 3) return 0;
  if (a->stages > 8) a->stages = 8;
  a->off_part = a->stages * ring;
  a->off_x = a->off_part + part;
  a->off_sum = a->off_x + xs;
  a->off_bars = a->off_sum + sums;
  return a->off_bars + tail;
}

}  // namespace

int run_linear_int4(const aicas_linear_int4_params* p, int sms, cudaStream_t stream, unsigned int* dev_err, char* err,
                    size_t errlen) {
  const bool pair = p->mode == AICAS_LINEAR_SWIGLU, bf16 = p->dtype == AICAS_DTYPE_BF16;
  Int4Args a;
  memset(&a, 0, sizeof(a));
  for (int j = 0; j < (pair ? 2 : 1); ++j) {
    if (!weight_map(&a.tm_w[j], p->w[j], p->out_features, p->in_features, pair ? 8 : 16, err, errlen))
      return AICAS_ERR_UNSUPPORTED;
    a.scales[j] = p->w[j].scales;
    a.zeros[j] = static_cast<const uint8_t*>(p->w[j].zeros);
  }
  a.norm_weight = p->norm_weight;
  a.x_stride = p->x_stride, a.res_stride = p->residual_stride, a.out_stride = p->out_stride;
  a.k = p->in_features, a.n = p->out_features, a.groups = p->in_features / p->group_size;
  a.mode = p->mode, a.eps = p->eps, a.err = dev_err;
  const int tile_n = pair ? 8 : 16;
  a.tiles = (p->out_features + tile_n - 1) / tile_n;
  // every row at once where x' fits on chip over a cluster of up to 8 CTAs, else fewer rows a launch
  const int columns = p->norm_weight != nullptr && !bf16 ? 2 : 1;  // a normalised x' for an fp16 result: two parts
  int batch = p->rows, nt = 0, smem = 0;
  for (;; batch = (batch + 1) / 2) {
    const int blocks = (batch * columns + 7) / 8;
    nt = blocks <= 1 ? 1 : blocks <= 2 ? 2 : blocks <= 4 ? 4 : 8;
    for (int s = 1; s <= 8 && smem == 0; s *= 2) smem = plan_int4(&a, nt, s, sms);
    if (smem != 0) break;
    if (batch == 1) {
      snprintf(err, errlen, "int4 linear: in_features %d is more than shared memory holds", p->in_features);
      return AICAS_ERR_UNSUPPORTED;
    }
  }
  for (int r = 0; r < p->rows; r += batch) {
    a.rows = p->rows - r < batch ? p->rows - r : batch;
    a.x = static_cast<const uint16_t*>(p->x) + r * p->x_stride;
    a.out = static_cast<uint16_t*>(p->out) + r * p->out_stride;
    a.residual = p->residual != nullptr ? static_cast<const uint16_t*>(p->residual) + r * p->residual_stride : nullptr;
    const cudaError_t e = bf16 ? dispatch_int4<__nv_bfloat16>(nt, p->group_size, a, smem, sms, stream)
                               : dispatch_int4<__half>(nt, p->group_size, a, smem, sms, stream);
    if (e != cudaSuccess) {
      snprintf(err, errlen, "int4 linear launch: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
      return AICAS_ERR_CUDA;
    }
  }
  return AICAS_OK;
}

}  // namespace aicas
