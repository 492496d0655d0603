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
constexpr int kVarBytes = 64 + 4 * 160;  // abort flag; rows' statistics, scales and their inverses

// Warps of a CTA: more of them hide the products' latency, fewer leave shared
// memory for the columns of many rows.
constexpr int warps_for(int nt) { return nt <= 2 ? 16 : 8; }

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

// W: 32-bit words of weights that a lane takes side by side (4 W lanes' words
// = 32 W of k share a group of g = 32 W).  NT: blocks of 8 columns.
template <typename T, int NT, int W>
__global__ void __launch_bounds__(warps_for(NT) * 32, 1) linear_int4_kernel(const __grid_constant__ Int4Args a) {
  constexpr int kWarps = warps_for(NT), kThreads = kWarps * 32;
  constexpr int kSegs = 8 / W;          // groups of a job
  constexpr int kHold = kSegs / 2;      // (scale, zero) pairs a lane holds of a job: two rows' kSegs over four lanes
  constexpr int kTileFloats = NT * 8 * kPitch;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, i = lane & 3;
  const bool pair = a.mode == AICAS_LINEAR_SWIGLU;
  const int tile_n = pair ? 8 : 16;     // output features of a tile
  const uint32_t ring = smem_u32(smem) + warp * a.stages * kJobBytes;
  const uint32_t bars = smem_u32(smem + a.off_bars) + warp * a.stages * 8;
  float* part = reinterpret_cast<float*>(smem + a.off_part);  // [tiles_round][kTileFloats], then [kWarps] heads
  float* heads = part + a.tiles_round * kTileFloats;
  uint8_t* xs = smem + a.off_x;
  float* xsum = reinterpret_cast<float*>(smem + a.off_sum);   // [group of this CTA's K][NT * 8 columns]
  int* s_abort = reinterpret_cast<int*>(smem + a.off_bars + kWarps * a.stages * 8);
  float* s_stat = reinterpret_cast<float*>(s_abort + 16);     // [(row, part), 32 at most][max, sums of squares]
  float* s_scale = s_stat + 96;                               // [32]
  float* s_inv = s_scale + 32;                                // [32]
  const int rank = a.s > 1 ? (int)cluster_rank() : 0;
  const int cluster = (int)blockIdx.x / a.s, clusters = (int)gridDim.x / a.s;
  const int kb0 = rank * a.kb;  // this CTA's first job along K
  const T* nw = static_cast<const T*>(a.norm_weight);
  const bool split = nw != nullptr && std::is_same<T, __half>::value;  // two parts a row

  if (tid == 0) *s_abort = 0;
  if (lane == 0) {
    for (int s = 0; s < a.stages; ++s) mbar_init(bars + 8 * s, 1);
    fence_mbar_init();
  }
  __syncwarp();
  grid_launch_dependents();

  const int tile0 = (int)((int64_t)cluster * a.tiles / clusters);
  const int tile_end = (int)((int64_t)(cluster + 1) * a.tiles / clusters);
  Jobs<kWarps> ld;
  ld.round = tile0;
  ld.cut(a, tile_end);
  Jobs<kWarps> job = ld;
  // the first weights into L2 (where every earlier write is seen) while the kernel before this one ends
  if (lane == 0) {
    Jobs<kWarps> pf = ld;
    for (int s = 0; s < a.stages && pf.settle(a, tile_end); ++s, pf.step(a)) {
      const int t = pf.round + pf.tile, x = (kb0 + pf.jk) * 128;
      tma_prefetch_l2_2d(&a.tm_w[0], x, t * tile_n);
      if (pair) tma_prefetch_l2_2d(&a.tm_w[1], x, t * tile_n);
    }
  }
  grid_dependency_wait();

  const uint64_t policy = l2_policy_evict_first();
  const auto issue = [&](int stage) -> int {
    if (!ld.settle(a, tile_end)) return 0;
    if (lane == 0) {
      const int t = ld.round + ld.tile, x = (kb0 + ld.jk) * 128;
      const uint32_t dst = ring + stage * kJobBytes, bar = bars + 8 * stage;
      mbar_arrive_expect_tx(bar, kJobBytes);
      tma_load_2d_hint(dst, &a.tm_w[0], x, t * tile_n, bar, policy);
      if (pair) tma_load_2d_hint(dst + 1024, &a.tm_w[1], x, t * tile_n, bar, policy);
    }
    ld.step(a);
    return 1;
  };
  int flying = 0;
#pragma unroll 1
  for (int s = 0; s < a.stages; ++s) flying += issue(s);

  // ---- (scale, zero) of a job: lane i of a row's four holds rows g + 8 (i / 2), groups (i % 2) kHold ..
  Jobs<kWarps> sj = job;  // next job whose scales are fetched
  const int my_row = tile_row(g), hi_row = i >> 1;
  const uint8_t* const my_zeros = pair && hi_row ? a.zeros[1] : a.zeros[0];
  const uint16_t* const my_scales = static_cast<const uint16_t*>(pair && hi_row ? a.scales[1] : a.scales[0]);
  const int n_off = my_row + (pair ? 0 : 8 * hi_row);
  const auto fetch = [&](uint32_t (&v)[kHold]) {
#pragma unroll
    for (int j = 0; j < kHold; ++j) v[j] = 0u;
    if (!sj.settle(a, tile_end)) return;
    const int n = (sj.round + sj.tile) * tile_n + n_off, grp0 = (kb0 + sj.jk) * kSegs + (i & 1) * kHold;
    sj.step(a);
    if (n >= a.n) return;
    const int64_t at = (int64_t)n * a.groups + grp0;
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      if (grp0 + j >= a.groups) continue;
      const float z = my_zeros != nullptr ? (float)my_zeros[at + j] : 8.f;
      union {
        T t;
        uint16_t u;
      } zb;
      zb.t = Elem<T>::from_float(z);  // 0..15: exact
      v[j] = my_scales[at + j] | (uint32_t)zb.u << 16;
    }
  };
  uint32_t sz0[kHold], sz1[kHold], sz2[kHold];
  fetch(sz0);
  fetch(sz1);
  fetch(sz2);

  // ---- rows' largest element (of this CTA's K) and sum of squares (of all K)
  const T* x = static_cast<const T*>(a.x);
  constexpr int kFly = NT <= 2 ? 4 : 8;  // vectors in flight a thread
  const int parts = a.rows >= kWarps ? 1 : kWarps / a.rows;  // warps a row
  const int vec0 = kb0 * (kJobK / 8), vecs = a.kb * (kJobK / 8), all_vecs = a.k / 8;
  for (int u = warp; u < a.rows * parts; u += kWarps) {
    const int r = u / parts, first = (u - r * parts) * 32 + lane;
    const uint4* row = reinterpret_cast<const uint4*>(x + r * a.x_stride);
    const int lo = nw != nullptr ? 0 : vec0, hi = nw != nullptr ? all_vecs : min(vec0 + vecs, all_vecs);
    float ss = 0.f, far = 0.f, top = 0.f;  // far: of elements times 2^-70, where squares pass fp32's range
    for (int v0 = lo + first; v0 < hi; v0 += kFly * parts * 32) {
      uint4 q[kFly], wq[kFly];
#pragma unroll
      for (int j = 0; j < kFly; ++j) {
        const int v = v0 + j * parts * 32;
        q[j] = wq[j] = make_uint4(0, 0, 0, 0);
        if (v < hi) {
          q[j] = row[v];
          if (nw != nullptr) wq[j] = reinterpret_cast<const uint4*>(nw)[v];
        }
      }
#pragma unroll
      for (int j = 0; j < kFly; ++j) {
        const int v = v0 + j * parts * 32;
        float f[8], w[8];
        Elem<T>::unpack(q[j], f);
        Elem<T>::unpack(wq[j], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ss = fmaf(f[e], f[e], ss);
          const float small = f[e] * 8.470329472543003e-22f;
          far = fmaf(small, small, far);
          if (nw != nullptr) f[e] *= w[e];
          if (v >= vec0 && v < vec0 + vecs) top = fmaxf(top, fabsf(f[e]));
        }
      }
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, off);
      far += __shfl_xor_sync(0xffffffffu, far, off);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    }
    if (lane == 0) s_stat[3 * u] = top, s_stat[3 * u + 1] = ss, s_stat[3 * u + 2] = far;
  }
  __syncthreads();
  if (tid < a.rows) {
    float ss = 0.f, far = 0.f, top = 0.f;
    for (int u = tid * parts; u < (tid + 1) * parts; ++u)
      top = fmaxf(top, s_stat[3 * u]), ss += s_stat[3 * u + 1], far += s_stat[3 * u + 2];
    float rstd = 1.f;
    if (nw != nullptr)
      rstd = ss < INFINITY ? rsqrtf(ss / (float)a.k + a.eps) : rsqrtf(far / (float)a.k) * 8.470329472543003e-22f;
    // 2^e that brings the largest element to [2^9, 2^10); 1 for a row of zeros or one with inf
    const uint32_t bits = __float_as_uint(top * rstd) >> 23;
    const int e = bits == 0u || bits >= 255u ? 0 : min(136 - (int)bits, 100);
    s_scale[tid] = rstd * __uint_as_float((uint32_t)(127 + e) << 23);
    s_inv[tid] = __uint_as_float((uint32_t)(127 - e) << 23);
  }
  __syncthreads();

  // ---- x' into shared memory, in the order in which the products take it
  for (int at0 = tid; at0 < a.rows * vecs; at0 += kFly * kThreads) {
    uint4 q[kFly], wq[kFly];
#pragma unroll
    for (int j = 0; j < kFly; ++j) {
      const int at = at0 + j * kThreads, r = at / vecs, v = vec0 + at - r * vecs;
      q[j] = wq[j] = make_uint4(0, 0, 0, 0);
      if (r < a.rows && v < all_vecs) {
        q[j] = reinterpret_cast<const uint4*>(x + r * a.x_stride)[v];
        if (nw != nullptr) wq[j] = reinterpret_cast<const uint4*>(nw)[v];
      }
    }
#pragma unroll
    for (int j = 0; j < kFly; ++j) {
      const int at = at0 + j * kThreads, r = at / vecs, v = at - r * vecs;
      if (r >= a.rows) break;  // whole warps: vecs is a multiple of 32
      float f[8], w[8], lo[8], sum = 0.f, low_sum = 0.f;
      Elem<T>::unpack(q[j], f);
      Elem<T>::unpack(wq[j], w);
      const float scale = s_scale[r];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = (nw != nullptr ? f[e] * w[e] : f[e]) * scale;
        f[e] = __half2float(__float2half_rn(y));
        lo[e] = split ? __half2float(__float2half_rn(y - f[e])) : 0.f;
        sum += f[e];
        low_sum += lo[e];
      }
      const int wd = v & 31, rem = wd % (4 * W);
      const int step = (v >> 5) * 8 + wd / (4 * W) * W + rem % W, li = rem / W;
      // pairs (k0, k4), (k1, k5) / 16, (k2, k6), (k3, k7) / 16
      const auto put = [&](int col, const float* y) {
        union {
          __half2 h[4];
          uint4 u;
        } d;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          d.h[e] = __floats2half2_rn(y[e] * (e & 1 ? 0.0625f : 1.f), y[e + 4] * (e & 1 ? 0.0625f : 1.f));
        *reinterpret_cast<uint4*>(xs + ((step * NT + (col >> 3)) * 32 + (col & 7) * 4 + li) * 16) = d.u;
      };
      put(split ? 2 * r : r, f);
      if (split) put(2 * r + 1, lo);
      // the group's sum: 4 W neighbouring lanes hold it
#pragma unroll
      for (int off = 2 * W; off >= 1; off >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, off);
        low_sum += __shfl_xor_sync(0xffffffffu, low_sum, off);
      }
      if (rem == 0) {
        float* d = xsum + (v / (4 * W)) * NT * 8 + (split ? 2 * r : r);
        d[0] = sum * 5.9604644775390625e-8f;  // 2^-24, as the weights
        if (split) d[1] = low_sum * 5.9604644775390625e-8f;
      }
    }
  }
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
        const uint32_t wrow = ring + stage * kJobBytes + my_row * 128;
        const uint8_t* xf = xs + (size_t)(job.jk * 8 * NT * 32 + lane) * 16;
        const float* gs = xsum + job.jk * kSegs * NT * 8 + 2 * i;
#pragma unroll
        for (int seg = 0; seg < kSegs; ++seg) {
          const uint32_t s_lo = __shfl_sync(0xffffffffu, sz0[seg % kHold], (lane & ~3) | seg / kHold);
          const uint32_t s_hi = __shfl_sync(0xffffffffu, sz0[seg % kHold], (lane & ~3) | 2 | seg / kHold);
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
#pragma unroll
        for (int j = 0; j < kHold; ++j) sz0[j] = sz1[j], sz1[j] = sz2[j];
        fetch(sz2);
      }
      const int tile = job.tile;
      job.step(a);
      fresh = job.jk == 0;
      if (fresh || job.left == 0) {
        float* dst = (head ? heads + warp * kTileFloats : part + tile * kTileFloats) + my_row;
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
    const int tiles = min(a.tiles_round, tile_end - job.round), total_jobs = tiles * a.kb;
    const int n0 = job.round * tile_n, width = min(tiles * tile_n, a.n - n0);
    for (int at = rank * kThreads + tid; at < width * a.rows; at += a.s * kThreads) {
      const int r = at / width, c = at - r * width, tile = c / tile_n, row = c - tile * tile_n;
      const int place = (split ? 2 * r : r) * kPitch + row;
      // warps that hold a head of this tile: those whose first job lies inside it
      int w0 = (tile * a.kb + 1) * kWarps / total_jobs;  // no smaller w begins after the tile's first job
      float y[2] = {0.f, 0.f};
      const auto add = [&](int where) {
        float v[2][2][8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (q >= a.s) break;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              v[m][h][q] = 0.f;
              if ((m == 1 && !pair) || (h == 1 && !split)) continue;
              const float* p = part + where + place + 8 * m + h * kPitch;
              v[m][h][q] = a.s > 1 ? ld_cluster(smem_u32(p), q) * ld_cluster(smem_u32(s_inv + r), q) : *p * s_inv[r];
            }
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (q >= a.s) break;
          y[0] += v[0][0][q] + v[0][1][q];
          y[1] += v[1][0][q] + v[1][1][q];
        }
      };
      add(tile * kTileFloats);
      for (int w = w0; w < kWarps; ++w) {
        const int begin = w * total_jobs / kWarps;
        if (begin >= (tile + 1) * a.kb) break;
        if (begin > tile * a.kb && begin < (w + 1) * total_jobs / kWarps) add((a.tiles_round + w) * kTileFloats);
      }
      float v = y[0];
      if (pair) v = v / (1.f + expf(-v)) * y[1];
      if (a.mode == AICAS_LINEAR_RESIDUAL)
        v += Elem<T>::to_float(static_cast<const T*>(a.residual)[r * a.res_stride + n0 + c]);
      static_cast<T*>(a.out)[r * a.out_stride + n0 + c] = Elem<T>::from_float(v);
    }
    job.round += a.tiles_round;
    if (job.round >= tile_end) break;
    job.cut(a, tile_end);
    if (a.s > 1) cluster_sync_all(); else __syncthreads();  // the partial tiles have been read
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
int plan_int4(Int4Args* a, int nt, int s) {
  const int jobs = (a->k + kJobK - 1) / kJobK;
  a->s = s;
  a->kb = (jobs + s - 1) / s;
  a->tiles_round = nt == 1 ? 16 : nt == 2 ? 8 : 4;
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
    for (int s = 1; s <= 8 && smem == 0; s *= 2) smem = plan_int4(&a, nt, s);
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
