// Decode-side products with 4-bit weights:
//   y[r, n] = sum_k x'[r, k] * scale[n, k / g] * (q[n, k] - zero[n, k / g])
// with x' = x or its RMSNorm, and a residual or SiLU(gate) * up epilogue.
//
// HBM bound by its bytes (N K / 2 of weights for at most 2 * 32 * N K flops).  One row of
// many features comes to 70 % of the copy rate, held back by the instructions of the
// product loop (47 % of the issue slots); small products are bound by the way to the
// first product (x, its statistics, x' in shared memory: 2.5 us) and the partial sums'
// way out (1 us, 2.5 over a cluster); many rows by the latency of reading x' from
// shared memory for every 32 rows of weights (tensor pipe 8 %, issue 19 %).
// Measured (bf16, groups of 128, norm where a layer has it; zero points but in the
// first two): 2048 -> 151936 at one row 35.9 us, 4480 GB/s, at 32 rows 133 us;
// 2048 -> 4096 at one row 5.9; SiLU * up 2048 -> 6144 at 8 rows 9.2 us; 6144 -> 2048 at
// 32 rows 13.4 us; 2048 -> 40000 at 32 rows 46 us (114 TFLOP/s).
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
//     element to [2^9, 2^10), as fp16.  16-bit x is exact so down to 2^20 (fp16) or
//     2^23 (bf16) below its row's largest element; smaller ones are off by up to
//     2^-30 of the largest, which is half of fp16's smallest step at an odd k.  (Of a
//     row below 2^-117, whose largest element gets no further than 2^126 times
//     itself, by up to 2^-147.)  A normalised x'
//     is carried as two fp16 parts in neighbouring columns where the result is fp16
//     or the parts of all rows fit one block of columns (run_linear_int4), and
//     rounded to fp16's 11 bits for the bf16 results of more rows.
//   * Sums: a group's sum over the whole numbers q in fp32, less zero point times
//     the group's sum of activations, times the scale in fp32; groups, warps and
//     CTAs are added up in fp32; one rounding at the end.  Rows with an infinity are
//     summed by the definition instead (define_rows): 135 us for one in 32 of 6144 -> 2048.
//   * Work: a cluster of S CTAs takes a run of 32-row tiles (16 gate + 16 up rows
//     for SiLU * up), each CTA one S-th of K, so that its share of x' fits beside
//     the ring (run_linear_int4 chooses S).  Tiles are taken in rounds; a
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
constexpr int kTileRows = 32;
constexpr int kJobBytes = kTileRows * 128;
constexpr int kPitch = 36;              // floats a column of a partial tile (32 rows; 36 keeps stores conflict free)
constexpr int kMaxSmem = 232448;

constexpr int kMaxRound = 40;           // tiles of a round
constexpr int kVarBytes = 64 + 3 * 32 * 4 + kMaxRound * 4 + 8 * 32 * 4;

// Warps of a CTA: more of them hide the products' latency, fewer leave shared
// memory for the columns of many rows.
constexpr int warps_for(int nt) { return nt <= 2 ? 12 : 8; }

// 16-byte vectors of x that a thread holds at once while x' is laid out.
constexpr int fly_for(int nt) { return nt <= 2 ? 6 : 12; }

struct Int4Args {
  CUtensorMap tm_w[2];
  const void* x;
  const void* norm_weight;
  const void* residual;
  void* out;
  const uint8_t* q[2];     // as under the tensor maps
  int64_t q_stride[2];
  const void* scales[2];
  const uint8_t* zeros[2];
  int64_t x_stride, res_stride, out_stride;
  int rows, k, n, groups;  // groups along K
  int mode;
  float eps;
  int s;                   // CTAs of a cluster
  int kb;                  // jobs of a tile for each of them
  int tiles, tiles_round;  // 32-row tiles of the launch; tiles of a round
  int out_quads;           // four outputs may be stored at once
  int whole;               // K is whole jobs and scales and zeros are aligned: vector loads
  int tiles_each, tiles_more;  // tiles of a cluster; the first tiles_more clusters take one more
  int stages;
  int off_part, off_recv, off_x, off_sum, off_bars;
  unsigned int* err;
};

__device__ __forceinline__ void mma_f16(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Element `odd` of a packed pair.
template <typename T>
__device__ __forceinline__ float half_of(uint32_t v, int odd) {
  union {
    uint16_t u[2];
    T t[2];
  } r;
  r.u[0] = (uint16_t)v, r.u[1] = (uint16_t)(v >> 16);
  return Elem<T>::to_float(r.t[odd]);
}

// Byte b of v as a float: its bits under those of 2^23, less 2^23.
__device__ __forceinline__ float byte_of(uint32_t v, int b) {
  return __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7440 | b)) - 8388608.f;
}

__device__ __forceinline__ void st_cluster(float* p, uint32_t rank, const float4& v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}
__device__ __forceinline__ void st_cluster(float* p, uint32_t rank, float v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}
// In two halves: every CTA of the cluster has started once the wait returns.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
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

// x' lies as 512 bytes a step of 16 k and block of 8 columns, a lane's 16 bytes
// after the other.  The lanes that write neighbouring vectors of a row write them
// to different steps; each step's lanes are turned so that these fall in
// different banks (without it four met in one).
template <int W>
__device__ __forceinline__ constexpr int turn(int step) {
  return W == 4 ? (step & 3) * 2 : (step & 1) * 4;
}

// A warp's jobs: those of each round's (tile, job along K) list that fall to it.
template <int WARPS>
struct Jobs {
  int round;       // first tile of the round
  int left;        // jobs of the round still this warp's
  int tile, jk;    // the next one: tile of the round, job along K

  __device__ __forceinline__ void cut(const Int4Args& a, int tile_end) {
    const int warp = threadIdx.x >> 5;
    const int total = min(a.tiles_round, tile_end - round) * a.kb;
    const int each = total / WARPS, more = total - each * WARPS;  // the first `more` warps take one more
    const int begin = warp * each + min(warp, more);
    left = each + (warp < more ? 1 : 0);
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

// Sum of squares of x * by over the vectors first, first + 32, .. below end, over the warp.
template <typename T>
__device__ __noinline__ float sum_squares(const T* row, int first, int end, float by) {
  float ss = 0.f;
#pragma unroll 4
  for (int v = first; v < end; v += 32) {
    float f[8];
    Elem<T>::unpack(reinterpret_cast<const uint4*>(row)[v], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = f[e] * by;
      ss = fmaf(y, y, ss);
    }
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
  return ss;
}

// Up to four neighbouring outputs' sums over [k0, k1) by the definition.
template <typename T>
__device__ __noinline__ float4 defined_sums(const Int4Args& a, int j, int r, int n, int count, int k0, int k1) {
  const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
  const int size = a.k / a.groups;
  float v[4] = {};
  for (int k = k0; k < k1; k += 8) {
    float f[8];
    Elem<T>::unpack(*reinterpret_cast<const uint4*>(x + k), f);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e >= count) break;
      const int64_t grp = (int64_t)(n + e) * a.groups + k / size;
      const uint32_t word = *reinterpret_cast<const uint32_t*>(a.q[j] + (n + e) * a.q_stride[j] + k / 2);
      const float s = Elem<T>::to_float(static_cast<const T*>(a.scales[j])[grp]);
      const int z = a.zeros[j] != nullptr ? a.zeros[j][grp] : 8;
#pragma unroll
      for (int b = 0; b < 8; ++b) v[e] = fmaf((float)((int)(word >> 4 * b & 15) - z) * s, f[b], v[e]);
    }
  }
  return make_float4(v[0], v[1], v[2], v[3]);
}

// Rows with an infinity: the products' sum q x' less zero point times sum x' is inf - inf there,
// where the definition has (q - zero) inf, an infinity unless q is the zero point.  Puts the definition's sums in
// the place of a round's partial ones, each thread for the outputs that it adds up next.
template <typename T, int THREADS>
__device__ __noinline__ void define_rows(const Int4Args& a, float* part, const int* heads, const uint32_t* top, int quads,
                                         int width, int n0, int k0, int k1) {
  const bool pair = a.mode == AICAS_LINEAR_SWIGLU;
  const int tile_n = pair ? 16 : 32, tile_floats = a.rows * kPitch;
  for (int at = threadIdx.x; at < quads * a.rows; at += THREADS) {
    const int r = at / quads, c = 4 * (at - r * quads), tile = c / tile_n;
    if (top[r] != 0x7f800000u) continue;
    const int place = r * kPitch + c - tile * tile_n, w0 = heads[tile] & 0xffff, w1 = heads[tile] >> 16;
    for (int j = 0; j < (pair ? 2 : 1); ++j) {
      *reinterpret_cast<float4*>(part + tile * tile_floats + place + 16 * j) =
          defined_sums<T>(a, j, r, n0 + c, min(4, width - c), k0, k1);
      for (int w = w0 + 1; w <= w1; ++w)
        *reinterpret_cast<float4*>(part + (a.tiles_round + w) * tile_floats + place + 16 * j) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
}

// CLUSTER: K is split over a cluster (a kernel of its own, so that calls of one row, bound by the way to their
// first instruction and back, do not carry the exchange).
// W: 32-bit words of weights that a lane takes side by side (4 W lanes' words
// = 32 W of k share a group of g = 32 W).  NT: blocks of 8 columns.  PARTS: a
// normalised row is two columns.
template <typename T, int NT, int W, bool CLUSTER, bool PARTS>
__global__ void __launch_bounds__(warps_for(NT) * 32, 1) linear_int4_kernel(const __grid_constant__ Int4Args a) {
  constexpr int kWarps = warps_for(NT), kThreads = kWarps * 32;
  constexpr int kSegs = 8 / W;          // groups of a job
  constexpr int kFly = fly_for(NT);     // vectors of x a thread holds at once
  constexpr int kAtOnce = 3;            // and works on side by side
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, i = lane & 3;
  const bool pair = a.mode == AICAS_LINEAR_SWIGLU;
  const int tile_n = pair ? 16 : 32;    // output features of a tile
  const uint32_t ring = smem_u32(smem) + warp * a.stages * kJobBytes;
  const uint32_t bars = smem_u32(smem + a.off_bars) + warp * a.stages * 8;
  float* part = reinterpret_cast<float*>(smem + a.off_part);  // [tiles_round][rows][kPitch], then [kWarps] heads
  float* s_sums = part;  // before the first round: a row's sums of squares, by blocks of 256
  float* recv = reinterpret_cast<float*>(smem + a.off_recv);  // cluster: [from rank][this CTA's share of the outputs]
  uint8_t* xs = smem + a.off_x;
  float* xsum = reinterpret_cast<float*>(smem + a.off_sum);   // [group of this CTA's K][NT * 8 columns]
  int* s_abort = reinterpret_cast<int*>(smem + a.off_bars + kWarps * a.stages * 8);
  int* s_infinite = s_abort + 1;                              // some row has an infinity
  uint32_t* s_top = reinterpret_cast<uint32_t*>(s_abort + 16);   // [32] a row's largest magnitude
  float* s_scale = reinterpret_cast<float*>(s_top + 32);      // [32]
  float* s_inv = s_scale + 32;                                // [32]
  float* s_ss = s_inv + 32;                                   // [8][32] cluster: [from rank] a row's sum of squares over its K
  int* s_heads = reinterpret_cast<int*>(s_ss + 8 * 32);       // [tile of the round] the warps after the tile's first
  const int rank = CLUSTER ? (int)cluster_rank() : 0;
  const int cluster = CLUSTER ? (int)blockIdx.x / a.s : (int)blockIdx.x;
  const int kb0 = rank * a.kb;  // this CTA's first job along K
  const T* nw = static_cast<const T*>(a.norm_weight);
  const bool split = PARTS && nw != nullptr;
  const int tile_floats = a.rows * kPitch;

  if (tid == 0) *s_abort = 0, *s_infinite = 0;
  if (tid < 32) s_top[tid] = 0u;
  if (CLUSTER) cluster_arrive();  // waited for before the first store to another CTA
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
  __syncthreads();
  grid_dependency_wait();

  // ---- x, ahead of the weights: blocks of 256 k of a row, a 16-byte vector a lane, kFly blocks a warp at once
  const T* x = static_cast<const T*>(a.x);
  const int all_vecs = a.k / 8;
  const bool once = a.rows * a.kb <= kFly * kWarps;  // the vectors stay in registers between statistics and staging
  uint4 xq[kFly], wq[kFly];
  int xr[kFly], xb[kFly];
  const auto load = [&](int block) {  // blocks block, block + kWarps, .. of rows of kb
    int r = block / a.kb, at = block - r * a.kb;
#pragma unroll
    for (int j = 0; j < kFly; ++j) {
      xr[j] = r, xb[j] = at;
      const int v = (kb0 + at) * 32 + lane;
      xq[j] = wq[j] = make_uint4(0, 0, 0, 0);
      if (r < a.rows && v < all_vecs) {
        xq[j] = reinterpret_cast<const uint4*>(x + r * a.x_stride)[v];
        if (nw != nullptr) wq[j] = reinterpret_cast<const uint4*>(nw)[v];
      }
      at += kWarps;
      while (at >= a.kb) at -= a.kb, ++r;
    }
  };
  load(warp);

  const uint64_t policy = l2_policy_evict_first();
  if (fill) {
    const uint32_t dst = ring + lane * kJobBytes, bar = bars + 8 * lane;
    mbar_arrive_expect_tx(bar, kJobBytes);
    tma_load_2d_hint(dst, &a.tm_w[0], fill_x, fill_n, bar, policy);
    if (pair) tma_load_2d_hint(dst + 2048, &a.tm_w[1], fill_x, fill_n, bar, policy);
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
      if (pair) tma_load_2d_hint(dst + 2048, &a.tm_w[1], xk, n, bar, policy);
    }
    ld.step(a);
    return 1;
  };
  // a first round with fewer jobs than stages: the next rounds' jobs fill the rest, so that
  // from here on the stage just read is the only free one, or nothing is left to copy
  while (flying < a.stages && issue(flying) != 0) ++flying;

  // ---- scales and zero points of a job: lane i of a lane group holds those of row my_row + 8 i;
  // fetched a job ahead, from L2 where the round before asked for them
  Jobs<kWarps> sj = job;  // next job whose scales are fetched
  const int my_row = tile_row(g);
  const bool up = pair && i >= 2;
  const uint8_t* const my_zeros = up ? a.zeros[1] : a.zeros[0];
  const uint16_t* const my_scales = static_cast<const uint16_t*>(up ? a.scales[1] : a.scales[0]);
  const int n_off = my_row + 8 * (pair ? i & 1 : i);
  uint32_t sc[kSegs / 2], zp[(kSegs + 3) / 4], next_s[kSegs / 2], next_z[(kSegs + 3) / 4];
  int64_t s_at = 0;     // of the next job's first group
  bool s_row = false;   // this lane's row exists
  bool s_new = true;    // the next job begins a tile, a round or the range
  const auto fetch = [&]() {
    if (sj.left == 0) {
      if (!sj.settle(a, tile_end)) return;
      s_new = true;
    }
    const int grp0 = (kb0 + sj.jk) * kSegs;
    if (s_new) {
      const int t = sj.round + sj.tile, n = t * tile_n + n_off;
      s_at = (int64_t)n * a.groups + grp0;
      s_row = n < a.n && grp0 < a.groups;  // K may end before the last CTA's share of it does
      if (t + a.tiles_round < tile_end && n + a.tiles_round * tile_n < a.n && grp0 < a.groups) {  // the next round's, a line of each kind
        const int64_t next = s_at + (int64_t)a.tiles_round * tile_n * a.groups;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(my_scales + next));
        if (my_zeros != nullptr) asm volatile("prefetch.global.L2 [%0];" ::"l"(my_zeros + next));
      }
    }
#pragma unroll
    for (int j = 0; j < (kSegs + 3) / 4; ++j) next_z[j] = 0x08080808u;
    if (s_row && a.whole && grp0 < a.groups) {
      // K is whole jobs: a row's groups of a job are one aligned vector
      if constexpr (kSegs == 2) {
        next_s[0] = *reinterpret_cast<const uint32_t*>(my_scales + s_at);
        if (my_zeros != nullptr) next_z[0] = *reinterpret_cast<const uint16_t*>(my_zeros + s_at);
      } else if constexpr (kSegs == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(my_scales + s_at);
        next_s[0] = v.x, next_s[1] = v.y;
        if (my_zeros != nullptr) next_z[0] = *reinterpret_cast<const uint32_t*>(my_zeros + s_at);
      } else {
        const uint4 v = *reinterpret_cast<const uint4*>(my_scales + s_at);
        next_s[0] = v.x, next_s[1] = v.y, next_s[2] = v.z, next_s[3] = v.w;
        if (my_zeros != nullptr) {
          const uint2 z = *reinterpret_cast<const uint2*>(my_zeros + s_at);
          next_z[0] = z.x, next_z[1] = z.y;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < kSegs / 2; ++j) next_s[j] = 0u;
#pragma unroll 1
      for (int j = 0; j < kSegs; ++j) {
        if (!s_row || grp0 + j >= a.groups) break;
        const uint32_t v = (uint32_t)my_scales[s_at + j] << (16 * (j & 1));
        const uint32_t z = my_zeros != nullptr ? (8u ^ my_zeros[s_at + j]) << (8 * (j & 3)) : 0u;
#pragma unroll
        for (int q = 0; q < kSegs / 2; ++q) next_s[q] |= q == j / 2 ? v : 0u;
#pragma unroll
        for (int q = 0; q < (kSegs + 3) / 4; ++q) next_z[q] ^= q == j / 4 ? z : 0u;
      }
    }
    s_at += kSegs;
    sj.step(a);
    s_new = sj.jk == 0;
  };
  const auto take = [&]() {  // the fetched ones become the next job's
#pragma unroll
    for (int j = 0; j < kSegs / 2; ++j) sc[j] = next_s[j];
#pragma unroll
    for (int j = 0; j < (kSegs + 3) / 4; ++j) zp[j] = next_z[j];
  };
  fetch();

  // ---- which warps share a tile of a full round, for the sums at its end
  const auto find_heads = [&](int tiles) {
    const int total = tiles * a.kb, each = total / kWarps, more = total - each * kWarps;
    const auto warp_of = [&](int j) {
      const int first = j / (each + 1);
      return first < more ? first : more + (j - more * (each + 1)) / max(each, 1);
    };
    if (tid < tiles) s_heads[tid] = warp_of(tid * a.kb) | warp_of((tid + 1) * a.kb - 1) << 16;
  };
  find_heads(min(a.tiles_round, tile_end - tile0));

  // ---- rows' largest element (of this CTA's K) and sum of squares (of all K)
  const auto row_scale = [&](int r, float top, float ss) {
    float rstd = 1.f;
    if (nw != nullptr) {
      rstd = rsqrtf(ss / (float)a.k + a.eps);
      if (!(ss < INFINITY)) {  // squares past fp32's range: of the elements times 2^-70
        const float by = 8.470329472543003e-22f;
        rstd = rsqrtf(sum_squares<T>(x + r * a.x_stride, lane, all_vecs, by) / (float)a.k) * by;
      }
    }
    // 2^e that brings the largest element to [2^9, 2^10), or as near as 2^126 does (2^-126 to 1); 1 for a row with inf
    // (or normalised to subnormal numbers, whose top may be far off)
    const uint32_t bits = __float_as_uint(top * rstd) >> 23;
    const int e = bits >= 255u || (bits == 0u && nw != nullptr) ? 0 : min(136 - (int)bits, 126);
    if (lane == 0) {
      s_scale[r] = nw != nullptr ? rstd : __uint_as_float((uint32_t)(127 + e) << 23);  // their product may be past fp32
      s_inv[r] = __uint_as_float((uint32_t)(127 - e) << 23);
      if (nw == nullptr && top == INFINITY) *s_infinite = 1;  // normalised, it is NaN, as the products make it
    }
  };
  for (int block = warp;;) {
#pragma unroll
    for (int j0 = 0; j0 < kFly; j0 += kAtOnce) {  // reductions side by side hide each other's latency
      if (xr[j0] >= a.rows) break;
      float ss[kAtOnce];
      uint32_t most[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        float f[8], top = 0.f;
        Elem<T>::unpack(xq[j0 + j], f);
        ss[j] = 0.f;
        if (nw != nullptr) {
          float w[8];
          Elem<T>::unpack(wq[j0 + j], w);
#pragma unroll
          for (int e = 0; e < 8; ++e) ss[j] = fmaf(f[e], f[e], ss[j]), f[e] *= w[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[e]));
        most[j] = __float_as_uint(top);  // magnitudes order as their bits
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) most[j] = __reduce_max_sync(0xffffffffu, most[j]);
      if (nw != nullptr)
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1)
#pragma unroll
          for (int j = 0; j < kAtOnce; ++j) ss[j] += __shfl_xor_sync(0xffffffffu, ss[j], off);
      if (lane == 0)
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          const int r = xr[j0 + j];
          if (r >= a.rows) break;
          if (nw != nullptr) s_sums[r * a.kb + xb[j0 + j]] = ss[j];
          atomicMax(s_top + r, most[j]);
        }
    }
    block += kFly * kWarps;
    if (block >= a.rows * a.kb) break;
    load(block);
  }
  __syncthreads();
  const auto row_sum = [&](int r) {
    float ss = 0.f;
    for (int e = lane; e < a.kb; e += 32) ss += s_sums[r * a.kb + e];
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    return ss;
  };
  const bool shared_rows = CLUSTER && nw != nullptr;  // the other CTAs have the rest of a row's squares
  if (shared_rows) {
    cluster_wait();
    for (int r = warp; r < a.rows; r += kWarps) {
      const float ss = row_sum(r);
      if (lane < a.s) st_cluster(s_ss + rank * 32 + r, lane, ss);
    }
    cluster_sync_all();
  }
  for (int r = warp; r < a.rows; r += kWarps) {
    float ss = 0.f;
    if (shared_rows)
      for (int q = 0; q < a.s; ++q) ss += s_ss[q * 32 + r];
    else if (nw != nullptr)
      ss = row_sum(r);
    row_scale(r, __uint_as_float(s_top[r]), ss);
  }
  __syncthreads();

  // ---- x' into shared memory, in the order in which the products take it
  const int my_step = lane / (4 * W) * W + lane % W, my_i = lane % (4 * W) / W;  // of this lane's vector of a block
  const int my_place = my_i ^ turn<W>(my_step);
  for (int block = warp;;) {
    if (!once) load(block);
#pragma unroll
    for (int j = 0; j < kFly; ++j) {
      if (xr[j] >= a.rows) break;
      float f[8];
      Elem<T>::unpack(xq[j], f);
      const float scale = s_scale[xr[j]], odd = scale * 0.0625f;  // odd k's times 2^-4
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= e & 1 ? odd : scale;
      if (nw != nullptr) {
        float w[8];
        Elem<T>::unpack(wq[j], w);
        const float power = __uint_as_float(0x7f000000u - __float_as_uint(s_inv[xr[j]]));  // the 2^e
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = f[e] * w[e] * power;
      }
      const auto put = [&](int col) {  // pairs (k0, k4), (k1, k5), (k2, k6), (k3, k7)
        union {
          __half2 h[4];
          uint4 u;
        } d;
#pragma unroll
        for (int e = 0; e < 4; ++e) d.h[e] = __floats2half2_rn(f[e], f[e + 4]);
        *reinterpret_cast<uint4*>(xs + (((xb[j] * 8 + my_step) * NT + (col >> 3)) * 32 + ((col & 7) * 4 ^ my_place)) * 16) = d.u;
      };
      if (split) {
        put(2 * xr[j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] -= __half2float(__float2half_rn(f[e]));
        put(2 * xr[j] + 1);
      } else {
        put(xr[j]);
      }
    }
    block += kFly * kWarps;
    if (block >= a.rows * a.kb) break;
  }
  __syncthreads();
  // a group's sums of x', times the weights' 2^-24: products with ones in the weights' place
  for (int grp = warp; grp < a.kb * kSegs; grp += kWarps) {
    float acc[NT][4] = {};
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 b = *reinterpret_cast<const uint4*>(xs + (((grp * W + w) * NT + n) * 32 + (lane ^ turn<W>(grp * W + w))) * 16);
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
    float tot[2][NT][4];  // rows my_row + 16 m, + 8; columns 8 n + 2 i, + 1
    bool head = job.jk != 0;  // a tile begun by an earlier warp is this warp's head; its own tiles have a place each
    bool fresh = true;
#pragma unroll 1
    while (job.left > 0) {
      if (fresh) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) tot[m][n][e] = 0.f;
      }
      if (!bad && !mbar_wait(bars + 8 * stage, phase, s_abort, a.err)) bad = true;  // computes no more, keeps to the barriers
      if (!bad) {
        fetch();
        const uint32_t wrow = ring + stage * kJobBytes + my_row * 128;
        const uint8_t* xf = xs + job.jk * 8 * NT * 512;
        const float* gs = xsum + job.jk * kSegs * NT * 8 + 2 * i;
#pragma unroll
        for (int seg = 0; seg < kSegs; ++seg) {
          // this lane's W words of rows my_row + 8 r
          uint32_t w[4][4];
          const int byte = (seg * 4 + i) * W * 4;
          const uint32_t at = wrow + ((byte & ~15) ^ (my_row << 4)) + (byte & 15);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (W == 4)
              asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                           : "=r"(w[r][0]), "=r"(w[r][1]), "=r"(w[r][2]), "=r"(w[r][3]) : "r"(at + 1024 * r));
            else if constexpr (W == 2)
              asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[r][0]), "=r"(w[r][1]) : "r"(at + 1024 * r));
            else
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[r][0]) : "r"(at + 1024 * r));
          }
          float acc[2][NT][4] = {};
#pragma unroll
          for (int j = 0; j < W; ++j) {
            uint32_t h[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) h[r] = w[r][j] >> 8;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint4 b = *reinterpret_cast<const uint4*>(xf + ((seg * W + j) * NT + n) * 512 + (lane ^ turn<W>(seg * W + j)) * 16);
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                const uint32_t p = w[2 * m][j], q = w[2 * m + 1][j];
                mma_f16(acc[m][n], p & 0x000f000fu, q & 0x000f000fu, p & 0x00f000f0u, q & 0x00f000f0u, b.x, b.y);
              }
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                const uint32_t p = h[2 * m], q = h[2 * m + 1];
                mma_f16(acc[m][n], p & 0x000f000fu, q & 0x000f000fu, p & 0x00f000f0u, q & 0x00f000f0u, b.z, b.w);
              }
            }
          }
          float f[4], z[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            f[r] = half_of<T>(__shfl_sync(0xffffffffu, sc[seg / 2], (lane & ~3) | r), seg & 1) * 16777216.f;  // the weights' 2^24
            z[r] = byte_of(__shfl_sync(0xffffffffu, zp[seg / 4], (lane & ~3) | r), seg & 3);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 xg = *reinterpret_cast<const float2*>(gs + (seg * NT + n) * 8);
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                tot[m][n][e] = fmaf(f[2 * m + e / 2], fmaf(-z[2 * m + e / 2], e & 1 ? xg.y : xg.x, acc[m][n][e]), tot[m][n][e]);
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
        float* dst = part + (head ? a.tiles_round + warp : tile) * tile_floats + my_row;
        head = false;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float* const at = dst + 16 * m + 8 * h;
              const float x0 = tot[m][n][2 * h], x1 = tot[m][n][2 * h + 1];
              if (split) {  // a row's two parts are this lane's two columns
                if (4 * n + i < a.rows) at[(4 * n + i) * kPitch] = x0 + x1;
              } else {
                if (8 * n + 2 * i < a.rows) at[(8 * n + 2 * i) * kPitch] = x0;
                if (8 * n + 2 * i + 1 < a.rows) at[(8 * n + 2 * i + 1) * kPitch] = x1;
              }
            }
      }
    }
    __syncthreads();

    if (CLUSTER && !shared_rows && job.round == tile0) cluster_wait();
    // ---- the round's outputs: the warps' partial tiles, then the CTAs', added in their order
    const int n0 = job.round * tile_n, width = min(min(a.tiles_round, tile_end - job.round) * tile_n, a.n - n0);
    // four neighbouring outputs a thread
    const int quads = (width + 3) / 4, count = quads * a.rows, share = CLUSTER ? (count + a.s - 1) / a.s : count;
    const float per_row = 1.f / (float)quads;
    const auto add4 = [](float4& y, const float* p) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      y.x += v.x, y.y += v.y, y.z += v.z, y.w += v.w;
    };
    const auto finish = [&](int r, int c, float4 y, const float4& u) {
      float v[4] = {y.x, y.y, y.z, y.w};
      const float w[4] = {u.x, u.y, u.z, u.w};
      T* out = static_cast<T*>(a.out) + r * a.out_stride + n0 + c;
      const T* res = static_cast<const T*>(a.residual) + r * a.res_stride + n0 + c;
      union {
        T t[4];
        uint2 u;
      } d;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (pair) v[e] = v[e] / (1.f + expf(-v[e])) * w[e];
        if (a.mode == AICAS_LINEAR_RESIDUAL && c + e < width) v[e] += Elem<T>::to_float(res[e]);
        d.t[e] = Elem<T>::from_float(v[e]);
      }
      if (a.out_quads && c + 3 < width) {
        *reinterpret_cast<uint2*>(out) = d.u;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < width) out[e] = d.t[e];
      }
    };
    if (*s_infinite != 0)
      define_rows<T, kThreads>(a, part, s_heads, s_top, quads, width, n0, kb0 * kJobK, min(a.k, (kb0 + a.kb) * kJobK));
    for (int at = tid; at < count; at += kThreads) {
      const int r = (int)((at + 0.5f) * per_row), c = 4 * (at - r * quads);  // at / quads: below 2^14 and 2^9
      const int tile = c / tile_n, place = r * kPitch + c - tile * tile_n;
      const int heads = s_heads[tile], w0 = heads & 0xffff, w1 = heads >> 16;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f), u = y;
      const float* const first = part + tile * tile_floats + place;
      const float* const heads_at = part + (a.tiles_round + w0) * tile_floats + place;
      const auto add_all = [&](float4& sum, int off) {  // up to four loads at once; few tiles have more
        float4 v[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          v[w] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (w <= w1 - w0) v[w] = *reinterpret_cast<const float4*>((w == 0 ? first : heads_at + w * tile_floats) + off);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) sum.x += v[w].x, sum.y += v[w].y, sum.z += v[w].z, sum.w += v[w].w;
#pragma unroll 1
        for (int w = 4; w <= w1 - w0; ++w) add4(sum, heads_at + w * tile_floats + off);
      };
      add_all(y, 0);
      if (pair) add_all(u, 16);
      const float inv = s_inv[r];
      y.x *= inv, y.y *= inv, y.z *= inv, y.w *= inv;
      u.x *= inv, u.y *= inv, u.z *= inv, u.w *= inv;
      if (!CLUSTER) {
        finish(r, c, y, u);
      } else {  // to the CTA that finishes these outputs
        const int owner = at / share, slot = rank * share + at - owner * share;
        st_cluster(recv + 4 * slot, owner, y);
        if (pair) st_cluster(recv + 4 * (a.s * share + slot), owner, u);
      }
    }
    if (CLUSTER) {
      cluster_sync_all();
      for (int at = rank * share + tid; at < min(count, (rank + 1) * share); at += kThreads) {
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f), u = y;
        for (int q = 0; q < a.s; ++q) {
          add4(y, recv + 4 * (q * share + at - rank * share));
          if (pair) add4(u, recv + 4 * ((a.s + q) * share + at - rank * share));
        }
        const int r = (int)((at + 0.5f) * per_row);
        finish(r, 4 * (at - r * quads), y, u);
      }
    }
    job.round += a.tiles_round;
    if (job.round >= tile_end) break;
    job.cut(a, tile_end);
    // the partial tiles have been read, the received ones in every CTA
    if (CLUSTER) cluster_sync_all(); else __syncthreads();
    if (tile_end - job.round < a.tiles_round) find_heads(tile_end - job.round);  // read after the next barrier
  }
  if (bad)
    for (; flying > 0; --flying) {  // leave once this warp's copies have landed (bounded again)
      mbar_wait(bars + 8 * stage, phase, nullptr, a.err);
      if (++stage == a.stages) stage = 0, phase ^= 1;
    }
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

template <typename T, int NT, int W, bool CLUSTER, bool PARTS>
cudaError_t launch_int4(Int4Args a, int smem, int sms, cudaStream_t st) {
  static bool attr_set[64] = {false};
  static int max_clusters[64][4] = {};  // by device and cluster size
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool known = dev >= 0 && dev < 64;
  if (!known || !attr_set[dev]) {
    e = cudaFuncSetAttribute(linear_int4_kernel<T, NT, W, CLUSTER, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
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
  cfg.numAttrs = CLUSTER ? 2 : 1;
  if (CLUSTER) {
    int* cached = known ? &max_clusters[dev][log2_of(a.s)] : nullptr;
    if (cached != nullptr && *cached > 0) {
      clusters = *cached;
    } else {
      cfg.gridDim = dim3((unsigned)a.s);
      cudaLaunchAttribute only = attr[1];
      cfg.attrs = &only;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&clusters, linear_int4_kernel<T, NT, W, CLUSTER, PARTS>, &cfg);
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
  return cudaLaunchKernelEx(&cfg, linear_int4_kernel<T, NT, W, CLUSTER, PARTS>, a);
}

template <typename T, int NT, bool PARTS>
cudaError_t dispatch_group(int group, const Int4Args& a, int smem, int sms, cudaStream_t st) {
  switch (group) {
    case 32: return a.s > 1 ? launch_int4<T, NT, 1, true, PARTS>(a, smem, sms, st) : launch_int4<T, NT, 1, false, PARTS>(a, smem, sms, st);
    case 64: return a.s > 1 ? launch_int4<T, NT, 2, true, PARTS>(a, smem, sms, st) : launch_int4<T, NT, 2, false, PARTS>(a, smem, sms, st);
    case 128: return a.s > 1 ? launch_int4<T, NT, 4, true, PARTS>(a, smem, sms, st) : launch_int4<T, NT, 4, false, PARTS>(a, smem, sms, st);
  }
  return cudaErrorInvalidValue;
}

// parts: the rows of bf16 calls are few enough for two parts, normalised or not (a layer's products share a kernel)
template <typename T>
cudaError_t dispatch_int4(int nt, bool parts, int group, const Int4Args& a, int smem, int sms, cudaStream_t st) {
  constexpr bool kHalf = std::is_same<T, __half>::value;
  switch (nt) {
    case 1:
      if constexpr (!kHalf)
        if (!parts) return dispatch_group<T, 1, false>(group, a, smem, sms, st);
      return dispatch_group<T, 1, true>(group, a, smem, sms, st);
    case 2: return dispatch_group<T, 2, kHalf>(group, a, smem, sms, st);
    case 4: return dispatch_group<T, 4, kHalf>(group, a, smem, sms, st);
  }
  if constexpr (kHalf)  // 32 rows in two parts
    if (nt == 8) return dispatch_group<T, 8, true>(group, a, smem, sms, st);
  return cudaErrorInvalidValue;
}

// Shared memory of a launch of nt column blocks with K split s ways and rings of at least `deep` jobs; 0: does
// not fit.  lean: x has to stay in registers and one round to do.
int plan_int4(Int4Args* a, int nt, int s, int rows, int cols, int deep, bool lean, int sms) {
  const int jobs = (a->k + kJobK - 1) / kJobK;
  a->s = s;
  a->kb = (jobs + s - 1) / s;
  const int warps = warps_for(nt), ring = warps * kJobBytes;
  const int jobs_cta = (int)(((int64_t)a->tiles * s + sms - 1) / sms) * a->kb, jobs_warp = (jobs_cta + warps - 1) / warps;
  // a ring need not hold more than a warp has: one row of 6144 -> 2048 goes over CTAs of their own, not pairs.  By
  // itself 7.9 us against 7.3; among a layer's other products, all of the same kernel then, 3.8 us a layer less.
  if (deep > jobs_warp) deep = jobs_warp;
  const int place = cols * kPitch * 4, recv_tile = s > 1 ? kTileRows * rows * 4 : 0;  // a tile's partial sums, received ones
  const int xs = a->kb * nt * 4096, sums = a->kb * (kJobK / (a->k / a->groups)) * nt * 32;
  const int tail = warps * 8 * 8 + kVarBytes + 16;
  // a round holds a cluster's tiles, if shared memory does beside rings of `deep` jobs; two jobs a warp at least
  const int most = cols <= 8 ? kMaxRound : kMaxRound * 8 / cols, want = (int)((int64_t)a->tiles * s * 4 / (3 * sms)) + 1;
  const int fixed = warps * place + (s > 1 ? 32 * s + 16 : 0) + xs + sums + tail, room = kMaxSmem - deep * ring - fixed;
  const int hold = room < 0 ? 0 : room / (place + recv_tile), least = (2 * warps + a->kb - 1) / a->kb;
  if (lean && (rows * a->kb > fly_for(nt) * warps || want > most || want > hold)) return 0;
  a->tiles_round = want < most ? want : most;
  if (a->tiles_round > hold) {
    if (hold < least || hold < 1) return 0;
    a->tiles_round = hold;
  }
  const int part = (a->tiles_round + warps) * place, recv = s > 1 ? a->tiles_round * recv_tile + 32 * s : 0;
  a->stages = (kMaxSmem - fixed - a->tiles_round * (place + recv_tile)) / ring;
  if (a->stages > 8) a->stages = 8;
  a->off_part = a->stages * ring;
  a->off_recv = a->off_part + part;
  a->off_x = a->off_recv + (recv + 15) / 16 * 16;
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
  a.whole = 1;
  for (int j = 0; j < (pair ? 2 : 1); ++j) {
    if (!weight_map(&a.tm_w[j], p->w[j], p->out_features, p->in_features, pair ? 16 : 32, err, errlen))
      return AICAS_ERR_UNSUPPORTED;
    a.q[j] = static_cast<const uint8_t*>(p->w[j].q);
    a.q_stride[j] = p->w[j].q_stride;
    a.scales[j] = p->w[j].scales;
    a.zeros[j] = static_cast<const uint8_t*>(p->w[j].zeros);
    const int segs = kJobK / p->group_size;
    if (p->in_features % kJobK != 0 || reinterpret_cast<uintptr_t>(a.scales[j]) % (2 * segs) != 0 ||
        reinterpret_cast<uintptr_t>(a.zeros[j]) % segs != 0)
      a.whole = 0;
  }
  a.norm_weight = p->norm_weight;
  a.x_stride = p->x_stride, a.res_stride = p->residual_stride, a.out_stride = p->out_stride;
  a.k = p->in_features, a.n = p->out_features, a.groups = p->in_features / p->group_size;
  a.mode = p->mode, a.eps = p->eps, a.err = dev_err;
  const int tile_n = pair ? 16 : 32;
  a.tiles = (p->out_features + tile_n - 1) / tile_n;
  // A normalised x' in two parts for an fp16 result, and for a bf16 one where both parts of every row fit the 8
  // columns that are multiplied anyway.  One part there changes a tenth of the results of 2048 terms by a unit in the
  // last place, two one in a hundred, for 0.2 us (one row of 2048 -> 4096 5.8 against 5.6 us, 2048 -> 151936 38.4
  // against 38.3; products without a norm, of the same kernel, 5.1 against 5.0 for 2048 -> 2048).  From 5 rows on two
  // parts are twice the columns: 8 rows of 2048 -> 4096 7.8 against 6.8 us, 32 of 2048 -> 4096 23.3 against 13.4, 8 of
  // 2048 -> 151936 81 against 42, 32 263 against 136 (16-bit weights: 181).
  const bool parts = !bf16 || p->rows <= 4;
  const int columns = parts && p->norm_weight != nullptr ? 2 : 1;
  // every row at once where x' fits on chip over a cluster of up to 8 CTAs, else fewer rows a launch
  int batch = p->rows, nt = 0, smem = 0;
  for (;; batch = (batch + 1) / 2) {
    const int blocks = (batch * columns + 7) / 8;
    nt = blocks <= 1 ? 1 : blocks <= 2 ? 2 : blocks <= 4 ? 4 : 8;
    // Rings of three jobs a warp, if some split leaves room for them.  Before that a split that lets x stay in
    // registers between its statistics and its place in shared memory, if the work is one round (else each round
    // pays for the split).  8 rows of 6144 -> 2048: 8.1 us over 4 CTAs, 10.3 over the 2 that would hold x'; 32 of
    // 2048 -> 2048: 10.1 over 4, 14.1 over 2; 32 of 4096 -> 4096 with the norm 19.5 over 8, 21.8 over 4; but 32 of
    // 2048 -> 40000 with the norm, several rounds: 57 over 4, 49 over 2.
    for (int lean = 1; lean >= 0 && smem == 0; --lean)
      for (int deep = 3; deep >= 2 && smem == 0; --deep)
        for (int s = 1; s <= 8 && smem == 0; s *= 2) smem = plan_int4(&a, nt, s, batch, batch * columns, deep, lean, sms);
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
    a.out_quads = reinterpret_cast<uintptr_t>(a.out) % 8 == 0 && (a.rows == 1 || p->out_stride % 4 == 0);
    a.residual = p->residual != nullptr ? static_cast<const uint16_t*>(p->residual) + r * p->residual_stride : nullptr;
    const cudaError_t e = bf16 ? dispatch_int4<__nv_bfloat16>(nt, parts, p->group_size, a, smem, sms, stream)
                               : dispatch_int4<__half>(nt, parts, p->group_size, a, smem, sms, stream);
    if (e != cudaSuccess) {
      snprintf(err, errlen, "int4 linear launch: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
      return AICAS_ERR_CUDA;
    }
  }
  return AICAS_OK;
}

}  // namespace aicas
