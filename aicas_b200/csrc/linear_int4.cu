// Decode-side products with 4-bit weights:
//   y[r, n] = sum_k x'[r, k] * scale[n, k / g] * (q[n, k] - zero[n, k / g])
// with x' = x or its RMSNorm, and a residual or SiLU(gate) * up epilogue.
//
// HBM bound: N K / 2 bytes of weights for at most 2 * 32 * N K flops.  What it
// takes is turning 4-bit numbers into tensor-core operands as fast as they come.
//
//   * Operands: mma.sync m16n8k16 with the weights as the 16 x 16 side, in
//     registers, and the activations as columns.  A 32-bit word of weights holds
//     k0..k7 of a row; (word >> 4 j) & 0x000f000f is the pair (k_j, k_{j+4}), and
//     or-ing the bits of 128 (bf16) or 1024 (fp16), whose units are 1, and
//     subtracting 128 + zero gives the exact q - zero.  The products do not care
//     in what order k goes by, so the weights stay as stored and the activations
//     are laid out in shared memory to match, once a CTA.  tcgen05 would need the
//     widened weights written back to shared or tensor memory: four times the
//     bytes that came from HBM.
//   * Sums: a group's products are summed in fp32 over whole numbers, multiplied
//     by the group's scale in fp32 and added up in fp32; one rounding at the end.
//     A normalised x' is carried as two 16-bit parts in neighbouring columns.
//   * Work: a cluster of S CTAs takes a run of 16-row tiles (8 gate + 8 up rows
//     for SiLU * up), each CTA one S-th of K, so that its share of x' fits beside
//     the ring (S = 1 wherever all of it does).  Tiles are taken in rounds; a
//     round's (tile, 256 k) jobs are cut evenly over the warps, whatever tile
//     they belong to, and the warps' and CTAs' partial sums are added in a fixed
//     order, so results repeat to the bit.  Each warp streams its own jobs through
//     a private TMA ring that runs on across rounds.
#include <cstdio>
#include <cstring>

#include "common.cuh"
#include "linear_int4.cuh"
#include "tma_host.cuh"

namespace aicas {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kJobK = 256;              // k of a job: 128 bytes of a row
constexpr int kJobBytes = 16 * 128;     // 16 rows
constexpr int kPitch = 20;              // floats a column of a partial tile (16 rows; 20 keeps stores conflict free)
constexpr int kMaxSmem = 232448;
constexpr int kTwoPerSm = 115712;       // shared memory of a CTA of which two fit on an SM

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
  int off_part, off_x, off_bars;
  unsigned int* err;
};

template <typename T> struct Int4Type;
template <> struct Int4Type<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x4300u;  // 128: its unit in the last place is 1
  __device__ __forceinline__ static uint32_t sub(uint32_t a, uint32_t b) {
    __nv_bfloat162 x = *reinterpret_cast<__nv_bfloat162*>(&a), y = *reinterpret_cast<__nv_bfloat162*>(&b);
    x = __hsub2(x, y);
    return *reinterpret_cast<uint32_t*>(&x);
  }
  __device__ __forceinline__ static void mma(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <> struct Int4Type<__half> {
  static constexpr uint32_t kMagic = 0x6400u;  // 1024: its unit in the last place is 1
  __device__ __forceinline__ static uint32_t sub(uint32_t a, uint32_t b) {
    __half2 x = *reinterpret_cast<__half2*>(&a), y = *reinterpret_cast<__half2*>(&b);
    x = __hsub2(x, y);
    return *reinterpret_cast<uint32_t*>(&x);
  }
  __device__ __forceinline__ static void mma(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

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
struct Jobs {
  int tile0, tile_end;  // tiles of the cluster
  int round;            // first tile of the round
  int at, end;          // jobs of the round: this warp's [at, end)

  __device__ __forceinline__ void cut(const Int4Args& a) {
    const int warp = threadIdx.x >> 5;
    const int total = min(a.tiles_round, tile_end - round) * a.kb;
    at = warp * total / kWarps;
    end = (warp + 1) * total / kWarps;
  }
  // Moves to the next job, over the rounds; false after the last.
  __device__ __forceinline__ bool settle(const Int4Args& a) {
    while (at >= end) {
      round += a.tiles_round;
      if (round >= tile_end) return false;
      cut(a);
    }
    return true;
  }
};

// W: 32-bit words of weights that a lane takes side by side (4 W lanes' words
// = 32 W of k share a group of g = 32 W).  NT: blocks of 8 columns.
template <typename T, int NT, int W>
__global__ void __launch_bounds__(kThreads, NT <= 4 ? 2 : 1) linear_int4_kernel(const __grid_constant__ Int4Args a) {
  using E = Int4Type<T>;
  constexpr int kSegs = 8 / W;          // groups of a job
  constexpr int kHold = kSegs / 2;      // (scale, zero) pairs a lane holds of a job: two rows' kSegs over four lanes
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, i = lane & 3;
  const bool pair = a.mode == AICAS_LINEAR_SWIGLU;
  const int tile_n = pair ? 8 : 16;     // output features of a tile
  const uint32_t ring = smem_u32(smem) + warp * a.stages * kJobBytes;
  const uint32_t bars = smem_u32(smem + a.off_bars) + warp * a.stages * 8;
  float* part = reinterpret_cast<float*>(smem + a.off_part);  // [tiles_round tiles][NT * 8][kPitch], then [kWarps] heads
  float* heads = part + a.tiles_round * NT * 8 * kPitch;
  uint8_t* xs = smem + a.off_x;
  int* s_abort = reinterpret_cast<int*>(smem + a.off_bars + kWarps * a.stages * 8);
  float* s_rstd = reinterpret_cast<float*>(s_abort + 1);
  const int rank = a.s > 1 ? (int)cluster_rank() : 0;
  const int cluster = (int)blockIdx.x / a.s, clusters = (int)gridDim.x / a.s;
  const int kb0 = rank * a.kb;  // this CTA's first job along K

  if (tid == 0) *s_abort = 0;
  if (lane == 0) {
    for (int s = 0; s < a.stages; ++s) mbar_init(bars + 8 * s, 1);
    fence_mbar_init();
  }
  __syncwarp();
  grid_launch_dependents();

  Jobs ld;
  ld.tile0 = (int)((int64_t)cluster * a.tiles / clusters);
  ld.tile_end = (int)((int64_t)(cluster + 1) * a.tiles / clusters);
  ld.round = ld.tile0;
  ld.cut(a);
  Jobs job = ld;
  // the first weights into L2 (where every earlier write is seen) while the kernel before this one ends
  if (lane == 0) {
    Jobs pf = ld;
    for (int s = 0; s < a.stages && pf.settle(a); ++s, ++pf.at) {
      const int t = pf.round + pf.at / a.kb, x = (kb0 + pf.at % a.kb) * 128;
      tma_prefetch_l2_2d(&a.tm_w[0], x, t * tile_n);
      if (pair) tma_prefetch_l2_2d(&a.tm_w[1], x, t * tile_n);
    }
  }
  grid_dependency_wait();

  const uint64_t policy = l2_policy_evict_first();
  const auto issue = [&](int stage) -> int {
    if (!ld.settle(a)) return 0;
    if (lane == 0) {
      const int t = ld.round + ld.at / a.kb, x = (kb0 + ld.at % a.kb) * 128;
      const uint32_t dst = ring + stage * kJobBytes, bar = bars + 8 * stage;
      mbar_arrive_expect_tx(bar, kJobBytes);
      tma_load_2d_hint(dst, &a.tm_w[0], x, t * tile_n, bar, policy);
      if (pair) tma_load_2d_hint(dst + 1024, &a.tm_w[1], x, t * tile_n, bar, policy);
    }
    ++ld.at;
    return 1;
  };
  int flying = 0;
#pragma unroll 1
  for (int s = 0; s < a.stages; ++s) flying += issue(s);

  // ---- (scale, zero) of a job: lane i of a row's four holds rows g + 8 (i / 2), groups (i % 2) kHold ..
  Jobs sj = job;  // next job whose scales are fetched
  const int my_row = tile_row(g), hi_row = i >> 1;
  const auto fetch = [&](uint32_t (&v)[kHold]) {
#pragma unroll
    for (int j = 0; j < kHold; ++j) v[j] = E::kMagic << 16;
    if (!sj.settle(a)) return;
    const int t = sj.round + sj.at / a.kb, jk = kb0 + sj.at % a.kb;
    const int n = t * tile_n + my_row + (pair ? 0 : 8 * hi_row);
    const bool up = pair && hi_row;
    const uint8_t* zeros = up ? a.zeros[1] : a.zeros[0];
    const uint16_t* scales = static_cast<const uint16_t*>(up ? a.scales[1] : a.scales[0]);
    ++sj.at;
    if (n >= a.n) return;
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      const int grp = jk * kSegs + (i & 1) * kHold + j;
      if (grp >= a.groups) continue;
      const int64_t at = (int64_t)n * a.groups + grp;
      const uint32_t z = zeros != nullptr ? zeros[at] : 8u;
      v[j] = scales[at] | (E::kMagic | z) << 16;
    }
  };
  uint32_t sz0[kHold], sz1[kHold], sz2[kHold];
  fetch(sz0);
  fetch(sz1);
  fetch(sz2);

  // ---- x' into shared memory, in the order in which the products take it
  const T* x = static_cast<const T*>(a.x);
  const T* nw = static_cast<const T*>(a.norm_weight);
  if (nw != nullptr) {
    for (int r = warp; r < a.rows; r += kWarps) {
      float ss = 0.f;
      for (int v = lane; v < a.k / 8; v += 32) {
        float f[8];
        Elem<T>::unpack(*reinterpret_cast<const uint4*>(x + r * a.x_stride + 8 * v), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
      }
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      if (lane == 0) s_rstd[r] = rsqrtf(ss / (float)a.k + a.eps);
    }
    __syncthreads();
  }
  const int vecs = a.kb * 32;
  for (int at = tid; at < a.rows * vecs; at += kThreads) {
    const int r = at / vecs, v = at - r * vecs;
    const int k = kb0 * kJobK + 8 * v;
    uint4 u = make_uint4(0, 0, 0, 0), lo = u;
    if (k < a.k) {
      u = *reinterpret_cast<const uint4*>(x + r * a.x_stride + k);
      if (nw != nullptr) {
        float f[8], w[8];
        Elem<T>::unpack(u, f);
        Elem<T>::unpack(*reinterpret_cast<const uint4*>(nw + k), w);
        union {
          T t[8];
          uint4 u;
        } h, l;
        const float rstd = s_rstd[r];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = f[e] * rstd * w[e];
          h.t[e] = Elem<T>::from_float(y);
          l.t[e] = Elem<T>::from_float(y - Elem<T>::to_float(h.t[e]));
        }
        u = h.u;
        lo = l.u;
      }
    }
    const int wd = v & 31, rem = wd % (4 * W);
    const int step = (v >> 5) * 8 + wd / (4 * W) * W + rem % W, li = rem / W;
    // pairs (k0, k4), (k1, k5), (k2, k6), (k3, k7)
    const auto put = [&](int col, const uint4& d) {
      *reinterpret_cast<uint4*>(xs + ((step * NT + (col >> 3)) * 32 + (col & 7) * 4 + li) * 16) =
          make_uint4(__byte_perm(d.x, d.z, 0x5410), __byte_perm(d.x, d.z, 0x7632), __byte_perm(d.y, d.w, 0x5410),
                     __byte_perm(d.y, d.w, 0x7632));
    };
    if (nw != nullptr) {
      put(2 * r, u);
      put(2 * r + 1, lo);
    } else {
      put(r, u);
    }
  }
  __syncthreads();

  // ---- rounds
  int stage = 0;
  uint32_t phase = 0;
  bool bad = false;
  for (;;) {
    const int first = job.at;
    float tot[NT][4];
#pragma unroll 1
    for (; job.at < job.end; ++job.at) {
      const int tile = job.at / a.kb, jk = job.at - tile * a.kb;
      if (job.at == first || jk == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) tot[n][e] = 0.f;
      }
      if (!bad && !mbar_wait(bars + 8 * stage, phase, s_abort, a.err)) bad = true;  // computes no more, keeps to the barriers
      if (!bad) {
        const uint32_t wrow = ring + stage * kJobBytes + my_row * 128;
        const uint8_t* xf = xs + (size_t)(jk * 8 * NT * 32 + lane) * 16;
#pragma unroll
        for (int seg = 0; seg < kSegs; ++seg) {
          const uint32_t s_lo = __shfl_sync(0xffffffffu, sz0[seg % kHold], (lane & ~3) | seg / kHold);
          const uint32_t s_hi = __shfl_sync(0xffffffffu, sz0[seg % kHold], (lane & ~3) | 2 | seg / kHold);
          const uint32_t z_lo = __byte_perm(s_lo, 0, 0x3232), z_hi = __byte_perm(s_hi, 0, 0x3232);
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
            uint32_t q0[4], q1[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              q0[j] = E::sub(((w0[w] >> (4 * j)) & 0x000f000fu) | E::kMagic * 0x10001u, z_lo);
              q1[j] = E::sub(((w1[w] >> (4 * j)) & 0x000f000fu) | E::kMagic * 0x10001u, z_hi);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint4 b = *reinterpret_cast<const uint4*>(xf + ((seg * W + w) * NT + n) * 512);
              E::mma(acc[n], q0[0], q1[0], q0[1], q1[1], b.x, b.y);
              E::mma(acc[n], q0[2], q1[2], q0[3], q1[3], b.z, b.w);
            }
          }
          const float f_lo = low_half<T>(s_lo), f_hi = low_half<T>(s_hi);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            tot[n][0] = fmaf(f_lo, acc[n][0], tot[n][0]), tot[n][1] = fmaf(f_lo, acc[n][1], tot[n][1]);
            tot[n][2] = fmaf(f_hi, acc[n][2], tot[n][2]), tot[n][3] = fmaf(f_hi, acc[n][3], tot[n][3]);
          }
        }
        __syncwarp();  // every lane has read the stage
        flying += issue(stage) - 1;
        if (++stage == a.stages) stage = 0, phase ^= 1;
#pragma unroll
        for (int j = 0; j < kHold; ++j) sz0[j] = sz1[j], sz1[j] = sz2[j];
        fetch(sz2);
      }
      if (jk == a.kb - 1 || job.at == job.end - 1) {
        // a tile begun by an earlier warp is this warp's head; its own tiles have a place each
        const bool head = job.at - jk < first;
        float* dst = (head ? heads + warp * NT * 8 * kPitch : part + tile * NT * 8 * kPitch) + my_row;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          dst[(8 * n + 2 * i) * kPitch] = tot[n][0], dst[(8 * n + 2 * i + 1) * kPitch] = tot[n][1];
          dst[(8 * n + 2 * i) * kPitch + 8] = tot[n][2], dst[(8 * n + 2 * i + 1) * kPitch + 8] = tot[n][3];
        }
      }
    }
    if (a.s > 1) cluster_sync_all(); else __syncthreads();

    // ---- the round's outputs: partial tiles of the warps and CTAs added in their order
    const int tiles = min(a.tiles_round, job.tile_end - job.round), total_jobs = tiles * a.kb;
    const int n0 = job.round * tile_n, width = min(tiles * tile_n, a.n - n0);
    const uint32_t part_at = smem_u32(part), heads_at = smem_u32(heads);
    for (int at = rank * kThreads + tid; at < width * a.rows; at += a.s * kThreads) {
      const int r = at / width, c = at - r * width, tile = c / tile_n, row = c - tile * tile_n;
      const int col = nw != nullptr ? 2 * r : r;
      float y[2] = {0.f, 0.f};
      for (int q = 0; q < a.s; ++q) {
        const auto add = [&](uint32_t base) {
          // the low parts of a normalised x' are the next column; up's rows come 8 after gate's
#pragma unroll
          for (int m = 0; m < 2; ++m)
            if (m == 0 || pair) {
              const uint32_t p = base + (col * kPitch + row + 8 * m) * 4;
              y[m] += a.s > 1 ? ld_cluster(p, q) : *reinterpret_cast<const float*>(smem + (p - smem_u32(smem)));
              if (nw != nullptr)
                y[m] += a.s > 1 ? ld_cluster(p + kPitch * 4, q)
                                : *reinterpret_cast<const float*>(smem + (p + kPitch * 4 - smem_u32(smem)));
            }
        };
        add(part_at + tile * NT * 8 * kPitch * 4);
        for (int w = 1; w < kWarps; ++w) {
          const int begin = w * total_jobs / kWarps, end = (w + 1) * total_jobs / kWarps;
          if (begin < end && begin > tile * a.kb && begin < (tile + 1) * a.kb) add(heads_at + w * NT * 8 * kPitch * 4);
        }
      }
      float v = y[0];
      if (pair) v = v / (1.f + expf(-v)) * y[1];
      if (a.mode == AICAS_LINEAR_RESIDUAL)
        v += Elem<T>::to_float(static_cast<const T*>(a.residual)[r * a.res_stride + n0 + c]);
      static_cast<T*>(a.out)[r * a.out_stride + n0 + c] = Elem<T>::from_float(v);
    }
    job.round += a.tiles_round;
    if (job.round >= job.tile_end) break;
    job.cut(a);
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
  static int max_clusters[64][4][2] = {};  // by device, cluster size and CTAs an SM
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool known = dev >= 0 && dev < 64;
  if (!known || !attr_set[dev]) {
    e = cudaFuncSetAttribute(linear_int4_kernel<T, NT, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
    if (e != cudaSuccess) return e;
    if (known) attr_set[dev] = true;
  }
  const bool two = smem <= kTwoPerSm;
  int clusters = sms * (two ? 2 : 1);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)a.s;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = a.s > 1 ? 2 : 1;
  if (a.s > 1) {
    int* cached = known ? &max_clusters[dev][log2_of(a.s)][two] : nullptr;
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
    case 8: return dispatch_group<T, 8>(group, a, smem, sms, st);
  }
  return cudaErrorInvalidValue;
}

// Shared memory of a launch of nt column blocks with K split s ways; 0: does not fit.
int plan_int4(Int4Args* a, int nt, int s) {
  const int jobs = (a->k + kJobK - 1) / kJobK;
  a->s = s;
  a->kb = (jobs + s - 1) / s;
  a->tiles_round = nt == 1 ? 16 : nt == 2 ? 8 : 4;
  const int part = (a->tiles_round + kWarps) * nt * 8 * kPitch * 4, xs = a->kb * nt * 4096, tail = 2048;
  const int rest = part + xs + tail, ring = kWarps * kJobBytes;
  a->stages = (kTwoPerSm - rest) / ring;  // two CTAs an SM, if their rings hold four jobs a warp
  if (a->stages < 4) a->stages = (kMaxSmem - rest) / ring;
  if (a->stages < 3) return 0;
  if (a->stages > 8) a->stages = 8;
  a->off_part = a->stages * ring;
  a->off_x = a->off_part + part;
  a->off_bars = a->off_x + xs;
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
  // every row at once where x' fits on chip over a cluster of up to 8 CTAs (K up to 14336 for 32 rows), else fewer
  const int columns = p->norm_weight != nullptr ? 2 : 1;
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
