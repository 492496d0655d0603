// What attention gave to each cached slot, added up for an eviction:
//   w[b, h, t] += sum over queries s and heads j of the group of 2^(c q[b, j, s].k[b, h, t] - lse[b, j, s]),
// c = scale log2(e), for the slots start <= t <= len - S + s that query s sees.
//
// A slot has one writer and its sum one order, so results repeat to the bit.
//
// 16-bit and 4-bit pages: mma.sync m16n8k16 with 16 slots as rows and 8 queries as columns;
// queries beyond 8 reuse K's fragments.  A sum over the dims may take them in any order,
// so 16-bit rows go from global memory straight into fragments (16 bytes of a row a lane,
// the next tile's on their way while a warp multiplies), with q's laid out to match.
// 4-bit rows, four times as many in flight for the same bytes, come through a ring in
// shared memory (paged_int4_tiles.cuh); the codes enter as paged_int4_decode.cu says.
//   * Work: the tiles of all (request, KV head) pairs in equal runs, cut on the device from
//     the lengths: a run a warp, or, with more than 8 queries, whose fragments the warps
//     of a CTA share, a run a CTA.
//   * Rounding: products of 16-bit numbers are exact, sums and weights fp32.
//   * Bound: HBM.  16 query and 8 KV heads of 128 in bf16: 64 16-bit caches of up to 4096 slots
//     52 us, 5.7 TB/s; 4 of 32768 48 us, 5.8; 4 4-bit ones of 65536 37 us, 4.3.  A window
//     of 16 queries over 4 4-bit caches of 16384 18.5 us, 4.1 for the bytes: the products, four
//     blocks of 8 columns a tile, and 32 exponentials a slot and head.
//   * Taken and dropped (64 of up to 4096): 3 CTAs an SM 52 -> 77 us (spills), tiles of 64 slots
//     63; rings of 4 or 6 stages no faster; for the window, queries as rows with 32 of them in a
//     warp's registers 18.4 -> 20.5 us, both 16 slots of a tile for one load of q 19.9 (spills).
//
// fp32 pages: a thread a slot, its row read once for each block of 8 queries (products of fp32
// numbers in full; the pages that float checks use).
#include <cstdio>
#include <cstring>
#include <type_traits>

#include "common.cuh"
#include "paged_int4.cuh"
#include "paged_int4_tiles.cuh"

namespace aicas {
namespace {

constexpr int kLogWarps = 3, kWarps = 1 << kLogWarps, kThreads = kWarps * 32;
constexpr int kCols = 8;        // queries a product
constexpr int kMostCols = 128;  // queries whose fragments shared memory holds at once

struct WeighArgs {
  aicas_paged_weights_params p;
  // what paged_split.cuh asks for
  const int32_t* lens;
  const int32_t* starts;
  int batch, hkv, row_blocks, cap, few;
  int group, cols;       // queries of a KV head: heads of the group times window
  Int4Source src;        // 4-bit pages; of 16-bit ones the division by the octets of a page
  float scale_log2;
};

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  __device__ __forceinline__ static void run(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <> struct Mma<__half> {
  __device__ __forceinline__ static void run(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// GD: groups a row of 4-bit pages; 0: 16-bit pages.  Of each 32 dims a lane has 8, as words
// of two dims or of 8 codes (of 16-bit heads of 16 it has 4 dims in all).
template <int D, int GD>
struct WeighCfg {
  static constexpr bool k4 = GD > 0;
  static constexpr int kG = k4 ? GD : 1;
  static constexpr int kMt = k4 ? 2 : 1;            // products' 16 slots a tile
  static constexpr int kTile = 16 * kMt;
  static constexpr int kWords = k4 ? D / 32 : D / 8;
  static constexpr int kSteps = D / 16;
  static constexpr int kFrag = 2 * kSteps;          // words of q's fragments a lane and 8 queries
  using Stage = Int4Stage<k4 ? D : 64, kG, 1>;
  static constexpr int kStages = 2;
  static constexpr int kRing = k4 ? kWarps * kStages * Stage::kStage : 0;
};

// What a lane has of a column of 8 queries: of its scores, factor, addends by group, -lse.
template <int G>
struct Column {
  float factor, least[G], minus_lse;
  int end;  // it sees slots below
};

// The fragments of query `col` of a pair (request b, head kvh), of which the four lanes i have a share each.
template <typename T, int D, int GD>
__device__ __forceinline__ void load_query(const WeighArgs& a, int b, int kvh, int len, int col, uint32_t* q,
                                           Column<WeighCfg<D, GD>::kG>& m) {
  using C = WeighCfg<D, GD>;
  const int i = threadIdx.x & 3, S = a.p.seq_len;
  const bool there = col < a.cols;
  const int j = there ? col / S : 0, s = there ? col - j * S : 0, head = kvh * a.group + j;
  const T* src = static_cast<const T*>(a.p.q) + b * a.p.q_stride_b + head * a.p.q_stride_h + s * a.p.q_stride_s;
  const float lse = a.p.lse[b * a.p.lse_stride_b + head * a.p.lse_stride_h + s * a.p.lse_stride_s];
  // a query that saw nothing, and columns that are none, add 2^-inf
  m.minus_lse = there && lse != -INFINITY ? -lse : -INFINITY;
  m.end = len - S + 1 + s;
  m.factor = a.scale_log2;
#pragma unroll
  for (int e = 0; e < C::kG; ++e) m.least[e] = 0.f;
  if constexpr (!C::k4) {
    if constexpr (D == 16) {
      const uint2 u = *reinterpret_cast<const uint2*>(src + 4 * i);
      q[0] = u.x, q[1] = u.y;
    } else {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const uint4 u = *reinterpret_cast<const uint4*>(src + 32 * c + 8 * i);
        q[4 * c] = u.x, q[4 * c + 1] = u.y, q[4 * c + 2] = u.z, q[4 * c + 3] = u.w;
      }
    }
  } else {
    float x[C::kWords][8], top = 0.f, sum[GD] = {};
#pragma unroll
    for (int w = 0; w < C::kWords; ++w) {
      Elem<T>::unpack(*reinterpret_cast<const uint4*>(src + 32 * w + 8 * i), x[w]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        top = fmaxf(top, fabsf(x[w][e]));
        sum[w * GD / C::kWords] += x[w][e];
      }
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
#pragma unroll
      for (int e = 0; e < GD; ++e) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], off);
    }
    // scaled by a power of two, so that the largest is in [2^14, 2^15): paged_int4_decode.cu
    const int E = (int)(__float_as_uint(top) >> 23) - 127;
    const int up = top > 0.f && E < 128 && E > -100 ? 14 - E : 0;
    const float by = __uint_as_float((uint32_t)(up + 127) << 23);
    m.factor = __uint_as_float((uint32_t)(127 - up) << 23) * kCodeUnit * a.scale_log2;
#pragma unroll
    for (int e = 0; e < GD; ++e) m.least[e] = sum[e] * a.scale_log2;
#pragma unroll
    for (int w = 0; w < C::kWords; ++w) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[w][e] *= by;
      q[4 * w] = pack_half(x[w][0], x[w][4]);
      q[4 * w + 1] = pack_half(x[w][1] * 0.0625f, x[w][5] * 0.0625f);
      q[4 * w + 2] = pack_half(x[w][2], x[w][6]);
      q[4 * w + 3] = pack_half(x[w][3] * 0.0625f, x[w][7] * 0.0625f);
    }
  }
}

// A lane's share of a tile: rows g and g + 8 of each 16 slots.
template <int D, int GD>
struct WeighTile {
  using C = WeighCfg<D, GD>;
  uint32_t k[C::kMt][2][C::kWords], pair[C::kMt][2][C::kG];

  // 16-bit rows.  page, row: of octet o of the tile in lane from + o.
  __device__ __forceinline__ void load(const WeighArgs& a, int head, int page, int row, int from) {
    const int g = (threadIdx.x & 31) >> 2, i = threadIdx.x & 3;
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const int pg = __shfl_sync(0xffffffffu, page, from + o), r = __shfl_sync(0xffffffffu, row, from + o) + g;
      uint32_t* w = k[0][o];
#pragma unroll
      for (int e = 0; e < C::kWords; ++e) w[e] = 0u;
      if (pg < 0) continue;
      const uint16_t* p = static_cast<const uint16_t*>(a.p.k_pages) + pg * a.p.kp_stride_p + head * a.p.kp_stride_h + r * a.p.kp_stride_t;
      if constexpr (D == 16) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p + 4 * i));
        w[0] = u.x, w[1] = u.y;
      } else {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(p + 32 * c + 8 * i));
          w[4 * c] = u.x, w[4 * c + 1] = u.y, w[4 * c + 2] = u.z, w[4 * c + 3] = u.w;
        }
      }
    }
  }

  // 4-bit rows from a stage.
  __device__ __forceinline__ void take(uint32_t at) {
    using St = typename C::Stage;
    const int lane = threadIdx.x & 31, mat = lane >> 3, r = lane & 7;
    // D = 128: chunk mat of rows 0..7; D = 64: chunk mat / 2 of rows 0..7 and 8..15
    const uint32_t from = at + (D == 128 ? r * St::kRow + 16 * swizzled<D>(r, mat)
                                         : (r + 8 * (mat & 1)) * St::kRow + 16 * swizzled<D>(r, mat >> 1));
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      uint32_t u[4];
      ldsm_x4(from + 16 * mt * St::kRow, u);
      if constexpr (D == 128) {
#pragma unroll
        for (int e = 0; e < 4; ++e) k[mt][0][e] = u[e];
        ldsm_x4(from + (16 * mt + 8) * St::kRow, u);
#pragma unroll
        for (int e = 0; e < 4; ++e) k[mt][1][e] = u[e];
      } else {
        k[mt][0][0] = u[0], k[mt][1][0] = u[1], k[mt][0][1] = u[2], k[mt][1][1] = u[3];
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t p = at + St::kOffPairs + (16 * mt + 8 * half + (lane >> 2)) * St::kPair;
        if constexpr (GD == 2)
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(pair[mt][half][0]), "=r"(pair[mt][half][1]) : "r"(p) : "memory");
        else
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(pair[mt][half][0]) : "r"(p) : "memory");
      }
    }
  }

  // The products' operand of 16 slots.
  __device__ __forceinline__ void operand(int mt, uint32_t (&f)[C::kSteps][4]) const {
#pragma unroll
    for (int s = 0; s < C::kSteps; ++s) {
      if constexpr (C::k4) {  // half a word of codes
        const uint32_t w0 = k[mt][0][s / 2] >> (s & 1 ? 8 : 0), w1 = k[mt][1][s / 2] >> (s & 1 ? 8 : 0);
        f[s][0] = w0 & 0x000f000fu, f[s][1] = w1 & 0x000f000fu, f[s][2] = w0 & 0x00f000f0u, f[s][3] = w1 & 0x00f000f0u;
      } else {
        f[s][0] = k[mt][0][2 * s], f[s][1] = k[mt][1][2 * s], f[s][2] = k[mt][0][2 * s + 1], f[s][3] = k[mt][1][2 * s + 1];
      }
    }
  }
};

// q(s): the words of steps s and s + 1 of q's fragments.
// Adds the weights of 8 queries (of which a lane has columns c[0] and c[1]) for 16 slots to s0 (row g) and s1 (row g + 8).
template <typename T, int D, int GD, typename Q>
__device__ __forceinline__ void add_columns(const uint32_t (&f)[WeighCfg<D, GD>::kSteps][4], const Q& q,
                                            const uint32_t (&pair)[2][WeighCfg<D, GD>::kG],
                                            const Column<WeighCfg<D, GD>::kG> (&c)[2], int slot, bool causal, float& s0, float& s1) {
  using C = WeighCfg<D, GD>;
  using M = typename std::conditional<C::k4, __half, T>::type;
  constexpr int kChains = C::kG == 2 || C::kSteps == 1 ? C::kG : 2;  // of products that wait for one another
  float acc[kChains][4] = {};
#pragma unroll
  for (int s = 0; s < C::kSteps; s += 2) {
    const uint4 u = q(s);  // of two steps
    Mma<M>::run(acc[s * kChains / C::kSteps], f[s][0], f[s][1], f[s][2], f[s][3], u.x, u.y);
    if (s + 1 < C::kSteps)
      Mma<M>::run(acc[(s + 1) * kChains / C::kSteps], f[s + 1][0], f[s + 1][1], f[s + 1][2], f[s + 1][3], u.z, u.w);
  }
  float s[2][2];
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float x = c[n].minus_lse;
      if constexpr (C::k4) {
#pragma unroll
        for (int e = 0; e < C::kG; ++e) {
          const float2 k = pair_of<T>(pair[half][e]);
          const float sum = C::kG == kChains ? acc[e][2 * half + n] : acc[0][2 * half + n] + acc[kChains - 1][2 * half + n];
          x = fmaf(sum * c[n].factor, k.x, fmaf(k.y, c[n].least[e], x));
        }
      } else {
        const float sum = kChains == 1 ? acc[0][2 * half + n] : acc[0][2 * half + n] + acc[kChains - 1][2 * half + n];
        x = fmaf(sum, c[n].factor, x);
      }
      s[half][n] = x;
    }
  if (causal) {  // the window's own tokens are in the tile
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int n = 0; n < 2; ++n)
        if (slot + 8 * half >= c[n].end) s[half][n] = -INFINITY;
  }
  s0 += exp2_fast(s[0][0]) + exp2_fast(s[0][1]);
  s1 += exp2_fast(s[1][0]) + exp2_fast(s[1][1]);
}

template <typename T, int D, int GD, bool MANY>
__global__ void __launch_bounds__(kThreads, 2) paged_weights_kernel(const __grid_constant__ WeighArgs a) {
  using C = WeighCfg<D, GD>;
  using Col = Column<C::kG>;
  extern __shared__ __align__(128) uint8_t smem[];
  // the ring of 4-bit rows; MANY: [8 queries][lane][kFrag] words of q, then the columns
  uint32_t* q_s = reinterpret_cast<uint32_t*>(smem + C::kRing);
  Col* col_s = reinterpret_cast<Col*>(smem + C::kRing + (MANY ? min(a.cols, kMostCols) + kCols - 1 : 0) / kCols * 32 * C::kFrag * 4);
  constexpr int kVec = C::kFrag < 4 ? C::kFrag : 4;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, i = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * C::kStages * C::Stage::kStage;
  grid_launch_dependents();
  grid_dependency_wait();
  Split<C::kTile> split = {};
  // a run a warp, or (MANY) a CTA
  split.template find<kLogWarps, kLogWarps, MANY ? 0 : (1 << 20), 1, 0>(a);
  if (!split.busy) return;
  const int team = 1 << split.log, rank = warp & (team - 1);
  for (int c0 = 0; c0 < a.cols; c0 += MANY ? kMostCols : kCols) {
    const int blocks = MANY ? (min(a.cols - c0, kMostCols) + kCols - 1) / kCols : 1;
    Segment<C::kTile> seg = split.seg;
    Cursor<C::k4 ? D : 64, C::kG, 1, WeighArgs> ahead;
    int stage = 0, turn = 0;  // turn: the warp that takes the segment's first tile
    if constexpr (C::k4) {
      ahead.begin(a, seg, rank, team);
#pragma unroll
      for (int k = 0; k < C::kStages; ++k) ahead.copy(a, ring + k * C::Stage::kStage, rank, team);
    }
    for (bool more = true; more; more = seg.next(a)) {
      if (seg.t0 == seg.t1) continue;
      const int kvh = seg.pair, b = seg.b;
      uint32_t q[C::kFrag];
      Col mine, c[2];
      if constexpr (MANY) {
        __syncthreads();  // the last ones are done with
        for (int n = warp; n < blocks; n += kWarps) {
          load_query<T, D, GD>(a, b, kvh, seg.len, c0 + n * kCols + g, q, mine);
#pragma unroll
          for (int e = 0; e < C::kFrag; ++e) q_s[(n * C::kFrag + e / kVec * kVec) * 32 + kVec * lane + e % kVec] = q[e];
          if (i == 0) col_s[n * kCols + g] = mine;
        }
        __syncthreads();
      } else {
        load_query<T, D, GD>(a, b, kvh, seg.len, c0 + g, q, mine);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int from = 4 * (2 * i + n);
          c[n].factor = __shfl_sync(0xffffffffu, mine.factor, from);
          c[n].minus_lse = __shfl_sync(0xffffffffu, mine.minus_lse, from);
          c[n].end = __shfl_sync(0xffffffffu, mine.end, from);
#pragma unroll
          for (int e = 0; e < C::kG; ++e) c[n].least[e] = __shfl_sync(0xffffffffu, mine.least[e], from);
        }
      }
      // the words of two steps of q's fragments
      const auto get = [&](int s) {
        return make_uint4(q[2 * s], q[2 * s + 1], 2 * s + 2 < C::kFrag ? q[(2 * s + 2) % C::kFrag] : 0u,
                          2 * s + 3 < C::kFrag ? q[(2 * s + 3) % C::kFrag] : 0u);
      };
      float* w = a.p.weights + b * a.p.w_stride_b + kvh * a.p.w_stride_h;
      // 16-bit pages: the page numbers of 16 tiles at once, octet lane % 2 of tile lane / 2
      int page = -1, row = 0, known = 0;
      const auto look = [&](int t) {
        const int n = (seg.first_tile + t + (lane >> 1) * team) * 2 + (lane & 1);
        const int at = (int)((__umulhi((uint32_t)n, a.src.octets_mul) + (uint32_t)n) >> a.src.octets_shift);
        row = 8 * (n - at * a.src.octets);
        page = -1;
        if (8 * n < seg.len && 8 * n + 8 > seg.start) page = a.p.page_table[b * a.p.table_stride + at];
        if (page >= a.p.num_pages) page = -1;
        known = 16;
      };
      // a lane writes the sum of one slot: row g of half a product, which of 2 kMt halves by i; what it holds so far
      const int place = 8 * i + g;
      const auto held = [&](int t) {
        const int own = (seg.first_tile + t) * C::kTile + place;
        return i < 2 * C::kMt && t < seg.t1 && own >= seg.start && own < seg.len ? w[own] : 0.f;
      };
      int t = seg.t0 + rank;
      if constexpr (C::k4) {  // in the order in which the tiles were asked for
        t = seg.t0 + ((rank - turn) & (team - 1));
        turn = (turn + seg.t1 - seg.t0) & (team - 1);
      }
      float old = held(t);
      WeighTile<D, GD> tile;
      if (!C::k4 && t < seg.t1) {
        look(t);
        tile.load(a, kvh, page, row, 32 - 2 * known--);
      }
#pragma unroll 1
      for (; t < seg.t1; t += team) {
        const int slot = (seg.first_tile + t) * C::kTile;
        const float coming = held(t + team);
        float mine_of_tile = 0.f;
        WeighTile<D, GD> next;
        if constexpr (C::k4) {
          asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
          __syncwarp();  // every lane's copies have landed
          const uint32_t at = ring + stage * C::Stage::kStage;
          tile.take(at);
          __syncwarp();  // every lane has read the stage
          ahead.copy(a, at, rank, team);
          if (++stage == C::kStages) stage = 0;
        } else if (t + team < seg.t1) {
          if (known == 0) look(t + team);
          next.load(a, kvh, page, row, 32 - 2 * known--);
        }
        const bool causal = a.p.seq_len > 1 && slot + C::kTile > seg.len - a.p.seq_len + 1;
#pragma unroll
        for (int mt = 0; mt < C::kMt; ++mt) {
          uint32_t f[C::kSteps][4];
          tile.operand(mt, f);
          float s0 = 0.f, s1 = 0.f;
          if constexpr (MANY) {
#pragma unroll 2
            for (int n = 0; n < blocks; ++n) {
              c[0] = col_s[n * kCols + 2 * i], c[1] = col_s[n * kCols + 2 * i + 1];
#pragma unroll
              for (int e = 0; e < C::kFrag; e += kVec) {
                const uint32_t* from = q_s + (n * C::kFrag + e) * 32 + kVec * lane;
                if constexpr (kVec == 4) {
                  const uint4 u = *reinterpret_cast<const uint4*>(from);
                  q[e] = u.x, q[e + 1] = u.y, q[e + 2] = u.z, q[e + 3] = u.w;
                } else {
                  const uint2 u = *reinterpret_cast<const uint2*>(from);
                  q[e] = u.x, q[e + 1] = u.y;
                }
              }
              add_columns<T, D, GD>(f, get, tile.pair[mt], c, slot + 16 * mt + g, causal, s0, s1);
            }
          } else {
            add_columns<T, D, GD>(f, get, tile.pair[mt], c, slot + 16 * mt + g, causal, s0, s1);
          }
          s0 += __shfl_xor_sync(0xffffffffu, s0, 1), s1 += __shfl_xor_sync(0xffffffffu, s1, 1);
          s0 += __shfl_xor_sync(0xffffffffu, s0, 2), s1 += __shfl_xor_sync(0xffffffffu, s1, 2);
          if ((i >> 1) == mt) mine_of_tile = i & 1 ? s1 : s0;
        }
        if (i < 2 * C::kMt && slot + place >= seg.start && slot + place < seg.len) w[slot + place] = old + mine_of_tile;
        old = coming;
        if constexpr (!C::k4) tile = next;
      }
    }
    if (MANY && c0 + kMostCols < a.cols) __syncthreads();  // the slots' sums so far, before others add to them
  }
}

// ------------------------------------------------------------------ fp32 pages

constexpr int kSlots32 = 128, kBlock32 = 8;

__global__ void __launch_bounds__(kSlots32) paged_weights_f32_kernel(const __grid_constant__ aicas_paged_weights_params a) {
  __shared__ float q_s[kBlock32][128], lse_s[kBlock32];
  __shared__ int end_s[kBlock32];
  const int group = a.num_q_heads / a.num_kv_heads, D = a.head_dim, cap = a.max_pages * a.page_size;
  const int chunks = (cap + kSlots32 - 1) / kSlots32;
  const int kvh = blockIdx.x / chunks % a.num_kv_heads, b = blockIdx.x / chunks / a.num_kv_heads;
  grid_launch_dependents();
  grid_dependency_wait();
  const int len = a.kv_lens != nullptr ? min(max(a.kv_lens[b], 0), cap) : cap;
  const int start = a.kv_starts != nullptr ? max(a.kv_starts[b], 0) : 0;
  const int t0 = blockIdx.x % chunks * kSlots32, t = t0 + threadIdx.x;
  if (t0 >= len || t0 + kSlots32 <= start) return;
  const bool mine = t >= start && t < len;
  const float* k = nullptr;
  if (mine) {
    const int i = t / a.page_size, page = a.page_table[b * a.table_stride + i];
    if (page >= 0 && page < a.num_pages)
      k = static_cast<const float*>(a.k_pages) + page * a.kp_stride_p + kvh * a.kp_stride_h + (t - i * a.page_size) * a.kp_stride_t;
  }
  const float c = a.sm_scale * 1.4426950408889634f;
  float sum = 0.f;
  for (int r0 = 0; r0 < group * a.seq_len; r0 += kBlock32) {
    __syncthreads();
    for (int x = threadIdx.x; x < kBlock32 * D; x += kSlots32) {
      const int r = r0 + x / D, j = kvh * group + r / a.seq_len, s = r % a.seq_len;
      const bool there = r < group * a.seq_len;
      q_s[x / D][x % D] = there ? static_cast<const float*>(a.q)[b * a.q_stride_b + j * a.q_stride_h + s * a.q_stride_s + x % D] : 0.f;
      if (x % D == 0) {
        lse_s[x / D] = there ? a.lse[b * a.lse_stride_b + j * a.lse_stride_h + s * a.lse_stride_s] : -INFINITY;
        end_s[x / D] = len - a.seq_len + 1 + s;
      }
    }
    __syncthreads();
    if (!mine) continue;
    float s[kBlock32] = {};
    if (k != nullptr)
      for (int d = 0; d < D; d += 4) {
        const float4 x = *reinterpret_cast<const float4*>(k + d);
#pragma unroll
        for (int r = 0; r < kBlock32; ++r) {
          const float4 y = *reinterpret_cast<const float4*>(&q_s[r][d]);
          s[r] = fmaf(y.x, x.x, fmaf(y.y, x.y, fmaf(y.z, x.z, fmaf(y.w, x.w, s[r]))));
        }
      }
#pragma unroll
    for (int r = 0; r < kBlock32; ++r)
      if (t < end_s[r] && lse_s[r] != -INFINITY) sum += exp2f(fmaf(s[r], c, -lse_s[r]));
  }
  if (mine) a.weights[b * a.w_stride_b + kvh * a.w_stride_h + t] += sum;
}

// ------------------------------------------------------------------ host side

template <typename T, int D, int GD>
cudaError_t launch_weigh(const WeighArgs& a, int sms, cudaStream_t st) {
  using C = WeighCfg<D, GD>;
  const auto launch = [&](auto kernel, dim3 grid, size_t smem, bool (&attr_set)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (smem > 48 * 1024 && (dev < 0 || dev >= 64 || !attr_set[dev])) {
      constexpr int kMost = C::kRing + kMostCols / kCols * 32 * C::kFrag * 4 + kMostCols * (int)sizeof(Column<C::kG>);
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
      if (e != cudaSuccess) return e;
      if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    return launch_pdl(kernel, grid, dim3(kThreads), smem, st, a);
  };
  static bool attr_few[64] = {false}, attr_many[64] = {false};
  const int64_t tiles = ((int64_t)a.cap + C::kTile - 1) / C::kTile * a.batch * a.hkv;
  const int64_t ctas = (tiles + kWarps - 1) / kWarps;
  const dim3 grid((unsigned)(ctas < 2 * sms ? ctas : 2 * sms));
  if (a.cols <= kCols) return launch(paged_weights_kernel<T, D, GD, false>, grid, C::kRing, attr_few);
  const int cols = ((a.cols < kMostCols ? a.cols : kMostCols) + kCols - 1) / kCols * kCols;
  const size_t smem = C::kRing + (size_t)cols / kCols * 32 * C::kFrag * 4 + (size_t)cols * sizeof(Column<C::kG>);
  return launch(paged_weights_kernel<T, D, GD, true>, grid, smem, attr_many);
}

template <typename T>
cudaError_t dispatch_weigh(const WeighArgs& a, int sms, cudaStream_t st) {
  const int D = a.p.head_dim;
  if (a.p.group_size != 0)
    return D == 64 ? launch_weigh<T, 64, 1>(a, sms, st) : a.p.group_size == 64 ? launch_weigh<T, 128, 2>(a, sms, st) : launch_weigh<T, 128, 1>(a, sms, st);
  switch (D) {
    case 16: return launch_weigh<T, 16, 0>(a, sms, st);
    case 32: return launch_weigh<T, 32, 0>(a, sms, st);
    case 64: return launch_weigh<T, 64, 0>(a, sms, st);
    case 128: return launch_weigh<T, 128, 0>(a, sms, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

int run_paged_weights(const aicas_paged_weights_params* p, int sms, cudaStream_t stream, char* err, size_t errlen) {
  cudaError_t e = cudaErrorInvalidValue;
  if (p->dtype == AICAS_DTYPE_F32) {
    const int64_t chunks = ((int64_t)p->max_pages * p->page_size + kSlots32 - 1) / kSlots32;
    e = launch_pdl(paged_weights_f32_kernel, dim3((unsigned)(chunks * p->batch * p->num_kv_heads)), dim3(kSlots32), 0, stream, *p);
  } else {
    WeighArgs a;
    memset(&a, 0, sizeof(a));
    a.p = *p;
    a.lens = p->kv_lens, a.starts = p->kv_starts;
    a.batch = p->batch, a.hkv = p->num_kv_heads, a.row_blocks = 1, a.cap = p->max_pages * p->page_size;
    a.group = p->num_q_heads / p->num_kv_heads, a.cols = a.group * p->seq_len;
    if (p->group_size != 0) {
      const aicas_int4_pages pages = {const_cast<void*>(p->k_pages), const_cast<void*>(p->k_scales), p->kp_stride_p, p->kp_stride_h,
                                      p->kp_stride_t, p->ks_stride_p, p->ks_stride_h, p->ks_stride_t};
      if (!a.src.set(&pages, 1, p->page_table, p->table_stride, p->head_dim, p->group_size, p->num_kv_heads, p->num_pages,
                     p->page_size, err, errlen))
        return AICAS_ERR_UNSUPPORTED;
    } else {
      a.src.set_division(p->page_size);
    }
    a.scale_log2 = p->sm_scale * 1.4426950408889634f;
    e = p->dtype == AICAS_DTYPE_F16 ? dispatch_weigh<__half>(a, sms, stream) : dispatch_weigh<__nv_bfloat16>(a, sms, stream);
  }
  if (e == cudaSuccess) return AICAS_OK;
  snprintf(err, errlen, "paged weights launch: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
  return AICAS_ERR_CUDA;
}

}  // namespace aicas
