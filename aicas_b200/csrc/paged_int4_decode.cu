// GQA decode attention (one query token per request) over a paged cache of 4-bit rows:
//   k_t = sk_t * ck_t + lk_t,  v_t = sv_t * cv_t + lv_t  (codes 0..15; scale and least a group)
//   o = softmax(scale * q K^T) V over the slots [start, len) of a request,
//   lse = log2(sum_j 2^(scale log2(e) q.k_j)).
//
// A row is a quarter of a 16-bit one and its products are as many, so what has to be kept
// low beside the bytes is the work on a code.  The codes enter mma.sync as they are:
//   q.k_t = sk_t (q.ck_t) + lk_t (sum q),   sum_t p_t v_t = sum_t (p_t sv_t) cv_t + sum_t p_t lv_t,
// so a code costs a mask (and half a shift): the 4 bits in the low end of an fp16 are the
// subnormal number code * 2^-24, 4 bits further up code * 2^-20, both exact, as are their
// products in the fp32 accumulators.  The 1 / 16 of the latter is taken on the other operand
// (q) or at the end (o).  Scales and least values act on a score or a probability, not on an
// element.
//
//   * Work: paged_split.cuh's equal ranges of tiles of 32 slots, one CTA an SM; partials of a
//     pair cut by ranges are joined by the last CTA to arrive, in CTA order, so results
//     repeat to the bit.
//   * Copies: each warp streams its tiles with 16-byte cp.async into a ring of its own,
//     rows swizzled so that the fragment loads below meet no bank twice.  A row is 64
//     bytes (D = 128) and a page may be 8 rows, too small for a tensor copy each.
//   * Products: m16n8k16 with K (16 slots) and V^T (16 dims) as the 16-row operand and the
//     heads as the 8 columns; a probability moves from the scores' accumulator layout to
//     the operand layout by a transposing 8 x 8 move in registers.
//   * Rounding: a 16-bit q enters as one fp16 after scaling by a power of two a head.  In the
//     dims that are taken by 1 / 16 an element is exact down to 2^-24 (of fp16; bf16 2^-27) of its
//     head's largest and off by at most 2^-35 of that below, in the others down to 2^-28 (2^-31)
//     and 2^-39.  A probability times its scale enters P V as two fp16 parts, 22 bits, or to
//     within 2^-25 of numbers that a power of two brings to 2^7 and more for the largest scale
//     of V so far: 2^-32 of that scale, whatever its slot's
//     probability.  Everything else is fp32, but a product's sum is cut off, not rounded, and
//     codes are all positive, so that a long chain of products into o drifts, and with values around
//     0 the sums of scale times code and of least cancel.  So o is emptied into a rounded sum
//     in shared memory every kHoldTiles tiles: 128 fp16 caches of 65536 slots 2.3e-4 off the 64-bit
//     result (its own rounding is 2.07e-4), without 1.5e-2; 4 of 131072 2.2e-4, 3.4e-4.
//   * Slots out of range: score -inf, V's scale and least 0.
//   * Bound: HBM, from a few thousand tiles on.  16 query and 8 KV heads of 128 in bf16: 4
//     caches of 131072 slots, groups of 64, 110 us, 5.5 TB/s; 64 of up to 4096, groups of 128,
//     38 us, 4.0 TB/s, of which about 5 us pass before the first products and 6 after the copies end.
//     One of 1024 7.3 us: the chain lengths, page table, rows, products, join.
//   * Taken and dropped (64 of up to 4096): masks after multiplies instead of shifts 41 -> 44
//     us; rings of 3 stages no faster than 2; 8 warps of twice the registers 10% slower; two
//     partial results joined at once 37 -> 52 (spills).  Against the drift of o, V's codes centred
//     at 8, by products with a constant (4 x 131072 111 us) or the lanes' own sums (109.5): codes
//     that do not average 8 drift on.
#include <cstdio>
#include <cstring>
#include <type_traits>

#include "common.cuh"
#include "paged_int4.cuh"
#include "paged_int4_tiles.cuh"

namespace aicas {
namespace {

constexpr int kTile = kInt4Tile;
// Ranges that a pair is cut into, about: 64 caches of up to 4096 slots, with 1 42.6 us, 2 38.9,
// 4 38.1, 8 38.9.
constexpr int kRanges = 4;
// What beginning and ending a pair costs a warp, in tiles: the same with 1 39.8, 3 38.1, 6 39.4;
// 256 caches of up to 512 31.4, 28.8, 31.0.
constexpr int kPairCost = 3;
// Most tiles a CTA of a launch that gives pairs whole teams: 8 caches of up to 2048 slots 10.4
// us, in equal ranges 11.9 (with 8 already), one of 8192 10.4, 11.0.
constexpr int kSmallTiles = 32;
constexpr int kLogWarps = 4, kMaxWarps = 1 << kLogWarps;
// Warps of a team in a small launch, as a power of two: one cache of 1024 slots with 2 8.2 us, 4 7.3, 16 8.5.
constexpr int kSmallLog = 2;
constexpr int kHeads = 8;      // query heads of a block
// Tiles of a warp whose products are added up in the tensor cores alone: 4 caches of 131072 slots
// 109.9 us with 8, 109.0 with 16, 105.3 without an end (64 of up to 4096 38.1, 37.8, 36.9).
constexpr int kHoldTiles = 8;
constexpr size_t kWsCounters = (size_t)1 << 20;  // counter region shared with the other decode kernels
struct Int4Args {
  Int4Source src;
  const void* q;
  void* out;
  float* lse;
  const int32_t* lens;
  const int32_t* starts;
  int64_t q_sb, q_sh, o_sb, o_sh;
  int batch, hq, hkv, group, row_blocks, cap;
  int few;                 // at most half as many pairs as CTAs
  int part_heads;          // heads that a partial result has room for
  float scale_log2;
  float* ws_o;             // [2 * teams][part_heads][D]
  float* ws_ml;            // [2 * teams][part_heads][2]
  unsigned int* ws_count;  // [teams]
};

template <int D, int GD>
struct Int4Cfg : Int4Stage<D, GD, 2> {
  static constexpr int kWarps = kMaxWarps, kThreads = kWarps * 32;
  static constexpr int kStages = 2;
  static constexpr int kRedRow = D + 4;
  static constexpr int kOffRed = kWarps * kStages * Int4Cfg::kStage;
  static constexpr int kOffVars = kOffRed + kWarps * kHeads * kRedRow * 4;
  static constexpr int kSmem = kOffVars + 4 * kWarps;
  static_assert(kSmem <= 232448, "shared memory");
  static_assert(32 * D <= kHeads * kRedRow * 4, "a warp's sums");
};

using Seg = Segment<kTile>;

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// hi = fp16(x), lo = fp16(x - hi) of two numbers: hi's and lo's packed.
__device__ __forceinline__ void split_half(float x, float y, uint32_t& hi, uint32_t& lo) {
  union {
    __half2 h;
    uint32_t u;
  } r;
  r.h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(r.h);
  hi = r.u;
  lo = pack_half(x - f.x, y - f.y);
}

// ------------------------------------------------------------------ a warp's state

// WIDE: up to 8 heads, a column each, lo parts in products of their own; else up to 4
// heads, head j's hi and lo parts in columns 2 j and 2 j + 1 of the same products (2 heads, 4
// caches of 131072 slots: 110 us, as WIDE 132).
// A lane's heads: WIDE 2 i and 2 i + 1, else i; its slots of 16: rows g and g + 8 of a product.
// K's fragments are words: lane i has 8 dims of each 32.  V's are 16-bit units of 4 dims,
// paired over two slots by the transposing load: lane g has units g of each 32.
template <typename T, int D, int GD, bool WIDE>
struct Int4State {
  using C = Int4Cfg<D, GD>;
  static constexpr int kN = WIDE ? 2 : 1;  // heads a lane
  static constexpr int kWords = D / 32;    // words of K a lane takes of a row: 8 dims each
  uint32_t q[kWords][4];  // of a word's dims (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16
  float fq[kN], qs[kN][GD];  // of the lane's heads: factor of q.code, sum of q, both with the softmax's scale
  float o[D / 16][4];
  float ref[kN];           // what scores are taken against; within kSlack of the largest so far, or above
  float l[kN], z[kN][GD];  // the lane's shares of sum p, sum p least
  float lift;              // power of two on scales of V
  float bound;             // the largest scale of V that lift is good for; -1: no tile yet
  bool holds;              // the warp's part of the reduction buffer has what was added up before o was last emptied

  // p stays below 2^kSlack: the reference is moved when a score passes it by more.
  static constexpr float kSlack = 4.f;

  uint32_t k_off, v_off, p_off;  // this lane's places in a stage: rows of the fragment loads, pairs

  // The lane's place in the warp's part of the reduction buffer, which is free until put.
  __device__ __forceinline__ static float4* place() {
    extern __shared__ __align__(128) uint8_t smem[];
    return reinterpret_cast<float4*>(smem + C::kOffRed + (threadIdx.x >> 5) * (kHeads * C::kRedRow * 4)) + (threadIdx.x & 31);
  }

  __device__ __forceinline__ void init() {
    const int lane = threadIdx.x & 31, mat = lane >> 3, r = lane & 7;
    // K, D = 128: chunk mat of rows 0..7; D = 64: chunk mat / 2 of rows 0..7 and 8..15
    k_off = D == 128 ? r * C::kRow + 16 * swizzled<D>(r, mat) : (r + 8 * (mat & 1)) * C::kRow + 16 * swizzled<D>(r, mat >> 1);
    v_off = C::kOffV + (r + 8 * (mat & 1)) * C::kRow + 16 * swizzled<D>(r, mat >> 1);
    p_off = C::kOffPairs + (lane >> 2) * 2 * C::kPair;
  }

  // Asks for the query heads of a segment's pair.
  __device__ __forceinline__ static void ask(const Int4Args& a, const Seg& s, uint4 (&raw)[kWords]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3;
    const int kvh = s.pair / a.row_blocks, h0 = (s.pair - kvh * a.row_blocks) * kHeads;
    const int heads = min(kHeads, a.group - h0);
    const int col = WIDE ? g : g >> 1;  // the head of column g
    const T* src = static_cast<const T*>(a.q) + s.b * a.q_sb + (int64_t)(kvh * a.group + h0 + min(col, heads - 1)) * a.q_sh;
#pragma unroll
    for (int c = 0; c < kWords; ++c) raw[c] = *reinterpret_cast<const uint4*>(src + 32 * c + 8 * i);
  }

  __device__ __forceinline__ void begin(const Int4Args& a, const uint4 (&raw)[kWords]) {
    const int i = threadIdx.x & 3;
    float x[kWords][8], top = 0.f, sum[GD] = {};
#pragma unroll
    for (int c = 0; c < kWords; ++c) {
      Elem<T>::unpack(raw[c], x[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        top = fmaxf(top, fabsf(x[c][e]));
        sum[c * GD / kWords] += x[c][e];
      }
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
#pragma unroll
      for (int e = 0; e < GD; ++e) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], off);
    }
    // top in [2^14, 2^15) after scaling: with an exponent E, times 2^(14 - E)
    const int E = (int)(__float_as_uint(top) >> 23) - 127;
    const bool plain = top > 0.f && E < 128 && E > -100;  // else 0, infinite, NaN, or so small that it may be lost
    const int up = plain ? 14 - E : 0;
    const float by = __uint_as_float((uint32_t)(up + 127) << 23);
    const float back = __uint_as_float((uint32_t)(127 - up) << 23) * kCodeUnit * a.scale_log2;
#pragma unroll
    for (int c = 0; c < kWords; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[c][e] *= by;
      q[c][0] = pack_half(x[c][0], x[c][4]);
      q[c][1] = pack_half(x[c][1] * 0.0625f, x[c][5] * 0.0625f);
      q[c][2] = pack_half(x[c][2], x[c][6]);
      q[c][3] = pack_half(x[c][3] * 0.0625f, x[c][7] * 0.0625f);
    }
    // from the lanes of column g to the lanes that hold the column's scores
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int from = 4 * (WIDE ? 2 * i + n : 2 * i);
      fq[n] = __shfl_sync(0xffffffffu, back, from);
#pragma unroll
      for (int e = 0; e < GD; ++e) qs[n][e] = __shfl_sync(0xffffffffu, sum[e], from) * a.scale_log2;
      ref[n] = 0.f, l[n] = 0.f;
#pragma unroll
      for (int e = 0; e < GD; ++e) z[n][e] = 0.f;
    }
    lift = 0.f, bound = -1.f, holds = false;
#pragma unroll
    for (int n = 0; n < D / 16; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  }

  // A score passes the reference by more than kSlack, or a scale of V the bound: both anew.
  __device__ __forceinline__ void move(float (&s)[2][2][kN], const float2 (&v)[2][2][GD]) {
    float f[kN], top = 0.f;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < GD; ++e) top = fmaxf(top, fabsf(v[a][b][e].x) < INFINITY ? fabsf(v[a][b][e].x) : 0.f);
    const uint32_t largest = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    const bool first = bound < 0.f;
    float again = 1.f;
    if (__uint_as_float(largest) > bound) {
      // the largest to [2^7, 2^8), so that it may grow 16-fold, and p to 2^kSlack, below 2^16
      const int E = min(max((int)(largest >> 23) - 127, -100), 127);
      const float to = __uint_as_float((uint32_t)(7 - E + 127) << 23);
      again = lift == 0.f ? 1.f : to / lift;
      lift = to;
      bound = __uint_as_float(min((uint32_t)(E + 4 + 127) << 23, 0x7f7fffffu));
    }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      float mt = fmaxf(fmaxf(s[0][0][n], s[0][1][n]), fmaxf(s[1][0][n], s[1][1][n]));
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, off));
      // scores are less the old reference; the first tile sets it, down too
      const float up = mt == -INFINITY ? 0.f : first ? mt : fmaxf(mt, 0.f);
      ref[n] += up;
      // nothing is added up before the first tile, and 2^-up overflows where its scores are far below 0
      const float alpha = first ? 1.f : exp2_fast(-up);
      l[n] *= alpha;
#pragma unroll
      for (int e = 0; e < GD; ++e) z[n][e] *= alpha;
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) s[a][b][n] -= up;
      f[n] = alpha * again;
    }
    if (first) return;  // nothing added up yet
#pragma unroll
    for (int n = 0; n < D / 16; ++n)
      o[n][0] *= f[0], o[n][1] *= f[kN - 1], o[n][2] *= f[0], o[n][3] *= f[kN - 1];
    if (holds) {
      float4* const held = place();
#pragma unroll 1
      for (int n = 0; n < D / 16; ++n) {
        const float4 x = held[32 * n];
        held[32 * n] = make_float4(x.x * f[0], x.y * f[kN - 1], x.z * f[0], x.w * f[kN - 1]);
      }
    }
  }

  // Adds o to what is held, rounding the sum, and empties it.
  __device__ __forceinline__ void hold() {
    float4* const held = place();
#pragma unroll
    for (int n = 0; n < D / 16; ++n) {
      float4 x = holds ? held[32 * n] : make_float4(0.f, 0.f, 0.f, 0.f);
      x.x += o[n][0], x.y += o[n][1], x.z += o[n][2], x.w += o[n][3];
      held[32 * n] = x;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
    }
    holds = true;
  }

  // One tile at shared-memory address `at`; lo..hi: its slots in range.
  __device__ __forceinline__ void tile(uint32_t at, int lo, int hi) {
    float s[2][2][kN];  // [16 slots][row half][head], less ref
    float2 v[2][2][GD];  // scale and least of V
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      float acc[GD][4] = {};
      uint32_t w[2][4];  // rows g and g + 8
      if constexpr (D == 128) {
        ldsm_x4(at + k_off + 16 * mt * C::kRow, w[0]);
        ldsm_x4(at + k_off + (16 * mt + 8) * C::kRow, w[1]);
      } else {
        uint32_t u[4];
        ldsm_x4(at + k_off + 16 * mt * C::kRow, u);
        w[0][0] = u[0], w[1][0] = u[1], w[0][1] = u[2], w[1][1] = u[3];
      }
#pragma unroll
      for (int c = 0; c < kWords; ++c) {
        float* t = acc[c * GD / kWords];
        const uint32_t w0 = w[0][c], w1 = w[1][c], u0 = w0 >> 8, u1 = w1 >> 8;
        mma(t, w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u, q[c][0], q[c][1]);
        mma(t, u0 & 0x000f000fu, u1 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x00f000f0u, q[c][2], q[c][3]);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t kp[GD], vp[GD];
        lds_pairs(at + p_off + (16 * mt + 8 * half) * 2 * C::kPair, kp, vp);
#pragma unroll
        for (int n = 0; n < kN; ++n) s[mt][half][n] = -ref[n];
#pragma unroll
        for (int e = 0; e < GD; ++e) {
          const float2 k = pair_of<T>(kp[e]);
          v[mt][half][e] = pair_of<T>(vp[e]);
#pragma unroll
          for (int n = 0; n < kN; ++n)
            s[mt][half][n] = fmaf(acc[e][2 * half + n] * fq[n], k.x, fmaf(k.y, qs[n][e], s[mt][half][n]));
        }
      }
    }
    if (lo > 0 || hi < kTile) {  // an end of the range
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = 16 * mt + 8 * half + ((threadIdx.x & 31) >> 2);
          if (r >= lo && r < hi) continue;
#pragma unroll
          for (int n = 0; n < kN; ++n) s[mt][half][n] = -INFINITY;
#pragma unroll
          for (int e = 0; e < GD; ++e) v[mt][half][e] = make_float2(0.f, 0.f);
        }
    }
    // ---- online softmax: a head's reference is agreed on by its eight lanes
    float top = 0.f, most = -INFINITY;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int n = 0; n < kN; ++n) most = fmaxf(most, s[a][b][n]);
#pragma unroll
        for (int e = 0; e < GD; ++e) top = fmaxf(top, fabsf(v[a][b][e].x));
      }
    if (__any_sync(0xffffffffu, most > kSlack || top > bound)) move(s, v);
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) l[n] += s[a][b][n] = exp2_fast(s[a][b][n]);
    // ---- o += V^T P^T
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      uint32_t ph[GD][2], pl[GD][2];  // operands of slots 0..7 and 8..15
#pragma unroll
      for (int e = 0; e < GD; ++e) {
        const float2 v0 = v[mt][0][e], v1 = v[mt][1][e];
        const float u0 = v0.x * lift, u1 = v1.x * lift;
#pragma unroll
        for (int n = 0; n < kN; ++n) z[n][e] = fmaf(s[mt][0][n], v0.y, fmaf(s[mt][1][n], v1.y, z[n][e]));
        uint32_t h, lw;
        if constexpr (WIDE) {
          split_half(s[mt][0][0] * u0, s[mt][0][1] * u0, h, lw);
          ph[e][0] = transposed(h), pl[e][0] = transposed(lw);
          split_half(s[mt][1][0] * u1, s[mt][1][1] * u1, h, lw);
          ph[e][1] = transposed(h), pl[e][1] = transposed(lw);
        } else {
          split_half(s[mt][0][0] * u0, s[mt][1][0] * u1, h, lw);
          ph[e][0] = transposed(__byte_perm(h, lw, 0x5410));
          ph[e][1] = transposed(__byte_perm(h, lw, 0x7632));
        }
      }
#pragma unroll
      for (int cp = 0; cp < D / 64; ++cp) {  // 64 dims: units of chunks 2 cp (rows 0..7 of the products) and 2 cp + 1
        const int e = GD == 2 ? cp : 0;
        uint32_t w[4];  // chunk 2 cp: slots 0..7, 8..15; chunk 2 cp + 1: the same
        ldsm_x4_t(at + (v_off ^ (32 * cp)) + 16 * mt * C::kRow, w);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t mask = t & 1 ? 0x00f000f0u : 0x000f000fu;
          mma(o[4 * cp + t], w[0] & mask, w[2] & mask, w[1] & mask, w[3] & mask, ph[e][0], ph[e][1]);
          if constexpr (WIDE) mma(o[4 * cp + t], w[0] & mask, w[2] & mask, w[1] & mask, w[3] & mask, pl[e][0], pl[e][1]);
          if (t == 1)
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] >>= 8;
        }
      }
    }
  }

  // A slot's pairs of K and V.
  __device__ __forceinline__ static void lds_pairs(uint32_t addr, uint32_t* k, uint32_t* v) {
    if constexpr (GD == 1) {
      asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(k[0]), "=r"(v[0]) : "r"(addr) : "memory");
    } else {
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(k[0]), "=r"(k[1]), "=r"(v[0]), "=r"(v[1]) : "r"(addr) : "memory");
    }
  }

  // The block's heads into this warp's part of the reduction buffer.
  __device__ __forceinline__ void put(int heads, float* red) {
    const int lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3;
    const float drop = lift == 0.f ? 0.f : 1.f / lift;  // times kCodeUnit it would overflow for scales of 2^111
    if (holds) {
      float4* const held = place();
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        const float4 x = held[32 * n];
        o[n][0] += x.x, o[n][1] += x.y, o[n][2] += x.z, o[n][3] += x.w;
      }
      __syncwarp();  // every lane has read its share of the buffer
    }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int h = WIDE ? 2 * i + n : i;
      float sum = l[n], least[GD];
#pragma unroll
      for (int e = 0; e < GD; ++e) least[e] = z[n][e];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, off);
#pragma unroll
        for (int e = 0; e < GD; ++e) least[e] += __shfl_xor_sync(0xffffffffu, least[e], off);
      }
      if (h >= heads) continue;
      float* row = red + h * C::kRedRow;
#pragma unroll
      for (int cp = 0; cp < D / 64; ++cp)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float x[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const float* c = o[4 * cp + t] + 2 * half;
            x[t] = fmaf((WIDE ? c[n] : c[0] + c[1]) * (t & 1 ? kCodeUnit / 16.f : kCodeUnit), drop, least[GD == 2 ? cp : 0]);
          }
          *reinterpret_cast<float4*>(row + 64 * cp + 32 * half + 4 * g) = make_float4(x[0], x[1], x[2], x[3]);
        }
      if (g == 0) *reinterpret_cast<float2*>(row + D) = make_float2(bound < 0.f ? -INFINITY : ref[n], sum);
    }
  }
};

// ------------------------------------------------------------------ the kernel

template <typename T>
__device__ __forceinline__ void write_result(const Int4Args& a, int b, int head, int d, float4 o4, float M, float L) {
  const float inv = L == 0.f ? 0.f : 1.f / L;
  union {
    T t[4];
    uint2 u;
  } r;
  r.t[0] = Elem<T>::from_float(o4.x * inv), r.t[1] = Elem<T>::from_float(o4.y * inv);
  r.t[2] = Elem<T>::from_float(o4.z * inv), r.t[3] = Elem<T>::from_float(o4.w * inv);
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + b * a.o_sb + head * a.o_sh + d) = r.u;
  if (a.lse != nullptr && d == 0) a.lse[(int64_t)b * a.hq + head] = L == 0.f ? -INFINITY : M + log2f(L);
}

template <typename T, int D, int GD, bool WIDE>
__global__ void __launch_bounds__(Int4Cfg<D, GD>::kThreads, 1) paged_decode_int4_kernel(const __grid_constant__ Int4Args a) {
  using C = Int4Cfg<D, GD>;
  extern __shared__ __align__(128) uint8_t smem[];
  int* s_last = reinterpret_cast<int*>(smem + C::kOffVars);  // of a team, at its first warp's place
  float* red = reinterpret_cast<float*>(smem + C::kOffRed);
  const int tid = threadIdx.x, warp = tid >> 5;
  grid_launch_dependents();
  grid_dependency_wait();
  Split<kTile> split = {};
  split.template find<kLogWarps, kSmallLog, kRanges, kPairCost, kSmallTiles>(a);
  const int team = 1 << split.log, rank = warp & (team - 1), threads = 32 * team, lane_id = tid & (threads - 1);
  const auto team_sync = [&] {
    if (team == 1) {
      __syncwarp();
    } else {
      asm volatile("bar.sync %0, %1;" ::"r"(1 + (warp >> split.log)), "r"(threads) : "memory");
    }
  };
  const uint32_t ring = smem_u32(smem) + warp * C::kStages * C::kStage;
  using State = Int4State<T, D, GD, WIDE>;
  uint4 raw[State::kWords];
  Cursor<D, GD, 2, Int4Args> ahead;
  if (split.busy) {
    State::ask(a, split.seg, raw);  // on its way while the tiles are asked for
    ahead.begin(a, split.seg, rank, team);
#pragma unroll
    for (int k = 0; k < C::kStages; ++k) ahead.copy(a, ring + k * C::kStage, rank, team);
  }
  if (split.empty_rows)  // requests with nothing to attend to: zeros
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
      int start, len, nt;
      request_bounds<kTile>(a, b, start, len, nt);
      if (nt == 0)
        for (int x = tid; x < a.hq * (D / 4); x += C::kThreads)
          write_result<T>(a, b, x / (D / 4), x % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f);
    }
  if (!split.busy) return;

  Seg seg = split.seg;
  const int chunk = split.chunk;
  const bool small = split.small;
  float* const team_red = red + (warp - rank) * kHeads * C::kRedRow;
  State st;
  st.init();
  int stage = 0, turn = 0;  // turn: the warp that takes the segment's first tile
  for (bool first = true;;) {
    if (seg.t0 == seg.t1) {
      if (!seg.next(a)) break;
      State::ask(a, seg, raw);
      continue;
    }
    st.begin(a, raw);
#pragma unroll 1
    for (int t = seg.t0 + ((rank - turn) & (team - 1)); t < seg.t1; t += team) {
      asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
      __syncwarp();  // every lane's copies have landed
      const uint32_t at = ring + stage * C::kStage;
      const int slot = (seg.first_tile + t) * kTile;
      st.tile(at, seg.start - slot, seg.len - slot);
      if ((~t & (kHoldTiles - 1) * team) == 0) st.hold();
      __syncwarp();  // every lane has read the stage
      ahead.copy(a, at, rank, team);
      if (++stage == C::kStages) stage = 0;
    }
    turn = (turn + seg.t1 - seg.t0) & (team - 1);

    // ---- the warps' states into one
    const int kvh = seg.pair / a.row_blocks, h0 = (seg.pair - kvh * a.row_blocks) * kHeads;
    const int heads = min(kHeads, a.group - h0), head0 = kvh * a.group + h0;
    const bool whole = seg.t0 == 0 && seg.t1 == seg.nt;
    // a pair that starts inside this range is its last: slot 1, unless it is the first, too
    const int64_t ws_row = ((int64_t)split.id * 2 + (first ? 0 : 1)) * a.part_heads;
    st.put(heads, red + warp * kHeads * C::kRedRow);
    team_sync();
    for (int x = lane_id; x < heads * (D / 4); x += threads) {
      const int r = x / (D / 4), d = x % (D / 4) * 4;
      float M = -INFINITY, L = 0.f;
#pragma unroll 4
      for (int w = 0; w < team; ++w) M = fmaxf(M, team_red[(w * kHeads + r) * C::kRedRow + D]);
      const float use = M == -INFINITY ? 0.f : M;
      float4 o4 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int w = 0; w < team; ++w) {
        const float* row = team_red + (w * kHeads + r) * C::kRedRow;
        const float2 ml = *reinterpret_cast<const float2*>(row + D);
        const float f = exp2_fast(ml.x - use);
        const float4 v = *reinterpret_cast<const float4*>(row + d);
        L = fmaf(f, ml.y, L);
        o4.x = fmaf(f, v.x, o4.x), o4.y = fmaf(f, v.y, o4.y);
        o4.z = fmaf(f, v.z, o4.z), o4.w = fmaf(f, v.w, o4.w);
      }
      if (whole) {
        write_result<T>(a, seg.b, head0 + r, d, o4, M, L);
      } else {
        *reinterpret_cast<float4*>(a.ws_o + (ws_row + r) * D + d) = o4;
        if (d == 0) *reinterpret_cast<float2*>(a.ws_ml + (ws_row + r) * 2) = make_float2(M, L);
      }
    }
    team_sync();

    // ---- a pair cut by ranges: the last team to arrive joins the partials in their order
    if (!whole) {
      const int pair0 = seg.pair_base();
      // the teams with tiles of it
      const int c0 = small ? split.first_id : (int)((uint32_t)(pair0 + seg.cost) / (uint32_t)chunk);
      const int c1 = small ? split.last_id : (int)((uint32_t)(pair0 + seg.units() - 1) / (uint32_t)chunk);
      unsigned int last = 0;
      if (lane_id < 32) {
        if (lane_id == 0) {
          unsigned int prev;
          // after the barrier, so cumulative over the team's stores of its partial
          asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(prev) : "l"(a.ws_count + c0) : "memory");
          last = prev == (unsigned int)(c1 - c0);
          if (last) a.ws_count[c0] = 0u;  // as the next call expects it
        }
        last = __shfl_sync(0xffffffffu, last, 0);
        if (team > 1 && lane_id == 0) s_last[warp] = last;
      }
      team_sync();  // lane 0's acquire holds for the team behind a barrier (a shuffle orders no memory)
      if (team > 1) last = s_last[warp - rank];
      if (last) {
        const int first_slot = small || c0 * chunk >= pair0 ? 0 : 1;  // of team c0; the others hold it as their first
        for (int x = lane_id; x < heads * (D / 4); x += threads) {
          const int r = x / (D / 4), d = x % (D / 4) * 4;
          float M = -INFINITY, L = 0.f;
          float4 o4 = make_float4(0.f, 0.f, 0.f, 0.f);
          constexpr int kMany = 4;  // partials in flight
          for (int c = c0; c <= c1; c += kMany) {
            float2 s[kMany];
            float4 v[kMany];
            float Mn = M;
#pragma unroll
            for (int k = 0; k < kMany; ++k) {
              s[k] = make_float2(-INFINITY, 0.f);
              v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (c + k <= c1) {
                const int64_t row = ((int64_t)(c + k) * 2 + (c + k == c0 ? first_slot : 0)) * a.part_heads + r;
                s[k] = __ldcg(reinterpret_cast<const float2*>(a.ws_ml + row * 2));
                v[k] = __ldcg(reinterpret_cast<const float4*>(a.ws_o + row * D + d));
              }
            }
#pragma unroll
            for (int k = 0; k < kMany; ++k) Mn = fmaxf(Mn, s[k].x);
            const float use = Mn == -INFINITY ? 0.f : Mn, old = exp2_fast(M - use);
            L *= old, o4.x *= old, o4.y *= old, o4.z *= old, o4.w *= old;
#pragma unroll
            for (int k = 0; k < kMany; ++k) {
              const float f = exp2_fast(s[k].x - use);
              L = fmaf(f, s[k].y, L);
              o4.x = fmaf(f, v[k].x, o4.x), o4.y = fmaf(f, v[k].y, o4.y);
              o4.z = fmaf(f, v[k].z, o4.z), o4.w = fmaf(f, v[k].w, o4.w);
            }
            M = Mn;
          }
          write_result<T>(a, seg.b, head0 + r, d, o4, M, L);
        }
      }
      if (team > 1) team_sync();  // s_last is free again
    }
    first = false;
    if (!seg.next(a)) break;
    State::ask(a, seg, raw);
  }
}

// ------------------------------------------------------------------ host side

int row_blocks_of(const aicas_paged_decode_int4_params* p) { return (p->num_q_heads / p->num_kv_heads + kHeads - 1) / kHeads; }

// CTAs of a launch: as many as the SMs hold, or fewer where even full caches have fewer tiles for their warps.
int decode_grid(const aicas_paged_decode_int4_params* p, int sms) {
  const int64_t cap_tiles = ((int64_t)p->max_pages * p->page_size + kTile - 1) / kTile;
  const int64_t pairs = (int64_t)p->batch * p->num_kv_heads * row_blocks_of(p);
  const int64_t runs = (cap_tiles * pairs + (1 << kSmallLog) - 1) / (1 << kSmallLog) + pairs;
  return (int)(runs < sms ? runs : sms);
}

int part_heads_of(const aicas_paged_decode_int4_params* p) {
  const int group = p->num_q_heads / p->num_kv_heads;
  return group < kHeads ? group : kHeads;
}

template <typename T, int D, int GD, bool WIDE>
cudaError_t launch_one(const Int4Args& a, int grid, cudaStream_t st) {
  using C = Int4Cfg<D, GD>;
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    e = cudaFuncSetAttribute(paged_decode_int4_kernel<T, D, GD, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  return launch_pdl(paged_decode_int4_kernel<T, D, GD, WIDE>, dim3(grid), dim3(C::kThreads), C::kSmem, st, a);
}

template <typename T>
cudaError_t dispatch(int head_dim, int group_size, const Int4Args& a, int grid, cudaStream_t st) {
  const bool wide = a.group > 4;
  if (head_dim == 64) return wide ? launch_one<T, 64, 1, true>(a, grid, st) : launch_one<T, 64, 1, false>(a, grid, st);
  if (group_size == 64) return wide ? launch_one<T, 128, 2, true>(a, grid, st) : launch_one<T, 128, 2, false>(a, grid, st);
  return wide ? launch_one<T, 128, 1, true>(a, grid, st) : launch_one<T, 128, 1, false>(a, grid, st);
}

}  // namespace

// Two partial results a team; the device makes teams no smaller than for all pairs.
size_t paged_decode_int4_workspace(const aicas_paged_decode_int4_params* p, int sms) {
  const int grid = decode_grid(p, sms);
  const int64_t pairs = (int64_t)p->batch * p->num_kv_heads * row_blocks_of(p);
  const int least = team_log<kLogWarps, kRanges>((int)(pairs < INT32_MAX ? pairs : INT32_MAX), grid);
  const int log = least < kSmallLog ? least : kSmallLog;
  return kWsCounters + ((size_t)grid << (kLogWarps - log)) * 2 * part_heads_of(p) * (p->head_dim + 2) * sizeof(float);
}

int run_paged_decode_int4(const aicas_paged_decode_int4_params* p, int sms, void* workspace, cudaStream_t stream, char* err,
                          size_t errlen) {
  const size_t workspace_bytes = paged_decode_int4_workspace(p, sms);
  Int4Args a;
  memset(&a, 0, sizeof(a));
  if (!a.src.set(p->kv, 2, p->page_table, p->table_stride, p->head_dim, p->group_size, p->num_kv_heads, p->num_pages,
                 p->page_size, err, errlen))
    return AICAS_ERR_UNSUPPORTED;
  a.q = p->q, a.out = p->out, a.lse = p->lse;
  a.lens = p->kv_lens, a.starts = p->kv_starts;
  a.q_sb = p->q_stride_b, a.q_sh = p->q_stride_h, a.o_sb = p->o_stride_b, a.o_sh = p->o_stride_h;
  a.batch = p->batch, a.hq = p->num_q_heads, a.hkv = p->num_kv_heads;
  a.group = p->num_q_heads / p->num_kv_heads;
  a.row_blocks = (a.group + kHeads - 1) / kHeads;
  a.cap = p->max_pages * p->page_size;
  a.scale_log2 = p->sm_scale * 1.4426950408889634f;
  const int grid = decode_grid(p, sms);
  a.few = 2 * (int64_t)a.batch * a.hkv * a.row_blocks <= grid;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.ws_count = reinterpret_cast<unsigned int*>(ws);
  a.ws_o = reinterpret_cast<float*>(ws + kWsCounters);
  a.part_heads = part_heads_of(p);
  a.ws_ml = a.ws_o + (workspace_bytes - kWsCounters) / sizeof(float) / (p->head_dim + 2) * p->head_dim;
  const cudaError_t e = p->dtype == AICAS_DTYPE_F16 ? dispatch<__half>(p->head_dim, p->group_size, a, grid, stream)
                                                    : dispatch<__nv_bfloat16>(p->head_dim, p->group_size, a, grid, stream);
  if (e == cudaSuccess) return AICAS_OK;
  snprintf(err, errlen, "paged 4-bit decode launch: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
  return AICAS_ERR_CUDA;
}

}  // namespace aicas
