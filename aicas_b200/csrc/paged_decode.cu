// GQA decode attention (one query token per request) over a paged KV cache:
//   o = softmax(scale * q K^T) V over the slots [start, len) of a request, slot
//   t being row t % page_size of page table[b, t / page_size];
//   lse = log2(sum_j 2^(scale log2(e) q.k_j)).
//
// HBM bound: every cached row is read once for up to 16 query heads of its group
// (a larger group reads it once for each block of 16) and used for 4 flops a head
// and pair of elements, far below what the tensor cores take, so the design is about
// keeping copies in flight.
//
//   * Work: the 16-slot tiles of all (request, KV head) pairs, numbered pair by
//     pair, are cut into equal ranges, one per CTA (one CTA an SM).  The cut is
//     made on the device from the lengths, so the host neither knows nor bounds
//     them and ragged batches balance to a tile; a pair counts kPairCost tiles more
//     for its beginning and end.  A pair inside one range is finished there; a pair
//     that crosses ranges leaves one fp32 partial a CTA (a CTA has at most two: its
//     first and its last pair), and the last CTA to arrive adds them in CTA order, so
//     results repeat to the bit.  A small launch of few pairs gives each pair CTAs of
//     its own.
//   * Copies: two warps stream the range's K and V tiles as TMA boxes, swizzled so
//     that ldmatrix reads them without bank conflicts, into a ring of its own for
//     each of the other warps, which take the tiles in turn; no warp waits for
//     another inside a pair.  (Warps that copied for themselves spent as long, 900
//     cycles a tile, at issuing the copies as at the products.)  A page number
//     outside the pool is an out-of-range box: zeros.
//   * Products: mma.sync m16n8k16 with the group's query heads as rows (a
//     larger group takes several blocks of 16).  At a few percent of the SM's
//     tensor rate the legacy path is not the bound, and it keeps scores and
//     output in registers, where the softmax is.  fp32 caches use the FMA pipes.
//   * Rounding: fp32 scores and statistics.  A probability enters P V as two
//     16-bit parts (hi + lo), so that only the result is rounded; with up to 8
//     heads the lo parts ride in the 8 unused rows of the same products.  fp16's
//     smallest step is 2^-24: there probabilities are held times 2^14 (up to the
//     end of the pair), so that a weight is within 2^-38 of the largest one.
//   * An infinite element of V in a live slot gives that infinity (split_pair), as long
//     as the slot's weight is one of the numbers above: not below 2^-38 of the
//     largest (fp16) or 2^-102 (bf16).
//   * Slots out of range: scores replaced by -inf and V's elements by 0 before
//     the products (0 * NaN), in the tiles at the range's ends only.
//
// Measured (16 query over 8 KV heads of 128, bf16): 4 caches of 131072 slots 326 us,
// 6590 GB/s; 64 ragged ones of up to 4096 slots 94.4 us, 6090 GB/s (the measured copy
// rate is 6450 GB/s); one cache of 1024 slots 7.9 us, which is a chain of latencies:
// lengths, page numbers, first tiles, a join over CTAs.
#include <cstdio>
#include <cstring>
#include <type_traits>

#include "common.cuh"
#include "paged.cuh"
#include "tma_host.cuh"

namespace aicas {
namespace {

constexpr int kTile = 16;       // slots a tile
// What beginning and ending a pair costs a CTA, in tiles.  3, 6, 10: 64 ragged caches of up to 4096 slots 94.6, 93.4,
// 93.6 us; 128 of 2048 with heads of 64 89.0, 86.3, 90.0.
constexpr int kPairCost = 6;
// Fewest tiles a CTA takes.  8, 16, 32: one cache of 1024 slots 7.2, 7.9, 9.2 us, one of 256 6.9, 5.7, 11.5.
constexpr int kMinChunk = 16;
// Most tiles a CTA of a launch that gives pairs whole CTAs.  16, 32, 64: one cache of 8192 slots 12.7, 10.6, 10.7 us, 8
// ragged ones of up to 2048 15.9, 15.9, 13.8, 128 of 2048 with heads of 64 89.2, 86.3, 89.2.
constexpr int kSmallTiles = 32;
constexpr int kRowsMax = 16;    // query heads of a block
constexpr size_t kWsCounters = (size_t)1 << 20;  // counter region shared with the contiguous decode

struct PagedArgs {
  CUtensorMap tm_k, tm_v;  // 5-D: (128 bytes of D, rows, parts of D, heads, pages), a box all of D of 16 (or 8) rows
  const void* q;
  void* out;
  float* lse;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;
  int64_t q_sb, q_sh, o_sb, o_sh, table_stride;
  int batch, hq, hkv, group, row_blocks;
  int page_size, cap;
  int few;                         // at most half as many pairs as CTAs
  int boxes;                       // boxes of a tile: 1 (16 rows) or 2 (8 rows: page sizes of 8, 24, ...)
  // a tile in shared memory: bytes from one 128-byte part of D to the next, and from rows 0..7 to rows 8..15
  int part_bytes, rows8_bytes;
  float scale_log2;
  float* ws_o;             // [2 * grid][kRowsMax][D]
  float* ws_ml;            // [2 * grid][kRowsMax][2]
  unsigned int* ws_count;  // [grid]
  unsigned int* err;
};

template <typename T, int D>
struct PagedCfg {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kRowBytes = D * (int)sizeof(T);
  static constexpr int kInner = kRowBytes < 128 ? kRowBytes : 128;  // bytes of a box's row (the swizzle's width)
  static constexpr int kSwzMask = kInner / 16 - 1;
  static constexpr int kTileBytes = kTile * kRowBytes;
  static constexpr int kStageBytes = 2 * kTileBytes;  // K tile, V tile
  static constexpr int kWarps = kF32 ? 4 : 8;              // warps at the products; two more copy K and V
  static constexpr int kConsumers = kWarps * 32, kThreads = kConsumers + 64;
  static constexpr int kRing = 196608 / kWarps / kStageBytes;
  static constexpr int kStages = kRing < 8 ? kRing : 8;
  static constexpr int kRedRow = D + 4;  // a row's output, its maximum and its sum
  static constexpr int kOffRed = kWarps * kStages * kStageBytes;
  static constexpr int kOffQ = kOffRed + kWarps * 8 * kRedRow * 4;  // fp32: the block's query rows
  static constexpr int kOffBars = kOffQ + (kF32 ? kRowsMax * D * 4 : 0);  // [warp][stage] full, then empty
  static constexpr int kOffVars = kOffBars + 2 * kWarps * kStages * 8;
  // no static shared memory beside it: the ring starts 1024-byte aligned, as the swizzle wants
  static constexpr int kSmem = kOffVars + 16;
  static_assert(kStages >= 3 && kSmem <= 232448, "shared memory");
};

// ------------------------------------------------------------------ fragments

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t r[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t r[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  __device__ __forceinline__ static void run(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Mma<__half> {
  __device__ __forceinline__ static void run(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Packed pairs hi = (x, y) cut to 16 bits and lo = what that left, rounded.  Both parts
// of a positive weight are positive (hi is cut, not rounded; a lo of 0 becomes the
// smallest part there is): with a 0 among them or opposite signs, an infinite element
// of V would make a NaN (0 inf, inf - inf) where the sum is that infinity.
template <typename T>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo);
template <>
__device__ __forceinline__ void split_pair<__nv_bfloat16>(float x, float y, uint32_t& hi, uint32_t& lo) {
  const uint32_t bx = __float_as_uint(x), by = __float_as_uint(y);
  hi = __byte_perm(bx, by, 0x7632);
  constexpr float kLeast = 5.9604644775390625e-08f;  // 2^-24 of the weight, far below lo's own rounding
  const float lx = fmaxf(x - __uint_as_float(bx & 0xffff0000u), x * kLeast);
  const float ly = fmaxf(y - __uint_as_float(by & 0xffff0000u), y * kLeast);
  union {
    __nv_bfloat162 b;
    uint32_t u;
  } l;
  l.b = __floats2bfloat162_rn(lx, ly);
  lo = l.u;
}
template <>
__device__ __forceinline__ void split_pair<__half>(float x, float y, uint32_t& hi, uint32_t& lo) {
  union {
    __half2 h;
    uint32_t u;
  } p, l;
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(p.u) : "f"(y), "f"(x));
  constexpr float kLeast = 5.9604644775390625e-08f;  // fp16's smallest step, 2^-24
  const float2 f = __half22float2(p.h);
  l.h = __floats2half2_rn(fmaxf(x - f.x, fminf(x, kLeast)), fmaxf(y - f.y, fminf(y, kLeast)));
  hi = p.u;
  lo = l.u;
}

// ------------------------------------------------------------------ the CTA's range

// Units of work: a pair counts its tiles and, before them, kPairCost units for
// beginning and ending it, so that a CTA with many short pairs gets fewer tiles.
//
// The tiles [t0, t1) of one pair (request, KV head and row block) in a CTA's
// range; none where the range ends in the pair's cost.  Tiles count from the one
// that holds the request's first slot.
struct Segment {
  int b, pair;        // request; KV head * row_blocks + row block
  int t0, t1, nt;     // this CTA's tiles, all tiles of the pair
  int first_tile;     // tile of the first slot
  int start, len;     // slots [start, len)
  int base;           // number of the request's first unit in the launch
  int left;           // units of the CTA's range after this segment

  __device__ __forceinline__ int units() const { return nt + kPairCost; }
  __device__ __forceinline__ int pair_base() const { return base + pair * units(); }
  // The pair's units [from, from + count), as far as it has them.
  __device__ __forceinline__ void take(int from, int count) {
    const int to = min(units(), from + count);
    left = count - (to - from);
    t0 = max(0, from - kPairCost);
    t1 = max(0, to - kPairCost);
  }
};

__device__ __forceinline__ void request_bounds(const PagedArgs& a, int b, int& start, int& len, int& nt) {
  len = a.lens != nullptr ? min(max(a.lens[b], 0), a.cap) : a.cap;
  start = a.starts != nullptr ? min(max(a.starts[b], 0), len) : 0;
  nt = len > start ? (len + kTile - 1) / kTile - start / kTile : 0;
}

__device__ __forceinline__ int request_units(const PagedArgs& a, int nt) {
  return nt == 0 ? 0 : (nt + kPairCost) * a.hkv * a.row_blocks;
}

// Fills a segment from unit `unit` of the launch, which lies in request s.b.
__device__ __forceinline__ void segment_at(const PagedArgs& a, Segment& s, int unit, int count) {
  request_bounds(a, s.b, s.start, s.len, s.nt);
  s.first_tile = s.start / kTile;
  const int off = unit - s.base;
  s.pair = off / s.units();
  s.take(off - s.pair * s.units(), count);
}

__device__ __forceinline__ bool segment_next(const PagedArgs& a, Segment& s) {
  if (s.left == 0) return false;
  if (++s.pair == a.hkv * a.row_blocks) {
    s.base += s.units() * a.hkv * a.row_blocks;
    s.pair = 0;
    do {
      ++s.b;  // units are left, so a request with some follows
      request_bounds(a, s.b, s.start, s.len, s.nt);
    } while (s.nt == 0);
    s.first_tile = s.start / kTile;
  }
  s.take(0, s.left);
  return true;
}

// The warps at the products among themselves.
template <int THREADS>
__device__ __forceinline__ void consumers_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}

// ------------------------------------------------------------------ the copying warps

__device__ __forceinline__ void copy_box(const CUtensorMap& m, uint32_t dst, int row, int head, int page, uint32_t bar,
                                         uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %2, %4, %5}], [%6], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(&m)), "r"(0), "r"(row), "r"(head), "r"(page),
      "r"(bar), "l"(policy)
      : "memory");
}

// A lane's tile of a batch of 32: page and row of its (up to) two boxes.
struct Pages {
  int page0, row0, page1, row1;
};

__device__ __forceinline__ Pages pages_of(const PagedArgs& a, const Segment& s, int t) {
  Pages p = {-1, 0, -1, 0};
  if (t < s.t1) {
    const int slot = (s.first_tile + t) * kTile;
    const int32_t* row = a.table + s.b * a.table_stride;
    const int i = slot / a.page_size;
    p.row0 = slot - i * a.page_size;
    p.page0 = row[i];
    if (a.boxes == 2 && slot + 8 < s.len) {
      const bool same = p.row0 + 8 < a.page_size;
      p.row1 = same ? p.row0 + 8 : 0;
      p.page1 = same ? p.page0 : row[i + 1];
    }
  }
  return p;
}

// Copies all K (or V) tiles of the CTA's range: tile number n of it to stage
// (n / kWarps) % kStages of warp n % kWarps.  A lane a tile, kWarps lanes at a time, so that the
// wait for a free stage and the page numbers' way are paid once for kWarps tiles
// (a tile at a time took 0.42 us each).  bars: full barriers, then empty ones.
template <typename T, int D>
__device__ void copy_range(const PagedArgs& a, const CUtensorMap& map, Segment seg, uint32_t ring, uint32_t bars,
                           volatile int* abort) {
  using C = PagedCfg<T, D>;
  const int lane = threadIdx.x & 31;
  const uint64_t policy = l2_policy_evict_first();
  const uint32_t empty = bars + C::kWarps * C::kStages * 8;
  int number = 0;  // of the segment's next tile
  int sent = 0;    // tiles copied by whole turns of kWarps lanes
  int last = -1;   // the lane's tile in a turn that was not whole
  bool ok = true;
  Pages at = pages_of(a, seg, seg.t0 + lane);
  while (ok) {
    const int head = seg.pair / a.row_blocks;
    Segment next = seg;
    bool more = true;
    for (int t = seg.t0; t < seg.t1 && ok; t += 32) {
      // the next batch's page numbers are on their way while this one is copied
      Pages ahead = {};
      if (t + 32 < seg.t1) {
        ahead = pages_of(a, seg, t + 32 + lane);
      } else {
        do more = segment_next(a, next);
        while (more && next.t0 == next.t1);
        if (more) ahead = pages_of(a, next, next.t0 + lane);
      }
      const int count = min(32, seg.t1 - t);
      const int n = number + lane, turn = n / C::kWarps, round = turn / C::kStages;
      const int place = n % C::kWarps * C::kStages + turn % C::kStages;
      const uint32_t dst = ring + place * C::kStageBytes, bar = bars + 8 * place;
      for (int first = 0; first < count && ok; first += C::kWarps) {
        if (lane >= first && lane < min(first + C::kWarps, count)) {
          if (round > 0) ok = mbar_wait(empty + 8 * place, (round - 1) & 1, abort, a.err);
          if (ok) {
            mbar_arrive_expect_tx(bar, C::kTileBytes);
            copy_box(map, dst, at.row0, head, at.page0, bar, policy);
            if (a.boxes == 2) copy_box(map, dst + C::kTileBytes / 2, at.row1, head, at.page1, bar, policy);
            last = n;
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        if (ok) sent = number + min(first + C::kWarps, count);
      }
      number += count;
      at = ahead;
    }
    if (seg.t0 == seg.t1) {  // the range begins in a pair's cost: nothing of it to copy
      more = segment_next(a, next);
      if (more) at = pages_of(a, next, next.t0 + lane);
    }
    if (!more) break;
    seg = next;
  }
  // Leave once this warp's last copies have landed: the products' warps wait for them too, unless a wait gave up.
  const auto landed = [&](int n) {
    const int turn = n / C::kWarps;
    mbar_wait(bars + 8 * (n % C::kWarps * C::kStages + turn % C::kStages), turn / C::kStages & 1, nullptr, a.err);
  };
  for (int n = max(0, sent - C::kWarps * C::kStages) + lane; n < sent; n += 32) landed(n);
  if (last >= sent) landed(last);
}

// ------------------------------------------------------------------ a warp's state, 16-bit caches

// RM: rows in use, 8 (the group fits 8 heads) or 16.
template <typename T, int D, int RM>
struct WarpState {
  using C = PagedCfg<T, D>;
  static constexpr int kSteps = D / 16;
  static constexpr int kH = RM / 8;  // row halves with heads in them
  // what probabilities, and with them o and l, are multiplied by
  static constexpr float kLift = std::is_same<T, __half>::value ? 16384.f : 1.f;
  uint32_t qf[kSteps][RM == 8 ? 2 : 4];
  float o[D / 8][4];
  float m[kH], l[kH];
  uint32_t k_off, v_off;  // this lane's row of the ldmatrix tiles, with its share of the swizzle
  uint32_t k_swz, v_swz;

  __device__ __forceinline__ void init(const PagedArgs& a, const uint8_t*) {
    const int lane = threadIdx.x & 31, mat = lane >> 3, r = lane & 7;
    k_off = (mat >> 1) * a.rows8_bytes + r * C::kInner;
    v_off = (mat & 1) * a.rows8_bytes + r * C::kInner + C::kTileBytes;
    k_swz = ((((r * C::kInner) >> 7) & C::kSwzMask) << 4) ^ ((mat & 1) << 4);
    v_swz = ((((r * C::kInner) >> 7) & C::kSwzMask) << 4) ^ ((mat >> 1) << 4);
  }

  __device__ __forceinline__ void begin(const PagedArgs& a, const Segment& s, uint8_t*) {
    const int lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3;
    const int kvh = s.pair / a.row_blocks, h0 = (s.pair - kvh * a.row_blocks) * kRowsMax;
    const int rows = min(kRowsMax, a.group - h0);
    const T* q = static_cast<const T*>(a.q) + s.b * a.q_sb + (int64_t)(kvh * a.group + h0 + g) * a.q_sh + 2 * i;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {  // dims 16 j + 8 c + 2 i
        const T* p = q + 16 * j + 8 * c;
        qf[j][RM == 8 ? c : 2 * c] = g < rows ? *reinterpret_cast<const uint32_t*>(p) : 0u;
        if constexpr (RM == 16)
          qf[j][2 * c + 1] = g + 8 < rows ? *reinterpret_cast<const uint32_t*>(p + 8 * a.q_sh) : 0u;
      }
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
#pragma unroll
    for (int h = 0; h < kH; ++h) m[h] = -INFINITY, l[h] = 0.f;
  }

  // One tile at shared-memory address `at`; lo..hi: its slots in range (0..16 inside a request).
  __device__ __forceinline__ void tile(const PagedArgs& a, uint32_t at, int lo, int hi) {
    const int i = threadIdx.x & 3;
    // ---- scores of 16 slots: s[n][0..1] = (row g, slots 8 n + 2 i, + 1), s[n][2..3] = row g + 8
    float s[2][4] = {}, s2[2][4] = {};  // even and odd steps: two shorter chains of products
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const uint32_t sub = (uint32_t)(j * 32 / C::kInner) * a.part_bytes;
      uint32_t kf[4];
      ldsm_x4(at + sub + k_off + (((j * 32) & (C::kInner - 1)) ^ k_swz), kf);
      uint32_t af[4];
      if constexpr (RM == 8) {
        af[0] = qf[j][0], af[1] = 0u, af[2] = qf[j][1], af[3] = 0u;
      } else {
        af[0] = qf[j][0], af[1] = qf[j][1], af[2] = qf[j][2], af[3] = qf[j][3];
      }
      Mma<T>::run(j & 1 ? s2[0] : s[0], af, kf[0], kf[1]);
      Mma<T>::run(j & 1 ? s2[1] : s[1], af, kf[2], kf[3]);
    }
    const bool edge = lo > 0 || hi < kTile;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2 * kH; ++e) {
        s[n][e] = (s[n][e] + s2[n][e]) * a.scale_log2;
        const int slot = 8 * n + 2 * i + (e & 1);
        if (edge && (slot < lo || slot >= hi)) s[n][e] = -INFINITY;
      }
    // ---- online softmax, one state a row (the four lanes of a row agree on m; l is this lane's share)
    float alpha[kH];
    bool moved = false;
#pragma unroll
    for (int h = 0; h < kH; ++h) {
      float mt = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
      const float mn = fmaxf(m[h], mt);
      const float use = mn == -INFINITY ? 0.f : mn;
      moved |= mn != m[h];
      alpha[h] = exp2f(m[h] - use);
      m[h] = mn;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[n][2 * h + e] = exp2f(s[n][2 * h + e] - use) * kLift;
          sum += s[n][2 * h + e];
        }
      l[h] = l[h] * alpha[h] + sum;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        o[n][0] *= alpha[0], o[n][1] *= alpha[0];
        o[n][2] *= alpha[kH - 1], o[n][3] *= alpha[kH - 1];
      }
    }
    // ---- o += P V, P in two 16-bit parts
    uint32_t ph[4], pl[4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      split_pair<T>(s[n][0], s[n][1], ph[2 * n], pl[2 * n]);
      if constexpr (RM == 16) {
        split_pair<T>(s[n][2], s[n][3], ph[2 * n + 1], pl[2 * n + 1]);
      } else {
        ph[2 * n + 1] = pl[2 * n];  // rows 8..15 carry the low parts
      }
    }
    // slots 2 i, 2 i + 1 (b0) and 2 i + 8, 2 i + 9 (b1) of V: 0 where out of range
    uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
    if (edge) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int slot = 8 * n + 2 * i;
        keep[n] = (slot >= lo && slot < hi ? 0x0000ffffu : 0u) | (slot + 1 >= lo && slot + 1 < hi ? 0xffff0000u : 0u);
      }
    }
#pragma unroll
    for (int c = 0; c < D / 8; c += 2) {
      const uint32_t sub = (uint32_t)(c * 16 / C::kInner) * a.part_bytes;
      uint32_t vf[4];
      ldsm_x4_t(at + sub + v_off + (((c * 16) & (C::kInner - 1)) ^ v_swz), vf);
#pragma unroll
      for (int e = 0; e < 4; ++e) vf[e] &= keep[e & 1];
      Mma<T>::run(o[c], ph, vf[0], vf[1]);
      Mma<T>::run(o[c + 1], ph, vf[2], vf[3]);
      if constexpr (RM == 16) {
        Mma<T>::run(o[c], pl, vf[0], vf[1]);
        Mma<T>::run(o[c + 1], pl, vf[2], vf[3]);
      }
    }
  }

  // Rows 8 h .. 8 h + 7 into this warp's part of the reduction buffer.
  __device__ __forceinline__ void put(int h, float* red) {
    const int lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3;
    float sum = l[RM == 8 ? 0 : h];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    float* row = red + g * C::kRedRow + 2 * i;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      float2 v;
      if constexpr (RM == 8) {
        v = make_float2(o[n][0] + o[n][2], o[n][1] + o[n][3]);
      } else {
        v = h == 0 ? make_float2(o[n][0], o[n][1]) : make_float2(o[n][2], o[n][3]);
      }
      *reinterpret_cast<float2*>(row + 8 * n) = make_float2(v.x * (1.f / kLift), v.y * (1.f / kLift));
    }
    if (i == 0) *reinterpret_cast<float2*>(red + g * C::kRedRow + D) = make_float2(m[RM == 8 ? 0 : h], sum * (1.f / kLift));
  }
};

// ------------------------------------------------------------------ a warp's state, fp32 caches

// Scores: lane = (slot, half of the 16-byte columns); P V: lane = (16-byte column, every kGroups-th slot).
template <int D, int RM>
struct WarpState<float, D, RM> {
  using C = PagedCfg<float, D>;
  static constexpr int kCols = D / 4, kGroups = 32 / kCols;
  float o[RM][4];
  float m[RM], l[RM];
  const float* qs;

  __device__ __forceinline__ void init(const PagedArgs&, const uint8_t* q_smem) { qs = reinterpret_cast<const float*>(q_smem); }

  // Every thread of the CTA copies a share of the block's query rows (zeros past the group).
  __device__ __forceinline__ void begin(const PagedArgs& a, const Segment& s, uint8_t* q_smem) {
    const int kvh = s.pair / a.row_blocks, h0 = (s.pair - kvh * a.row_blocks) * kRowsMax;
    const int rows = min(kRowsMax, a.group - h0);
    const float* q = static_cast<const float*>(a.q) + s.b * a.q_sb + (int64_t)(kvh * a.group + h0) * a.q_sh;
    float* dst = reinterpret_cast<float*>(q_smem);
    for (int x = threadIdx.x; x < RM * D; x += C::kConsumers) dst[x] = x / D < rows ? q[(x / D) * a.q_sh + x % D] : 0.f;
    consumers_sync<C::kConsumers>();
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[r][e] = 0.f;
    }
  }

  __device__ __forceinline__ static uint32_t at_col(const PagedArgs& a, int row, int col) {  // byte offset of a 16-byte column
    const int byte = col * 16, r = row & 7;
    return byte / C::kInner * a.part_bytes + (row >> 3) * a.rows8_bytes + r * C::kInner +
           (byte % C::kInner ^ ((((r * C::kInner) >> 7) & C::kSwzMask) << 4));
  }

  __device__ __forceinline__ static float4 lds4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
  }

  __device__ __forceinline__ void tile(const PagedArgs& a, uint32_t at, int lo, int hi) {
    const int lane = threadIdx.x & 31, slot = lane & 15, half = lane >> 4;
    float s[RM] = {};
    for (int c = half; c < kCols; c += 2) {
      const float4 k = lds4(at + at_col(a, slot, c));
#pragma unroll
      for (int r = 0; r < RM; ++r) {
        const float4 q = *reinterpret_cast<const float4*>(qs + r * D + 4 * c);
        s[r] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[r]))));
      }
    }
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      s[r] += __shfl_xor_sync(0xffffffffu, s[r], 16);
      s[r] = slot < lo || slot >= hi ? -INFINITY : s[r] * a.scale_log2;
      float mt = s[r];
#pragma unroll
      for (int off = 8; off >= 1; off >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, off));
      const float mn = fmaxf(m[r], mt), use = mn == -INFINITY ? 0.f : mn;
      const float alpha = exp2f(m[r] - use);
      s[r] = exp2f(s[r] - use);
      l[r] = l[r] * alpha + (half == 0 ? s[r] : 0.f);
      m[r] = mn;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[r][e] *= alpha;
    }
    const int col = lane % kCols, kg = lane / kCols;
    for (int t0 = 0; t0 < kTile; t0 += kGroups) {
      const int t = t0 + kg;
      float4 v = lds4(at + C::kTileBytes + at_col(a, t, col));
      if (t < lo || t >= hi) v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int r = 0; r < RM; ++r) {
        const float p = __shfl_sync(0xffffffffu, s[r], t);
        o[r][0] = fmaf(p, v.x, o[r][0]), o[r][1] = fmaf(p, v.y, o[r][1]);
        o[r][2] = fmaf(p, v.z, o[r][2]), o[r][3] = fmaf(p, v.w, o[r][3]);
      }
    }
  }

  __device__ __forceinline__ void put(int h, float* red) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      if (r / 8 != h) continue;
      float sum = l[r];
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int off = kCols; off < 32; off <<= 1) o[r][e] += __shfl_xor_sync(0xffffffffu, o[r][e], off);
      if (lane < kCols) *reinterpret_cast<float4*>(red + (r & 7) * C::kRedRow + 4 * lane) =
          make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
      if (lane == 0) *reinterpret_cast<float2*>(red + (r & 7) * C::kRedRow + D) = make_float2(m[r], sum);
    }
  }
};

// ------------------------------------------------------------------ the kernel

template <typename T>
__device__ __forceinline__ void store4(T* dst, float4 v) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(dst) = v;
  } else {
    union {
      T t[4];
      uint2 u;
    } r;
    r.t[0] = Elem<T>::from_float(v.x), r.t[1] = Elem<T>::from_float(v.y);
    r.t[2] = Elem<T>::from_float(v.z), r.t[3] = Elem<T>::from_float(v.w);
    *reinterpret_cast<uint2*>(dst) = r.u;
  }
}

// A pair's result: o4 = sum of p V over its slots at statistics (M, L), 4 columns of one head.
template <typename T>
__device__ __forceinline__ void write_result(const PagedArgs& a, int b, int head, int d, float4 o4, float M, float L) {
  const float inv = L == 0.f ? 0.f : 1.f / L;
  store4<T>(static_cast<T*>(a.out) + b * a.o_sb + head * a.o_sh + d,
            make_float4(o4.x * inv, o4.y * inv, o4.z * inv, o4.w * inv));
  if (a.lse != nullptr && d == 0) a.lse[(int64_t)b * a.hq + head] = L == 0.f ? -INFINITY : M + log2f(L);
}

template <typename T, int D, int RM>
__global__ void __launch_bounds__(PagedCfg<T, D>::kThreads, 1) paged_decode_kernel(const __grid_constant__ PagedArgs a) {
  using C = PagedCfg<T, D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  int* vars = reinterpret_cast<int*>(smem + C::kOffVars);
  int& s_abort = vars[0];
  int& s_last = vars[1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const uint32_t all_bars = smem_u32(smem + C::kOffBars);
  float* red = reinterpret_cast<float*>(smem + C::kOffRed);
  if (tid == 0) s_abort = 0;
  if (tid < 2 * C::kWarps * C::kStages) mbar_init(all_bars + 8 * tid, tid < C::kWarps * C::kStages ? 2 : 1);  // K and V; the reader
  fence_mbar_init();
  grid_launch_dependents();
  __syncthreads();
  grid_dependency_wait();

  // ---- the launch's units before each lane's requests (a run of requests a lane; every warp for itself)
  const int run = (a.batch + 31) / 32, per = a.hkv * a.row_blocks, pairs = a.batch * per;
  const int b0 = min(a.batch, lane * run), b1 = min(a.batch, b0 + run);
  int tiles = 0, full_pairs = 0;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    int start, len, nt;
    request_bounds(a, b, start, len, nt);
    tiles += nt * per;
    full_pairs += nt > 0 ? per : 0;
  }
  tiles = __reduce_add_sync(0xffffffffu, tiles);
  full_pairs = __reduce_add_sync(0xffffffffu, full_pairs);
  // A small launch of few pairs: whole CTAs a pair, as short as they go (latency); else equal ranges (bandwidth).
  const bool small = a.few && tiles <= (int)gridDim.x * kSmallTiles;
  const int ctas = (int)gridDim.x - (small ? pairs : 0);  // small: at most tiles / chunk + pairs are needed
  const int units = tiles + (small ? 0 : full_pairs * kPairCost);
  int chunk = max((units + ctas - 1) / ctas, kMinChunk);  // units of a CTA; small: its tiles
  if (small) chunk = (chunk + C::kWarps - 1) / C::kWarps * C::kWarps;
  // what a request counts: units, or (small) CTAs
  const auto share = [&](int nt) { return small ? (nt + chunk - 1) / chunk * per : request_units(a, nt); };
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    int start, len, nt;
    request_bounds(a, b, start, len, nt);
    mine += share(nt);
  }
  int before = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, off);
    if (lane >= off) before += v;
  }
  const int total = __shfl_sync(0xffffffffu, before, 31);
  before -= mine;
  const int64_t r64 = small ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * chunk;
  const bool busy = r64 < total;

  Segment seg;
  int split_first = 0, split_last = 0;  // small: the CTAs of this CTA's pair
  if (busy) {
    const int r0 = (int)r64;
    int b = 0, at = before;
    const bool here = r0 >= before && r0 < before + mine;
    if (here)
      for (b = b0;; ++b) {
        int start, len, nt;
        request_bounds(a, b, start, len, nt);
        if (r0 < at + share(nt)) break;
        at += share(nt);
      }
    const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    seg.b = __shfl_sync(0xffffffffu, b, src);
    seg.base = __shfl_sync(0xffffffffu, at, src);
    if (small) {
      request_bounds(a, seg.b, seg.start, seg.len, seg.nt);
      seg.first_tile = seg.start / kTile;
      const int splits = (seg.nt + chunk - 1) / chunk, off = r0 - seg.base;
      seg.pair = off / splits;
      seg.t0 = (off - seg.pair * splits) * chunk;
      seg.t1 = min(seg.nt, seg.t0 + chunk);
      seg.left = 0;
      split_first = seg.base + seg.pair * splits;
      split_last = split_first + splits - 1;
    } else {
      segment_at(a, seg, r0, min(chunk, total - r0));
    }
    if (warp >= C::kWarps) {
      const bool v = warp > C::kWarps;
      copy_range<T, D>(a, v ? a.tm_v : a.tm_k, seg, smem_u32(smem) + (v ? C::kTileBytes : 0), all_bars, &s_abort);
      return;
    }
  } else if (warp >= C::kWarps) {
    return;
  }

  if (full_pairs < pairs)  // requests with nothing to attend to: zeros
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
      int start, len, nt;
      request_bounds(a, b, start, len, nt);
      if (nt == 0)
        for (int x = tid; x < a.hq * (D / 4); x += C::kConsumers)
          write_result<T>(a, b, x / (D / 4), x % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f);
    }
  if (!busy) return;

  const uint32_t ring = smem_u32(smem) + warp * C::kStages * C::kStageBytes;
  const uint32_t full = all_bars + warp * C::kStages * 8, empty = full + C::kWarps * C::kStages * 8;
  WarpState<T, D, RM> st;
  st.init(a, smem + C::kOffQ);
  int stage = 0, turn = 0;  // turn: the warp that takes the segment's first tile
  uint32_t phase = 0;
  bool bad = false;
  for (bool first = true;;) {
    if (seg.t0 == seg.t1) {
      if (!segment_next(a, seg)) break;
      continue;
    }
    st.begin(a, seg, smem + C::kOffQ);
#pragma unroll 1
    for (int t = seg.t0 + (warp - turn + C::kWarps) % C::kWarps; t < seg.t1; t += C::kWarps) {
      if (bad) continue;
      if (!mbar_wait(full + 8 * stage, phase, &s_abort, a.err)) {
        bad = true;  // this warp computes no more, but keeps to the barriers below
        continue;
      }
      const int slot = (seg.first_tile + t) * kTile;
      st.tile(a, ring + stage * C::kStageBytes, seg.start - slot, seg.len - slot);
      __syncwarp();  // every lane has read the stage
      if (lane == 0) mbar_arrive(empty + 8 * stage);
      if (++stage == C::kStages) stage = 0, phase ^= 1;
    }
    turn = (turn + seg.t1 - seg.t0) % C::kWarps;

    // ---- the warps' states into one, 8 rows a round
    const int kvh = seg.pair / a.row_blocks, h0 = (seg.pair - kvh * a.row_blocks) * kRowsMax;
    const int rows = min(kRowsMax, a.group - h0), head0 = kvh * a.group + h0;
    const bool whole = seg.t0 == 0 && seg.t1 == seg.nt;
    // a pair that starts inside this range is its last: slot 1, unless it is the first, too
    const int64_t ws_row = ((int64_t)blockIdx.x * 2 + (first ? 0 : 1)) * kRowsMax;
#pragma unroll
    for (int h = 0; h < RM / 8; ++h) {
      if (h * 8 >= rows) break;
      st.put(h, red + warp * 8 * C::kRedRow);
      consumers_sync<C::kConsumers>();
      for (int x = tid; x < min(8, rows - 8 * h) * (D / 4); x += C::kConsumers) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < C::kWarps; ++w) M = fmaxf(M, red[(w * 8 + r) * C::kRedRow + D]);
        const float use = M == -INFINITY ? 0.f : M;
        float4 o4 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < C::kWarps; ++w) {
          const float* row = red + (w * 8 + r) * C::kRedRow;
          const float2 ml = *reinterpret_cast<const float2*>(row + D);
          const float f = exp2f(ml.x - use);
          const float4 v = *reinterpret_cast<const float4*>(row + d);
          L = fmaf(f, ml.y, L);
          o4.x = fmaf(f, v.x, o4.x), o4.y = fmaf(f, v.y, o4.y);
          o4.z = fmaf(f, v.z, o4.z), o4.w = fmaf(f, v.w, o4.w);
        }
        if (whole) {
          write_result<T>(a, seg.b, head0 + 8 * h + r, d, o4, M, L);
        } else {
          *reinterpret_cast<float4*>(a.ws_o + (ws_row + 8 * h + r) * D + d) = o4;
          if (d == 0) *reinterpret_cast<float2*>(a.ws_ml + (ws_row + 8 * h + r) * 2) = make_float2(M, L);
        }
      }
      consumers_sync<C::kConsumers>();
    }

    // ---- a pair cut by ranges: the last CTA to arrive joins the partials in CTA order
    if (!whole) {
      const int pair0 = seg.pair_base();
      // the CTAs with tiles of it
      const int c0 = small ? split_first : (pair0 + kPairCost) / chunk;
      const int c1 = small ? split_last : (pair0 + seg.units() - 1) / chunk;
      if (tid == 0) {
        unsigned int prev;
        // after the barrier, so cumulative over the CTA's stores of its partial
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(prev) : "l"(a.ws_count + c0) : "memory");
        s_last = prev == (unsigned int)(c1 - c0);
        if (s_last) a.ws_count[c0] = 0u;  // as the next call expects it
      }
      consumers_sync<C::kConsumers>();
      if (s_last) {
        const int first_slot = small || c0 * chunk >= pair0 ? 0 : 1;  // of CTA c0; the others hold it as their first
        for (int x = tid; x < rows * (D / 4); x += C::kConsumers) {
          const int r = x / (D / 4), d = x % (D / 4) * 4;
          float M = -INFINITY, L = 0.f;
          float4 o4 = make_float4(0.f, 0.f, 0.f, 0.f);
          constexpr int kMany = 8;  // partials in flight
          for (int c = c0; c <= c1; c += kMany) {
            float2 s[kMany];
            float4 v[kMany];
            float Mn = M;
#pragma unroll
            for (int k = 0; k < kMany; ++k) {
              s[k] = make_float2(-INFINITY, 0.f);
              v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (c + k <= c1) {
                const int64_t row = ((int64_t)(c + k) * 2 + (c + k == c0 ? first_slot : 0)) * kRowsMax + r;
                s[k] = __ldcg(reinterpret_cast<const float2*>(a.ws_ml + row * 2));
                v[k] = __ldcg(reinterpret_cast<const float4*>(a.ws_o + row * D + d));
              }
            }
#pragma unroll
            for (int k = 0; k < kMany; ++k) Mn = fmaxf(Mn, s[k].x);
            const float use = Mn == -INFINITY ? 0.f : Mn, old = exp2f(M - use);
            L *= old, o4.x *= old, o4.y *= old, o4.z *= old, o4.w *= old;
#pragma unroll
            for (int k = 0; k < kMany; ++k) {
              const float f = exp2f(s[k].x - use);
              L = fmaf(f, s[k].y, L);
              o4.x = fmaf(f, v[k].x, o4.x), o4.y = fmaf(f, v[k].y, o4.y);
              o4.z = fmaf(f, v[k].z, o4.z), o4.w = fmaf(f, v[k].w, o4.w);
            }
            M = Mn;
          }
          write_result<T>(a, seg.b, head0 + r, d, o4, M, L);
        }
      }
    }
    first = false;
    if (!segment_next(a, seg)) break;
  }
}

// ------------------------------------------------------------------ host side

bool pages_map(CUtensorMap* m, const void* ptr, const aicas_paged_decode_params* p, int64_t sp, int64_t sh, int64_t st,
               int box_rows, char* err, size_t errlen) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (enc == nullptr) {
    snprintf(err, errlen, "cuTensorMapEncodeTiled is unavailable from the driver");
    return false;
  }
  const int eb = p->dtype == AICAS_DTYPE_F32 ? 4 : 2;
  // a dimension of one entry may carry any stride: give it a valid one
  if (p->num_kv_heads == 1) sh = st * p->page_size;
  if (p->num_pages == 1) sp = st * p->page_size + sh * p->num_kv_heads;
  const int row_bytes = p->head_dim * eb, inner = row_bytes < 128 ? row_bytes : 128;
  const cuuint64_t dims[5] = {(cuuint64_t)(inner / eb), (cuuint64_t)p->page_size, (cuuint64_t)(row_bytes / inner),
                              (cuuint64_t)p->num_kv_heads, (cuuint64_t)p->num_pages};
  const cuuint64_t strides[4] = {(cuuint64_t)st * eb, (cuuint64_t)inner, (cuuint64_t)sh * eb, (cuuint64_t)sp * eb};
  const cuuint32_t box[5] = {(cuuint32_t)(inner / eb), (cuuint32_t)box_rows, (cuuint32_t)(row_bytes / inner), 1u, 1u};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType type = p->dtype == AICAS_DTYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : p->dtype == AICAS_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle swz = inner == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                 : inner == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                               : CU_TENSOR_MAP_SWIZZLE_32B;
  const CUresult r = enc(m, type, 5, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    snprintf(err, errlen, "cuTensorMapEncodeTiled failed (%d) for pages of strides %lld, %lld, %lld", (int)r,
             (long long)sp, (long long)sh, (long long)st);
    return false;
  }
  return true;
}

// CTAs of a launch: as many as the SMs hold, or fewer where even full caches have fewer runs of kMinChunk tiles.
int paged_grid(const aicas_paged_decode_params* p, int sms) {
  const int64_t cap_tiles = ((int64_t)p->max_pages * p->page_size + kTile - 1) / kTile;
  const int blocks = (p->num_q_heads / p->num_kv_heads + kRowsMax - 1) / kRowsMax;
  const int64_t pairs = (int64_t)p->batch * p->num_kv_heads * blocks;
  const int64_t runs = (cap_tiles * pairs + kMinChunk - 1) / kMinChunk + pairs;
  return (int)(runs < sms ? runs : sms);
}

template <typename T, int D, int RM>
cudaError_t launch_paged(const PagedArgs& a, int grid, cudaStream_t st) {
  using C = PagedCfg<T, D>;
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    e = cudaFuncSetAttribute(paged_decode_kernel<T, D, RM>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  return launch_pdl(paged_decode_kernel<T, D, RM>, dim3(grid), dim3(C::kThreads), C::kSmem, st, a);
}

template <typename T>
cudaError_t dispatch_paged(int head_dim, const PagedArgs& a, int grid, cudaStream_t st) {
  const bool small = a.group <= 8;
  switch (head_dim) {
    case 16: return small ? launch_paged<T, 16, 8>(a, grid, st) : launch_paged<T, 16, 16>(a, grid, st);
    case 32: return small ? launch_paged<T, 32, 8>(a, grid, st) : launch_paged<T, 32, 16>(a, grid, st);
    case 64: return small ? launch_paged<T, 64, 8>(a, grid, st) : launch_paged<T, 64, 16>(a, grid, st);
    case 128: return small ? launch_paged<T, 128, 8>(a, grid, st) : launch_paged<T, 128, 16>(a, grid, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

// The same for every call (3.5 MB on 148 SMs), so that a stream's buffer never has to grow for another shape.
size_t paged_decode_workspace(int sms) {
  return kWsCounters + (size_t)sms * 2 * kRowsMax * (128 + 2) * sizeof(float);
}

int run_paged_decode(const aicas_paged_decode_params* p, int sms, void* workspace, cudaStream_t stream,
                     unsigned int* dev_err, char* err, size_t errlen) {
  PagedArgs a;
  memset(&a, 0, sizeof(a));
  const int box_rows = p->page_size % kTile == 0 ? kTile : 8;
  if (!pages_map(&a.tm_k, p->k_pages, p, p->kp_stride_p, p->kp_stride_h, p->kp_stride_t, box_rows, err, errlen) ||
      !pages_map(&a.tm_v, p->v_pages, p, p->vp_stride_p, p->vp_stride_h, p->vp_stride_t, box_rows, err, errlen))
    return AICAS_ERR_UNSUPPORTED;
  a.q = p->q, a.out = p->out, a.lse = p->lse;
  a.table = p->page_table, a.lens = p->kv_lens, a.starts = p->kv_starts;
  a.q_sb = p->q_stride_b, a.q_sh = p->q_stride_h, a.o_sb = p->o_stride_b, a.o_sh = p->o_stride_h;
  a.table_stride = p->table_stride;
  a.batch = p->batch, a.hq = p->num_q_heads, a.hkv = p->num_kv_heads;
  a.group = p->num_q_heads / p->num_kv_heads;
  a.row_blocks = (a.group + kRowsMax - 1) / kRowsMax;
  a.page_size = p->page_size;
  a.cap = p->max_pages * p->page_size;
  a.boxes = kTile / box_rows;
  const int row_bytes = p->head_dim * (p->dtype == AICAS_DTYPE_F32 ? 4 : 2), inner = row_bytes < 128 ? row_bytes : 128;
  a.part_bytes = box_rows * inner;
  a.rows8_bytes = a.boxes == 2 ? 8 * row_bytes : 8 * inner;
  a.scale_log2 = p->sm_scale * 1.4426950408889634f;
  const int grid = paged_grid(p, sms);
  a.few = 2 * (int64_t)a.batch * a.hkv * a.row_blocks <= grid;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.ws_count = reinterpret_cast<unsigned int*>(ws);
  a.ws_o = reinterpret_cast<float*>(ws + kWsCounters);
  a.ws_ml = a.ws_o + (size_t)grid * 2 * kRowsMax * p->head_dim;
  a.err = dev_err;
  cudaError_t e = cudaErrorInvalidValue;
  switch (p->dtype) {
    case AICAS_DTYPE_F32: e = dispatch_paged<float>(p->head_dim, a, grid, stream); break;
    case AICAS_DTYPE_F16: e = dispatch_paged<__half>(p->head_dim, a, grid, stream); break;
    case AICAS_DTYPE_BF16: e = dispatch_paged<__nv_bfloat16>(p->head_dim, a, grid, stream); break;
  }
  if (e != cudaSuccess) {
    snprintf(err, errlen, "paged decode launch: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
    return AICAS_ERR_CUDA;
  }
  return AICAS_OK;
}

}  // namespace aicas
