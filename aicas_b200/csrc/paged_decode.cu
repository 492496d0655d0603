// GQA decode attention (one query token per request) over a paged KV cache:
//   o = softmax(scale * q K^T) V over the slots [start, len) of a request, slot
//   t being row t % page_size of page table[b, t / page_size];
//   lse = log2(sum_j 2^(scale log2(e) q.k_j)).
//
// HBM bound: every cached row is read once for the whole group of query heads
// and used for 4 G flops a pair of elements, far below what the tensor cores
// take, so the design is about keeping copies in flight.
//
//   * Work: the 16-slot tiles of all (request, KV head) pairs, numbered pair by
//     pair, are cut into equal ranges, one per CTA (one CTA an SM).  The cut is
//     made on the device from the lengths, so the host neither knows nor bounds
//     them and ragged batches balance to a tile.  A pair inside one range is
//     finished there; a pair that crosses ranges leaves one fp32 partial a CTA
//     (a CTA has at most two: its first and its last pair), and the last CTA to
//     arrive adds them in CTA order, so results repeat to the bit.
//   * Copies: each warp streams its own tiles (every kWarps-th of the CTA's
//     range) through a private ring of TMA boxes, swizzled so that ldmatrix
//     reads them without bank conflicts; no warp waits for another inside a
//     pair.  Page numbers for the next 32 tiles are fetched by the lanes at
//     once.  A page number outside the pool is an out-of-range box: zeros.
//   * Products: mma.sync m16n8k16 with the group's query heads as rows (a
//     larger group takes several blocks of 16).  At a few percent of the SM's
//     tensor rate the legacy path is not the bound, and it keeps scores and
//     output in registers, where the softmax is.  fp32 caches use the FMA pipes.
//   * Rounding: fp32 scores and statistics.  A probability enters P V as two
//     16-bit parts (hi + lo), so that only the result is rounded; with up to 8
//     heads the lo parts ride in the 8 unused rows of the same products.
//   * Slots out of range: scores replaced by -inf and V's elements by 0 before
//     the products (0 * NaN), in the tiles at the range's ends only.
#include <cstdio>
#include <cstring>

#include "common.cuh"
#include "paged.cuh"
#include "tma_host.cuh"

namespace aicas {
namespace {

constexpr int kTile = 16;       // slots a tile
constexpr int kMinChunk = 16;   // fewest tiles a CTA takes
constexpr int kRowsMax = 16;    // query heads of a block
constexpr size_t kWsCounters = (size_t)1 << 20;  // counter region shared with the contiguous decode

struct PagedArgs {
  CUtensorMap tm_k, tm_v;
  const void* q;
  void* out;
  float* lse;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;
  int64_t q_sb, q_sh, o_sb, o_sh, table_stride;
  int batch, hq, hkv, group, row_blocks;
  int page_size, cap;
  int k_rows_first, v_rows_first;  // 1: map dims (D, rows, heads, pages); 0: (D, heads, rows, pages)
  int boxes;                       // boxes of a tile: 1 (16 rows) or 2 (8 rows: page sizes of 8, 24, ...)
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
  static constexpr int kHalves = kRowBytes / kInner;                // boxes along D
  static constexpr int kSwzMask = kInner / 16 - 1;
  static constexpr int kTileBytes = kTile * kRowBytes;
  static constexpr int kStageBytes = 2 * kTileBytes;  // K tile, V tile
  static constexpr int kWarps = kF32 ? 4 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kRing = 196608 / kWarps / kStageBytes;
  static constexpr int kStages = kRing < 8 ? kRing : 8;
  static constexpr int kRedRow = D + 8;  // the 8 keeps the fragment stores free of bank conflicts
  static constexpr int kOffRed = kWarps * kStages * kStageBytes;
  static constexpr int kOffMl = kOffRed + kWarps * 8 * kRedRow * 4;
  static constexpr int kOffQ = kOffMl + kWarps * 8 * 2 * 4;  // fp32: the block's query rows
  static constexpr int kOffBars = kOffQ + (kF32 ? kRowsMax * D * 4 : 0);
  static constexpr int kOffVars = kOffBars + kWarps * kStages * 8;
  // no static shared memory beside it: the ring starts 1024-byte aligned, as the swizzle wants
  static constexpr int kSmem = kOffVars + 64;
  static_assert(kStages >= 3 && kSmem <= 232448, "shared memory");
};

// ------------------------------------------------------------------ fragments

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t r[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t r[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  __device__ __forceinline__ static void run(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Mma<__half> {
  __device__ __forceinline__ static void run(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// hi = (T(x), T(y)) and lo = what that rounding left, as packed pairs.
template <typename T>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
  union {
    T t[2];
    uint32_t u;
  } h, l;
  h.t[0] = Elem<T>::from_float(x);
  h.t[1] = Elem<T>::from_float(y);
  l.t[0] = Elem<T>::from_float(x - Elem<T>::to_float(h.t[0]));
  l.t[1] = Elem<T>::from_float(y - Elem<T>::to_float(h.t[1]));
  hi = h.u;
  lo = l.u;
}

// ------------------------------------------------------------------ the CTA's range

// The tiles [t0, t1) of one (request, KV head, row block) in a CTA's range.
// Tiles count from the one that holds the request's first slot.
struct Segment {
  int b, pair;        // request; KV head * row_blocks + row block
  int t0, t1, nt;     // this CTA's tiles, all tiles of the pair
  int first_tile;     // tile of the first slot
  int start, len;     // slots [start, len)
  int base;           // number of the request's first tile in the launch
  int left;           // tiles of the CTA's range after this segment
};

__device__ __forceinline__ void request_bounds(const PagedArgs& a, int b, int& start, int& len, int& nt) {
  len = a.lens != nullptr ? min(max(a.lens[b], 0), a.cap) : a.cap;
  start = a.starts != nullptr ? min(max(a.starts[b], 0), len) : 0;
  nt = len > start ? (len + kTile - 1) / kTile - start / kTile : 0;
}

// Fills a segment from tile `tile` of the launch, which lies in request s.b.
__device__ __forceinline__ void segment_at(const PagedArgs& a, Segment& s, int tile, int count) {
  request_bounds(a, s.b, s.start, s.len, s.nt);
  s.first_tile = s.start / kTile;
  const int off = tile - s.base;
  s.pair = off / s.nt;
  s.t0 = off - s.pair * s.nt;
  s.t1 = min(s.nt, s.t0 + count);
  s.left = count - (s.t1 - s.t0);
}

__device__ __forceinline__ bool segment_next(const PagedArgs& a, Segment& s) {
  if (s.left == 0) return false;
  if (++s.pair == a.hkv * a.row_blocks) {
    s.base += s.nt * a.hkv * a.row_blocks;
    s.pair = 0;
    do {
      ++s.b;  // tiles are left, so a request with some follows
      request_bounds(a, s.b, s.start, s.len, s.nt);
    } while (s.nt == 0);
    s.first_tile = s.start / kTile;
  }
  s.t0 = 0;
  s.t1 = min(s.nt, s.left);
  s.left -= s.t1;
  return true;
}

// ------------------------------------------------------------------ a warp's copies

template <typename T, int D>
struct Loader {
  using C = PagedCfg<T, D>;
  Segment seg;
  int tile;          // next tile of the segment to copy
  int batch;         // tile whose page this warp's lane 0 holds
  int page0, row0, page1, row1;  // this lane's tile: page and row of its (up to) two boxes
  bool done;

  __device__ __forceinline__ void fetch_pages(const PagedArgs& a) {
    const int lane = threadIdx.x & 31;
    batch = tile;
    const int t = tile + lane * C::kWarps;
    page0 = page1 = -1;
    row0 = row1 = 0;
    if (t < seg.t1) {
      const int slot = (seg.first_tile + t) * kTile;
      const int32_t* row = a.table + seg.b * a.table_stride;
      const int i = slot / a.page_size;
      row0 = slot - i * a.page_size;
      page0 = row[i];
      if (a.boxes == 2 && slot + 8 < seg.len) {
        const bool same = row0 + 8 < a.page_size;
        row1 = same ? row0 + 8 : 0;
        page1 = same ? page0 : row[i + 1];
      }
    }
  }

  // Copies this warp's next tile into a stage; false when none is left.
  __device__ __forceinline__ bool issue(const PagedArgs& a, uint32_t dst, uint32_t bar, uint64_t policy) {
    if (done) return false;
    const int warp = threadIdx.x >> 5;
    while (tile >= seg.t1) {
      if (!segment_next(a, seg)) {
        done = true;
        return false;
      }
      tile = seg.t0 + warp;
      fetch_pages(a);
    }
    if (tile - batch >= 32 * C::kWarps) fetch_pages(a);
    const int src = (tile - batch) / C::kWarps;
    const int p0 = __shfl_sync(0xffffffffu, page0, src), r0 = __shfl_sync(0xffffffffu, row0, src);
    const int p1 = __shfl_sync(0xffffffffu, page1, src), r1 = __shfl_sync(0xffffffffu, row1, src);
    if ((threadIdx.x & 31) == 0) {
      mbar_arrive_expect_tx(bar, C::kStageBytes);
      const int head = seg.pair / a.row_blocks;
#pragma unroll
      for (int h = 0; h < C::kHalves; ++h) {
        const int x = h * (C::kInner / (int)sizeof(T));
        const uint32_t d = dst + h * kTile * C::kInner;
        box(a.tm_k, a.k_rows_first, d, x, r0, head, p0, bar, policy);
        box(a.tm_v, a.v_rows_first, d + C::kTileBytes, x, r0, head, p0, bar, policy);
        if (a.boxes == 2) {
          box(a.tm_k, a.k_rows_first, d + 8 * C::kInner, x, r1, head, p1, bar, policy);
          box(a.tm_v, a.v_rows_first, d + C::kTileBytes + 8 * C::kInner, x, r1, head, p1, bar, policy);
        }
      }
    }
    tile += C::kWarps;
    return true;
  }

  __device__ __forceinline__ static void box(const CUtensorMap& m, int rows_first, uint32_t dst, int x, int row,
                                             int head, int page, uint32_t bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(&m)), "r"(x), "r"(rows_first ? row : head), "r"(rows_first ? head : row),
        "r"(page), "r"(bar), "l"(policy)
        : "memory");
  }
};

// ------------------------------------------------------------------ a warp's state, 16-bit caches

// RM: rows in use, 8 (the group fits 8 heads) or 16.
template <typename T, int D, int RM>
struct WarpState {
  using C = PagedCfg<T, D>;
  static constexpr int kSteps = D / 16;
  static constexpr int kH = RM / 8;  // row halves with heads in them
  uint32_t qf[kSteps][RM == 8 ? 2 : 4];
  float o[D / 8][4];
  float m[kH], l[kH];
  uint32_t k_off, v_off;  // this lane's row of the ldmatrix tiles, with its share of the swizzle
  uint32_t k_swz, v_swz;

  __device__ __forceinline__ void init(const uint8_t*) {
    const int lane = threadIdx.x & 31, mat = lane >> 3, r = lane & 7;
    const int krow = (mat >> 1) * 8 + r, vrow = (mat & 1) * 8 + r;
    k_off = krow * C::kInner;
    v_off = vrow * C::kInner;
    k_swz = ((((krow * C::kInner) >> 7) & C::kSwzMask) << 4) ^ ((mat & 1) << 4);
    v_swz = ((((vrow * C::kInner) >> 7) & C::kSwzMask) << 4) ^ ((mat >> 1) << 4);
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
    float s[2][4] = {};
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const uint32_t sub = (uint32_t)(j * 32 / C::kInner) * kTile * C::kInner;
      uint32_t kf[4];
      ldsm_x4(at + sub + k_off + (((j * 32) & (C::kInner - 1)) ^ k_swz), kf);
      uint32_t af[4];
      if constexpr (RM == 8) {
        af[0] = qf[j][0], af[1] = 0u, af[2] = qf[j][1], af[3] = 0u;
      } else {
        af[0] = qf[j][0], af[1] = qf[j][1], af[2] = qf[j][2], af[3] = qf[j][3];
      }
      Mma<T>::run(s[0], af, kf[0], kf[1]);
      Mma<T>::run(s[1], af, kf[2], kf[3]);
    }
    const bool edge = lo > 0 || hi < kTile;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2 * kH; ++e) {
        s[n][e] *= a.scale_log2;
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
          s[n][2 * h + e] = exp2f(s[n][2 * h + e] - use);
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
      const uint32_t sub = (uint32_t)(c * 16 / C::kInner) * kTile * C::kInner;
      uint32_t vf[4];
      ldsm_x4_t(at + C::kTileBytes + sub + v_off + (((c * 16) & (C::kInner - 1)) ^ v_swz), vf);
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
  __device__ __forceinline__ void put(int h, float* red, float* ml) {
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
      *reinterpret_cast<float2*>(row + 8 * n) = v;
    }
    if (i == 0) ml[2 * g] = m[RM == 8 ? 0 : h], ml[2 * g + 1] = sum;
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

  __device__ __forceinline__ void init(const uint8_t* q_smem) { qs = reinterpret_cast<const float*>(q_smem); }

  // Every thread of the CTA copies a share of the block's query rows (zeros past the group).
  __device__ __forceinline__ void begin(const PagedArgs& a, const Segment& s, uint8_t* q_smem) {
    const int kvh = s.pair / a.row_blocks, h0 = (s.pair - kvh * a.row_blocks) * kRowsMax;
    const int rows = min(kRowsMax, a.group - h0);
    const float* q = static_cast<const float*>(a.q) + s.b * a.q_sb + (int64_t)(kvh * a.group + h0) * a.q_sh;
    float* dst = reinterpret_cast<float*>(q_smem);
    for (int x = threadIdx.x; x < RM * D; x += C::kThreads) dst[x] = x / D < rows ? q[(x / D) * a.q_sh + x % D] : 0.f;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RM; ++r) {
      m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[r][e] = 0.f;
    }
  }

  __device__ __forceinline__ static uint32_t at_col(int row, int col) {  // byte offset of a 16-byte column
    const int byte = col * 16, sub = byte / C::kInner, in = byte % C::kInner;
    return sub * kTile * C::kInner + row * C::kInner + (in ^ ((((row * C::kInner) >> 7) & C::kSwzMask) << 4));
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
      const float4 k = lds4(at + at_col(slot, c));
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
      float4 v = lds4(at + C::kTileBytes + at_col(t, col));
      if (t < lo || t >= hi) v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int r = 0; r < RM; ++r) {
        const float p = __shfl_sync(0xffffffffu, s[r], t);
        o[r][0] = fmaf(p, v.x, o[r][0]), o[r][1] = fmaf(p, v.y, o[r][1]);
        o[r][2] = fmaf(p, v.z, o[r][2]), o[r][3] = fmaf(p, v.w, o[r][3]);
      }
    }
  }

  __device__ __forceinline__ void put(int h, float* red, float* ml) {
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
      if (lane == 0) ml[2 * (r & 7)] = m[r], ml[2 * (r & 7) + 1] = sum;
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
  int* s_find = vars + 2;
  int* s_warp = vars + 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const uint32_t ring = smem_u32(smem) + warp * C::kStages * C::kStageBytes;
  const uint32_t bars = smem_u32(smem + C::kOffBars) + warp * C::kStages * 8;
  float* red = reinterpret_cast<float*>(smem + C::kOffRed);
  float* ml = reinterpret_cast<float*>(smem + C::kOffMl);
  if (tid == 0) s_abort = 0;
  if (lane == 0) {
    for (int s = 0; s < C::kStages; ++s) mbar_init(bars + 8 * s, 1);
    fence_mbar_init();
  }
  grid_launch_dependents();
  grid_dependency_wait();

  // ---- the launch's tiles before each thread's requests (a run of requests a thread)
  const int per = a.hkv * a.row_blocks;
  const int run = (a.batch + C::kThreads - 1) / C::kThreads;
  const int b0 = min(a.batch, tid * run), b1 = min(a.batch, b0 + run);
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    int start, len, nt;
    request_bounds(a, b, start, len, nt);
    mine += nt * per;
    if (nt == 0 && b % (int)gridDim.x == (int)blockIdx.x) {
      // nothing to attend to: zeros (few requests: one thread a request)
      for (int x = 0; x < a.hq * D / 4; ++x)
        write_result<T>(a, b, x / (D / 4), x % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f);
    }
  }
  int before = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, off);
    if (lane >= off) before += v;
  }
  if (lane == 31) s_warp[warp] = before;
  __syncthreads();
  int total = 0;
  before -= mine;
#pragma unroll
  for (int w = 0; w < C::kWarps; ++w) {
    if (w < warp) before += s_warp[w];
    total += s_warp[w];
  }
  const int chunk = max((total + (int)gridDim.x - 1) / (int)gridDim.x, kMinChunk);
  const int64_t r64 = (int64_t)blockIdx.x * chunk;
  if (r64 >= total) return;  // the same for every thread of the CTA
  const int r0 = (int)r64, count = min(chunk, total - r0);
  if (r0 >= before && r0 < before + mine) {
    int at = before;
    for (int b = b0; b < b1; ++b) {
      int start, len, nt;
      request_bounds(a, b, start, len, nt);
      if (r0 < at + nt * per) {
        s_find[0] = b;
        s_find[1] = at;
        break;
      }
      at += nt * per;
    }
  }
  __syncthreads();

  Segment seg;
  seg.b = s_find[0];
  seg.base = s_find[1];
  segment_at(a, seg, r0, count);

  // ---- fill the ring
  const uint64_t policy = l2_policy_evict_first();
  Loader<T, D> ld;
  ld.seg = seg;
  ld.tile = seg.t0 + warp;
  ld.done = false;
  ld.fetch_pages(a);
  int flying = 0;  // copies issued and not yet waited for
#pragma unroll 1
  for (int s = 0; s < C::kStages; ++s) flying += ld.issue(a, ring + s * C::kStageBytes, bars + 8 * s, policy);

  WarpState<T, D, RM> st;
  st.init(smem + C::kOffQ);
  int stage = 0;
  uint32_t phase = 0;
  bool bad = false;
  for (bool first = true;; first = false) {
    st.begin(a, seg, smem + C::kOffQ);
#pragma unroll 1
    for (int t = seg.t0 + warp; t < seg.t1; t += C::kWarps) {
      if (bad) continue;
      if (!mbar_wait(bars + 8 * stage, phase, &s_abort, a.err)) {
        bad = true;  // this warp computes and copies no more, but keeps to the barriers below
        continue;
      }
      const int slot = (seg.first_tile + t) * kTile;
      st.tile(a, ring + stage * C::kStageBytes, seg.start - slot, seg.len - slot);
      __syncwarp();  // every lane has read the stage
      flying += ld.issue(a, ring + stage * C::kStageBytes, bars + 8 * stage, policy) - 1;
      if (++stage == C::kStages) stage = 0, phase ^= 1;
    }

    // ---- the warps' states into one, 8 rows a round
    const int kvh = seg.pair / a.row_blocks, h0 = (seg.pair - kvh * a.row_blocks) * kRowsMax;
    const int rows = min(kRowsMax, a.group - h0), head0 = kvh * a.group + h0;
    const bool whole = seg.t0 == 0 && seg.t1 == seg.nt;
    // a pair that starts inside this range is its last: slot 1, unless it is the first, too
    const int64_t ws_row = ((int64_t)blockIdx.x * 2 + (first ? 0 : 1)) * kRowsMax;
#pragma unroll
    for (int h = 0; h < RM / 8; ++h) {
      if (h * 8 >= rows) break;
      st.put(h, red + warp * 8 * C::kRedRow, ml + warp * 16);
      __syncthreads();
      for (int x = tid; x < min(8, rows - 8 * h) * (D / 4); x += C::kThreads) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < C::kWarps; ++w) M = fmaxf(M, ml[w * 16 + 2 * r]);
        const float use = M == -INFINITY ? 0.f : M;
        float4 o4 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < C::kWarps; ++w) {
          const float f = exp2f(ml[w * 16 + 2 * r] - use);
          const float4 v = *reinterpret_cast<const float4*>(red + (w * 8 + r) * C::kRedRow + d);
          L = fmaf(f, ml[w * 16 + 2 * r + 1], L);
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
      __syncthreads();
    }

    // ---- a pair cut by ranges: the last CTA to arrive joins the partials in CTA order
    if (!whole) {
      const int pair0 = seg.base + seg.pair * seg.nt;                     // the pair's first tile in the launch
      const int c0 = pair0 / chunk, c1 = (pair0 + seg.nt - 1) / chunk;    // the CTAs it crosses
      if (tid == 0) {
        unsigned int prev;
        // after the barrier, so cumulative over the CTA's stores of its partial
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(prev) : "l"(a.ws_count + c0) : "memory");
        s_last = prev == (unsigned int)(c1 - c0);
        if (s_last) a.ws_count[c0] = 0u;  // as the next call expects it
      }
      __syncthreads();
      if (s_last) {
        const int first_slot = pair0 % chunk == 0 ? 0 : 1;  // of CTA c0; the others hold it as their first
        for (int x = tid; x < rows * (D / 4); x += C::kThreads) {
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
    if (!segment_next(a, seg)) break;
  }
  // a warp that gave up leaves once its copies have landed (bounded again)
  if (bad)
    for (; flying > 0; --flying) {
      mbar_wait(bars + 8 * stage, phase, nullptr, a.err);
      if (++stage == C::kStages) stage = 0, phase ^= 1;
    }
}

// ------------------------------------------------------------------ host side

bool pages_map(CUtensorMap* m, const void* ptr, const aicas_paged_decode_params* p, int64_t sp, int64_t sh, int64_t st,
               int box_rows, int* rows_first, char* err, size_t errlen) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (enc == nullptr) {
    snprintf(err, errlen, "cuTensorMapEncodeTiled is unavailable from the driver");
    return false;
  }
  const int eb = p->dtype == AICAS_DTYPE_F32 ? 4 : 2;
  // a dimension of one entry may carry any stride: give it a valid one
  if (p->num_kv_heads == 1) sh = st * p->page_size;
  if (p->num_pages == 1) sp = st * p->page_size + sh * p->num_kv_heads;
  *rows_first = st <= sh;
  const cuuint64_t rows = (cuuint64_t)p->page_size, heads = (cuuint64_t)p->num_kv_heads;
  const cuuint64_t dims[4] = {(cuuint64_t)p->head_dim, *rows_first ? rows : heads, *rows_first ? heads : rows,
                              (cuuint64_t)p->num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)(*rows_first ? st : sh) * eb, (cuuint64_t)(*rows_first ? sh : st) * eb,
                                 (cuuint64_t)sp * eb};
  const int row_bytes = p->head_dim * eb, inner = row_bytes < 128 ? row_bytes : 128;
  const cuuint32_t box[4] = {(cuuint32_t)(inner / eb), *rows_first ? (cuuint32_t)box_rows : 1u,
                             *rows_first ? 1u : (cuuint32_t)box_rows, 1u};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = p->dtype == AICAS_DTYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : p->dtype == AICAS_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle swz = inner == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                 : inner == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                               : CU_TENSOR_MAP_SWIZZLE_32B;
  const CUresult r = enc(m, type, 4, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    snprintf(err, errlen, "cuTensorMapEncodeTiled failed (%d) for pages of strides %lld, %lld, %lld", (int)r,
             (long long)sp, (long long)sh, (long long)st);
    return false;
  }
  return true;
}

// CTAs of a launch: an SM each, or fewer where even full caches have fewer runs of kMinChunk tiles.
int paged_grid(const aicas_paged_decode_params* p, int sms) {
  const int64_t cap_tiles = ((int64_t)p->max_pages * p->page_size + kTile - 1) / kTile;
  const int blocks = (p->num_q_heads / p->num_kv_heads + kRowsMax - 1) / kRowsMax;
  const int64_t runs = (cap_tiles * p->batch * p->num_kv_heads * blocks + kMinChunk - 1) / kMinChunk;
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

size_t paged_decode_workspace(const aicas_paged_decode_params* p, int sms) {
  return kWsCounters + (size_t)paged_grid(p, sms) * 2 * kRowsMax * (p->head_dim + 2) * sizeof(float);
}

int run_paged_decode(const aicas_paged_decode_params* p, int sms, void* workspace, cudaStream_t stream,
                     unsigned int* dev_err, char* err, size_t errlen) {
  PagedArgs a;
  memset(&a, 0, sizeof(a));
  const int box_rows = p->page_size % kTile == 0 ? kTile : 8;
  if (!pages_map(&a.tm_k, p->k_pages, p, p->kp_stride_p, p->kp_stride_h, p->kp_stride_t, box_rows, &a.k_rows_first, err,
                 errlen) ||
      !pages_map(&a.tm_v, p->v_pages, p, p->vp_stride_p, p->vp_stride_h, p->vp_stride_t, box_rows, &a.v_rows_first, err,
                 errlen))
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
  a.scale_log2 = p->sm_scale * 1.4426950408889634f;
  const int grid = paged_grid(p, sms);
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
