// Tiles of 32 slots of 4-bit pages: their way into shared memory, a warp by itself, and what
// the kernels that multiply them share.
#pragma once
#include <stdio.h>
#include <type_traits>

#include "common.cuh"
#include "paged_split.cuh"

namespace aicas {

constexpr int kInt4Tile = 32;  // slots a tile
// A code in an fp16's low bits is the subnormal number code / kCodeUnit, 4 bits further up 16 times that.
constexpr float kCodeUnit = 16777216.f;  // 2^24

// One side's pages: strides of the codes in 16 bytes, of the pairs in bytes of a row's pairs.
struct Side {
  const uint8_t* codes;
  const uint8_t* pairs;
  uint32_t cs_p, cs_h, cs_t, ss_p, ss_h, ss_t;
};

// The pages of a call: what its kernel's arguments derive from.
struct Int4Source {
  Side kv[2];
  const int32_t* table;
  int64_t table_stride;
  int num_pages;
  int octets;              // of 8 rows a page has
  uint32_t octets_mul;     // n / octets = (umulhi(n, octets_mul) + n) >> octets_shift
  int octets_shift;
  // Rows follow one another within a page and head, both sides have the same strides, and
  // places in them, in units of 16 bytes and of a row's pairs, fit 32 bits.
  int dense;

  // Of `sides` sides; false, with a message, for strides that are too large.
  bool set(const aicas_int4_pages* pages, int sides, const int32_t* page_table, int64_t stride, int head_dim, int group_size,
           int heads, int pages_in_pool, int page_size, char* err, size_t errlen) {
    dense = 1;
    for (int i = 0; i < sides; ++i) {
      const aicas_int4_pages& from = pages[i];
      const int64_t pair = 2 * (head_dim / group_size);  // elements
      const int64_t st[] = {from.cs_p / 16, from.cs_h / 16, from.cs_t / 16, from.ss_p / pair, from.ss_h / pair, from.ss_t / pair};
      for (int64_t s : st)
        if (s > (int64_t)UINT32_MAX) {
          snprintf(err, errlen, "page strides of 64 GB or more are not supported");
          return false;
        }
      kv[i] = {static_cast<const uint8_t*>(from.codes), static_cast<const uint8_t*>(from.scales), (uint32_t)st[0], (uint32_t)st[1],
               (uint32_t)st[2], (uint32_t)st[3], (uint32_t)st[4], (uint32_t)st[5]};
      const Side &a = kv[0], &b = kv[i];
      dense &= b.cs_t == (uint32_t)head_dim / 32 && b.ss_t == 1 && a.cs_p == b.cs_p && a.cs_h == b.cs_h && a.ss_p == b.ss_p && a.ss_h == b.ss_h;
      // the last row's place; products of numbers below 2^32
      const double last = (double)pages_in_pool * b.cs_p + (double)heads * b.cs_h + (double)page_size * b.cs_t;
      const double last_pair = (double)pages_in_pool * b.ss_p + (double)heads * b.ss_h + (double)page_size * b.ss_t;
      dense &= last < 4e9 && last_pair < 4e9;
    }
    table = page_table, table_stride = stride, num_pages = pages_in_pool;
    set_division(page_size);
    return true;
  }

  // n / d for n < 2^28: with s = ceil(log2 d), (n + floor(n M / 2^32)) >> s, M = floor(2^32 (2^s - d) / d) + 1
  void set_division(int page_size) {
    octets = page_size / 8;
    octets_shift = 0;
    while ((1ll << octets_shift) < octets) ++octets_shift;
    octets_mul = (uint32_t)((((1ull << octets_shift) - octets) << 32) / octets + 1);
  }
};

#if defined(__CUDACC__)

// A stage in shared memory: the codes of K (and V), then a slot's pairs of K (and V).
template <int D, int GD, int SIDES>
struct Int4Stage {
  static constexpr int kRow = D / 2;          // bytes of a row's codes
  static constexpr int kChunks = kRow / 16;   // its 16-byte chunks
  static constexpr int kPair = 4 * GD;        // bytes of a row's pairs
  static constexpr int kOffV = kInt4Tile * kRow;
  static constexpr int kOffPairs = SIDES * kInt4Tile * kRow;
  static constexpr int kStage = kOffPairs + SIDES * kInt4Tile * kPair;
};

// The 16-byte chunk where chunk c of row r is kept: the same chunk of 8 rows, which a
// fragment load takes, lies in all banks once.
template <int D>
__device__ __forceinline__ int swizzled(int r, int c) {
  return c ^ (D == 128 ? (r >> 1) & 3 : (r >> 2) & 1);
}

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

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool there) {
  if constexpr (BYTES == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(there ? BYTES : 0)
                 : "memory");
  }
}

__device__ __forceinline__ void mma(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half(float x, float y) {
  union {
    __half2 h;
    uint32_t u;
  } r;
  r.h = __floats2half2_rn(x, y);
  return r.u;
}

template <typename T>
__device__ __forceinline__ float2 pair_of(uint32_t u) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
}

// A warp's way through its tiles, ahead of the products.  The pages of 8 of its tiles are
// looked up at once, a lane an octet (8 rows) of slots, so that the page table's way and the
// division are paid once for them.
// A: a kernel's arguments, what paged_split.cuh asks for and `src`.
template <int D, int GD, int SIDES, typename A>
struct Cursor {
  using C = Int4Stage<D, GD, SIDES>;
  using Seg = Segment<kInt4Tile>;
  Seg seg;
  int t;      // its next tile, in seg
  int turn;   // the warp that takes seg's first tile
  int known;  // tiles from t on whose pages are looked up; -1: no tile left
  // Of the lane's octet lane % 4 of the tile lane / 4 of those 8: page number (-1: nothing to
  // copy) and first row in the page; of dense pages the places of its codes (-1) and pairs.
  int page, row;

  __device__ __forceinline__ uint32_t head(const A& a) const { return a.row_blocks == 1 ? seg.pair : seg.pair / a.row_blocks; }

  __device__ __forceinline__ void look(const A& a, int team) {
    const int lane = threadIdx.x & 31;
    const int n = (seg.first_tile + t + (lane >> 2) * team) * (kInt4Tile / 8) + (lane & 3);
    const int i = (int)((__umulhi((uint32_t)n, a.src.octets_mul) + (uint32_t)n) >> a.src.octets_shift);
    row = 8 * (n - i * a.src.octets);
    page = -1;
    if (8 * n < seg.len && 8 * n + 8 > seg.start) page = a.src.table[seg.b * a.src.table_stride + i];
    if (page >= a.src.num_pages || page < 0) {
      page = -1;
    } else if (a.src.dense) {
      const Side& p = a.src.kv[0];
      const uint32_t at = page, h = head(a);
      page = (int)(at * p.cs_p + h * p.cs_h + (uint32_t)row * C::kChunks);
      row = (int)(at * p.ss_p + h * p.ss_h + (uint32_t)row);
    }
    known = 8;
  }

  // To the warp's first tile at or after the segment.
  __device__ __forceinline__ void settle(const A& a, int rank, int team) {
    for (;;) {
      t = seg.t0 + ((rank - turn) & (team - 1));
      if (t < seg.t1) return look(a, team);
      turn = (turn + seg.t1 - seg.t0) & (team - 1);
      if (!seg.next(a)) {
        known = -1;
        return;
      }
    }
  }

  __device__ __forceinline__ void begin(const A& a, const Seg& first, int rank, int team) {
    seg = first, turn = 0;
    settle(a, rank, team);
  }

  // One tile's rows: page and row of the lane's octet, as above.
  template <bool DENSE>
  __device__ __forceinline__ void rows(const A& a, uint32_t stage, int pg, int first_row) {
    const int lane = threadIdx.x & 31, o = lane >> 3, sub = lane & 7;
    const bool there = pg != -1;
    constexpr int kAtOnce = 8 / C::kChunks;  // rows of an octet in one go
    const int r = sub / C::kChunks, c = sub % C::kChunks;
    const uint32_t h = DENSE ? 0u : head(a);
#pragma unroll
    for (int side = 0; side < SIDES; ++side) {
      const Side& p = a.src.kv[side];
      const uint8_t *codes = p.codes, *pair = p.pairs;
      uint64_t step = kAtOnce * C::kRow;
      if constexpr (DENSE) {
        // this lane's 16 bytes of the octet are the sub-th, and 8 further ones each
        codes += 16ull * (uint32_t)(there ? pg + sub : 0);
        pair += (uint64_t)C::kPair * (uint32_t)(there ? first_row + sub : 0);
      } else {
        const uint32_t at = there ? pg : 0;
        codes += 16 * ((uint64_t)at * p.cs_p + (uint64_t)h * p.cs_h + (uint64_t)(uint32_t)(first_row + r) * p.cs_t + c);
        pair += C::kPair * ((uint64_t)at * p.ss_p + (uint64_t)h * p.ss_h + (uint64_t)(uint32_t)(first_row + sub) * p.ss_t);
        step = (uint64_t)p.cs_t * (16 * kAtOnce);
      }
      const uint32_t dst = stage + side * C::kOffV + (8 * o + r) * C::kRow;
#pragma unroll
      for (int k = 0; k < C::kChunks; ++k)
        copy_async<16>(dst + kAtOnce * k * C::kRow + 16 * swizzled<D>(r + kAtOnce * k, c), codes + k * step, there);
      copy_async<C::kPair>(stage + C::kOffPairs + (SIDES * lane + side) * C::kPair, pair, there);
    }
  }

  // Asks for the tile and goes on to the next one.
  __device__ __forceinline__ void copy(const A& a, uint32_t stage, int rank, int team) {
    if (known >= 0) {
      const int from = 4 * (8 - known) + ((threadIdx.x & 31) >> 3);
      const int pg = __shfl_sync(0xffffffffu, page, from), first_row = __shfl_sync(0xffffffffu, row, from);
      if (a.src.dense)
        rows<true>(a, stage, pg, first_row);
      else
        rows<false>(a, stage, pg, first_row);
      t += team;
      if (t >= seg.t1) {
        turn = (turn + seg.t1 - seg.t0) & (team - 1);
        if (seg.next(a))
          settle(a, rank, team);
        else
          known = -1;
      } else if (--known == 0) {
        look(a, team);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
};

#endif  // __CUDACC__

}  // namespace aicas
