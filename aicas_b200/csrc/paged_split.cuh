// How a decode attention over a paged cache is cut over the warps of a launch.
//
// The TILE-slot tiles of all pairs (request, KV head, block of query heads), numbered
// pair by pair, are cut into equal ranges, one per team of warps, on the device and from
// the lengths, so the host neither knows nor bounds them and ragged batches balance to a
// tile.  A pair counts `cost` units more, before its tiles, for beginning and ending it, so
// that a team with many short pairs gets fewer tiles.
//
// Teams are of 1 to 16 warps: as small as leaves a pair in few ranges.  Small teams wait
// for no one at a pair's ends, and lose nothing to tiles that do not divide by the warps;
// large ones leave fewer partial results to join.
//
// A: a kernel's arguments, with lens, starts, cap, batch, hkv, row_blocks and few.
#pragma once
#include <stdint.h>

namespace aicas {

// A request's slots [start, len) and how many tiles hold them.
template <int TILE, typename A>
__device__ __forceinline__ void request_bounds(const A& a, int b, int& start, int& len, int& nt) {
  len = a.lens != nullptr ? min(max(a.lens[b], 0), a.cap) : a.cap;
  start = a.starts != nullptr ? min(max(a.starts[b], 0), len) : 0;
  nt = len > start ? (int)((uint32_t)(len + TILE - 1) / TILE - (uint32_t)start / TILE) : 0;
}

// The tiles [t0, t1) of one pair in a team's range; none where the range ends in the pair's
// cost.  Tiles count from the one that holds the request's first slot.
template <int TILE>
struct Segment {
  int b, pair;        // request; KV head * row_blocks + row block
  int t0, t1, nt;     // this team's tiles, all tiles of the pair
  int first_tile;     // tile of the first slot
  int start, len;     // slots [start, len)
  int base;           // number of the request's first unit in the launch
  int left;           // units of the range after this segment
  int cost;

  __device__ __forceinline__ int units() const { return nt + cost; }
  __device__ __forceinline__ int pair_base() const { return base + pair * units(); }

  // The pair's units [from, from + count), as far as it has them.
  __device__ __forceinline__ void take(int from, int count) {
    const int to = min(units(), from + count);
    left = count - (to - from);
    t0 = max(0, from - cost);
    t1 = max(0, to - cost);
  }

  template <typename A>
  __device__ __forceinline__ bool next(const A& a) {
    if (left == 0) return false;
    if (++pair == a.hkv * a.row_blocks) {
      base += units() * a.hkv * a.row_blocks;
      pair = 0;
      do {
        ++b;  // units are left, so a request with some follows
        request_bounds<TILE>(a, b, start, len, nt);
      } while (nt == 0);
      first_tile = (uint32_t)start / TILE;
    }
    take(0, left);
    return true;
  }
};

// Warps of a team, as a power of two, for so many pairs: the least that leaves a pair about RANGES ranges.
template <int LOG_WARPS, int RANGES>
__host__ __device__ __forceinline__ int team_log(int pairs, int ctas) {
  int log = 0;
#pragma unroll
  for (int k = 0; k < LOG_WARPS; ++k) log += (int64_t)pairs * RANGES << k < (int64_t)ctas << LOG_WARPS;
  return log;
}

// A team's place in the launch.  Small launches of few pairs (a.few, and at most MOST tiles
// a CTA) give each pair whole teams, as short as the warps' tiles allow, of 1 << SMALL warps
// where that leaves each team a CTA: latency; the others equal ranges: bandwidth.
template <int TILE>
struct Split {
  bool small, busy, empty_rows;  // empty_rows: some request has no slot
  int log;                       // warps of a team: 1 << log
  int id;                        // this team's number
  int chunk;                     // units of a range; small: its tiles
  int first_id, last_id;         // small: the teams of this team's pair
  Segment<TILE> seg;             // this team's first, if it is busy

  // Every warp for itself, a run of requests a lane.  The chain of a launch of few
  // tiles, so loads and divisions are few.  COST: a pair's, for each warp of a team.
  template <int LOG_WARPS, int SMALL, int RANGES, int COST, int MOST, typename A>
  __device__ __forceinline__ void find(const A& a) {
    const int lane = threadIdx.x & 31, per = a.hkv * a.row_blocks;
    const int run = (a.batch + 31) >> 5, b0 = min(a.batch, lane * run), b1 = min(a.batch, b0 + run);
    int start = 0, len = 0, nt0 = 0;  // of the lane's first request
    if (b0 < b1) request_bounds<TILE>(a, b0, start, len, nt0);
    int tiles = nt0, full = nt0 > 0;
    for (int b = b0 + 1; b < b1; ++b) {
      int st, ln, nt;
      request_bounds<TILE>(a, b, st, ln, nt);
      tiles += nt;
      full += nt > 0;
    }
    tiles = __reduce_add_sync(0xffffffffu, tiles) * per;
    full = __reduce_add_sync(0xffffffffu, full);
    empty_rows = full < a.batch;
    full *= per;
    const int grid = (int)gridDim.x;
    small = a.few && tiles <= grid * MOST;
    log = small ? (tiles <= grid << SMALL ? SMALL : LOG_WARPS) : team_log<LOG_WARPS, RANGES>(full, grid);
    const int teams = grid << (LOG_WARPS - log);
    const int of_cta = (int)(threadIdx.x >> (5 + log));
    id = small ? (int)blockIdx.x + grid * of_cta : (int)(blockIdx.x << (LOG_WARPS - log)) + of_cta;
    const int ranges = teams - (small ? a.batch * per : 0);  // small: at most tiles / chunk + pairs are needed
    const int cost = small ? 0 : COST << log;
    const uint32_t units = (uint32_t)(tiles + full * cost);
    chunk = max((int)((units + ranges - 1) / (uint32_t)ranges), 1 << log);
    if (small) chunk = (chunk + (1 << log) - 1) & -(1 << log);
    const float inv = 1.f / (float)chunk;
    // what a request counts: units, or (small; numbers below 2^16, so the quotient is exact) teams
    const auto share = [&](int nt) {
      return small ? (int)(((float)(nt + chunk - 1) + 0.5f) * inv) * per : nt == 0 ? 0 : (nt + cost) * per;
    };
    int mine = b0 < b1 ? share(nt0) : 0;
    for (int b = b0 + 1; b < b1; ++b) {
      int st, ln, nt;
      request_bounds<TILE>(a, b, st, ln, nt);
      mine += share(nt);
    }
    int before = mine;
    if (a.batch > 1)
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, off);
        if (lane >= off) before += v;
      }
    const int total = __shfl_sync(0xffffffffu, before, 31 < a.batch - 1 ? 31 : a.batch - 1);
    before -= mine;
    const int64_t r64 = small ? (int64_t)id : (int64_t)id * chunk;
    busy = r64 < total;
    if (!busy) return;
    const int r0 = (int)r64;
    int b = b0, at = before, nt = nt0;
    const bool here = r0 >= before && r0 < before + mine;
    if (here)
      while (r0 >= at + share(nt)) {
        at += share(nt);
        request_bounds<TILE>(a, ++b, start, len, nt);
      }
    const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    seg.b = __shfl_sync(0xffffffffu, b, src);
    seg.base = __shfl_sync(0xffffffffu, at, src);
    seg.start = __shfl_sync(0xffffffffu, start, src);
    seg.len = __shfl_sync(0xffffffffu, len, src);
    seg.nt = __shfl_sync(0xffffffffu, nt, src);
    seg.first_tile = (uint32_t)seg.start / TILE;
    seg.cost = cost;
    const uint32_t off = (uint32_t)(r0 - seg.base);
    if (small) {
      const uint32_t splits = (uint32_t)(((float)(seg.nt + chunk - 1) + 0.5f) * inv);
      seg.pair = (int)(off / splits);
      seg.t0 = (int)(off - seg.pair * splits) * chunk;
      seg.t1 = min(seg.nt, seg.t0 + chunk);
      seg.left = 0;
      first_id = seg.base + seg.pair * (int)splits;
      last_id = first_id + (int)splits - 1;
    } else {
      seg.pair = (int)(off / (uint32_t)seg.units());
      seg.take((int)off - seg.pair * seg.units(), min(chunk, total - r0));
    }
  }
};

}  // namespace aicas
