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
  nt = len > start ? (len + TILE - 1) / TILE - start / TILE : 0;
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

  // From unit `unit` of the launch, which lies in request b.
  template <typename A>
  __device__ __forceinline__ void at(const A& a, int unit, int count) {
    request_bounds<TILE>(a, b, start, len, nt);
    first_tile = start / TILE;
    const int off = unit - base;
    pair = off / units();
    take(off - pair * units(), count);
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
      first_tile = start / TILE;
    }
    take(0, left);
    return true;
  }
};

// Warps of a team for so many pairs: the least that leaves a pair about RANGES ranges.
template <int WARPS, int RANGES>
__host__ __device__ __forceinline__ int team_warps(int pairs, int ctas) {
  int team = 1;
  while (team < WARPS && (int64_t)pairs * RANGES * team < (int64_t)ctas * WARPS) team *= 2;
  return team;
}

// A team's place in the launch.  Small launches of few pairs (a.few, and at most MOST tiles
// a CTA) give each pair whole CTAs, as short as WARPS tiles allow: latency; the others
// equal ranges: bandwidth.
template <int TILE>
struct Split {
  bool small, busy, empty_rows;  // empty_rows: some request has no slot
  int team;                      // warps of a team, a power of two
  int id;                        // this team's number
  int chunk;                     // units of a range; small: its tiles
  int first_id, last_id;         // small: the teams of this team's pair
  Segment<TILE> seg;             // this team's first, if it is busy

  // Every warp for itself: a run of requests a lane.  LEAST: fewest tiles a warp; COST: a pair's, for each warp of a team.
  template <int WARPS, int RANGES, int LEAST, int COST, int MOST, typename A>
  __device__ __forceinline__ void find(const A& a) {
    const int lane = threadIdx.x & 31, per = a.hkv * a.row_blocks, pairs = a.batch * per;
    const int run = (a.batch + 31) / 32, b0 = min(a.batch, lane * run), b1 = min(a.batch, b0 + run);
    int tiles = 0, full_pairs = 0;
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
      int start, len, nt;
      request_bounds<TILE>(a, b, start, len, nt);
      tiles += nt * per;
      full_pairs += nt > 0 ? per : 0;
    }
    tiles = __reduce_add_sync(0xffffffffu, tiles);
    full_pairs = __reduce_add_sync(0xffffffffu, full_pairs);
    empty_rows = full_pairs < pairs;
    small = a.few && tiles <= (int)gridDim.x * MOST;
    team = small ? WARPS : team_warps<WARPS, RANGES>(full_pairs, (int)gridDim.x);
    const int teams = (int)gridDim.x * (WARPS / team);
    id = (int)blockIdx.x * (WARPS / team) + (int)(threadIdx.x >> 5) / team;
    const int ranges = teams - (small ? pairs : 0);  // small: at most tiles / chunk + pairs are needed
    const int cost = small ? 0 : COST * team;
    const int units = tiles + full_pairs * cost;
    chunk = max((units + ranges - 1) / ranges, LEAST * team);
    if (small) chunk = (chunk + WARPS - 1) / WARPS * WARPS;
    // what a request counts: units, or (small) teams
    const auto share = [&](int nt) {
      return small ? (nt + chunk - 1) / chunk * per : nt == 0 ? 0 : (nt + cost) * per;
    };
    int mine = 0;
    for (int b = b0; b < b1; ++b) {
      int start, len, nt;
      request_bounds<TILE>(a, b, start, len, nt);
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
    const int64_t r64 = small ? (int64_t)id : (int64_t)id * chunk;
    busy = r64 < total;
    if (!busy) return;
    const int r0 = (int)r64;
    int b = 0, at = before;
    const bool here = r0 >= before && r0 < before + mine;
    if (here)
      for (b = b0;; ++b) {
        int start, len, nt;
        request_bounds<TILE>(a, b, start, len, nt);
        if (r0 < at + share(nt)) break;
        at += share(nt);
      }
    const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    seg.b = __shfl_sync(0xffffffffu, b, src);
    seg.base = __shfl_sync(0xffffffffu, at, src);
    seg.cost = cost;
    if (small) {
      request_bounds<TILE>(a, seg.b, seg.start, seg.len, seg.nt);
      seg.first_tile = seg.start / TILE;
      const int splits = (seg.nt + chunk - 1) / chunk, off = r0 - seg.base;
      seg.pair = off / splits;
      seg.t0 = (off - seg.pair * splits) * chunk;
      seg.t1 = min(seg.nt, seg.t0 + chunk);
      seg.left = 0;
      first_id = seg.base + seg.pair * splits;
      last_id = first_id + splits - 1;
    } else {
      seg.at(a, r0, min(chunk, total - r0));
    }
  }
};

}  // namespace aicas
