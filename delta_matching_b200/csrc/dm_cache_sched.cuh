// Even division of the cache's live blocks over a grid.
//
// A unit is (sequence, kv head, tile of query rows); it has as many blocks of 32 tokens as its sequence holds.  All blocks of all units,
// in order, are one flat range of `total` blocks; CTA c of G takes blocks [c total / G, (c + 1) total / G), whatever the lengths are.  So
// a unit may be cut between CTAs: each cut leaves a partial result in a slot of the CTA (2 c for the CTA's first segment, else 2 c + 1),
// which cache_join_kernel joins.  The division depends on the lengths and the grid alone: the same call gives the same bits.
#pragma once
#include "dm_cache.cuh"

namespace dm {

struct FlatRange {
  int total;
  int chunk;              // sequences per entry of cum
  const int* cum;         // blocks before entry i's sequences, i = 0 ... 128
};

// Executed by all 128 threads; `cum`: 129 ints + 4 of scratch.
__device__ __forceinline__ FlatRange flat_range(const CacheView& c, int units, int* cum) {
  const int tid = threadIdx.x, lane = tid & 31, chunk = (c.B + 127) / 128;
  int mine = 0;
  for (int i = tid * chunk; i < min(c.B, (tid + 1) * chunk); ++i) mine += (cache_length(c, i) + 31) / 32 * units;
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += o;
  }
  if (lane == 31) cum[129 + (tid >> 5)] = incl;
  __syncthreads();
  for (int w = 0; w < (tid >> 5); ++w) incl += cum[129 + w];
  cum[tid + 1] = incl;
  if (tid == 0) cum[0] = 0;
  __syncthreads();
  return FlatRange{cum[128], chunk, cum};
}
__device__ __forceinline__ int range_start(int cta, int grid, int total) {
  return static_cast<int>(static_cast<int64_t>(cta) * total / grid);
}
// The CTA that holds flat block f: the largest c with c total / G <= f.
__device__ __forceinline__ int range_owner(int f, int grid, int total) {
  return static_cast<int>(((static_cast<int64_t>(f) + 1) * grid - 1) / total);
}
// Flat blocks before sequence b.
__device__ __forceinline__ int blocks_before(const CacheView& c, int units, const FlatRange& r, int b) {
  const int i = b / r.chunk;
  int f = r.cum[i];
  for (int k = i * r.chunk; k < b; ++k) f += (cache_length(c, k) + 31) / 32 * units;
  return f;
}

// One CTA's piece of a unit.
struct Segment {
  int b, unit, n, blocks;         // sequence, unit within it, its length and blocks
  int blk0, blk1;                 // blocks of this piece
  int f1;                         // flat end of the piece
};
__device__ __forceinline__ void segment_at(Segment& s, int off, int f, int f_end) {
  s.unit = off / s.blocks;
  s.blk0 = off - s.unit * s.blocks;
  s.blk1 = min(s.blocks, s.blk0 + f_end - f);
  s.f1 = f + s.blk1 - s.blk0;
}
// The piece that begins at flat block f < f_end.
__device__ __forceinline__ Segment first_segment(const CacheView& c, int units, const FlatRange& r, int f, int f_end) {
  int lo = 0, hi = 128;           // cum[lo] <= f < cum[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (r.cum[mid] <= f) lo = mid; else hi = mid;
  }
  Segment s;
  int off = f - r.cum[lo];
  s.b = lo * r.chunk;
  for (;; ++s.b) {
    s.n = cache_length(c, s.b);
    s.blocks = (s.n + 31) / 32;
    if (off < s.blocks * units) break;
    off -= s.blocks * units;
  }
  segment_at(s, off, f, f_end);
  return s;
}
__device__ __forceinline__ bool next_segment(const CacheView& c, int units, Segment& s, int f_end) {
  if (s.f1 >= f_end) return false;
  int off = 0;
  if (s.unit + 1 < units) {
    off = (s.unit + 1) * s.blocks;
  } else {
    do {
      s.n = cache_length(c, ++s.b);
      s.blocks = (s.n + 31) / 32;
    } while (s.blocks == 0);
  }
  segment_at(s, off, s.f1, f_end);
  return true;
}

// One warp's way through its CTA's blocks: every fourth block of each segment.
struct Cursor {
  Segment s;
  int kb, page;                   // page of block kb, looked up when the cursor comes to it
  bool live;
};
__device__ __forceinline__ void cursor_settle(const CacheView& c, int units, Cursor& k, int warp, int f_end) {
  while (k.kb >= k.s.blk1) {
    if (!next_segment(c, units, k.s, f_end)) {
      k.live = false;
      return;
    }
    k.kb = k.s.blk0 + warp;
  }
  k.page = __ldg(c.table + k.s.b * c.t_row + k.kb / (c.page / 32));
}
__device__ __forceinline__ Cursor cursor_start(const CacheView& c, int units, const Segment& s, int warp, int f_end) {
  Cursor k{s, s.blk0 + warp, 0, true};
  cursor_settle(c, units, k, warp, f_end);
  return k;
}
__device__ __forceinline__ void cursor_next(const CacheView& c, int units, Cursor& k, int warp, int f_end) {
  k.kb += 4;
  cursor_settle(c, units, k, warp, f_end);
}

}  // namespace dm
