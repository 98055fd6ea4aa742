// Even division of the cache's live blocks over the warps of a grid.
//
// A unit is (sequence, kv head, tile of query rows); it costs as many steps as its sequence holds blocks of 32 tokens, and kUnitCost more for
// its queries and its output.  The steps of all units, in order, are one flat range; warp w of G takes steps [w total / G, (w + 1) total / G),
// whatever the lengths are (G: the grid's warps, or as many as there are steps).  So a unit may be cut between warps: a cut leaves a partial
// result in a slot of its warp (2 w for the warp's first piece, else 2 w + 1), which cache_join_kernel joins.  The division depends on the
// lengths and the grid alone: the same call gives the same bits.
#pragma once
#include "dm_cache.cuh"

namespace dm {

// us of a call with 1, 3 and 6: H=32 Hk=8, B=16 with 1000 - 4096 tokens, four new ones 36.0, 33.5 and 34.9; head_dim 256, H=16 Hk=16, B=8 with 4001 - 8192
// 76.8, 76.8 and 76.6.
constexpr int kUnitCost = 3;

struct FlatRange {
  int total;
  int chunk;              // sequences per entry of cum
  const int* cum;         // steps before entry i's sequences, i = 0 ... 128
};

__device__ __forceinline__ int sequence_steps(int n, int units) { return n > 0 ? ((n + 31) / 32 + kUnitCost) * units : 0; }

// Executed by all 128 threads; `cum`: 129 ints + 4 of scratch.
__device__ __forceinline__ FlatRange flat_range(const CacheView& c, int units, int* cum) {
  const int tid = threadIdx.x, lane = tid & 31, chunk = (c.B + 127) / 128;
  int mine = 0;
  for (int i = tid * chunk; i < min(c.B, (tid + 1) * chunk); ++i) mine += sequence_steps(cache_length(c, i), units);
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
// w total / workers, without 64-bit division (workers^2 < 2^32).
__device__ __forceinline__ int range_start(int w, int workers, int total) {
  const unsigned q = static_cast<unsigned>(total) / workers, r = static_cast<unsigned>(total) - q * workers;
  return static_cast<int>(w * q + w * r / workers);
}

// A warp's piece of a unit.
struct Piece {
  int b, unit, n, blocks;         // sequence, unit within it, its length and blocks
  int blk0, blk1;                 // blocks of the piece; none where only steps of the unit's own cost are left to the warp
  int f1;                         // flat end of the piece
};
__device__ __forceinline__ void piece_at(Piece& s, int off, int f, int f_end) {
  const int cost = s.blocks + kUnitCost;
  s.unit = off / cost;
  const int at = off - s.unit * cost;
  s.f1 = min(f_end, f + cost - at);
  s.blk0 = max(0, at - kUnitCost);
  s.blk1 = max(0, at + s.f1 - f - kUnitCost);
}
// The piece that begins at step f < f_end; it may be empty.
__device__ __forceinline__ Piece first_piece(const CacheView& c, int units, const FlatRange& r, int f, int f_end) {
  int lo = 0, hi = 128;           // cum[lo] <= f < cum[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (r.cum[mid] <= f) lo = mid; else hi = mid;
  }
  Piece s;
  int off = f - r.cum[lo];
  s.b = lo * r.chunk;
  for (;; ++s.b) {
    s.n = cache_length(c, s.b);
    const int steps = sequence_steps(s.n, units);
    if (off < steps) break;
    off -= steps;
  }
  s.blocks = (s.n + 31) / 32;
  piece_at(s, off, f, f_end);
  return s;
}
__device__ __forceinline__ bool next_piece(const CacheView& c, int units, Piece& s, int f_end) {
  if (s.f1 >= f_end) return false;
  const int f = s.f1;
  if (s.unit + 1 < units) {       // a unit begins: no division needed
    ++s.unit;
  } else {
    do {
      s.n = cache_length(c, ++s.b);
    } while (s.n == 0);
    s.blocks = (s.n + 31) / 32;
    s.unit = 0;
  }
  s.f1 = min(f_end, f + s.blocks + kUnitCost);
  s.blk0 = 0;
  s.blk1 = max(0, s.f1 - f - kUnitCost);
  return true;
}

// The blocks of a warp's pieces in order, with their pages: what its loads run ahead on.  Pages are looked up for 32 blocks at a time, one a
// lane, so that a block costs no load and no division of its own.
struct Cursor {
  Piece s;
  int kb, window;                 // block; first block of the window
  int page, sub;                  // of block window + lane: its page, and its place in it
  bool live;
};
__device__ __forceinline__ void cursor_window(const CacheView& c, Cursor& k) {
  const int bpp = c.page / 32, blk = k.kb + (threadIdx.x & 31), entry = blk / bpp;
  k.window = k.kb;
  k.sub = blk - entry * bpp;
  k.page = blk < k.s.blk1 ? __ldg(c.table + k.s.b * c.t_row + entry) : 0;
}
__device__ __forceinline__ void cursor_enter(const CacheView& c, int units, Cursor& k, int f_end) {
  while (k.s.blk0 >= k.s.blk1) {
    if (!next_piece(c, units, k.s, f_end)) {
      k.live = false;
      return;
    }
  }
  k.kb = k.s.blk0;
  cursor_window(c, k);
}
__device__ __forceinline__ Cursor cursor_start(const CacheView& c, int units, const Piece& s, int f_end) {
  Cursor k{s, 0, 0, 0, 0, true};
  cursor_enter(c, units, k, f_end);
  return k;
}
__device__ __forceinline__ void cursor_next(const CacheView& c, int units, Cursor& k, int f_end) {
  if (++k.kb < k.s.blk1) {
    if (k.kb - k.window == 32) cursor_window(c, k);
    return;
  }
  k.s.blk0 = k.s.blk1;            // done with this piece
  cursor_enter(c, units, k, f_end);
}
// Page and place of the cursor's block, for the whole warp; a page that is none is reported and replaced by page 0.
__device__ __forceinline__ int2 cursor_at(const CacheView& c, const Cursor& k) {
  const int page = __shfl_sync(0xffffffffu, k.page, k.kb - k.window), sub = __shfl_sync(0xffffffffu, k.sub, k.kb - k.window);
  return make_int2(max(0, checked_page(c, page)), sub);
}

}  // namespace dm
