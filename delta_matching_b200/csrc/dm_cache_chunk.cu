// Attention of many new queries over the 8-bit cache (chunks of a prompt): the same result as dm_cache_attn.cu, on tcgen05.
//
//   S = Q K^T and O += P V as f16 tcgen05 chains with fp32 accumulators in TMEM.  The codes are exact in f16, q is brought to f16 with a power
//   of two per row; K's block scales go into the factors of the logits, V's into the exponent of P.  P is f16 with the row's largest product of a
//   probability and a V scale at 2^12 (11 bits, never closer than 2^-36 of it): blocks that a row does not see, or gives no weight, cost it no bits.
//
// A unit is (sequence, kv head, 256 rows); rows are (new token, head of the group).  The key tiles of 128 tokens of all units are one flat
// range, divided evenly over one CTA per SM (as the warps' blocks are in dm_cache_sched.cuh); pieces of cut units are joined by a second kernel.
// Warps 0-3 and 4-7: softmax of the unit's two row tiles (thread = row = TMEM lane).  Warps 8-11: codes -> f16 operand tiles in shared
// memory, shared by both row tiles.  Warp 12: TMA of the code tiles from the pages.  Warp 13: MMA.  Warp 14: TMA of the
// queries, which a small kernel has brought to f16 in the order of the row tiles.  The two row tiles take turns: while one is in its softmax the
// tensor cores work for the other.
//
// TMEM: S0 0-127, S1 128-255 (P of a tile over the first 64 columns of its S), O0 256-383, O1 384-511.
// The references (of the sum, and of the products) move only when a row exceeds them by more than 2^3.9 (P then still fits f16's range), so O is seldom
// rescaled: a move costs its row tile about 3000 cycles, and with a reference that follows within a factor of two some warp moved it in most
// tiles (6800 cycles a tile).
//
// Head_dim 256: a unit is 128 rows, the two softmax groups take half of a tile's keys each and half of O, S has two buffers (0-127, 128-255) and
// O the columns 256-511.
//
// Bound by the chain of a tile at head_dim 128: softmax 2000 - 2500 cycles, P V and the next S 1300 - 1700 until seen, beside which the other row tile
// works; its exponentials alone are 2048 cycles for both row tiles.  512 new tokens, H=32 Hk=8, B=2 with 4096 - 8192 tokens: 128 - 132 us =
// 750 - 770 TFLOP/s (cuBLAS in bf16: 1635).  At head_dim 256 by the conversion of the codes, 4400 cycles a tile, and their loads, for which 32 KB are left:
// H=16 Hk=4 147 us = 670 TFLOP/s.
#include <type_traits>
#include "dm_cache.cuh"
#include "dm_kernels.h"

namespace dm {

namespace {

// Key tiles that a unit's queries and output are worth.  us with 1, 3 and 6 at H=32 Hk=8: 512 new tokens, B=2 with 4096 - 8192 133.1, 129.8 and 133.0; 128
// new ones, B=4 with 512 37.0, 34.3 and 34.2.
constexpr int kChunkCost = 3;
constexpr int kPBase = 12;                  // log2 of P at the reference,
constexpr float kHeadroom = 3.9f;           // and what a row may exceed it by: P stays below 2^16
constexpr float kExact = 4194304.f;         // references up to this size plus a whole number are exact sums

// D = 256: as D = 128, but one row tile, whose two softmax groups take half of the keys each, and O of 256 columns.
template <int kD>
struct ChunkCfg {
  static constexpr int D = kD;
  static constexpr bool kWide = D == 256;
  static constexpr int kThreads = 512;                        // four warpgroups
  static constexpr int kRegsSoftmax = 168, kRegsOther = 88;
  static_assert(256 * kRegsSoftmax + 256 * kRegsOther <= kThreads * 128, "a split above the launch's own registers would wait for ever");
  static constexpr int kRows = kWide ? 128 : 256;
  static constexpr int kPanels = D / 64;                      // of 64 columns, of an f16 operand tile
  static constexpr int kCols = kWide ? 64 : 128;              // keys of a tile that a softmax group looks after
  static constexpr int kTile = 128 * 128;                     // 128 keys x 128 codes; also an f16 panel of 128 rows
  static constexpr int kVBufs = kWide ? 1 : 2;
  static constexpr int kSmemQ = 0;                            // row tiles x panels
  static constexpr int kSmemK = 4 * kTile;                    // between the uses of two tiles lies a softmax, longer than a conversion
  static constexpr int kSmemV = kSmemK + kPanels * kTile;
  static constexpr int kSmemCode = kSmemV + 4 * kTile;        // two pieces: a load takes 2000 cycles, a conversion 1200; with four it was not faster
  // output staging, 4 KB a softmax warp: with 256 columns over the queries, which then wait for it
  static constexpr int kSmemOut = kWide ? kSmemQ : kSmemCode + 2 * kTile;
  static constexpr int kSmemBars = kSmemCode + (kWide ? 2 : 4) * kTile;
  static constexpr int kSmemScales = kSmemBars + 416;         // 8 tiles x (4 K scales, 4 V scales)
  static constexpr int kSmemRows = kSmemScales + 8 * 32;      // what the two groups tell each other of their rows
  static constexpr int kSmem = kSmemRows + (kWide ? 1024 + 256 : 0) + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
};

// ------------------------------------------------------------------------------------------------ schedule
// Rows and key tiles of a sequence's units.
struct ChunkSeq {
  int n, count, units;                      // units per head
};
__device__ __forceinline__ ChunkSeq chunk_seq(const CacheAttnParams& p, int b) {
  ChunkSeq s;
  s.n = cache_length(p.c, b);
  s.count = checked_count(p.c.status, p.counts, b, p.Nq);
  s.units = (s.count * p.rep + (1 << p.unit_shift) - 1) >> p.unit_shift;
  return s;
}
// Keys that row r of the sequence sees.
__device__ __forceinline__ int row_limit(const CacheAttnParams& p, const ChunkSeq& s, int r) {
  const int i = r / p.rep;
  return i >= s.count ? 0 : p.causal ? max(0, s.n - s.count + i + 1) : s.n;
}
__device__ __forceinline__ int unit_tiles(const CacheAttnParams& p, const ChunkSeq& s, int rt) {
  return (row_limit(p, s, min(s.count * p.rep, (rt + 1) << p.unit_shift) - 1) + 127) / 128;
}
__device__ __forceinline__ int unit_steps(const CacheAttnParams& p, const ChunkSeq& s, int rt) {
  const int tiles = unit_tiles(p, s, rt);
  return tiles > 0 ? tiles + kChunkCost : 0;
}
// Steps of one head of a sequence.
__device__ __forceinline__ int head_steps(const CacheAttnParams& p, int b) {
  const ChunkSeq s = chunk_seq(p, b);
  int steps = 0;
  for (int rt = 0; rt < s.units; ++rt) steps += unit_steps(p, s, rt);
  return steps;
}

// Steps before each group of sequences, 128 groups; executed by the first 128 threads (barrier 1).
__device__ __forceinline__ void chunk_range(const CacheAttnParams& p, int* cum, int tid) {
  const int lane = tid & 31, chunk = (p.c.B + 127) / 128;
  int incl = 0;
  for (int i = tid * chunk; i < min(p.c.B, (tid + 1) * chunk); ++i) incl += head_steps(p, i) * p.c.Hk;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += o;
  }
  if (lane == 31) cum[129 + (tid >> 5)] = incl;
  bar_sync(1, 128);
  for (int w = 0; w < (tid >> 5); ++w) incl += cum[129 + w];
  cum[tid + 1] = incl;
  if (tid == 0) cum[0] = 0;
}
__device__ __forceinline__ int share_start(int cta, int grid, int total) { return static_cast<int>(static_cast<int64_t>(cta) * total / grid); }
// A CTA's piece of a unit: key tiles t0 ... t1 - 1.
struct ChunkPiece {
  int b, hk, rt;
  ChunkSeq s;
  int tiles, t0, t1, f1;
  // Row tiles (head_dim 128): two, but for the last unit of a head.
  __device__ __forceinline__ int groups(const CacheAttnParams& p) const { return s.count * p.rep - (rt << 8) <= 128 ? 1 : 2; }
};
__device__ __forceinline__ void chunk_cut(const CacheAttnParams& p, ChunkPiece& x, int at, int f, int f_end) {
  x.tiles = unit_tiles(p, x.s, x.rt);
  x.f1 = min(f_end, f + x.tiles + kChunkCost - at);
  x.t0 = max(0, at - kChunkCost);
  x.t1 = max(0, at + x.f1 - f - kChunkCost);
}
__device__ __forceinline__ ChunkPiece first_chunk(const CacheAttnParams& p, const int* cum, int chunk, int f, int f_end) {
  int lo = 0, hi = 128;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (cum[mid] <= f) lo = mid; else hi = mid;
  }
  ChunkPiece x;
  int off = f - cum[lo];
  x.b = lo * chunk;
  int steps;
  for (;; ++x.b) {
    steps = head_steps(p, x.b);
    if (off < steps * p.c.Hk) break;
    off -= steps * p.c.Hk;
  }
  x.s = chunk_seq(p, x.b);
  x.hk = off / steps;
  off -= x.hk * steps;
  for (x.rt = 0;; ++x.rt) {
    const int u = unit_steps(p, x.s, x.rt);
    if (off < u) break;
    off -= u;
  }
  chunk_cut(p, x, off, f, f_end);
  return x;
}
__device__ __forceinline__ bool next_chunk(const CacheAttnParams& p, ChunkPiece& x, int f_end) {
  if (x.f1 >= f_end) return false;
  do {
    if (++x.rt >= x.s.units) {
      x.rt = 0;
      if (++x.hk == p.c.Hk) {
        x.hk = 0;
        do {
          x.s = chunk_seq(p, ++x.b);
        } while (x.s.units == 0);
      }
    }
  } while (unit_tiles(p, x.s, x.rt) == 0);
  chunk_cut(p, x, 0, x.f1, f_end);
  return true;
}

// What a CTA begins with: made once per call by the queries' kernel (8000 cycles in each CTA of the main kernel otherwise).
struct ChunkStart {
  ChunkPiece x;
  int f0, f_end;
};
__device__ __forceinline__ void chunk_starts(const CacheAttnParams& p, int* cum) {
  const int tid = threadIdx.x, chunk = (p.c.B + 127) / 128;
  if (tid < 128) chunk_range(p, cum, tid);
  __syncthreads();
  const int total = cum[128], sharers = min(p.grid, total);   // each has a step at least
  for (int c = tid; c < p.grid; c += blockDim.x) {
    ChunkStart s{};
    if (c < sharers) {
      s.f0 = share_start(c, sharers, total);
      s.f_end = share_start(c + 1, sharers, total);
      s.x = first_chunk(p, cum, chunk, s.f0, s.f_end);
    }
    reinterpret_cast<ChunkStart*>(p.starts)[c] = s;
  }
}

// ------------------------------------------------------------------------------------------------ instructions
// kind::f16, f16 operands, fp32 accumulator: the descriptor's fields are those of kind::f8f6f4 with type code 0.
__device__ __forceinline__ void mma_h_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc ? 1u : 0u), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_h_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(acc ? 1u : 0u), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
               "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}

enum ChunkBar : int {
  kCodeFull = 0, kCodeEmpty = 4,            // of the ring of pieces
  kKFull = 8, kKEmpty = 9,
  kVFull = 10, kVEmpty = 12,                // by parity of the running tile
  kQFull = 14, kQFree = 16, kSFull = 18, kPHalf = 20, kPFull = 22, kPvDone = 24,      // by row tile; kSFull, kPFull and kPvDone of 256 columns by tile
  // 256 columns, by pair of warps (the two of the same rows): a row's maximum has moved, by parity of the tile; maxima and sums lie ready
  kVote = 26, kTell = 34,
  kScales = 38,                             // of running tile g: entry g % 8 (the loads are at most five tiles ahead of the softmax)
  kBars = 46,                               // behind them the TMEM slot, the abort flag and two words of votes
};

// ------------------------------------------------------------------------------------------------ queries
// q (bf16, any strides) -> f16 rows with a power of two per row, in the order of the row tiles (b, kv head, new token, head of the group; rows
// of a head filled up to whole tiles with zeros), and the factor of each row's logits.  Tokens beyond the sequence's count are zeros too: their q
// may hold anything, and the weights kernel drops such rows by a sum of infinity, which a logit that is NaN or infinite would outlive.  Eight
// elements a lane.  In the main kernel this took its softmax warps 7000 cycles a unit, and a warp of its own 40000 and more.  The first CTA makes
// the division of the tiles instead.
template <int D>
__global__ void __launch_bounds__(256) cache_chunk_queries_kernel(const CacheAttnParams p) {
  constexpr int kLanes = D / 8;
  __shared__ int cum[136];
  grid_dep_wait();
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) *p.marked = 0;
    chunk_starts(p, cum);
    return;
  }
  const int lane = threadIdx.x & (kLanes - 1), R = p.Nq * p.rep, padded = (R + 127) / 128 * 128;
  const int64_t row = static_cast<int64_t>(blockIdx.x - 1) * (256 / kLanes) + threadIdx.x / kLanes;       // the grid is whole tiles
  const int bh = static_cast<int>(row / padded), r = static_cast<int>(row - static_cast<int64_t>(bh) * padded), b = bh / p.c.Hk, hk = bh - b * p.c.Hk;
  const int tok = r / p.rep, head = hk * p.rep + r - tok * p.rep;
  uint4 w = make_uint4(0, 0, 0, 0);
  if (tok < checked_count(p.c.status, p.counts, b, p.Nq)) w = __ldg(reinterpret_cast<const uint4*>(p.q + b * p.q_sb + tok * p.q_sn + head * p.q_sh) + lane);
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) amax = max3(amax, fabsf(__uint_as_float(v[j] << 16)), fabsf(__uint_as_float(v[j] & 0xFFFF0000u)));
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const uint32_t eb = min(254u, max(14u, __float_as_uint(amax) >> 23));
  const float up = sb_to_scale(267u - eb);                    // largest element to [2^13, 2^14)
  uint32_t h[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = pack_f16x2(__uint_as_float(v[j] << 16) * up, __uint_as_float(v[j] & 0xFFFF0000u) * up);
  reinterpret_cast<uint4*>(p.q16 + row * D)[lane] = make_uint4(h[0], h[1], h[2], h[3]);
  if (lane == 0) {
    const float f = sb_to_scale(eb - 13u) * p.scale * kLog2e;
    p.factors[row] = f;
    if (p.row_ml != nullptr) p.row_ml[row] = make_float2(f, CUDART_INF_F);      // sees nothing, until its sum is known
  }
}

// ------------------------------------------------------------------------------------------------ main kernel
template <int kD>
__global__ void __launch_bounds__(ChunkCfg<kD>::kThreads, 1)
cache_chunk_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tq,
                   const CacheAttnParams p) {
  using C = ChunkCfg<kD>;
  constexpr int D = C::D;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023) & ~1023u) - raw);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kSmemBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kBars + 1);
  float* scales = reinterpret_cast<float*>(smem + C::kSmemScales);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + kVFull + i, 4);
      mbar_init(bars + kVEmpty + i, 1);
      mbar_init(bars + kQFull + i, 1);
      mbar_init(bars + kQFree + i, C::kWide ? 8 : 1);
      mbar_init(bars + kSFull + i, 1);
      mbar_init(bars + kPHalf + i, 4);
      mbar_init(bars + kPFull + i, C::kWide ? 8 : 4);
      mbar_init(bars + kPvDone + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + kCodeFull + i, 1);
      mbar_init(bars + kCodeEmpty + i, 4);
    }
    mbar_init(bars + kKFull, 4);
    mbar_init(bars + kKEmpty, 1);
    for (int i = 0; i < 8; ++i) mbar_init(bars + kVote + i, 2);
    for (int i = 0; i < 4; ++i) mbar_init(bars + kTell + i, 2);
    for (int i = 0; i < 8; ++i) mbar_init(bars + kScales + i, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
    tma_prefetch_desc(&tq);
  }
  if (warp == 13) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  grid_dep_wait();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int cta = blockIdx.x;
  const ChunkStart start = reinterpret_cast<const ChunkStart*>(p.starts)[cta];
  const int f_end = start.f_end;
  bool ok = true;
  auto bar = [&](int i) { return smem_u32(bars + i); };

  if (start.f0 < f_end) {
    ChunkPiece x = start.x;
    if (warp >= 12) {
      reg_dec<C::kRegsOther>();
    }
    if (warp == 12) {
      // ---------------------------------------------------------------------------------------- TMA: code tiles and their scales
      // Lane i < 4 looks after block i of a tile.  A tile's pages are asked for two tiles ahead of its loads and its scales one tile ahead, so
      // that the loads wait for free buffers alone.
      struct Ahead {
        bool live, held;
        int hk, page, sub;
        float ks, vs;
      };
      const int bpp = p.c.page / 32;
      int t = x.t0;
      bool more = true;                                       // (x, t) is the next tile to be looked up
      auto look_up = [&]() {
        Ahead a{};
        while (more && t >= x.t1) {
          more = next_chunk(p, x, f_end);
          t = x.t0;
        }
        a.live = more;
        if (!more) return a;
        const int blk = 4 * t++ + lane;
        a.held = lane < 4 && blk * 32 < x.s.n;
        a.hk = x.hk;
        if (a.held) {
          const int entry = blk / bpp;
          a.sub = blk - entry * bpp;
          a.page = __ldg(p.c.table + x.b * p.c.t_row + entry);
        }
        return a;
      };
      auto ask_scales = [&](Ahead& a) {
        if (!a.held) return;
        a.page = max(0, checked_page(p.c, a.page));
        const int64_t at = a.page * p.c.s_page + a.hk * p.c.s_head + a.sub;
        a.ks = __ldg(p.c.ks + at);
        a.vs = __ldg(p.c.vs + at);
      };
      int g = 0, j = 0;                                       // running tile, running piece of codes
      auto load = [&](const Ahead& a, bool is_v) {
        const int boxes = __popc(__ballot_sync(0xffffffffu, a.held));
        for (int c = 0; c < D / 128 && ok; ++c, ++j) {
          const int buf = j & 1;
          if (j >= 2 && !(ok = wait_warp(bar(kCodeEmpty + buf), ((j >> 1) - 1) & 1, abort_flag))) break;
          if (lane == 0) mbar_expect_tx(bars + kCodeFull + buf, boxes * 4096);
          __syncwarp();
          if (a.held)
            tma_load_4d(sbase + C::kSmemCode + buf * C::kTile + lane * 4096, is_v ? &tv : &tk, bar(kCodeFull + buf), 128 * c, a.sub * 32, a.hk, a.page);
        }
      };
      Ahead now = look_up(), next = look_up();
      ask_scales(now);
      bool first = C::kWide && now.live;
      for (; now.live && ok; ++g) {
        const Ahead after = look_up();
        ask_scales(next);
        if (lane < 4) {
          scales[(g & 7) * 8 + lane] = now.ks;                // zero where there is no block
          scales[(g & 7) * 8 + 4 + lane] = static_cast<float>(static_cast<int>(scale_to_sb(now.vs)) - 127);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + kScales + (g & 7));
        // K of the next tile before V with 256 columns: its S is computed while the softmax is at this one.  (One place calls load: with more of
        // them the kernel outgrew its instruction cache.)
#pragma unroll 1
        for (int i = first ? 0 : 1; i < 3; ++i) {
          const bool ahead = C::kWide && i == 1;
          if ((ahead ? next.live : true) && ok) load(ahead ? next : now, i == 2);
        }
        first = false;
        now = next;
        next = after;
      }
      if (!ok) {
        if (lane == 0) raise_abort(abort_flag, p.c.status, kStatusTimeoutProducer + kInCache);
        // what is in flight lands before the shared memory goes
        for (int k = 1; k <= 2; ++k)
          if (j >= k) wait_or_abort(bar(kCodeFull + ((j - k) & 1)), ((j - k) >> 1) & 1, abort_flag);
      }
    } else if (warp == 13) {
      // ---------------------------------------------------------------------------------------- MMA
      if (elect_one()) {
        constexpr uint32_t kIdescS = idesc_f8(128, 128, false, false), kIdescO = idesc_f8(128, D, false, true);
        const uint32_t q_lo = desc_lo(sbase + C::kSmemQ), k_lo = desc_lo(sbase + C::kSmemK);
        // V's panels of 64 columns lie kTile apart: the leading offset of an operand wider than 128 bytes
        const uint32_t v_lo = (((sbase + C::kSmemV) & 0x3FFFFu) >> 4) | (static_cast<uint32_t>(C::kTile >> 4) << 16);
        int g = 0;                                            // running tile
        // S of a row tile, or (256 columns) into S buffer r
        auto issue_s = [&](int r, bool last) {
          const uint32_t a = q_lo + (C::kWide ? 0 : r * (2 * C::kTile >> 4)), b = k_lo;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k >> 2) * (C::kTile >> 4) + (k & 3) * 2;
            mma_h_ss(tmem + 128 * r, a + off, b + off, kIdescS, k > 0);
          }
          if (last) tc_commit(bars + kKEmpty);
          tc_commit(bars + kSFull + r);
        };
        if constexpr (C::kWide) {
          int units = 0;
          do {
            if (x.t0 >= x.t1) continue;
            const int n = x.t1 - x.t0;
            if (!(ok = wait_or_abort(bar(kQFull), units++ & 1, abort_flag) && wait_or_abort(bar(kKFull), g & 1, abort_flag))) break;
            tc_fence_after();
            issue_s(g & 1, true);
            for (int i = 0; i < n && ok; ++i, ++g) {
              if (i + 1 < n) {                                // the next S, while the softmax is at this one
                // its buffer held the P of the tile before this one, and the products of different shapes need not keep their order
                if (!(ok = wait_or_abort(bar(kKFull), (g + 1) & 1, abort_flag) && (i == 0 || wait_or_abort(bar(kPvDone + ((g - 1) & 1)), ((g - 1) >> 1) & 1, abort_flag)))) break;
                tc_fence_after();
                issue_s((g + 1) & 1, true);
              }
              // both groups' P before any product: both may have rescaled O
              if (!(ok = wait_or_abort(bar(kPFull + (g & 1)), (g >> 1) & 1, abort_flag) && wait_or_abort(bar(kVFull), g & 1, abort_flag))) break;
              tc_fence_after();
#pragma unroll
              for (int k = 0; k < 8; ++k)
                mma_h_ts(tmem + 256, tmem + 128 * (g & 1) + 64 * (k >> 2) + 8 * (k & 3), v_lo + k * (2048 >> 4), kIdescO, i > 0 || k > 0);
              tc_commit(bars + kVEmpty);
              tc_commit(bars + kPvDone + (g & 1));
            }
          } while (ok && next_chunk(p, x, f_end));
        } else {
          int tiles[2] = {0, 0}, units[2] = {0, 0};           // tiles and units of each row tile
          do {
            if (x.t0 >= x.t1) continue;
            const int n = x.t1 - x.t0, groups = x.groups(p);
            for (int r = 0; r < groups; ++r) {
              if (r == 0 && !(ok = wait_or_abort(bar(kKFull), g & 1, abort_flag))) break;
              if (!(ok = wait_or_abort(bar(kQFull + r), units[r]++ & 1, abort_flag))) break;
              tc_fence_after();
              issue_s(r, r == groups - 1);
              if (n == 1) tc_commit(bars + kQFree + r);       // the row tile's last S of the unit
            }
            for (int i = 0; i < n && ok; ++i, ++g) {
              for (int r = 0; r < groups; ++r) {
                // 16 keys a step: 8 columns of P, 16 rows of V; the first half of the keys while the softmax is at the second
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  if (!(ok = wait_or_abort(bar((half == 0 ? kPHalf : kPFull) + r), tiles[r] & 1, abort_flag))) break;
                  if (r == 0 && half == 0 && !(ok = wait_or_abort(bar(kVFull + (g & 1)), (g >> 1) & 1, abort_flag))) break;
                  tc_fence_after();
#pragma unroll
                  for (int k = 4 * half; k < 4 * half + 4; ++k)
                    mma_h_ts(tmem + 256 + 128 * r, tmem + 128 * r + 8 * k, v_lo + (g & 1) * (2 * C::kTile >> 4) + k * (2048 >> 4), kIdescO, i > 0 || k > 0);
                }
                if (!ok) break;
                ++tiles[r];
                if (r == groups - 1) tc_commit(bars + kVEmpty + (g & 1));
                tc_commit(bars + kPvDone + r);
                if (i + 1 < n) {
                  if (r == 0 && !(ok = wait_or_abort(bar(kKFull), (g + 1) & 1, abort_flag))) break;
                  tc_fence_after();
                  issue_s(r, r == groups - 1);                // over the P just read: products of one shape run in the order of their issue
                  if (i + 2 >= n) tc_commit(bars + kQFree + r);
                }
              }
            }
          } while (ok && next_chunk(p, x, f_end));
        }
        if (!ok) raise_abort(abort_flag, p.c.status, kStatusTimeoutMma + kInCache);
      }
    } else if (warp == 14) {
      // ---------------------------------------------------------------------------------------- queries of the next unit
      if (elect_one()) {
        int units[2] = {0, 0};
        const int tiles_of_head = (p.Nq * p.rep + 127) / 128;
        do {
          if (x.t0 >= x.t1) continue;
          for (int r = 0; r < (C::kWide ? 1 : x.groups(p)) && ok; ++r) {
            if (units[r] > 0) ok = wait_or_abort(bar(kQFree + r), (units[r] - 1) & 1, abort_flag);
            if (!ok) break;
            ++units[r];
            mbar_expect_tx(bars + kQFull + r, C::kPanels * C::kTile);
            const int row = ((x.b * p.c.Hk + x.hk) * tiles_of_head + (C::kWide ? x.rt : 2 * x.rt + r)) * 128;
            for (int panel = 0; panel < C::kPanels; ++panel)
              tma_load_2d(smem + C::kSmemQ + (2 * r + panel) * C::kTile, &tq, bars + kQFull + r, 128 * panel, row);        // x in bytes
          }
        } while (ok && next_chunk(p, x, f_end));
        if (!ok) {
          raise_abort(abort_flag, p.c.status, kStatusTimeoutProducer + kInCache);
          for (int r = 0; r < 2; ++r)                         // what is in flight lands before the shared memory goes
            if (units[r] > 0) wait_or_abort(bar(kQFull + r), (units[r] - 1) & 1, abort_flag);
        }
      }
    } else if (warp >= 8 && warp < 12) {
      reg_dec<C::kRegsOther>();
      // ---------------------------------------------------------------------------------------- codes -> f16 operand tiles
      const int ct = tid - 256, c = ct & 7;                   // a thread takes 16-byte pieces c of keys ct / 8, + 16, ...
      // a piece's two halves of eight elements: which goes first is chosen so that the stores of eight lanes fall on different banks
      const int panel = c >> 2, flip = panel;
      int j = 0;                                              // running piece of codes
      // K or V of running tile g; V's slots beyond the length hold anything, NaN codes too: zeros
      auto convert = [&](bool is_v, int g, int held) {
        const int vbuf = C::kVBufs == 2 ? g & 1 : 0;
#pragma unroll 1
        for (int part = 0; part < D / 128 && ok; ++part, ++j) {
          const int buf = j & 1;
          ok = wait_warp(bar(kCodeFull + buf), (j >> 1) & 1, abort_flag);
          if (!ok) break;
          const uint32_t src = sbase + C::kSmemCode + buf * C::kTile;
          const uint32_t dst = sbase + (is_v ? C::kSmemV + vbuf * C::kPanels * C::kTile : C::kSmemK) + (2 * part + panel) * C::kTile;
          auto piece_of = [&](int i) {
            const int key = (ct >> 3) + 16 * i;
            return lds_f4(src + key * 128 + ((c ^ (key & 7)) << 4));
          };
          // With 256 columns, whose pieces outnumber their buffers, all of one into registers: its buffer is free for the next load during the
          // conversion (512 new tokens 173 -> 145 us; with 128 126 -> 128).
          float4 in[8];
          if (C::kWide) {
#pragma unroll
            for (int i = 0; i < 8; ++i) in[i] = piece_of(i);
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + kCodeEmpty + buf);
          }
          if (part == 0 && !is_v && g >= 1) ok = wait_warp(bar(kKEmpty), (g - 1) & 1, abort_flag);
          if (part == 0 && is_v && g >= C::kVBufs) ok = wait_warp(bar(kVEmpty + vbuf), (g / C::kVBufs - 1) & 1, abort_flag);
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = (ct >> 3) + 16 * i;
            const float4 w4 = C::kWide ? in[i] : piece_of(i);
            uint32_t w[4] = {__float_as_uint(w4.x), __float_as_uint(w4.y), __float_as_uint(w4.z), __float_as_uint(w4.w)};
            if (key >= held) w[0] = w[1] = w[2] = w[3] = 0;
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              h[2 * e] = e4m3_lo_f16x2(w[e]);
              h[2 * e + 1] = e4m3_hi_f16x2(w[e]);
            }
            const int cc = (c & 3) * 2;
            const uint32_t row = dst + key * 128;
            const uint32_t first = row + (((cc + flip) ^ (key & 7)) << 4), second = row + (((cc + 1 - flip) ^ (key & 7)) << 4);
            if (flip) {
              sts_u4(first, h[4], h[5], h[6], h[7]);
              sts_u4(second, h[0], h[1], h[2], h[3]);
            } else {
              sts_u4(first, h[0], h[1], h[2], h[3]);
              sts_u4(second, h[4], h[5], h[6], h[7]);
            }
          }
          if (part < D / 128 - 1) continue;
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(bars + (is_v ? kVFull + vbuf : kKFull));
            if (!C::kWide) mbar_arrive(bars + kCodeEmpty + buf);
          }
        }
      };
      int t = x.t0;
      auto find = [&]() {                                     // from tile t of the piece on: is there one?
        while (t >= x.t1) {
          if (!next_chunk(p, x, f_end)) return false;
          t = x.t0;
        }
        return true;
      };
      int held = 0;                                           // of the tile whose V is next
      bool live = true;
      for (int g = 0; live && ok; ++g) {                      // in the order of the loads: K of tile g, V of the same or (256 columns) the one before
        live = find();
        const int held_g = live ? x.s.n - 128 * t++ : 0;
        if (!C::kWide) held = held_g;
#pragma unroll 1
        for (int kv = 0; kv < 2 && ok; ++kv)
          if (C::kWide && kv == 1 ? g > 0 : live) convert(kv == 1, C::kWide ? g - kv : g, kv == 1 ? held : 128);
        held = held_g;
      }
      if (!ok && lane == 0) raise_abort(abort_flag, p.c.status, kStatusTimeoutCompute + kInCache);
    } else if (warp < 8) {
      reg_inc<C::kRegsSoftmax>();
      // ---------------------------------------------------------------------------------------- softmax and output
      const int r = warp >> 2, in_tile = (warp & 3) * 32 + lane;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t t_o = tmem + lanes + 256 + 128 * r;      // of 256 columns, the half that this group rescales and writes
      volatile int8_t* told_d = reinterpret_cast<volatile int8_t*>(smem + C::kSmemRows + 1024) + in_tile;        // the same, a second value
      volatile float* told = reinterpret_cast<volatile float*>(smem + C::kSmemRows) + in_tile;        // by group 0 of this row; by group 1 128 values on
      const uint32_t stage = sbase + C::kSmemOut + warp * 4096;
      int g = 0, mine = 0, asked = 0, tells = 0;              // running tile; tiles of this row tile; votes and values that the pair has exchanged
      int slot = 2 * cta;
      do {
        if (x.t0 >= x.t1) continue;
        if (!C::kWide && r >= x.groups(p)) {
          g += x.t1 - x.t0;
          slot = 2 * cta + 1;
          continue;
        }
        const int row = x.rt * C::kRows + (C::kWide ? 0 : r * 128) + in_tile, limit = row_limit(p, x.s, row);
        const int i_tok = row / p.rep, head = x.hk * p.rep + row - i_tok * p.rep;
        // A row that sees nothing is not written here: its logits need no mask (one of them had its warp take the masked path in all tiles), and a warp
        // of such rows makes none, whatever its P holds.
        const int sees = limit > 0 ? limit : INT_MAX;
        const bool idle = !__any_sync(0xffffffffu, limit > 0);
        // of the row's logits, K's scale aside
        const int64_t padded_row = (static_cast<int64_t>(x.b) * p.c.Hk + x.hk) * ((p.Nq * p.rep + 127) / 128 * 128) + row;
        const float f = fabsf(__ldg(p.factors + padded_row));
        // Of the row, whole numbers: m, the reference of the sum l; m + v, that of the products of a probability and its V scale: O counts in
        // 2^(m + v - kPBase).  The largest logit, and logit + log2 of its V scale, are at most kHeadroom above them.
        float m = kNone, v = 0.f, l = 0.f;
        // P V of this group's tile i is in O.  With 256 columns the softmax may be two tiles ahead of the products, so that these have two barriers.
        auto products_of = [&](int i) { return C::kWide ? wait_warp(bar(kPvDone + (i & 1)), (i >> 1) & 1, abort_flag) : wait_warp(bar(kPvDone + r), i & 1, abort_flag); };
        // What the two warps of a row's two groups know of it (256 columns): the other's value.
        auto tell = [&](float mine_v, float& other) -> bool {
          told[128 * r] = mine_v;
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + kTell + (warp & 3));
          if (!wait_warp(bar(kTell + (warp & 3)), tells++ & 1, abort_flag)) return false;
          other = told[128 * (r ^ 1)];
          return true;
        };
        // One key tile.  kCut: some row of the warp does not see all its keys (a compile-time variant: no select per element elsewhere).
        auto tile = [&](int t, auto cut_tag) -> bool {
          constexpr bool kCut = decltype(cut_tag)::value;
          const int entry = (g + t - x.t0) & 7;
          const float4 ks = lds_f4(sbase + C::kSmemScales + entry * 32), vs = lds_f4(sbase + C::kSmemScales + entry * 32 + 16);
          const uint32_t t_s = tmem + lanes + (C::kWide ? 128 * (mine & 1) + 64 * r : 128 * r);
          const float fc[4] = {f * (C::kWide && r ? ks.z : ks.x), f * (C::kWide && r ? ks.w : ks.y), f * ks.z, f * ks.w};
          const float ev[4] = {C::kWide && r ? vs.z : vs.x, C::kWide && r ? vs.w : vs.y, vs.z, vs.w};
          const int seen = sees - 128 * t - (C::kWide ? 64 * r : 0);         // keys of the tile, from this group's first on, that the row sees
          // 32 columns at a time, the next ones in flight; what a row does not see is -inf
          uint32_t s_buf[2][32];
          auto columns = [&](int c) {
            tmem_wait_ld();
            if (c < C::kCols / 32 - 1) tmem_ld32(t_s + 32 * (c + 1), s_buf[(c + 1) & 1]);
            if (kCut) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (32 * c + e >= seen) s_buf[c & 1][e] = 0xff800000u;
            }
          };
          auto pair = [&](int c, int e) { return make_float2(__uint_as_float(s_buf[c & 1][2 * e]), __uint_as_float(s_buf[c & 1][2 * e + 1])); };
          float top = -CUDART_INF_F, top2 = -CUDART_INF_F;    // of the tile: logit, and logit + log2 of V's scale
          auto moves_row = [&]() { return top > m + kHeadroom || top2 > m + v + kHeadroom; };
          tmem_ld32(t_s, s_buf[0]);
#pragma unroll
          for (int c = 0; c < C::kCols / 32; ++c) {
            columns(c);
            float2 s2[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) s2[e] = pair(c, e);
            const float top_s = max32(s2);
            const float top_c = kCut && top_s == -CUDART_INF_F ? top_s : top_s * fc[c];        // the factor may be zero
            top = fmaxf(top, top_c);
            top2 = fmaxf(top2, top_c + ev[c]);
          }
          if (C::kWide) {
            // a common reference: seldom does a row move, so that the pair first tell each other whether any does
            const bool moves = __any_sync(0xffffffffu, moves_row());
            volatile uint8_t* votes = smem + C::kSmemBars + 8 * (kBars + 2 + (asked & 1));      // behind the TMEM slot and the abort flag
            const int vote = kVote + 2 * (warp & 3) + (asked & 1);
            if (lane == 0) {
              votes[warp] = moves;
              mbar_arrive(bars + vote);
            }
            if (!wait_warp(bar(vote), (asked++ >> 1) & 1, abort_flag)) return false;
            if (moves || votes[warp ^ 4]) {
              float other;
              // the second value as its distance from the first, rounded up: the same in both groups
              const float d = fminf(fmaxf(ceilf(top2 - top), -128.f), 127.f);
              told_d[128 * r] = static_cast<int8_t>(d);
              if (!tell(top, other)) return false;
              top2 = fmaxf(top + d, other + static_cast<float>(told_d[128 * (r ^ 1)]));
              top = fmaxf(top, other);
            }
          }
          tmem_ld32(t_s, s_buf[0]);
          if (__any_sync(0xffffffffu, moves_row())) {
            float keep = 1.f;
            if (moves_row()) {
              // a row of larger logits than fp32 can add whole numbers to: marked, for the join to make it by itself
              if (fabsf(top) > kExact) {
                p.factors[padded_row] = -f;
                *p.marked = 1;
              }
              const float m_old = m, u_old = m + v, u = top2 > u_old + kHeadroom ? ceilf(top2) : u_old;
              if (top > m + kHeadroom) m = ceilf(top);
              v = u - m;
              l *= ex2_approx(m_old - m);
              keep = ex2_approx(u_old - u);
            }
            if (t > x.t0) {
              if (!products_of(mine - 1)) return false;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                tmem_ld32(t_o + 32 * c, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                tmem_st32(t_o + 32 * c, o);
              }
            }
          }
#pragma unroll
          for (int c = 0; c < C::kCols / 32; ++c) {
            // P comes out as 2^(s - m + off), below 2^16; where the products are 2^-57 of the largest they vanish anyway, but the sum must not
            const float off = fmaxf(kPBase + ev[c] - v, -45.f);
            const float2 f2 = splat2(fc[c]), sub = splat2(off - m);
            columns(c);
            float2 sum = make_float2(0.f, 0.f);
            uint32_t h[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float2 y = fma2(pair(c, e), f2, sub);
              if (kCut) {                                     // zero times infinity is none
                if (32 * c + 2 * e >= seen) y.x = -CUDART_INF_F;
                if (32 * c + 2 * e + 1 >= seen) y.y = -CUDART_INF_F;
              }
              y = ex2_2(y);
              sum = add2(sum, y);
              h[e] = pack_f16x2(y.x, y.y);
            }
            l = fmaf(sum.x + sum.y, ex2_approx(-off), l);        // a power of two; zero where p is below 2^-111 of the largest
            tmem_st16(t_s + 16 * c, h);                       // over columns that have been read: 16 c + 15 < 32 c + 32
            if (!C::kWide && c == 1) {                        // the first half of the keys: the tensor cores may begin
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bars + kPHalf + r);
            }
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + kPFull + (C::kWide ? mine & 1 : r));
          return true;
        };
        for (int t = x.t0; t < x.t1; ++t, ++mine) {
          const int gt = g + t - x.t0;
          ok = (idle || wait_warp(bar(kScales + (gt & 7)), (gt >> 3) & 1, abort_flag)) &&
               (C::kWide ? wait_warp(bar(kSFull + (mine & 1)), (mine >> 1) & 1, abort_flag) : wait_warp(bar(kSFull + r), mine & 1, abort_flag));
          if (!ok) break;
          tc_fence_after();
          if (idle) {
            if (lane == 0) {
              if (!C::kWide) mbar_arrive(bars + kPHalf + r);
              mbar_arrive(bars + kPFull + (C::kWide ? mine & 1 : r));
            }
            continue;
          }
          const bool cut = __any_sync(0xffffffffu, sees < 128 * (t + 1));
          if (!(ok = cut ? tile(t, std::true_type{}) : tile(t, std::false_type{}))) break;
        }
        g += x.t1 - x.t0;
        if (!ok) break;
        ok = idle || products_of(mine - 1);
        if (ok && !idle && C::kWide) {                                 // the sum over both halves of the keys
          float other = 0.f;
          ok = tell(l, other);
          l += other;
        }
        if (!ok) break;
        tc_fence_after();
        const bool whole = x.t0 == 0 && x.t1 == x.tiles;
        const float scale = whole ? exp2f(v - kPBase) / l : 1.f;
        // where a row that sees something goes
        const int64_t out_row = limit == 0 ? -1 : ((static_cast<int64_t>(x.b) * p.Nq + i_tok) * p.H + head) * D;
        // Through shared memory, so that the lanes of a store write whole rows (a row a thread, 16 bytes at a time, took 11000 cycles a piece):
        // 32 rows x 128 bytes at a time, 16-byte pieces XORed with the row.
        const int64_t part0 = static_cast<int64_t>(slot) * C::kRows + (C::kWide ? 0 : r * 128) + (warp & 3) * 32;
        const int col0 = C::kWide ? 128 * r : 0;
        float any_nan = 0.f;                                  // NaN where a value is
#pragma unroll 1
        for (int c = idle ? 4 : 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(t_o + 32 * c, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) any_nan += __uint_as_float(o[e]);
          if (whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const __nv_bfloat162 b2 = __floats2bfloat162_rn(__uint_as_float(o[8 * e + 2 * j]) * scale, __uint_as_float(o[8 * e + 2 * j + 1]) * scale);
                w[j] = *reinterpret_cast<const uint32_t*>(&b2);
              }
              sts_u4(stage + lane * 128 + ((((4 * c + e) & 7) ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
            }
            if ((c & 1) == 0) continue;                       // 64 columns make 128 bytes
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              sts_u4(stage + lane * 128 + ((e ^ (lane & 7)) << 4), __float_as_uint(__uint_as_float(o[4 * e]) * scale), __float_as_uint(__uint_as_float(o[4 * e + 1]) * scale),
                     __float_as_uint(__uint_as_float(o[4 * e + 2]) * scale), __float_as_uint(__uint_as_float(o[4 * e + 3]) * scale));
          }
          __syncwarp();
          const int piece = lane & 7;
          float4 v[8];                                        // of rows lane / 8, + 4, ...: four rows a store, eight lanes each
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row32 = 4 * i + (lane >> 3);
            v[i] = lds_f4(stage + row32 * 128 + ((piece ^ (row32 & 7)) << 4));
          }
          if (whole) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int64_t at = __shfl_sync(0xffffffffu, out_row, 4 * i + (lane >> 3));
              if (at >= 0) reinterpret_cast<float4*>(p.o + at + col0 + 64 * (c >> 1))[piece] = v[i];
            }
          } else {                                            // rows that see nothing too: their slots are not read
            float4* to = reinterpret_cast<float4*>(p.part_o + (part0 + (lane >> 3)) * D + col0 + 32 * c) + piece;
#pragma unroll
            for (int i = 0; i < 8; ++i) to[4 * i * (D / 4)] = v[i];
          }
          __syncwarp();
        }
        // A NaN may be that of a value whose token this row does not see, times zero: the row is marked too.
        if (p.causal && limit > 0 && any_nan != any_nan) {
          p.factors[padded_row] = -f;
          *p.marked = 1;
        }
        // where the join finds the unit: the slot of its first piece, and the last CTA that has one (the pieces between are first ones)
        if (r == 0 && in_tile == 0) {
          int2* u = p.unit_slots + (static_cast<int64_t>(x.b) * p.c.Hk + x.hk) * ((p.Nq * p.rep + C::kRows - 1) / C::kRows) + x.rt;
          if (x.t0 == 0) u->x = whole ? -1 : slot;
          if (x.t1 == x.tiles) u->y = cta;
        }
        if (limit > 0 && (!C::kWide || r == 0)) {
          if (whole) {
            p.lse[(static_cast<int64_t>(x.b) * p.H + head) * p.Nq + i_tok] = (m + log2f(l)) * kLn2;
            if (p.row_ml != nullptr) p.row_ml[padded_row] = make_float2(f, m + log2f(l));
          } else {
            p.part_ml[part0 + lane] = make_float4(m, l, v, 0.f);
          }
        }
        tc_fence_before();
        if (C::kWide) {                                       // the staging has been read: the next queries may come
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + kQFree);
        }
        slot = 2 * cta + 1;
      } while (next_chunk(p, x, f_end));
      if (!ok && lane == 0) raise_abort(abort_flag, p.c.status, kStatusTimeoutCompute + kInCache);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------------ join
// A row that the main kernel marked, by one warp and from the definition: a key after the other, all in fp32, the logits' differences exact whatever their
// size.  `factor`: of the logits, of the query as the main kernel has it.  Writes o (this lane's four channels of each 128); -> maximum (log2 domain), sum.
template <int D>
__device__ __forceinline__ float2 one_row(const CacheAttnParams& p, int b, int hk, int head, int i_tok, int limit, float factor, __nv_bfloat162* o) {
  constexpr int kVecs = D / 128;
  const int lane = threadIdx.x & 31, bpp = p.c.page / 32;
  const __half2* q = reinterpret_cast<const __half2*>(p.q16 + ((static_cast<int64_t>(b) * p.c.Hk + hk) * ((p.Nq * p.rep + 127) / 128 * 128) +
                                                               static_cast<int64_t>(i_tok) * p.rep + head - hk * p.rep) * D) + 2 * lane;
  float4 qv[kVecs], acc[kVecs] = {};
#pragma unroll
  for (int x = 0; x < kVecs; ++x) {
    const float2 a = __half22float2(q[64 * x]), c = __half22float2(q[64 * x + 1]);
    qv[x] = make_float4(a.x, a.y, c.x, c.y);
  }
  float m = kNone, l = 0.f;
  for (int j = 0; j < limit; ++j) {
    const int blk = j / 32, page = max(0, checked_page(p.c, __ldg(p.c.table + b * p.c.t_row + blk / bpp))), sub = blk % bpp;
    const int64_t code = page * p.c.c_page + hk * p.c.c_head + (sub * 32 + j % 32) * p.c.c_slot + 4 * lane, scale = page * p.c.s_page + hk * p.c.s_head + sub;
    float s = 0.f;
    float4 v[kVecs];
    const float vs = __ldg(p.c.vs + scale);
#pragma unroll
    for (int x = 0; x < kVecs; ++x) {
      const uint32_t k4 = __ldg(reinterpret_cast<const uint32_t*>(p.c.k8 + code + 128 * x)), v4 = __ldg(reinterpret_cast<const uint32_t*>(p.c.v8 + code + 128 * x));
      const float2 k0 = f16x2_to_float2(e4m3_lo_f16x2(k4)), k1 = f16x2_to_float2(e4m3_hi_f16x2(k4)), v0 = f16x2_to_float2(e4m3_lo_f16x2(v4)), v1 = f16x2_to_float2(e4m3_hi_f16x2(v4));
      s = fmaf(qv[x].x, k0.x, fmaf(qv[x].y, k0.y, fmaf(qv[x].z, k1.x, fmaf(qv[x].w, k1.y, s))));
      v[x] = make_float4(v0.x * vs, v0.y * vs, v1.x * vs, v1.y * vs);
    }
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    s = __fmul_rn(s, __fmul_rn(factor, __ldg(p.c.ks + scale)));
    const float m_new = fmaxf(m, s), keep = exp2f(m - m_new), w = exp2f(s - m_new);
    m = m_new;
    l = fmaf(l, keep, w);
#pragma unroll
    for (int x = 0; x < kVecs; ++x)
      acc[x] = make_float4(fmaf(acc[x].x, keep, w * v[x].x), fmaf(acc[x].y, keep, w * v[x].y), fmaf(acc[x].z, keep, w * v[x].z), fmaf(acc[x].w, keep, w * v[x].w));
  }
#pragma unroll
  for (int x = 0; x < kVecs; ++x) {
    o[64 * x] = __floats2bfloat162_rn(acc[x].x / l, acc[x].y / l);
    o[64 * x + 1] = __floats2bfloat162_rn(acc[x].z / l, acc[x].w / l);
  }
  return make_float2(m, l);
}

// Rows of units that were cut, rows that see nothing, marked rows: a warp a row, four of a (sequence, head) a CTA.
template <int D>
__global__ void __launch_bounds__(128, D == 128 ? 12 : 10) cache_chunk_join_kernel(const CacheAttnParams p) {
  constexpr int kRows = ChunkCfg<D>::kRows, kVecs = D / 128;
  grid_dep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int R = p.Nq * p.rep, groups = (R + 3) / 4, unit_tiles_max = (R + kRows - 1) / kRows;
  const int r = static_cast<int>(blockIdx.x % groups) * 4 + warp, bh = static_cast<int>(blockIdx.x / groups), hk = bh % p.c.Hk, b = bh / p.c.Hk;
  if (r >= R) return;
  const int2 unit = p.unit_slots[static_cast<int64_t>(bh) * unit_tiles_max + r / kRows];
  const int marked = *p.marked;                           // any row of the call
  const ChunkSeq s = chunk_seq(p, b);
  const int i_tok = r / p.rep, head = hk * p.rep + r - i_tok * p.rep;
  __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(p.o + ((static_cast<int64_t>(b) * p.Nq + i_tok) * p.H + head) * D) + 2 * lane;
  float* lse = p.lse + (static_cast<int64_t>(b) * p.H + head) * p.Nq + i_tok;
  const int64_t padded_row = static_cast<int64_t>(bh) * ((R + 127) / 128 * 128) + r;
  if (row_limit(p, s, r) == 0) {
#pragma unroll
    for (int x = 0; x < kVecs; ++x) o[64 * x] = o[64 * x + 1] = __floats2bfloat162_rn(0.f, 0.f);
    if (lane == 0) *lse = -CUDART_INF_F;
    return;
  }
  if (marked != 0 && p.factors[padded_row] < 0.f) {
    const float factor = p.factors[padded_row];
    const float2 ml = one_row<D>(p, b, hk, head, i_tok, row_limit(p, s, r), -factor, o);
    if (lane == 0) {
      *lse = (ml.x + log2f(ml.y)) * kLn2;
      if (p.row_ml != nullptr) p.row_ml[padded_row] = make_float2(-factor, ml.x + log2f(ml.y));
    }
    return;
  }
  const JoinSlots slots = join_slots_of_ctas(unit, p.grid);
  if (slots.none()) return;                               // whole: written by its CTA (or given up)
  float top = kNone, v_top = 0.f, sum = 0.f;
  float4 acc[kVecs] = {};
  const int n = slots.count;
  // 32 results at a time, a lane each: their maxima and sums together, then the values of those that count
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int i = i0 + lane, at = slots.slot(i) * kRows + (r & (kRows - 1));
    const float4 ml = i < n ? p.part_ml[at] : make_float4(kNone, 0.f, 0.f, 0.f);       // kNone: a piece of which the row sees nothing
    float top_new = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top_new = fmaxf(top_new, __shfl_xor_sync(0xffffffffu, top_new, o));
    top_new = fmaxf(top, top_new);
    const float fall = ml.x - top_new, old = v_top + (top - top_new);
    float l = ml.y * ex2_approx(fall);
    v_top = ml.z + fall;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      l += __shfl_xor_sync(0xffffffffu, l, o);
      v_top = fmaxf(v_top, __shfl_xor_sync(0xffffffffu, v_top, o));
    }
    v_top = fmaxf(v_top, old);
    const float a = ex2_approx(old - v_top), w = ex2_approx(ml.z + fall - v_top);
    sum = sum * ex2_approx(top - top_new) + l;
    top = top_new;
#pragma unroll
    for (int x = 0; x < kVecs; ++x) acc[x] = make_float4(acc[x].x * a, acc[x].y * a, acc[x].z * a, acc[x].w * a);
    const uint32_t counts = __ballot_sync(0xffffffffu, ml.x > kNone);
#pragma unroll 8
    for (int k = 0; k < min(32, n - i0); ++k) {
      const float w_k = __shfl_sync(0xffffffffu, w, k);
      const int64_t at_k = __shfl_sync(0xffffffffu, at, k);
      if (!((counts >> k) & 1)) continue;
#pragma unroll
      for (int x = 0; x < kVecs; ++x) {
        const float4 v = reinterpret_cast<const float4*>(p.part_o + at_k * D)[32 * x + lane];
        acc[x] = make_float4(acc[x].x + v.x * w_k, acc[x].y + v.y * w_k, acc[x].z + v.z * w_k, acc[x].w + v.w * w_k);
      }
    }
  }
  const float inv = exp2f(v_top - kPBase) / sum;
#pragma unroll
  for (int x = 0; x < kVecs; ++x) {
    o[64 * x] = __floats2bfloat162_rn(acc[x].x * inv, acc[x].y * inv);
    o[64 * x + 1] = __floats2bfloat162_rn(acc[x].z * inv, acc[x].w * inv);
  }
  if (lane == 0) {
    *lse = (top + log2f(sum)) * kLn2;
    if (p.row_ml != nullptr) p.row_ml[padded_row] = make_float2(fabsf(p.factors[padded_row]), top + log2f(sum));
  }
}

// ------------------------------------------------------------------------------------------------ weights
// weights[b, hk, j] (+)= sum over the rows r that see token j of exp(s_rj) / sum_r = 2^(f_r ks s_rj - c_r), c_r = log2 of the row's sum.
// S^T = K Q^T on tcgen05 with 128 tokens as M and up to 128 rows as N: a token's sum stays in its thread (TMEM lane) over all row tiles, in
// the order of the rows.  An item is a key tile of a (sequence, head): its codes become an f16 tile once, the row tiles pass by.  Where a
// head has but one row tile it stays for the next items of the head.  Warps 0-3 and 4-7 take row tiles in turn (32 rows each of an only one);
// warp 8: TMA, warp 9: MMA.  Four S^T buffers of 128 columns.
// The first row that sees token j.
__device__ __forceinline__ int first_row(const CacheAttnParams& p, const ChunkSeq& s, int j) { return p.causal ? max(0, j - s.n + s.count) * p.rep : 0; }

template <int D>
struct ChunkWeightsCfg {
  static constexpr int kThreads = 320;
  static constexpr int kRows = 128;                           // of a row tile
  static constexpr int kPanels = D / 64;
  static constexpr int kTile = 128 * 128;
  static constexpr int kQBytes = kPanels * kTile;             // of a row tile
  static constexpr int kQBufs = D == 128 ? 4 : 2, kQShift = D == 128 ? 2 : 1;
  static constexpr int kSmemK = kQBufs * kQBytes;             // panels
  static constexpr int kChunks = D / 128;                     // pieces of kTile in which an item's codes come
  static constexpr int kCodeBufs = D == 128 ? 3 : 1;          // what fits of them
  static constexpr int kSmemCode = kSmemK + kPanels * kTile;
  static constexpr int kSmemRows = kSmemCode + kCodeBufs * kTile;     // (factor, log2 sum) of the rows, by row tile buffer
  static constexpr int kSmemSums = kSmemRows + kQBufs * kRows * 8;    // by parity of the item
  static constexpr int kSmemBars = kSmemSums + 2 * 128 * 4;
  static constexpr int kSmem = kSmemBars + 256 + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
};
enum ChunkWeightsBar : int { kwCode = 0, kwCodeFree = 3, kwQ = 6, kwQFree = 10, kwS = 14, kwSFree = 18, kwK = 22, kwSums = 23, kwSumsFree = 25, kwBars = 27 };

template <int D>
__global__ void __launch_bounds__(ChunkWeightsCfg<D>::kThreads, 1)
cache_chunk_weights_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tq, const CacheAttnParams p, const int tiles_of_row,
                           const int run) {
  using C = ChunkWeightsCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023) & ~1023u) - raw);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kSmemBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kwBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kwBars + 1);
  float* sums = reinterpret_cast<float*>(smem + C::kSmemSums);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(bars + kwQ + i, 1);
      mbar_init(bars + kwQFree + i, 9);                       // the MMA, and the warps that read the rows' constants
      mbar_init(bars + kwS + i, 1);
      mbar_init(bars + kwSFree + i, 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + kwSums + i, 4);
      mbar_init(bars + kwSumsFree + i, 4);
    }
    for (int i = 0; i < C::kCodeBufs; ++i) {
      mbar_init(bars + kwCode + i, 1);
      mbar_init(bars + kwCodeFree + i, 8);
    }
    mbar_init(bars + kwK, 8);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tq);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  grid_dep_wait();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto bar = [&](int i) { return smem_u32(bars + i); };
  const int R = p.Nq * p.rep, row_tiles_max = (R + 127) / 128;
  const int items = p.c.B * p.c.Hk * tiles_of_row;            // 128 weights each: they fit
  bool ok = true;
  // Item i: a key tile that exists, and its row tiles that see any of it: rt0 ... rt1 - 1.
  struct Item {
    int b, hk, t, n, rt0, rt1;
    ChunkSeq s;
  };
  auto item_at = [&](int i, Item& x) {
    const int bh = i / tiles_of_row;
    x.t = i - bh * tiles_of_row;
    x.b = bh / p.c.Hk;
    x.hk = bh - x.b * p.c.Hk;
    x.s = chunk_seq(p, x.b);
    x.n = x.s.n;
    x.rt1 = (x.s.count * p.rep + C::kRows - 1) / C::kRows;
    x.rt0 = min(x.rt1, first_row(p, x.s, 128 * x.t) / C::kRows);
    return 128 * x.t < x.n;
  };
  // The CTA's items that some row sees, one by one: runs of them, a grid apart (n: where it stands, k: in the run).
  struct Place {
    int n, k;
  };
  const int runs = (items + run - 1) / run;
  auto find = [&](Place& at, Item& x, auto&& unseen) {
    while (at.n < runs) {
      const int i = at.n * run + at.k;
      if (++at.k == run) {
        at.k = 0;
        at.n += gridDim.x;
      }
      if (i >= items) continue;
      if (item_at(i, x) && x.rt0 < x.rt1) return true;
      unseen(x);
    }
    return false;
  };
  // y's row tile is x's, the only one of both: it stays where it is.
  auto same_rows = [](const Item& x, const Item& y) { return x.b == y.b && x.hk == y.hk && x.rt0 == y.rt0 && x.rt1 - x.rt0 == 1 && y.rt1 - y.rt0 == 1; };
  auto none = [](const Item&) {};
  Place n{static_cast<int>(blockIdx.x), 0};
  int q = 0;                                                  // row tiles loaded
  bool fresh = true;                                          // this item's are loaded for it
  Item x, y;                                                  // this item, the next one
  bool live = find(n, x, none);
  if (warp == 8) {
    // ------------------------------------------------------------------------------------------ TMA
    const int bpp = p.c.page / 32;
    int j = 0;                                                // running piece of codes
    auto load_codes = [&](const Item& x) {
      const int blk = 4 * x.t + lane, entry = blk / bpp;
      const bool held = lane < 4 && blk * 32 < x.n;
      const int page = held ? max(0, checked_page(p.c, __ldg(p.c.table + x.b * p.c.t_row + entry))) : 0;
      const int boxes = __popc(__ballot_sync(0xffffffffu, held));
      for (int c = 0; c < C::kChunks; ++c, ++j) {
        const int buf = j % C::kCodeBufs;
        if (j >= C::kCodeBufs && !(ok = wait_warp(bar(kwCodeFree + buf), (j / C::kCodeBufs - 1) & 1, abort_flag))) return;
        if (lane == 0) mbar_expect_tx(bars + kwCode + buf, boxes * 4096);
        __syncwarp();
        if (held) tma_load_4d(sbase + C::kSmemCode + buf * C::kTile + lane * 4096, &tk, bar(kwCode + buf), 128 * c, (blk - entry * bpp) * 32, x.hk, page);
      }
    };
    if (live) load_codes(x);
    while (live && ok) {
      const bool more = find(n, y, none);
      if (C::kChunks <= C::kCodeBufs && more) load_codes(y);  // (otherwise its second piece would wait for this item's end)
      for (int rt = x.rt0; rt < x.rt1 && fresh && ok; ++rt, ++q) {
        const int qb = q & (C::kQBufs - 1);
        if (q >= C::kQBufs && !(ok = wait_warp(bar(kwQFree + qb), ((q >> C::kQShift) - 1) & 1, abort_flag))) break;
        if (lane == 0) {
          const int tile = (x.b * p.c.Hk + x.hk) * row_tiles_max + rt;
          mbar_expect_tx(bars + kwQ + qb, C::kQBytes + 1024);
          for (int panel = 0; panel < C::kPanels; ++panel)
            tma_load_2d(smem + qb * C::kQBytes + panel * C::kTile, &tq, bars + kwQ + qb, 128 * panel, tile * 128);
          bulk_load_1d(smem + C::kSmemRows + qb * 1024, p.row_ml + static_cast<int64_t>(tile) * 128, 1024, bars + kwQ + qb);
        }
        __syncwarp();
      }
      if (C::kChunks > C::kCodeBufs && more && ok) load_codes(y);
      fresh = more && !same_rows(x, y);
      x = y;
      live = more;
    }
    if (!ok) {
      if (lane == 0) raise_abort(abort_flag, p.c.status, kStatusTimeoutProducer + kInCache);
      for (int k = 1; k <= C::kCodeBufs; ++k)                 // what is in flight lands before the shared memory goes
        if (j >= k) wait_or_abort(bar(kwCode + (j - k) % C::kCodeBufs), (j - k) / C::kCodeBufs & 1, abort_flag);
      for (int k = 1; k <= C::kQBufs; ++k)
        if (q >= k) wait_or_abort(bar(kwQ + ((q - k) & (C::kQBufs - 1))), ((q - k) >> C::kQShift) & 1, abort_flag);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------------------------------ MMA
    if (elect_one()) {
      const uint32_t k_lo = desc_lo(sbase + C::kSmemK), q_lo = desc_lo(sbase);
      int s = 0;                                              // running product
      for (int g = 0; live && ok; ++g) {
        const bool more = find(n, y, none), stays = more && same_rows(x, y);
        if (!(ok = wait_or_abort(bar(kwK), g & 1, abort_flag))) break;
        for (int rt = x.rt0; rt < x.rt1; ++rt, ++s) {
          if (fresh && !(ok = wait_or_abort(bar(kwQ + (q & (C::kQBufs - 1))), (q >> C::kQShift) & 1, abort_flag))) break;
          q += fresh;
          if (s >= 4 && !(ok = wait_or_abort(bar(kwSFree + (s & 3)), ((s >> 2) - 1) & 1, abort_flag))) break;
          tc_fence_after();
          const int qb = (q - 1) & (C::kQBufs - 1), rows = min(C::kRows, x.s.count * p.rep - rt * C::kRows);
          const uint32_t idesc = idesc_f8(128, (rows + 31) / 32 * 32, false, false);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k >> 2) * (C::kTile >> 4) + (k & 3) * 2;
            mma_h_ss(tmem + 128 * (s & 3), k_lo + off, q_lo + qb * (C::kQBytes >> 4) + off, idesc, k > 0);
          }
          if (!stays) tc_commit(bars + kwQFree + qb);
          tc_commit(bars + kwS + (s & 3));
        }
        fresh = !stays;
        x = y;
        live = more;
      }
      if (!ok) raise_abort(abort_flag, p.c.status, kStatusTimeoutMma + kInCache);
    }
  } else {
    // ------------------------------------------------------------------------------------------ codes, exponentials, sums
    const int half = warp >> 2, key = (warp & 3) * 32 + lane;           // token of a tile = TMEM lane
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    auto weight_at = [&](const Item& x) { return p.weights + x.b * p.w_sb + x.hk * p.w_sh + 128 * x.t + key; };
    auto zeros = [&](const Item& x) {
      if (half == 0 && !p.accumulate && 128 * x.t + key < p.W) *weight_at(x) = 0.f;
    };
    int j = 0;                                                // running piece of codes
    // An item's codes as its f16 tile, as in the main kernel: 16-byte pieces c of keys tid / 8, + 32, ...  All products of the last item have been seen.
    auto convert = [&]() {
#pragma unroll 1
      for (int part = 0; part < C::kChunks && ok; ++part, ++j) {
        const int buf = j % C::kCodeBufs;
        if (!(ok = wait_warp(bar(kwCode + buf), j / C::kCodeBufs & 1, abort_flag))) break;
        const int c = tid & 7, panel = c >> 2, cc = (c & 3) * 2;
        const uint32_t src = sbase + C::kSmemCode + buf * C::kTile, dst = sbase + C::kSmemK + (2 * part + panel) * C::kTile;
        float4 in[4];                                         // then the buffer is free for the next load
#pragma unroll
        for (int k = 0; k < 4; ++k) in[k] = lds_f4(src + ((tid >> 3) + 32 * k) * 128 + ((c ^ ((tid >> 3) & 7)) << 4));
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + kwCodeFree + buf);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = (tid >> 3) + 32 * k;
          const float4 w4 = in[k];
          const uint32_t w[4] = {__float_as_uint(w4.x), __float_as_uint(w4.y), __float_as_uint(w4.z), __float_as_uint(w4.w)};
          uint32_t h[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            h[2 * e] = e4m3_lo_f16x2(w[e]);
            h[2 * e + 1] = e4m3_hi_f16x2(w[e]);
          }
          const int flip = panel;                             // which half first: eight lanes' stores on different banks
          sts_u4(dst + row * 128 + (((cc + flip) ^ (row & 7)) << 4), flip ? h[4] : h[0], flip ? h[5] : h[1], flip ? h[6] : h[2], flip ? h[7] : h[3]);
          sts_u4(dst + row * 128 + (((cc + 1 - flip) ^ (row & 7)) << 4), flip ? h[0] : h[4], flip ? h[1] : h[5], flip ? h[2] : h[6], flip ? h[3] : h[7]);
        }
        if (part < C::kChunks - 1) continue;
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + kwK);
      }
    };
    // Of this thread's token: its page, and the scale of its block.  Each is asked for long before it is looked at, page an item ahead.
    auto page_of = [&](const Item& x) { return __ldg(p.c.table + x.b * p.c.t_row + min(128 * x.t + key, x.n - 1) / p.c.page); };
    auto scale_of = [&](const Item& x, int page) {
      const int tok = min(128 * x.t + key, x.n - 1);
      return __ldg(p.c.ks + max(0, checked_page(p.c, page)) * p.c.s_page + x.hk * p.c.s_head + tok % p.c.page / 32);
    };
    // of the last item: this half's sum, where it goes, whether the token exists
    float mine = 0.f;
    float* at = nullptr;
    bool held = false;
    int last = -1;
    auto finish = [&](int g) -> bool {
      if (!wait_warp(bar(kwSums + (g & 1)), (g >> 1) & 1, abort_flag)) return false;
      mine += sums[128 * (g & 1) + key];
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + kwSumsFree + (g & 1));
      if (at != nullptr) *at = !held ? 0.f : p.accumulate ? *at + mine : mine;
      return true;
    };
    n = Place{static_cast<int>(blockIdx.x), 0};
    live = find(n, x, zeros);
    int page = live ? page_of(x) : 0;
    int s = 0;                                                // running product
    for (int g = 0; live && ok; ++g) {
      const float ks = scale_of(x, page);
      convert();
      if (!ok) break;
      // while the first product is under way
      const bool more = find(n, y, zeros), stays = more && same_rows(x, y);
      if (more) page = page_of(y);
      const int tok = 128 * x.t + key;
      float total = 0.f;
      for (int rt = x.rt0; rt < x.rt1; ++rt, ++s) {
        q += fresh;
        const int qb = (q - 1) & (C::kQBufs - 1);
        // the products; and the rows' constants, seen by this warp itself
        if (!(ok = wait_warp(bar(kwS + (s & 3)), (s >> 2) & 1, abort_flag) && wait_warp(bar(kwQ + qb), ((q - 1) >> C::kQShift) & 1, abort_flag))) break;
        tc_fence_after();
        const int parts = (min(C::kRows, x.s.count * p.rep - rt * C::kRows) + 31) / 32;    // of 32 rows
        const int from_row = first_row(p, x.s, tok) - rt * C::kRows;      // of the row tile, the first that sees this token
        const bool cut = __any_sync(0xffffffffu, from_row > 0);
        const uint32_t from = tmem + lanes + 128 * (s & 3), rows = sbase + C::kSmemRows + qb * 1024;
        uint32_t s_buf[2][32];
        auto part_sum = [&](int c, const uint32_t (&v)[32], auto cut_tag) {
          constexpr bool kCut = decltype(cut_tag)::value;     // some token of the warp is not seen by all rows
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int e8 = 0; e8 < 16; e8 += 8) {
            float4 fc[8];                                     // factors and log2 sums of two rows each, asked for together
#pragma unroll
            for (int e = 0; e < 8; ++e) fc[e] = lds_f4(rows + (32 * c + 2 * (e8 + e)) * 8);
            float2 z[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              z[e] = fma2(mul2(make_float2(__uint_as_float(v[2 * (e8 + e)]), __uint_as_float(v[2 * (e8 + e) + 1])), make_float2(fc[e].x, fc[e].z)), splat2(ks),
                          make_float2(-fc[e].y, -fc[e].w));
              if (kCut) {
                if (32 * c + 2 * (e8 + e) < from_row) z[e].x = -CUDART_INF_F;
                if (32 * c + 2 * (e8 + e) + 1 < from_row) z[e].y = -CUDART_INF_F;
              }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = ex2_2(z[e]);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = add2(sum, z[e]);
          }
          // (no sum of probabilities is above their number; logits so large that their last bit counts powers of two would make it one)
          const float both = sum.x + sum.y;
          total += both > 32.f ? 32.f : both;
        };
        auto parts_from = [&](int c, int step, auto cut_tag) {
          if (c < parts) tmem_ld32(from + 32 * c, s_buf[0]);
#pragma unroll 1
          for (; c < parts; c += 2 * step) {
            tmem_wait_ld();
            if (c + step < parts) tmem_ld32(from + 32 * (c + step), s_buf[1]);
            part_sum(c, s_buf[0], cut_tag);
            if (c + step >= parts) break;
            tmem_wait_ld();
            if (c + 2 * step < parts) tmem_ld32(from + 32 * (c + 2 * step), s_buf[0]);
            part_sum(c + step, s_buf[1], cut_tag);
          }
        };
        // the two groups of warps: halves of an only row tile, or every second one
        const bool only = x.rt1 - x.rt0 == 1;
        const int first = only ? half : (rt - x.rt0 & 1) == half ? 0 : parts, step = only ? 2 : 1;
        if (cut) parts_from(first, step, std::true_type{});
        else parts_from(first, step, std::false_type{});
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bars + kwSFree + (s & 3));
          if (!stays) mbar_arrive(bars + kwQFree + qb);
        }
      }
      if (!ok) break;
      // The two halves' sums: the second leaves its own, the first picks it up an item later.
      if (half == 1) {
        if (g >= 2 && !(ok = wait_warp(bar(kwSumsFree + (g & 1)), ((g >> 1) - 1) & 1, abort_flag))) break;
        sums[128 * (g & 1) + key] = total;
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + kwSums + (g & 1));
      } else {
        if (g > 0 && !(ok = finish(g - 1))) break;
        mine = total;
        at = tok < x.n || (!p.accumulate && tok < p.W) ? weight_at(x) : nullptr;
        held = tok < x.n;
      }
      last = g;
      fresh = !stays;
      x = y;
      live = more;
    }
    if (ok && half == 0 && last >= 0) ok = finish(last);
    if (!ok && lane == 0) raise_abort(abort_flag, p.c.status, kStatusTimeoutCompute + kInCache);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

int cache_chunk_rows(int D) { return D == 128 ? ChunkCfg<128>::kRows : ChunkCfg<256>::kRows; }
int64_t cache_chunk_start_bytes() { return (sizeof(ChunkStart) + 7) / 8 * 8; }
int64_t cache_chunk_query_rows(int B, int Hk, int R) { return static_cast<int64_t>(B) * Hk * ((R + 127) / 128 * 128); }

template <int D>
static cudaError_t launch_chunk(const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tq, const CacheAttnParams& p, cudaStream_t stream) {
  using C = ChunkCfg<D>;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    cudaFuncAttributes attr;
    cudaError_t e = cudaFuncGetAttributes(&attr, cache_chunk_kernel<D>);
    if (e != cudaSuccess) return e;
    if (attr.numRegs * C::kThreads < 256 * (C::kRegsSoftmax + C::kRegsOther)) return cudaErrorLaunchOutOfResources;
    e = cudaFuncSetAttribute(cache_chunk_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(cache_chunk_weights_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkWeightsCfg<D>::kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const unsigned row_tiles = static_cast<unsigned>(p.c.B) * p.c.Hk * ((p.Nq * p.rep + 127) / 128);
  count_launch();
  cudaError_t e = launch_chained(cache_chunk_queries_kernel<D>, dim3(row_tiles * (D / 16) + 1), 256, 0, stream, p);      // 2048 / D rows a CTA
  if (e != cudaSuccess) return e;
  count_launch();
  e = launch_chained(cache_chunk_kernel<D>, dim3(p.grid), C::kThreads, C::kSmem, stream, tk, tv, tq, p);
  if (e != cudaSuccess) return e;
  count_launch();
  const int groups = (p.Nq * p.rep + 3) / 4;
  e = launch_chained(cache_chunk_join_kernel<D>, dim3(static_cast<unsigned>(p.c.B) * p.c.Hk * groups), 128, 0, stream, p);
  if (e != cudaSuccess || p.weights == nullptr) return e;
  const int tiles_of_row = (p.W + 127) / 128;                 // what lies beyond the length too: its weights are zeros
  const int64_t items = static_cast<int64_t>(p.c.B) * p.c.Hk * tiles_of_row;
  // One row tile stays where it is for a run of four items; several pass by in any case, and items one by one divide more evenly.
  const int run = p.Nq * p.rep <= 128 && items >= 16ll * sm_count() ? 4 : 1;
  const int64_t n_runs = (items + run - 1) / run;
  count_launch();
  return launch_chained(cache_chunk_weights_kernel<D>, dim3(static_cast<unsigned>(n_runs < sm_count() ? n_runs : sm_count())), ChunkWeightsCfg<D>::kThreads,
                        ChunkWeightsCfg<D>::kSmem, stream, tk, tq, p, tiles_of_row, run);
}

cudaError_t launch_cache_chunk(int D, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tq, const CacheAttnParams& p, cudaStream_t stream) {
  return D == 128 ? launch_chunk<128>(tk, tv, tq, p, stream) : launch_chunk<256>(tk, tv, tq, p, stream);
}

}  // namespace dm
