// Attention of many new queries over the 8-bit cache (chunks of a prompt): the same result as dm_cache_attn.cu, on tcgen05.
//
//   S = Q K^T and O += P V as f16 tcgen05 chains with fp32 accumulators in TMEM.  The codes are exact in f16, q is brought to f16 with a power
//   of two per row, P is f16 with the row's reference maximum at 2^15 (11 bits, never closer than 2^-40 of the row's largest); K's
//   block scales go into the factors of the logits, V's into the exponent of P relative to the largest the row tile has met.
//
// A unit is (sequence, kv head, 256 rows); rows are (new token, head of the group).  The key tiles of 128 tokens of all units are one flat
// range, divided evenly over one CTA per SM (as the warps' blocks are in dm_cache_sched.cuh); pieces of cut units are joined by a second kernel.
// Warps 0-3 and 4-7: softmax of the unit's two row tiles (thread = row = TMEM lane).  Warps 8-11: codes -> f16 operand tiles in shared
// memory, shared by both row tiles.  Warp 12: TMA of the code tiles from the pages.  Warp 13: MMA.  The two row tiles take turns: while
// one is in its softmax the tensor cores work for the other.
//
// TMEM: S0 0-127, S1 128-255 (P of a tile over the first 64 columns of its S), O0 256-383, O1 384-511.
// The maximum moves only when a row exceeds its reference by a factor of two (P then still fits f16's range), so O is seldom rescaled.
#include "dm_cache.cuh"
#include "dm_kernels.h"

namespace dm {

namespace {

constexpr int kChunkCost = 2;               // key tiles that a unit's queries and output are worth

struct ChunkCfg {
  static constexpr int D = 128;
  static constexpr int kThreads = 512;                        // four warpgroups, the last two of its warps idle
  static constexpr int kRegsSoftmax = 168, kRegsOther = 88;
  static_assert(256 * kRegsSoftmax + 256 * kRegsOther <= kThreads * 128, "a split above the launch's own registers would wait for ever");
  static constexpr int kRows = 256;
  static constexpr int kTile = 128 * 128;                     // a code tile; also a 64-column f16 panel of 128 rows
  static constexpr int kSmemQ = 0;                            // two row tiles x two panels
  static constexpr int kSmemK = 4 * kTile;                    // two buffers x two panels
  static constexpr int kSmemV = kSmemK + 4 * kTile;
  static constexpr int kSmemCode = kSmemV + 4 * kTile;        // K codes, V codes
  static constexpr int kSmemBars = kSmemCode + 2 * kTile;
  static constexpr int kSmemScales = kSmemBars + 256;         // 8 tiles x (4 K scales, 4 V scales)
  static constexpr int kSmemCum = kSmemScales + 8 * 32;
  static constexpr int kSmem = kSmemCum + 136 * 4 + 64 + 1024;
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
  s.units = (s.count * p.rep + ChunkCfg::kRows - 1) / ChunkCfg::kRows;
  return s;
}
// Keys that row r of the sequence sees.
__device__ __forceinline__ int row_limit(const CacheAttnParams& p, const ChunkSeq& s, int r) {
  const int i = r / p.rep;
  return i >= s.count ? 0 : p.causal ? max(0, s.n - s.count + i + 1) : s.n;
}
__device__ __forceinline__ int unit_tiles(const CacheAttnParams& p, const ChunkSeq& s, int rt) {
  return (row_limit(p, s, min(s.count * p.rep, (rt + 1) * ChunkCfg::kRows) - 1) + 127) / 128;
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
__device__ __forceinline__ int chunk_range(const CacheAttnParams& p, int* cum, int tid) {
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
  return chunk;
}
__device__ __forceinline__ int share_start(int cta, int grid, int total) { return static_cast<int>(static_cast<int64_t>(cta) * total / grid); }
__device__ __forceinline__ int share_owner(int f, int grid, int total) {
  return static_cast<int>(((static_cast<int64_t>(f) + 1) * grid - 1) / total);
}

// A CTA's piece of a unit: key tiles t0 ... t1 - 1.
struct ChunkPiece {
  int b, hk, rt;
  ChunkSeq s;
  int tiles, t0, t1, f1;
  __device__ __forceinline__ int row_tiles(const CacheAttnParams& p) const { return s.count * p.rep - rt * ChunkCfg::kRows > 128 ? 2 : 1; }
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
  kCodeFull = 0, kCodeEmpty = 2,            // K codes, V codes
  kKFull = 4, kKEmpty = 6, kVFull = 8, kVEmpty = 10,          // by parity of the running tile
  kQFull = 12, kSFull = 14, kPFull = 16, kPvDone = 18,        // by row tile
  kScales = 20,                             // of running tile g: entry g % 8 (the loads are at most four tiles ahead of the softmax)
  kBars = 28,
};

// ------------------------------------------------------------------------------------------------ main kernel
__global__ void __launch_bounds__(ChunkCfg::kThreads, 1)
cache_chunk_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const CacheAttnParams p) {
  using C = ChunkCfg;
  constexpr int D = C::D;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023) & ~1023u) - raw);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kSmemBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kBars + 1);
  float* scales = reinterpret_cast<float*>(smem + C::kSmemScales);
  int* cum = reinterpret_cast<int*>(smem + C::kSmemCum);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + kCodeFull + i, 1);
      mbar_init(bars + kCodeEmpty + i, 4);
      mbar_init(bars + kKFull + i, 4);
      mbar_init(bars + kKEmpty + i, 1);
      mbar_init(bars + kVFull + i, 4);
      mbar_init(bars + kVEmpty + i, 1);
      mbar_init(bars + kQFull + i, 4);
      mbar_init(bars + kSFull + i, 1);
      mbar_init(bars + kPFull + i, 4);
      mbar_init(bars + kPvDone + i, 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(bars + kScales + i, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (warp == 13) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  grid_dep_wait();
  const int chunk = (p.c.B + 127) / 128;
  if (tid < 128) chunk_range(p, cum, tid);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int total = cum[128];
  const int f0 = share_start(blockIdx.x, p.grid, total), f_end = share_start(blockIdx.x + 1, p.grid, total);
  bool ok = true;
  auto bar = [&](int i) { return smem_u32(bars + i); };

  if (f0 < f_end) {
    ChunkPiece x = first_chunk(p, cum, chunk, f0, f_end);
    if (warp >= 12) {
      reg_dec<C::kRegsOther>();
    }
    if (warp == 12) {
      // ---------------------------------------------------------------------------------------- TMA: code tiles and their scales
      int g = 0;                                              // running tile
      const int bpp = p.c.page / 32;
      do {
        for (int t = x.t0; t < x.t1 && ok; ++t, ++g) {
          // lane i < 4: block 4 t + i of the sequence, its page and scales
          const int blk = 4 * t + lane;
          const bool held = lane < 4 && blk * 32 < x.s.n;
          int page = 0, sub = 0;
          if (held) {
            const int entry = blk / bpp;
            sub = blk - entry * bpp;
            page = max(0, checked_page(p.c, __ldg(p.c.table + x.b * p.c.t_row + entry)));
          }
          const int boxes = __popc(__ballot_sync(0xffffffffu, held));
          for (int kv = 0; kv < 2; ++kv) {
            if (g > 0) ok = ok && wait_warp(bar(kCodeEmpty + kv), (g - 1) & 1, abort_flag);
            if (!ok) break;
            if (lane == 0) mbar_expect_tx(bars + kCodeFull + kv, boxes * 4096);
            __syncwarp();
            if (held) tma_load_4d(sbase + C::kSmemCode + kv * C::kTile + lane * 4096, kv ? &tv : &tk, bar(kCodeFull + kv), 0, sub * 32, x.hk, page);
          }
          if (!ok) break;
          if (lane < 4) {
            const int64_t at = page * p.c.s_page + x.hk * p.c.s_head + sub;
            scales[(g & 7) * 8 + lane] = held ? __ldg(p.c.ks + at) : 0.f;
            scales[(g & 7) * 8 + 4 + lane] = held ? __ldg(p.c.vs + at) : 0.f;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + kScales + (g & 7));
        }
      } while (ok && next_chunk(p, x, f_end));
      if (!ok) {
        if (lane == 0) raise_abort(abort_flag, p.c.status, kStatusTimeoutProducer + kInCache);
        // what is in flight lands before the shared memory goes
        for (int kv = 0; kv < 2; ++kv)
          if (g > 0) wait_or_abort(bar(kCodeFull + kv), (g - 1) & 1, abort_flag);
      }
    } else if (warp == 13) {
      // ---------------------------------------------------------------------------------------- MMA
      if (elect_one()) {
        constexpr uint32_t kIdescS = idesc_f8(128, 128, false, false), kIdescO = idesc_f8(128, 128, false, true);
        const uint32_t q_lo = desc_lo(sbase + C::kSmemQ), k_lo = desc_lo(sbase + C::kSmemK);
        // V's panels of 64 columns lie kTile apart: the leading offset of an operand wider than 128 bytes
        const uint32_t v_lo = (((sbase + C::kSmemV) & 0x3FFFFu) >> 4) | (static_cast<uint32_t>(C::kTile >> 4) << 16);
        int g = 0, tiles[2] = {0, 0}, units[2] = {0, 0};      // running tile; tiles and units of each row tile
        auto issue_s = [&](int r, int gi, bool last) {
          const uint32_t a = q_lo + r * (2 * C::kTile >> 4), b = k_lo + (gi & 1) * (2 * C::kTile >> 4);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t off = (k >> 2) * (C::kTile >> 4) + (k & 3) * 2;
            mma_h_ss(tmem + 128 * r, a + off, b + off, kIdescS, k > 0);
          }
          if (last) tc_commit(bars + kKEmpty + (gi & 1));
          tc_commit(bars + kSFull + r);
        };
        do {
          if (x.t0 >= x.t1) continue;
          const int nr = x.row_tiles(p);
          ok = wait_or_abort(bar(kKFull + (g & 1)), (g >> 1) & 1, abort_flag);
          for (int r = 0; r < nr && ok; ++r) {
            if (!(ok = wait_or_abort(bar(kQFull + r), units[r]++ & 1, abort_flag))) break;
            tc_fence_after();
            issue_s(r, g, r == nr - 1);
          }
          for (int t = x.t0; t < x.t1 && ok; ++t, ++g) {
            const uint32_t v = v_lo + (g & 1) * (2 * C::kTile >> 4);
            for (int r = 0; r < nr; ++r) {
              if (!(ok = wait_or_abort(bar(kPFull + r), tiles[r]++ & 1, abort_flag))) break;
              if (r == 0 && !(ok = wait_or_abort(bar(kVFull + (g & 1)), (g >> 1) & 1, abort_flag))) break;
              tc_fence_after();
#pragma unroll
              for (int k = 0; k < 8; ++k)                     // 16 keys: 8 columns of P, 16 rows of V
                mma_h_ts(tmem + 256 + 128 * r, tmem + 128 * r + 8 * k, v + k * (2048 >> 4), kIdescO, t > x.t0 || k > 0);
              if (r == nr - 1) tc_commit(bars + kVEmpty + (g & 1));
              tc_commit(bars + kPvDone + r);
              if (t + 1 < x.t1) {
                if (r == 0 && !(ok = wait_or_abort(bar(kKFull + ((g + 1) & 1)), ((g + 1) >> 1) & 1, abort_flag))) break;
                tc_fence_after();
                issue_s(r, g + 1, r == nr - 1);
              }
            }
          }
        } while (ok && next_chunk(p, x, f_end));
        if (!ok) raise_abort(abort_flag, p.c.status, kStatusTimeoutMma + kInCache);
      }
    } else if (warp >= 8 && warp < 12) {
      reg_dec<C::kRegsOther>();
      // ---------------------------------------------------------------------------------------- codes -> f16 operand tiles
      const int ct = tid - 256, c = ct & 7;                   // a thread takes 16-byte pieces c of keys ct / 8, + 16, ...
      // a piece's two halves of eight elements: which goes first is chosen so that the stores of eight lanes fall on different banks
      const int panel = c >> 2, flip = panel;
      int g = 0;
      do {
        for (int t = x.t0; t < x.t1 && ok; ++t, ++g) {
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv) {
            ok = wait_warp(bar(kCodeFull + kv), g & 1, abort_flag);
            if (ok && g >= 2) ok = wait_warp(bar((kv ? kVEmpty : kKEmpty) + (g & 1)), ((g >> 1) - 1) & 1, abort_flag);
            if (!ok) break;
            const uint32_t src = sbase + C::kSmemCode + kv * C::kTile;
            const uint32_t dst = sbase + (kv ? C::kSmemV : C::kSmemK) + (g & 1) * 2 * C::kTile + panel * C::kTile;
            const int held = kv ? x.s.n - 128 * t : 128;      // V's slots beyond the length hold anything, NaN codes too: zeros
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int key = (ct >> 3) + 16 * i;
              const float4 w4 = lds_f4(src + key * 128 + ((c ^ (key & 7)) << 4));
              uint32_t w[4] = {__float_as_uint(w4.x), __float_as_uint(w4.y), __float_as_uint(w4.z), __float_as_uint(w4.w)};
              if (key >= held) w[0] = w[1] = w[2] = w[3] = 0;
              uint32_t h[8];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                h[2 * j] = e4m3_lo_f16x2(w[j]);
                h[2 * j + 1] = e4m3_hi_f16x2(w[j]);
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
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(bars + (kv ? kVFull : kKFull) + (g & 1));
              mbar_arrive(bars + kCodeEmpty + kv);
            }
          }
        }
      } while (ok && next_chunk(p, x, f_end));
      if (!ok && lane == 0) raise_abort(abort_flag, p.c.status, kStatusTimeoutCompute + kInCache);
    } else if (warp < 8) {
      reg_inc<C::kRegsSoftmax>();
      // ---------------------------------------------------------------------------------------- softmax and output
      const int r = warp >> 2, in_tile = (warp & 3) * 32 + lane;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t t_s = tmem + lanes + 128 * r, t_o = tmem + lanes + 256 + 128 * r;
      const uint32_t q_row = sbase + C::kSmemQ + r * 2 * C::kTile + in_tile * 128;
      int g = 0, mine = 0;                                    // running tile, those of this row tile
      int slot = 2 * blockIdx.x;
      do {
        if (x.t0 >= x.t1) continue;
        if (r >= x.row_tiles(p)) {
          g += x.t1 - x.t0;
          slot = 2 * blockIdx.x + 1;
          continue;
        }
        const int row = x.rt * C::kRows + r * 128 + in_tile, limit = row_limit(p, x.s, row);
        const int i_tok = row / p.rep, head = x.hk * p.rep + row - i_tok * p.rep;
        float f;                                              // factor of the row's logits, K's scale aside
        {
          const __nv_bfloat16* src = p.q + x.b * p.q_sb + i_tok * p.q_sn + head * p.q_sh;
          uint4 w[16];
          float amax = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            w[i] = row < x.s.count * p.rep ? __ldg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0, 0, 0, 0);
            const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(v[j] << 16)), fabsf(__uint_as_float(v[j] & 0xFFFF0000u))));
          }
          const uint32_t eb = min(254u, max(14u, __float_as_uint(amax) >> 23));
          const float up = sb_to_scale(267u - eb);            // largest element to [2^13, 2^14)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) h[j] = pack_f16x2(__uint_as_float(v[j] << 16) * up, __uint_as_float(v[j] & 0xFFFF0000u) * up);
            sts_u4(q_row + (i >> 3) * C::kTile + (((i & 7) ^ (in_tile & 7)) << 4), h[0], h[1], h[2], h[3]);
          }
          f = sb_to_scale(eb - 13u) * p.scale * kLog2e;
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + kQFull + r);

        float m = -CUDART_INF_F, l = 0.f;
        int vexp = -1000;
        for (int t = x.t0; t < x.t1; ++t, ++g, ++mine) {
          ok = wait_warp(bar(kScales + (g & 7)), (g >> 3) & 1, abort_flag) && wait_warp(bar(kSFull + r), mine & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const float4 ks = lds_f4(sbase + C::kSmemScales + (g & 7) * 32), vs = lds_f4(sbase + C::kSmemScales + (g & 7) * 32 + 16);
          const float fc[4] = {f * ks.x, f * ks.y, f * ks.z, f * ks.w};
          const int ev[4] = {static_cast<int>(scale_to_sb(vs.x)) - 127, static_cast<int>(scale_to_sb(vs.y)) - 127, static_cast<int>(scale_to_sb(vs.z)) - 127,
                             static_cast<int>(scale_to_sb(vs.w)) - 127};
          const int seen = limit - 128 * t;                   // keys of the tile that the row sees
          const bool cut = __any_sync(0xffffffffu, seen < 128);
          float top = -CUDART_INF_F;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t s[32];
            tmem_ld32(t_s + 32 * c, s);
            tmem_wait_ld();
            if (cut) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (32 * c + e >= seen) s[e] = 0xff800000u;
            }
            float2 s2[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) s2[e] = make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
            const float top_c = max32(s2);
            top = fmaxf(top, top_c == -CUDART_INF_F ? top_c : top_c * fc[c]);
          }
          // the reference moves where the row exceeds it by a factor of two: P stays below 2^16
          const float m_new = top > m + 0.999f ? top : m;
          const int v_new = max(max(vexp, max(ev[0], ev[1])), max(ev[2], ev[3]));
          const float mu = m_new == -CUDART_INF_F ? 0.f : m_new;
          const float keep = ex2_approx(m - mu);
          if (__any_sync(0xffffffffu, m_new != m || v_new != vexp)) {
            if (t > x.t0) {
              ok = wait_warp(bar(kPvDone + r), (mine - 1) & 1, abort_flag);
              if (!ok) break;
              tc_fence_after();
              const float a = keep * exp2f(static_cast<float>(vexp - v_new));
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                tmem_ld32(t_o + 32 * c, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
                tmem_st32(t_o + 32 * c, o);
              }
              tmem_wait_st();
            }
            l *= keep;
            m = m_new;
            vexp = v_new;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t s[32];
            tmem_ld32(t_s + 32 * c, s);
            // P comes out as 2^off exp(s - m); where V's scale is 2^-60 of another's the product vanishes anyway, but the sum must not
            const int off = max(15 + ev[c] - vexp, -45);
            const float2 f2 = splat2(fc[c]), sub = splat2(static_cast<float>(off) - mu);
            float2 sum = make_float2(0.f, 0.f);
            uint32_t h[16];
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float2 y = fma2(make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), f2, sub);
              if (cut) {
                if (32 * c + 2 * e >= seen) y.x = -CUDART_INF_F;
                if (32 * c + 2 * e + 1 >= seen) y.y = -CUDART_INF_F;
              }
              y = ex2_2(y);
              sum = add2(sum, y);
              h[e] = pack_f16x2(y.x, y.y);
            }
            l = fmaf(sum.x + sum.y, __uint_as_float(static_cast<uint32_t>(127 - off) << 23), l);
            tmem_st16(t_s + 16 * c, h);
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + kPFull + r);
        }
        if (!ok) break;
        ok = wait_warp(bar(kPvDone + r), (mine - 1) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const bool whole = x.t0 == 0 && x.t1 == x.tiles;
        const float unit_exp = exp2f(static_cast<float>(vexp - 15));
        const float scale = whole ? unit_exp / l : unit_exp;
        __nv_bfloat16* o16 = p.o + ((static_cast<int64_t>(x.b) * p.Nq + i_tok) * p.H + head) * D;
        const int64_t part = static_cast<int64_t>(slot) * C::kRows + r * 128 + in_tile;
        float* o32 = p.part_o + part * D;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(t_o + 32 * c, o);
          tmem_wait_ld();
          float v[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(o[e]) * scale;
          if (whole) {
            if (limit > 0) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const __nv_bfloat162 b2 = __floats2bfloat162_rn(v[8 * e + 2 * j], v[8 * e + 2 * j + 1]);
                  w[j] = *reinterpret_cast<const uint32_t*>(&b2);
                }
                *reinterpret_cast<uint4*>(o16 + 32 * c + 8 * e) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            }
          } else if (limit > 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) *reinterpret_cast<float4*>(o32 + 32 * c + 4 * e) = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
          }
        }
        if (limit > 0) {
          if (whole) {
            p.lse[(static_cast<int64_t>(x.b) * p.H + head) * p.Nq + i_tok] = (m + log2f(l)) * kLn2;
            if (p.row_ml != nullptr) p.row_ml[(static_cast<int64_t>(x.b) * p.c.Hk + x.hk) * p.Nq * p.rep + row] = make_float2(m, 1.f / l);
          } else {
            p.part_ml[part] = make_float2(m, l);
          }
        }
        tc_fence_before();
        slot = 2 * blockIdx.x + 1;
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
// Rows of units that were cut, and rows that see nothing: one CTA per 32 rows of a (sequence, head), a warp a row at a time.
__global__ void __launch_bounds__(128) cache_chunk_join_kernel(const CacheAttnParams p) {
  constexpr int D = ChunkCfg::D;
  __shared__ int cum[136];
  grid_dep_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int R = p.Nq * p.rep, groups = (R + 31) / 32;
  const int r0 = static_cast<int>(blockIdx.x % groups) * 32, hk = static_cast<int>(blockIdx.x / groups % p.c.Hk), b = static_cast<int>(blockIdx.x / groups / p.c.Hk);
  const int chunk = chunk_range(p, cum, tid);
  __syncthreads();
  const int total = cum[128], grid = p.grid;
  const ChunkSeq s = chunk_seq(p, b);
  int c0 = 0, c1 = 0, f0 = 0;
  if (r0 < s.count * p.rep) {
    f0 = cum[b / chunk];
    for (int k = b / chunk * chunk; k < b; ++k) f0 += head_steps(p, k) * p.c.Hk;
    f0 += hk * head_steps(p, b);
    const int rt = r0 / ChunkCfg::kRows;
    for (int k = 0; k < rt; ++k) f0 += unit_steps(p, s, k);
    const int steps = unit_steps(p, s, rt);
    if (steps > 0) {
      c0 = share_owner(f0 + kChunkCost, grid, total);
      c1 = share_owner(f0 + steps - 1, grid, total);
    }
  }
  for (int r = r0 + warp; r < min(R, r0 + 32); r += 4) {
    const int i_tok = r / p.rep, head = hk * p.rep + r - i_tok * p.rep;
    __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(p.o + ((static_cast<int64_t>(b) * p.Nq + i_tok) * p.H + head) * D) + 2 * lane;
    float* lse = p.lse + (static_cast<int64_t>(b) * p.H + head) * p.Nq + i_tok;
    float2* row_ml = p.row_ml == nullptr ? nullptr : p.row_ml + (static_cast<int64_t>(b) * p.c.Hk + hk) * R + r;
    if (row_limit(p, s, r) == 0) {
      o[0] = o[1] = __floats2bfloat162_rn(0.f, 0.f);
      if (lane == 0) {
        *lse = -CUDART_INF_F;
        if (row_ml != nullptr) *row_ml = make_float2(0.f, 0.f);
      }
      continue;
    }
    if (c0 == c1) continue;                                   // whole: written by its CTA
    float top = -CUDART_INF_F, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = c0; c <= c1; ++c) {
      const int start = share_start(c, grid, total);
      if (start == share_start(c + 1, grid, total)) continue;
      const int64_t at = static_cast<int64_t>(2 * c + (start >= f0 ? 0 : 1)) * ChunkCfg::kRows + (r & (ChunkCfg::kRows - 1));
      const float2 ml = p.part_ml[at];
      if (ml.x == -CUDART_INF_F) continue;
      const float4 v = reinterpret_cast<const float4*>(p.part_o + at * D)[lane];
      const float top_new = fmaxf(top, ml.x), a = exp2f(top - top_new), w = exp2f(ml.x - top_new);
      sum = sum * a + ml.y * w;
      acc = make_float4(acc.x * a + v.x * w, acc.y * a + v.y * w, acc.z * a + v.z * w, acc.w * a + v.w * w);
      top = top_new;
    }
    const float inv = 1.f / sum;
    o[0] = __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
    o[1] = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
    if (lane == 0) {
      *lse = (top + log2f(sum)) * kLn2;
      if (row_ml != nullptr) *row_ml = make_float2(top, inv);
    }
  }
}

}  // namespace

int cache_chunk_rows() { return ChunkCfg::kRows; }

cudaError_t launch_cache_chunk(const CUtensorMap& tk, const CUtensorMap& tv, const CacheAttnParams& p, cudaStream_t stream) {
  using C = ChunkCfg;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    cudaFuncAttributes attr;
    cudaError_t e = cudaFuncGetAttributes(&attr, cache_chunk_kernel);
    if (e != cudaSuccess) return e;
    if (attr.numRegs * C::kThreads < 256 * (C::kRegsSoftmax + C::kRegsOther)) return cudaErrorLaunchOutOfResources;
    e = cudaFuncSetAttribute(cache_chunk_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  count_launch();
  const cudaError_t e = launch_chained(cache_chunk_kernel, dim3(p.grid), C::kThreads, C::kSmem, stream, tk, tv, p);
  if (e != cudaSuccess) return e;
  count_launch();
  const int groups = (p.Nq * p.rep + 31) / 32;
  return launch_chained(cache_chunk_join_kernel, dim3(static_cast<unsigned>(p.c.B) * p.c.Hk * groups), 128, 0, stream, p);
}

}  // namespace dm
