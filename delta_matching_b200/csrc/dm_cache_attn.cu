// Attention of few new queries over the 8-bit cache.
//
//   s_rj = scale q_r . (ks code_j);  o_r = sum_j exp(s_rj - m_r) vs code_j / sum_j exp(s_rj - m_r)  over the keys j that row r sees
//
// Rows are (new token, head of the kv head's group): they share one pass over the codes, which is what the kernel is bound by.  K^T Q is
// made with the keys as M (16) and the rows as N (8 a tile) of mma.m16n8k16, so that a group of up to 8 rows wastes nothing and the
// transposed product V^T P needs P in the layout that it comes in, up to one movmatrix.  The codes are exact in f16; q is brought to f16 with
// a power of two per row (bf16's 8 bits fit f16's 11), p = exp2(x) is rounded to f16's 11 bits; sums, maxima and accumulators are fp32.  The
// power-of-two scale of V's block goes into the exponent of p, relative to the largest product of a probability and a scale that the row has met
// (blocks that it does not see, or gives no weight, cost it no bits), and the scale of K's block into the factor of the logits, so no code is
// ever multiplied by a scale.
//
// Every warp works for itself: it takes an even share of the blocks of 32 tokens of the whole call (dm_cache_sched.cuh), one after the other, with
// its own maximum, sum and accumulator, and fills its own ring of TMA boxes (32 rows x 128 bytes, 128-byte swizzle, straight from the pages),
// K and V of a block in turn, each refilled as soon as it has been read.  Units that one warp holds whole are written at once; the pieces
// of the others are joined by a second kernel.
//
// Bound by its bytes where there are many blocks a warp: one new token, H=32 Hk=8, B=64 with 17 - 8191 tokens 101 us = 5.4 TB/s of codes and
// scales (the card copies at 6.5); H=64 Hk=8, one sequence of 131071 tokens 57 us = 4.7 TB/s; head_dim 256, H=16 Hk=16, B=8 with 4001 - 8192 73 us
// = 5.5 TB/s.  Small calls are bound by the chain from the lengths through the block table to the first codes (about 6700 cycles), 2300 cycles a
// block and the join (3000 - 6000): B=4 with 3601 - 4096 15.4 us, one sequence of 255 tokens 7.1 us.
#include <cooperative_groups.h>
#include "dm_cache_sched.cuh"
#include "dm_kernels.h"

namespace dm {

namespace {

namespace cg = cooperative_groups;

constexpr int kMaxCluster = 8;

template <int D, int NT>
struct AttnCfg {
  static constexpr int kWarps = 4;
  static constexpr int kRows = 8 * NT;
  static constexpr int kSlotBytes = 32 * D;                   // K or V of a block
  static constexpr int kCtasPerSm = D == 128 && NT == 1 ? 3 : 2;
  static constexpr int kSlots = D == 128 ? (NT == 2 ? 6 : 4) : 3;
  static constexpr int kRing = kWarps * kSlots * kSlotBytes;
  static constexpr int kStats = kWarps * kRows * 16;          // m, l and v of a warp's rows, for the CTA's own join
  static constexpr int kSmem = 1024 + kRing + kStats + kWarps * kSlots * 8 + 136 * 4 + 64;
  static_assert(NT * D * 32 <= kSlots * kSlotBytes, "a warp leaves its accumulator in its ring");
};

// Row r of a unit's tile rt: new token i, head, and how many keys it sees.
struct RowInfo {
  int i, head, limit;
};
__device__ __forceinline__ RowInfo row_info(const CacheAttnParams& p, int r, int hk, int n, int count) {
  RowInfo x;
  x.i = r / p.rep;
  x.head = hk * p.rep + r - x.i * p.rep;
  const bool valid = x.i < count;
  x.limit = !valid ? 0 : p.causal ? max(0, n - count + x.i + 1) : n;
  return x;
}

// Query fragments of a row tile: row 8 j + g, elements 16 c + 4 t ... + 3.  In two steps, so that other loads can be sent off between them:
// the bf16 values; then the same as f16, scaled by a power of two per row, with the factors of this thread's accumulator rows 8 j + 2 t and
// + 1 (softmax scale and log2 e included) in f.
template <int D, int NT>
__device__ __forceinline__ void ask_queries(const CacheAttnParams& p, int b, int hk, int rt, int count, uint32_t (&qf)[NT][D / 16][2]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = rt * 8 * NT + 8 * j + g;
    const int i = r / p.rep, head = hk * p.rep + r - i * p.rep;
    const bool valid = i < count;                             // rows beyond the call's: zeros
    const __nv_bfloat16* src = p.q + b * p.q_sb + i * p.q_sn + head * p.q_sh + 4 * t;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const uint2 raw = valid ? __ldg(reinterpret_cast<const uint2*>(src + 16 * c)) : make_uint2(0, 0);
      qf[j][c][0] = raw.x;
      qf[j][c][1] = raw.y;
    }
  }
}
template <int D, int NT>
__device__ __forceinline__ void scale_queries(const CacheAttnParams& p, uint32_t (&qf)[NT][D / 16][2], float2 (&f)[NT]) {
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        amax = max3(amax, fabsf(__uint_as_float(qf[j][c][i] << 16)), fabsf(__uint_as_float(qf[j][c][i] & 0xFFFF0000u)));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const uint32_t eb = min(254u, max(14u, __float_as_uint(amax) >> 23));
    const float up = sb_to_scale(267u - eb);                  // largest element to [2^13, 2^14)
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        qf[j][c][i] = pack_f16x2(__uint_as_float(qf[j][c][i] << 16) * up, __uint_as_float(qf[j][c][i] & 0xFFFF0000u) * up);
    const float back = sb_to_scale(eb - 13u) * p.scale * kLog2e;
    f[j] = make_float2(__shfl_sync(0xffffffffu, back, 8 * t), __shfl_sync(0xffffffffu, back, 8 * t + 4));
  }
}
// S^T of a block: acc[j][mt] rows: keys 16 mt + g (elements 0, 1) and + 8 (2, 3); columns: query rows 8 j + 2 t, + 1.
template <int D, int NT>
__device__ __forceinline__ void keys_times_queries(uint32_t kbase, const uint32_t (&qf)[NT][D / 16][2], float (&s)[NT][2][4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[j][mt][i] = 0.f;
  // even and odd chunks in accumulators of their own where registers allow: a chain of dependent MMAs is what a block waits for
  constexpr bool kTwo = NT == 1;
  float s2[kTwo ? NT : 1][2][4] = {};
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    uint32_t r[4];
    ldmatrix4(kbase + (c >> 3) * 4096 + lane * 128 + (((c & 7) ^ (lane & 7)) << 4), r);
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = e4m3_lo_f16x2(r[i]);
      hi[i] = e4m3_hi_f16x2(r[i]);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint32_t q0 = qf[j][c][0], q1 = qf[j][c][1];
      mma_f16(kTwo && (c & 1) ? s2[kTwo ? j : 0][0] : s[j][0], lo[0], lo[1], hi[0], hi[1], q0, q1);
      mma_f16(kTwo && (c & 1) ? s2[kTwo ? j : 0][1] : s[j][1], lo[2], lo[3], hi[2], hi[3], q0, q1);
    }
  }
  if (kTwo) {
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[0][mt][i] += s2[0][mt][i];
  }
}

// ------------------------------------------------------------------------------------------------ main kernel
// kCluster: a cluster of CTAs per unit instead of the even division, its results joined through distributed shared memory: nothing is left
// to a second kernel.
template <int D, int NT, bool kCluster>
__global__ void __launch_bounds__(128, AttnCfg<D, NT>::kCtasPerSm)
cache_attn_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const CacheAttnParams p, const int row_tiles) {
  using C = AttnCfg<D, NT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023) & ~1023u) - raw);
  float4* stats = reinterpret_cast<float4*>(smem + C::kRing);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kRing + C::kStats);
  int* cum = reinterpret_cast<int*>(bars + C::kWarps * C::kSlots);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(cum + 134);
  __shared__ int left_unit[C::kWarps], left_end[C::kWarps];   // what a warp leaves to the CTA's join: its unit (-1: nothing), its last block

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (tid == 0) {
    *abort_flag = 0;
    for (int i = 0; i < C::kWarps * C::kSlots; ++i) mbar_init(bars + i, 1);
    mbar_fence_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  grid_dep_wait();
  const int units = p.c.Hk * row_tiles;
  Piece seg{};
  int worker = warp, f_end = 0;
  bool have;                                                  // this warp has a piece
  int blk_first = 0, blk_step = 1;                            // block kb of it is block blk_first + kb blk_step of the sequence
  int page = 0, sub = 0;
  if constexpr (kCluster) {
    // The warps take the blocks in turn: which ones does not depend on the length, so that their pages are looked up beside it (in a call of a few
    // blocks a warp every load of this chain counts).  A warp has no more than kClusterBlocks of them.
    const int cl = p.cluster, unit = blockIdx.x / cl;
    seg.b = unit / units;
    seg.unit = unit - seg.b * units;
    blk_first = (blockIdx.x - unit * cl) * C::kWarps + warp;
    blk_step = cl * C::kWarps;
    const int bpp = p.c.page / 32, blk = blk_first + min(lane, 8) * blk_step, entry = blk / bpp;
    sub = blk - entry * bpp;
    if (entry < p.c.T) page = __ldg(p.c.table + seg.b * p.c.t_row + entry);
    seg.n = cache_length(p.c, seg.b);
    seg.blocks = (seg.n + 31) / 32;
    seg.blk1 = max(0, (seg.blocks - blk_first + blk_step - 1) / blk_step);
    have = seg.blk1 > 0;
    __syncthreads();                                          // publishes the mbarriers
  } else {
    const FlatRange range = flat_range(p.c, units, cum);      // its barriers publish the mbarriers too
    worker = blockIdx.x * C::kWarps + warp;
    const int workers = min(p.grid * C::kWarps, range.total); // each has a step at least
    have = worker < workers;
    if (have) {
      const int f0 = range_start(worker, workers, range.total);
      f_end = range_start(worker + 1, workers, range.total);
      seg = first_piece(p.c, units, range, f0, f_end);
    }
  }
  // the first piece's queries, then its pages: the loads are under way together
  while (have && seg.blk0 >= seg.blk1) have = next_piece(p.c, units, seg, f_end);       // no blocks: nothing but a unit's own cost
  uint32_t qf[NT][D / 16][2];
  Cursor ahead{};
  if (have) {
    const int hk = seg.unit / row_tiles;
    ask_queries<D, NT>(p, seg.b, hk, seg.unit - hk * row_tiles, checked_count(p.c.status, p.counts, seg.b, p.Nq), qf);
    if constexpr (kCluster) ahead = Cursor{seg, 0, 0, page, sub, true};
    else ahead = cursor_start(p.c, units, seg, f_end);
  }

  const uint32_t ring = smem_u32(smem) + warp * C::kSlots * C::kSlotBytes;
  const uint32_t my_bars = smem_u32(bars + warp * C::kSlots);
  float ks_reg = 0.f, vs_reg = 0.f;                           // lane i % 8: the scales of the i-th block of this warp
  int issued = 0, used = 0;                                   // boxes: K and V of a block in turn
  int put = 0, get = 0;                                       // their places in the ring
  uint32_t parity = 0;
  // The next box of this warp into its ring, if there is one.
  auto issue = [&]() {
    if (!ahead.live) return;
    const int2 at = cursor_at(p.c, ahead);                    // page, place
    const int hk = row_tiles == 1 ? ahead.s.unit : ahead.s.unit / row_tiles;
    const bool is_v = issued & 1;
    if (lane == 0) {
      const uint32_t bar = my_bars + 8 * put, dst = ring + put * C::kSlotBytes;
      asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(C::kSlotBytes) : "memory");
#pragma unroll
      for (int x = 0; x < D; x += 128) tma_load_4d(dst + x * 32, is_v ? &tv : &tk, bar, x, at.y * 32, hk, at.x);
    }
    if (is_v) {
      cursor_next(p.c, units, ahead, f_end);
    } else if (lane == ((issued >> 1) & 7)) {
      const int64_t scale = at.x * p.c.s_page + hk * p.c.s_head + at.y;
      ks_reg = __ldg(p.c.ks + scale);
      vs_reg = __ldg(p.c.vs + scale);
    }
    ++issued;
    if (++put == C::kSlots) put = 0;
  };
  for (int i = 0; i < C::kSlots; ++i) issue();

  bool ok = true;
  auto arrived = [&]() {
    if (ok && !wait_warp(my_bars + 8 * get, parity, abort_flag)) {
      ok = false;
      raise_abort(abort_flag, p.c.status, kStatusTimeoutCompute + kInCache);
    }
  };
  auto release = [&]() {
    __syncwarp();
    ++used;
    if (++get == C::kSlots) {
      get = 0;
      parity ^= 1;
    }
    if (ok) issue();
  };
  float m[NT][2], l[NT][2], acc[NT][D / 16][4];
  // of a row, whole numbers: m, at most 1 below the largest logit, which l is the sum beside; v, such that m + v is at most 0.99 below the largest logit
  // + log2 of its V scale: the accumulator counts in 2^(m + v - 15).  All is reckoned by differences of logits, so that it holds for large ones too.
  float v[NT][2];
  int slot = 2 * worker;
  // Of a finished piece: the rows' sums, complete in every lane.
  auto settle = [&]() {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], o);
  };
  // The results of a warp: to where they belong, or to a slot for the join.  `one`: only this sixteenth of head_dim, held in the first.
  auto write_out = [&](bool whole, int to_slot, int one) {
    const int hk = seg.unit / row_tiles, rt = seg.unit - hk * row_tiles, count = checked_count(p.c.status, p.counts, seg.b, p.Nq);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int in_tile = 8 * j + 2 * t + e, r = rt * C::kRows + in_tile;
        if (r >= p.Nq * p.rep) continue;
        if (whole) {
          const RowInfo ri = row_info(p, r, hk, seg.n, count);
          const bool any = ri.limit > 0;
          const float inv_l = any ? 1.f / l[j][e] : 0.f, inv = inv_l * exp2f(v[j][e] - 15.f);
          __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(p.o + ((static_cast<int64_t>(seg.b) * p.Nq + ri.i) * p.H + ri.head) * D + 2 * g);
          if (kCluster) {
            o[8 * one] = any ? __floats2bfloat162_rn(acc[j][0][e] * inv, acc[j][0][2 + e] * inv) : __floats2bfloat162_rn(0.f, 0.f);
          } else {
#pragma unroll
            for (int c = 0; c < D / 16; ++c)
              o[8 * c] = any ? __floats2bfloat162_rn(acc[j][c][e] * inv, acc[j][c][2 + e] * inv) : __floats2bfloat162_rn(0.f, 0.f);
          }
          if (g == 0 && one == 0) {
            p.lse[(static_cast<int64_t>(seg.b) * p.H + ri.head) * p.Nq + ri.i] = any ? (m[j][e] + log2f(l[j][e])) * kLn2 : -CUDART_INF_F;
            if (p.row_ml != nullptr)
              p.row_ml[(static_cast<int64_t>(seg.b) * p.c.Hk + hk) * p.Nq * p.rep + r] = make_float2(any ? m[j][e] : 0.f, inv_l);
          }
        } else {
          const int64_t row = static_cast<int64_t>(to_slot) * C::kRows + in_tile;
          float2* o = reinterpret_cast<float2*>(p.part_o + row * D + 2 * g);
#pragma unroll
          for (int c = 0; c < D / 16; ++c) o[8 * c] = make_float2(acc[j][c][e], acc[j][c][2 + e]);
          if (g == 0) p.part_ml[row] = make_float4(m[j][e], l[j][e], v[j][e], 0.f);
        }
      }
  };
  bool pending = false;                                       // the last piece waits for the CTA's join
  bool asked = true;                                          // the piece's queries are on their way
  while (have) {
    if (seg.blk0 >= seg.blk1) {                               // nothing but the unit's own cost
      if (!next_piece(p.c, units, seg, f_end)) break;
      continue;
    }
    const int hk = seg.unit / row_tiles, rt = seg.unit - hk * row_tiles;
    const int count = checked_count(p.c.status, p.counts, seg.b, p.Nq);
    float2 f[NT];
    if (!asked) ask_queries<D, NT>(p, seg.b, hk, rt, count, qf);
    asked = false;
    scale_queries<D, NT>(p, qf, f);
    // keys that this thread's row 8 j + 2 t + e sees: made where a block is cut (registers are what a block has least of)
    auto lim = [&](int j, int e) { return row_info(p, rt * C::kRows + 8 * j + 2 * t + e, hk, seg.n, count).limit; };
    int lim_min = seg.n;
    if (p.causal) lim_min = seg.n - count + 1;                // of the rows that are any
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      m[j][0] = m[j][1] = kNone;
      v[j][0] = v[j][1] = 0.f;
      l[j][0] = l[j][1] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) acc[j][c][0] = acc[j][c][1] = acc[j][c][2] = acc[j][c][3] = 0.f;
    }

    for (int kb = seg.blk0; kb < seg.blk1; ++kb) {
      const int at = (used >> 1) & 7;
      arrived();
      if (!ok) break;
      const float ks = __shfl_sync(0xffffffffu, ks_reg, at), vs = __shfl_sync(0xffffffffu, vs_reg, at);
      float s[NT][2][4];
      keys_times_queries<D, NT>(ring + get * C::kSlotBytes, qf, s);
      const int key0 = (kCluster ? blk_first + kb * blk_step : kb) * 32;
      const bool cut = key0 + 32 > lim_min;                   // some row does not see all keys of the block
      const float e_blk = static_cast<float>(static_cast<int>(scale_to_sb(vs)) - 127);
      uint32_t pb[NT][2][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float2 fs = make_float2(f[j].x * ks, f[j].y * ks);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[j][mt][i] = __fmul_rn(s[j][mt][i], (i & 1) ? fs.y : fs.x);       // one value for the maximum and for p, however large
        if (cut) {
          const int seen[2] = {lim(j, 0) - key0 - g, lim(j, 1) - key0 - g};
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (16 * mt + 8 * (i >> 1) >= seen[i & 1]) s[j][mt][i] = -CUDART_INF_F;
        }
        const int logit_rows = NT == 1 ? p.logit_rows : C::kRows;
        if (p.logits != nullptr && 8 * j + 2 * t < logit_rows) {        // for the weights: (b, kv head, token, row of the tile)
          float* to = p.logits + ((static_cast<int64_t>(seg.b) * p.c.Hk + hk) * p.c.T * p.c.page + key0 + g) * logit_rows + 8 * j + 2 * t;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              *reinterpret_cast<float2*>(to + (16 * mt + 8 * i) * logit_rows) = make_float2(s[j][mt][2 * i], s[j][mt][2 * i + 1]);
        }
        float2 mx = make_float2(fmaxf(fmaxf(s[j][0][0], s[j][0][2]), fmaxf(s[j][1][0], s[j][1][2])),
                                fmaxf(fmaxf(s[j][0][1], s[j][0][3]), fmaxf(s[j][1][1], s[j][1][3])));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          mx.x = fmaxf(mx.x, __shfl_xor_sync(0xffffffffu, mx.x, o));
          mx.y = fmaxf(mx.y, __shfl_xor_sync(0xffffffffu, mx.y, o));
        }
        const float2 over = make_float2(mx.x - m[j][0], mx.y - m[j][1]);
        if (__any_sync(0xffffffffu, over.x > 1.f || over.y > 1.f || over.x + e_blk > v[j][0] + 0.99f || over.y + e_blk > v[j][1] + 0.99f)) {
          float keep[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mx_e = e ? mx.y : mx.x, m_new = (e ? over.y : over.x) > 1.f ? ceilf(mx_e) : m[j][e];
            const float fall = m[j][e] - m_new, v_old = v[j][e] + fall, pv = mx_e - m_new + e_blk;
            m[j][e] = m_new;
            v[j][e] = pv > v_old + 0.99f ? ceilf(pv) : v_old;
            l[j][e] *= ex2_approx(fall);
            keep[e] = ex2_approx(v_old - v[j][e]);
          }
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            acc[j][c][0] *= keep[0];
            acc[j][c][1] *= keep[1];
            acc[j][c][2] *= keep[0];
            acc[j][c][3] *= keep[1];
          }
        }
        float off[2], back[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // p comes out as 2^(s - m + off), below 2^16; where the products are 2^-60 of the largest they vanish anyway, but the sum must not
          off[e] = fmaxf(15.f + e_blk - v[j][e], -45.f);
          back[e] = ex2_approx(-off[e]);                      // zero where p is below 2^-111 of the largest
        }
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          float e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[i] = ex2_approx(s[j][mt][i] - m[j][i & 1] + off[i & 1]);
            if (i & 1) sum.y += e[i]; else sum.x += e[i];
          }
          pb[j][mt][0] = movmatrix_trans(pack_f16x2(e[0], e[1]));
          pb[j][mt][1] = movmatrix_trans(pack_f16x2(e[2], e[3]));
        }
        l[j][0] = fmaf(sum.x, back[0], l[j][0]);
        l[j][1] = fmaf(sum.y, back[1], l[j][1]);
      }
      release();
      arrived();
      if (!ok) break;
      const uint32_t vbase = ring + get * C::kSlotBytes;
      // slots beyond the length hold anything, NaN codes too: zero times NaN must not reach the sums
      uint32_t sel[4] = {0x3120u, 0x3120u, 0x3120u, 0x3120u};
      if (key0 + 32 > seg.n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = key0 + 8 * i + 2 * t;
          sel[i] = k + 1 < seg.n ? 0x3120u : k < seg.n ? 0x4140u : 0x4444u;
        }
      }
      // A NaN code belongs to the rows that see its token; the others would multiply it by zero.  Where some row does not see all that is held: which rows see
      // one, by products of ones (token seen) and ones (code NaN), and zeros in its place.
      if (key0 + 32 > lim_min && lim_min < seg.n) {
        const uint32_t slot = vbase + lane * 128;             // a lane a token (its pieces in an order of its own: different banks)
        uint32_t found = 0;
#pragma unroll 1
        for (int x = 0; x < D / 16; ++x) {
          const float4 w = lds_f4(slot + (x >> 3) * 4096 + (((x ^ lane) & 7) << 4));
          found |= nan_codes(__float_as_uint(w.x)) | nan_codes(__float_as_uint(w.y)) | nan_codes(__float_as_uint(w.z)) | nan_codes(__float_as_uint(w.w));
        }
        if (__any_sync(0xffffffffu, found != 0 && key0 + lane < seg.n)) {
          uint32_t sees[NT][2][2];
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int k = key0 + 8 * i + g;
              sees[j][i >> 1][i & 1] = movmatrix_trans(pack_f16x2(k < lim(j, 0) ? 1.f : 0.f, k < lim(j, 1) ? 1.f : 0.f));
            }
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t r[4], lo[4], hi[4];
            ldmatrix4_trans(vbase + (c >> 3) * 4096 + lane * 128 + (((c & 7) ^ (lane & 7)) << 4), r);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              r[i] = nan_codes(prmt(r[i], 0u, sel[i])) & 0x38383838u;         // one
              lo[i] = e4m3_lo_f16x2(r[i]);
              hi[i] = e4m3_hi_f16x2(r[i]);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              float seen[4] = {0.f, 0.f, 0.f, 0.f};
              mma_f16(seen, lo[0], hi[0], lo[1], hi[1], sees[j][0][0], sees[j][0][1]);
              mma_f16(seen, lo[2], hi[2], lo[3], hi[3], sees[j][1][0], sees[j][1][1]);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (seen[i] > 0.f) acc[j][c][i] = CUDART_NAN_F;
            }
          }
          __syncwarp();
#pragma unroll 1
          for (int x = 0; x < D / 16; ++x) {
            const uint32_t at = slot + (x >> 3) * 4096 + (((x ^ lane) & 7) << 4);
            const float4 f4 = lds_f4(at);
            const uint32_t w[4] = {__float_as_uint(f4.x), __float_as_uint(f4.y), __float_as_uint(f4.z), __float_as_uint(f4.w)};
            sts_u4(at, w[0] & ~nan_codes(w[0]), w[1] & ~nan_codes(w[1]), w[2] & ~nan_codes(w[2]), w[3] & ~nan_codes(w[3]));
          }
          fence_async_smem();                                 // before the next box comes here
          __syncwarp();
        }
      }
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        uint32_t r[4], lo[4], hi[4];
        ldmatrix4_trans(vbase + (c >> 3) * 4096 + lane * 128 + (((c & 7) ^ (lane & 7)) << 4), r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          r[i] = prmt(r[i], 0u, sel[i]);
          lo[i] = e4m3_lo_f16x2(r[i]);
          hi[i] = e4m3_hi_f16x2(r[i]);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma_f16(acc[j][c], lo[0], hi[0], lo[1], hi[1], pb[j][0][0], pb[j][0][1]);
          mma_f16(acc[j][c], lo[2], hi[2], lo[3], hi[3], pb[j][1][0], pb[j][1][1]);
        }
      }
      release();
    }
    if (!ok) break;

    settle();
    const bool whole = seg.blk0 == 0 && seg.blk1 == seg.blocks, last = seg.f1 >= f_end;
    if (kCluster || (last && !whole)) {
      pending = true;
      break;
    }
    if (lane == 0) {                                          // for the join (see unit_slots): a whole unit, or the end of one
      int2* u = p.unit_slots + (static_cast<int64_t>(seg.b) * units + seg.unit);
      if (whole) u->x = -1;
      u->y = 2 * worker + 1;
    }
    write_out(whole, slot, 0);
    slot = 2 * worker + 1;
    if (!next_piece(p.c, units, seg, f_end)) break;
  }
  // given up: the copies in flight must land before the shared memory goes
  for (; used < issued; ++used) {
    wait_or_abort(my_bars + 8 * get, parity, abort_flag);
    if (++get == C::kSlots) {
      get = 0;
      parity ^= 1;
    }
  }

  // The CTA's join.  Neighbouring warps that end in one unit: the first of them takes over the others' results, in their order, from their
  // rings (which are done with).  In a cluster all warps are of one unit, those without blocks too.
  float4* parked = reinterpret_cast<float4*>(smem + warp * C::kSlots * C::kSlotBytes);
  if (kCluster && !pending) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      m[j][0] = m[j][1] = kNone;
      v[j][0] = v[j][1] = 0.f;
      l[j][0] = l[j][1] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) acc[j][c][0] = acc[j][c][1] = acc[j][c][2] = acc[j][c][3] = 0.f;
    }
  }
  if (lane == 0) {
    left_unit[warp] = kCluster ? 0 : pending ? seg.b * units + seg.unit : -1;
    left_end[warp] = seg.blk1;
  }
  __syncthreads();
  const bool follows = warp > 0 && left_unit[warp] >= 0 && left_unit[warp - 1] == left_unit[warp];
  auto park = [&]() {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (g == 0) {
        stats[warp * C::kRows + 8 * j + 2 * t] = make_float4(m[j][0], l[j][0], v[j][0], 0.f);
        stats[warp * C::kRows + 8 * j + 2 * t + 1] = make_float4(m[j][1], l[j][1], v[j][1], 0.f);
      }
#pragma unroll
      for (int c = 0; c < D / 16; ++c) parked[(j * (D / 16) + c) * 32 + lane] = make_float4(acc[j][c][0], acc[j][c][1], acc[j][c][2], acc[j][c][3]);
    }
  };
  // Parked results, by their base and statistics, into this warp's.
  auto take_over = [&](const float4* from, const float4* st) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float2 mine, theirs;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float4 x = st[8 * j + 2 * t + e];
        const float top = fmaxf(m[j][e], x.x), fall = m[j][e] - top, their_fall = x.x - top, v_new = fmaxf(v[j][e] + fall, x.z + their_fall);
        l[j][e] = l[j][e] * ex2_approx(fall) + x.y * ex2_approx(their_fall);
        (e ? mine.y : mine.x) = ex2_approx(v[j][e] + fall - v_new);
        (e ? theirs.y : theirs.x) = ex2_approx(x.z + their_fall - v_new);
        m[j][e] = top;
        v[j][e] = v_new;
      }
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const float4 x = from[(j * (D / 16) + c) * 32 + lane];
        acc[j][c][0] = acc[j][c][0] * mine.x + x.x * theirs.x;
        acc[j][c][1] = acc[j][c][1] * mine.y + x.y * theirs.y;
        acc[j][c][2] = acc[j][c][2] * mine.x + x.z * theirs.x;
        acc[j][c][3] = acc[j][c][3] * mine.y + x.w * theirs.y;
      }
    }
  };
  if (follows) park();
  __syncthreads();
  if constexpr (kCluster) {
    if (warp == 0) {
      for (int w = 1; w < C::kWarps; ++w) take_over(reinterpret_cast<const float4*>(smem + w * C::kSlots * C::kSlotBytes), stats + w * C::kRows);
      park();
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    // CTA r of the cluster joins and writes its share of the sixteenths of head_dim, a warp a sixteenth, over the CTAs in order
    const int cl = p.cluster, rank = blockIdx.x % cl, c1 = (rank + 1) * (D / 16) / cl;
    for (int c = rank * (D / 16) / cl + warp; c < c1; c += C::kWarps) {
      // Lane (g, t) looks at CTA g's statistics of its rows; these and the values are all on their way together.
      float4 st[NT][2], x[NT][kMaxCluster];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          st[j][e] = g < cl ? cluster.map_shared_rank(stats, g)[8 * j + 2 * t + e] : make_float4(kNone, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
          if (r < cl) x[j][r] = cluster.map_shared_rank(reinterpret_cast<float4*>(smem), r)[(j * (D / 16) + c) * 32 + lane];
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = st[j][e].x;
#pragma unroll
          for (int i = 4; i < 32; i <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
          const float fall = st[j][e].x - top, mine = st[j][e].z + fall;
          float v_top = mine, sum = st[j][e].y * ex2_approx(fall);
#pragma unroll
          for (int i = 4; i < 32; i <<= 1) v_top = fmaxf(v_top, __shfl_xor_sync(0xffffffffu, v_top, i));
          const float w = ex2_approx(mine - v_top);
#pragma unroll
          for (int i = 4; i < 32; i <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
#pragma unroll
          for (int r = 0; r < kMaxCluster; ++r) {
            if (r >= cl) continue;
            const float w_r = __shfl_sync(0xffffffffu, w, 4 * r + t);
            o[e] = fmaf(e ? x[j][r].y : x[j][r].x, w_r, o[e]);
            o[2 + e] = fmaf(e ? x[j][r].w : x[j][r].z, w_r, o[2 + e]);
          }
          m[j][e] = top;
          l[j][e] = sum;
          v[j][e] = v_top;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][0][i] = o[i];
      }
      write_out(true, 0, c);
    }
    cluster.sync();                                           // shared memory stays until all have read it
  } else {
    if (pending && !follows) {
      int end = seg.blk1, last = worker;
      for (int w = warp + 1; w < C::kWarps && left_unit[w] == left_unit[warp]; ++w) {
        take_over(reinterpret_cast<const float4*>(smem + w * C::kSlots * C::kSlotBytes), stats + w * C::kRows);
        end = left_end[w];
        ++last;
      }
      const bool whole = seg.blk0 == 0 && end == seg.blocks;
      if (lane == 0) {
        int2* u = p.unit_slots + (static_cast<int64_t>(seg.b) * units + seg.unit);
        if (seg.blk0 == 0) u->x = whole ? -1 : slot;
        if (end == seg.blocks) u->y = 2 * last;
      }
      write_out(whole, slot, 0);
    }
  }
}

// ------------------------------------------------------------------------------------------------ join
// The partial results of units that were cut: one CTA per (sequence, head, new token), four warps that take every fourth slot.
// Also rows of sequences that hold nothing.
template <int D>
__global__ void __launch_bounds__(128) cache_join_kernel(const CacheAttnParams p, const int row_tiles, const int row_tile) {
  __shared__ float part[4][D];
  __shared__ float factors[128], red[4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  grid_dep_wait();
  const int R = p.Nq * p.rep;
  const int64_t item = blockIdx.x;                            // (b, hk, r)
  const int bh = static_cast<int>(item / R), r = static_cast<int>(item - static_cast<int64_t>(bh) * R), hk = bh % p.c.Hk, b = bh / p.c.Hk, rt = r / row_tile;
  const int2 unit = p.unit_slots[static_cast<int64_t>(bh) * row_tiles + rt];
  const int n = cache_length(p.c, b);
  const int count = checked_count(p.c.status, p.counts, b, p.Nq);
  const RowInfo ri = row_info(p, r, hk, n, count);
  __nv_bfloat16* o = p.o + ((static_cast<int64_t>(b) * p.Nq + ri.i) * p.H + ri.head) * D;
  float* lse = p.lse + (static_cast<int64_t>(b) * p.H + ri.head) * p.Nq + ri.i;
  if (ri.limit == 0) {
    for (int d = tid; d < D; d += 128) o[d] = __float2bfloat16(0.f);
    if (tid == 0) {
      *lse = -CUDART_INF_F;
      if (p.row_ml != nullptr) p.row_ml[item] = make_float2(0.f, 0.f);
    }
    return;
  }
  const JoinSlots slots = join_slots_of_warps(unit, p.grid);
  if (slots.none()) return;                                   // whole: written by its warp (or given up)
  const int pieces = slots.count, in_tile = r - rt * row_tile;
  auto row_of = [&](int i) { return static_cast<int64_t>(slots.slot(i)) * row_tile + in_tile; };
  // over the CTA's threads
  auto block_max = [&](float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    __syncthreads();
    if (lane == 0) red[warp] = x;
    __syncthreads();
    return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  };
  float top = kNone, v_top = kNone;
  for (int i = tid; i < pieces; i += 128) top = fmaxf(top, p.part_ml[row_of(i)].x);
  top = block_max(top);
  for (int i = tid; i < pieces; i += 128) {
    const float4 x = p.part_ml[row_of(i)];
    v_top = fmaxf(v_top, x.x - top + x.z);
  }
  v_top = block_max(v_top);
  float sum = 0.f, acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  for (int i0 = 0; i0 < pieces; i0 += 128) {                  // 128 pieces at a time: their factors, then their rows
    float f = 0.f;
    if (i0 + tid < pieces) {
      const float4 x = p.part_ml[row_of(i0 + tid)];
      f = ex2_approx(x.x - top + x.z - v_top);
      sum = fmaf(x.y, ex2_approx(x.x - top), sum);
    }
    if (i0 > 0) __syncthreads();
    factors[tid] = f;
    __syncthreads();
#pragma unroll 8
    for (int i = warp; i < min(128, pieces - i0); i += 4) {
      const float f_i = factors[i];
      const float4* src = reinterpret_cast<const float4*>(p.part_o + row_of(i0 + i) * D) + lane;
#pragma unroll
      for (int x = 0; x < D / 128; ++x) {
        const float4 v = src[32 * x];
        acc[4 * x] = fmaf(v.x, f_i, acc[4 * x]);
        acc[4 * x + 1] = fmaf(v.y, f_i, acc[4 * x + 1]);
        acc[4 * x + 2] = fmaf(v.z, f_i, acc[4 * x + 2]);
        acc[4 * x + 3] = fmaf(v.w, f_i, acc[4 * x + 3]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < D / 128; ++i)
    *reinterpret_cast<float4*>(&part[warp][128 * i + 4 * lane]) = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) red[warp] = sum;
  __syncthreads();
  sum = (red[0] + red[1]) + (red[2] + red[3]);
  const float inv_l = 1.f / sum, inv = inv_l * exp2f(v_top - 15.f);
  for (int d = tid; d < D; d += 128) o[d] = __float2bfloat16(((part[0][d] + part[1][d]) + (part[2][d] + part[3][d])) * inv);
  if (tid == 0) {
    *lse = (top + log2f(sum)) * kLn2;
    if (p.row_ml != nullptr) p.row_ml[item] = make_float2(top, inv_l);
  }
}

// ------------------------------------------------------------------------------------------------ weights
// weights[b, hk, j] (+)= sum over the group's rows of exp(s_rj - m_r) / l_r, with the rows' m and l from the kernels before.  No result is shared between
// warps or threads, and the sum's order is that of the rows.
// Up to 16 rows the main kernel leaves its logits (16 - 64 bytes a token instead of K's 128 or 256, and no products), and
// cache_weights_of_logits_kernel adds their exponentials, one thread a token: a call with weights at H=32 Hk=8, B=16 with 2049 - 4096 tokens takes 35 us
// with one new token (59 with K read again) and 46 with four (66).  For 17 to 32 rows of head_dim 128 cache_weights_kernel reads K once more, a
// block of 32 tokens a warp, all rows on it.
__global__ void __launch_bounds__(256) cache_weights_of_logits_kernel(const CacheAttnParams p, const int pieces) {
  __shared__ float2 ml[16];
  grid_dep_wait();
  const int bh = blockIdx.x / pieces, j = (blockIdx.x - bh * pieces) * 256 + threadIdx.x, b = bh / p.c.Hk, hk = bh - b * p.c.Hk, R = p.Nq * p.rep;
  // the first logits before it is known whether the token exists (its place does): the loads are under way together
  const float4* x = reinterpret_cast<const float4*>(p.logits + (static_cast<int64_t>(bh) * p.c.T * p.c.page + j) * p.logit_rows);
  const float4 first = j < p.c.T * p.c.page ? *x : make_float4(0.f, 0.f, 0.f, 0.f);
  const int n = cache_length(p.c, b);
  if (threadIdx.x < R) ml[threadIdx.x] = p.row_ml[static_cast<int64_t>(bh) * R + threadIdx.x];
  __syncthreads();
  if (j >= p.W) return;
  float* at = p.weights + b * p.w_sb + hk * p.w_sh + j;
  if (j >= n) {                                               // beyond the length: zero, unless the sums go on
    if (!p.accumulate) *at = 0.f;
    return;
  }
  float w = 0.f;
#pragma unroll
  for (int r = 0; r < 16; r += 4) {
    if (r >= R) break;
    const float4 y = r == 0 ? first : x[r / 4];
    // of a row that sees anything (1 / sum is not zero): those of others are logits of zeros, NaN where K is
    const auto p_of = [&](float s, float2 row) { return row.y != 0.f ? ex2_approx(s - row.x) * row.y : 0.f; };
    w += p_of(y.x, ml[r]);
    if (r + 1 < R) w += p_of(y.y, ml[r + 1]);
    if (r + 2 < R) w += p_of(y.z, ml[r + 2]);
    if (r + 3 < R) w += p_of(y.w, ml[r + 3]);
  }
  *at = p.accumulate ? *at + w : w;
}

__global__ void __launch_bounds__(128) cache_weights_kernel(const __grid_constant__ CUtensorMap tk, const CacheAttnParams p) {
  constexpr int D = 128, NT = 4, kStages = 4, kStageBytes = 32 * D;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023) & ~1023u) - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 4 * kStages * kStageBytes);
  int* cum = reinterpret_cast<int*>(bars + 4 * kStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(cum + 134);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (tid == 0) {
    *abort_flag = 0;
    for (int i = 0; i < 4 * kStages; ++i) mbar_init(bars + i, 1);
    mbar_fence_init();
    tma_prefetch_desc(&tk);
  }
  grid_dep_wait();
  // what lies beyond the lengths: zero, unless the sums go on
  if (!p.accumulate) {
    const int pieces = (p.W + 1023) / 1024;
    for (int64_t x = blockIdx.x; x < static_cast<int64_t>(p.c.B) * p.c.Hk * pieces; x += gridDim.x) {
      const int piece = static_cast<int>(x % pieces), hk = static_cast<int>(x / pieces % p.c.Hk), b = static_cast<int>(x / pieces / p.c.Hk);
      const int n = cache_length(p.c, b);
      for (int j = max(n, piece * 1024) + tid; j < min(p.W, (piece + 1) * 1024); j += 128) p.weights[b * p.w_sb + hk * p.w_sh + j] = 0.f;
    }
  }
  const int units = p.c.Hk;
  const FlatRange range = flat_range(p.c, units, cum);
  const int worker = blockIdx.x * 4 + warp, workers = gridDim.x * 4;
  const int f0 = range_start(worker, workers, range.total), f_end = range_start(worker + 1, workers, range.total);
  if (f0 >= f_end) return;
  Piece seg = first_piece(p.c, units, range, f0, f_end);
  Cursor ahead = cursor_start(p.c, units, seg, f_end);
  const uint32_t ring = smem_u32(smem) + warp * kStages * kStageBytes, my_bars = smem_u32(bars + warp * kStages);
  float ks_reg = 0.f;
  auto issue = [&](int st) {
    const int2 where = cursor_at(p.c, ahead);
    const int page = where.x, sub = where.y, hk = ahead.s.unit;
    if (lane == 0) {
      const uint32_t bar = my_bars + 8 * st, dst = ring + st * kStageBytes;
      asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(kStageBytes) : "memory");
      tma_load_4d(dst, &tk, bar, 0, sub * 32, hk, page);
    }
    if (lane == st) ks_reg = __ldg(p.c.ks + page * p.c.s_page + hk * p.c.s_head + sub);
  };
  int issued = 0, used = 0;
  for (int st = 0; st < kStages && ahead.live; ++st) {
    issue(st);
    ++issued;
    cursor_next(p.c, units, ahead, f_end);
  }
  bool ok = true;
  int st = 0;
  uint32_t parity = 0;
  const int R = p.Nq * p.rep;
  for (;;) {
    const int hk = seg.unit, count = checked_count(p.c.status, p.counts, seg.b, p.Nq);
    const float2* row_ml = p.row_ml + (static_cast<int64_t>(seg.b) * p.c.Hk + hk) * R;
    uint32_t qf[NT][D / 16][2];
    float2 f[NT];
    ask_queries<D, NT>(p, seg.b, hk, 0, count, qf);
    scale_queries<D, NT>(p, qf, f);
    for (int kb = seg.blk0; kb < seg.blk1; ++kb) {
      if (ok && !wait_warp(my_bars + 8 * st, parity, abort_flag)) {
        ok = false;
        raise_abort(abort_flag, p.c.status, kStatusTimeoutCompute + kInCache);
      }
      if (ok) {
        const float ks = __shfl_sync(0xffffffffu, ks_reg, st);
        const int key0 = kb * 32;
        float w[4] = {0.f, 0.f, 0.f, 0.f};                    // of keys key0 + g + 8 i
        float s[NT][2][4];
        keys_times_queries<D, NT>(ring + st * kStageBytes, qf, s);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 8 * j + 2 * t + e;
            const float2 ml = r < R ? row_ml[r] : make_float2(0.f, 0.f);
            const int limit = row_info(p, r, hk, seg.n, count).limit;
            const float fs = (e ? f[j].y : f[j].x) * ks;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x = __fmul_rn(s[j][i >> 1][(i & 1) * 2 + e], fs) - ml.x;         // as in the main kernel
              w[i] += key0 + g + 8 * i < limit ? ex2_approx(x) * ml.y : 0.f;
            }
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] += __shfl_xor_sync(0xffffffffu, w[i], 1);
          w[i] += __shfl_xor_sync(0xffffffffu, w[i], 2);
        }
        const float mine = t == 0 ? w[0] : t == 1 ? w[1] : t == 2 ? w[2] : w[3];
        const int key = key0 + g + 8 * t;
        if (key < seg.n) {
          float* at = p.weights + seg.b * p.w_sb + hk * p.w_sh + key;
          *at = p.accumulate ? *at + mine : mine;
        }
      }
      __syncwarp();
      ++used;
      if (ok && ahead.live) {
        issue(st);
        ++issued;
        cursor_next(p.c, units, ahead, f_end);
      }
      if (++st == kStages) {
        st = 0;
        parity ^= 1;
      }
    }
    if (!next_piece(p.c, units, seg, f_end)) break;
  }
  if (!ok) {
    for (; used < issued; ++used) wait_or_abort(my_bars + 8 * (used % kStages), (used / kStages) & 1, abort_flag);
  }
}

// Once per kernel and device: the driver call takes longer than a launch.
template <auto kKernel>
cudaError_t allow_smem(int bytes) {
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && done[dev]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
  return e;
}

template <int D, int NT>
cudaError_t launch_main(const CUtensorMap& tk, const CUtensorMap& tv, const CacheAttnParams& p, int row_tiles, cudaStream_t stream) {
  using C = AttnCfg<D, NT>;
  if (p.cluster > 0) {
    const cudaError_t e = allow_smem<cache_attn_kernel<D, NT, true>>(C::kSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.grid);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    count_launch();
    return cudaLaunchKernelEx(&cfg, cache_attn_kernel<D, NT, true>, tk, tv, p, row_tiles);
  }
  cudaError_t e = allow_smem<cache_attn_kernel<D, NT, false>>(C::kSmem);
  if (e != cudaSuccess) return e;
  count_launch();
  e = launch_chained(cache_attn_kernel<D, NT, false>, dim3(p.grid), 128, C::kSmem, stream, tk, tv, p, row_tiles);
  if (e != cudaSuccess) return e;
  count_launch();
  return launch_chained(cache_join_kernel<D>, dim3(static_cast<unsigned>(static_cast<int64_t>(p.c.B) * p.H * p.Nq)), 128, 0, stream, p, row_tiles, C::kRows);
}

cudaError_t launch_weights(const CUtensorMap& tk, const CacheAttnParams& p, cudaStream_t stream) {
  constexpr int smem = 1024 + 4 * 4 * 32 * 128 + 4 * 4 * 8 + 136 * 4 + 64;
  const cudaError_t e = allow_smem<cache_weights_kernel>(smem);
  if (e != cudaSuccess) return e;
  // a wave, and no more warps than there can be blocks
  const int64_t most = (static_cast<int64_t>(p.c.B) * p.c.Hk * p.c.T * (p.c.page / 32) + 3) / 4, wave = sm_count() * 2ll;
  count_launch();
  return launch_chained(cache_weights_kernel, dim3(static_cast<unsigned>(most < wave ? most : wave)), 128, smem, stream, tk, p);
}

// Blocks of a warp up to which a cluster takes a unit, joining its warps' results itself, instead of the even division with a kernel that joins.  us with and
// without, H=32 Hk=8, one new token: B=1 with 4096 tokens 12.7 and 14.8, B=4 with 3601 - 4096 15.5 and 18.5, B=8 with 2048 15.5 and 18.8; with
// 16 instead of 8, B=1 with 16384 tokens took 25.0 against 19.4.
constexpr int kClusterBlocks = 8;
// A tile of 32 rows reads the codes once where two of 16 read them twice (the second time from L2), but its accumulators leave fewer warps in flight:
// us with 32 and 16 at H=32 Hk=8, 8 new tokens: B=64 with 17 - 8191 tokens 232 and 243, B=8 with 4096 - 8192 56.4 and 54.7, B=1 with 1000
// 15.0 and 10.8.
int small_row_tile(int R) { return R <= 8 ? 8 : 16; }

}  // namespace

// Rows (new tokens x heads of a group) from which the tcgen05 form is taken.  us of this form and of that: at head_dim 128, H=32 Hk=8, 32 rows B=8 with
// 4096 - 8192 tokens 59.4 and 65.6, B=1 with 8192 26.5 and 31.6, 36 rows 78.2 and 65.9, 27.0 and 31.6; at head_dim 256, where this form takes two
// passes over 17 rows, H=16 Hk=4, 16 rows B=8 44.5 and 57.0, 24 rows 69.4 and 57.2, B=1 36.4 and 37.5, B=64 with 17 - 8191 296 and 217.
int cache_chunk_from(int D) { return D == 128 ? 33 : 17; }

CacheAttnPlan plan_cache_attn(int B, int Nq, int H, int Hk, int D, int T, int page, bool weights) {
  CacheAttnPlan x;
  const int R = Nq * (H / Hk);
  x.chunk = R >= cache_chunk_from(D);
  x.row_tile = x.chunk ? cache_chunk_rows(D) : small_row_tile(R);
  x.row_tiles = (R + x.row_tile - 1) / x.row_tile;
  const int64_t blocks = static_cast<int64_t>(T) * (page / 32), units = static_cast<int64_t>(B) * Hk * x.row_tiles;       // of a sequence; in all
  const int ctas = x.chunk ? 1 : D == 128 && x.row_tile == 8 ? AttnCfg<128, 1>::kCtasPerSm : AttnCfg<128, 2>::kCtasPerSm;
  const int64_t wave = static_cast<int64_t>(sm_count()) * ctas;
  // A cluster per unit where a warp of it has at most kClusterBlocks blocks and all clusters are resident at a time.
  x.cluster = 0;
  if (!x.chunk) {
    int cl = 1;
    while (cl < 8 && units * cl * 2 <= wave && cl * 4 < blocks) cl *= 2;
    if (units * cl <= wave && blocks <= static_cast<int64_t>(kClusterBlocks) * 4 * cl) x.cluster = cl;
  }
  // otherwise one wave, and no more workers than there can be blocks (tiles of four blocks for a CTA of the tcgen05 form)
  const int64_t most = (units * blocks + 3) / 4;
  x.grid = x.cluster > 0 ? static_cast<int>(units) * x.cluster : static_cast<int>(most < wave ? most : wave);
  const int64_t slots = x.cluster > 0 ? 0 : 2ll * x.grid * (x.chunk ? 1 : 4);
  x.part_o_bytes = slots * x.row_tile * D * 4;
  x.part_ml_bytes = slots * x.row_tile * 16;
  const int64_t q_rows = x.chunk ? cache_chunk_query_rows(B, Hk, R) : 0;
  x.q16_bytes = q_rows * D * 2;
  x.mark_bytes = x.chunk ? 16 : 0;
  x.factor_bytes = q_rows * 4;
  x.start_bytes = x.chunk ? x.grid * cache_chunk_start_bytes() : 0;
  x.unit_bytes = static_cast<int64_t>(B) * Hk * x.row_tiles * 8;
  // logits for the weights, where they are fewer bytes than K
  x.logit_rows = R <= 4 ? 4 : x.row_tile;
  x.logit_bytes = weights && R <= 16 ? static_cast<int64_t>(B) * Hk * T * page * x.logit_rows * 4 : 0;
  x.row_ml_bytes = !weights ? 0 : x.chunk ? q_rows * 8 : static_cast<int64_t>(B) * Hk * R * 8;
  return x;
}

cudaError_t launch_cache_attn(int D, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tq, const CacheAttnParams& p, cudaStream_t stream) {
  const int R = p.Nq * p.rep, tile = small_row_tile(R), row_tiles = (R + tile - 1) / tile;
  if (p.unit_shift > 0) return launch_cache_chunk(D, tk, tv, tq, p, stream);
  cudaError_t e;
  if (D == 128) {
    e = tile == 8 ? launch_main<128, 1>(tk, tv, p, row_tiles, stream) : launch_main<128, 2>(tk, tv, p, row_tiles, stream);
  } else {
    e = tile == 8 ? launch_main<256, 1>(tk, tv, p, row_tiles, stream) : launch_main<256, 2>(tk, tv, p, row_tiles, stream);
  }
  if (e != cudaSuccess || p.weights == nullptr) return e;
  if (p.logits != nullptr) {
    const int pieces = (p.W + 255) / 256;
    count_launch();
    return launch_chained(cache_weights_of_logits_kernel, dim3(static_cast<unsigned>(p.c.B) * p.c.Hk * pieces), 256, 0, stream, p, pieces);
  }
  return launch_weights(tk, p, stream);                      // head_dim 256 has its logits or the form for many rows
}

}  // namespace dm
