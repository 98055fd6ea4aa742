// Attention of a tree of drafted tokens over the 8-bit cache.
//
//   s_rj = scale q_r . (ks code_j);  o_r = sum_j exp(s_rj - m_r) vs code_j / sum_j exp(s_rj - m_r)  over the keys j that row r sees:
//   all tokens held before the drafted ones, and of these its node's own ancestors and itself
//
// Rows are (drafted token, head of the kv head's group); a unit is (sequence, kv head, up to 128 rows).  The codes of K and V go to the tensor cores as
// they lie in the pages, no code is ever converted: S = Q K^T is the sum of two kind::f8f6f4 chains with q in two codes, e4m3 and what that leaves in e5m2
// (4 and 3 significant bits, of bf16's 8 with the signs: exact down to 2^-13 of the row's largest element, 2^-21 of that off below), and O += P V the sum
// of two block-scaled chains with P in two e4m3 codes relative to the largest of its 32 keys (off by 2^-8 of itself at most, 2^-17 of that largest one where it is
// small).  The power-of-two scale of V's block goes into P's scale byte and that of K's block into the factor of the logits.
//
// The key tiles of 128 tokens of all units are one flat range, divided evenly over the CTAs of one wave; pieces of cut units are joined by a second kernel.
// Warps 0-3: queries, softmax and output (thread = TMEM lane).  Warp 4: TMA of the code tiles from the pages.  Warp 5: MMA.  At head_dim 128 two CTAs
// share an SM (TMEM: S 0-127, O 128-255 each), at head_dim 256 one CTA has two S buffers (0-127, 128-255) and O at 256-511.
//
// kCopies: where a unit has at most 64 or 32 rows, they stand twice or four times in the 128 lanes, and copy c looks after its share of a tile's blocks of 32
// keys (P is zero in the others), with a reference, a sum and an accumulator of its own, which the CTA adds up at the end: the softmax of a tile is as much
// shorter, and the tensor cores, which take 128 rows whatever is in them, have no more to do.
#include <type_traits>
#include "dm_cache.cuh"
#include "dm_drafts.h"
#include "dm_kernels.h"

namespace dm {

namespace {

// Key tiles that a unit's queries and output are worth.
constexpr int kTreeCost = 2;
constexpr float kExact = 4194304.f;         // logits (log2) up to this size: whole numbers beside them are exact
constexpr float kReach = 40.f;              // what a row's logits may exceed its references by, in powers of two: fp32 has room for it

template <int kD>
struct TreeCfg {
  static constexpr int D = kD;
  static constexpr int kPanels = D / 128;                     // of 128 bytes, of a row of codes
  static constexpr int kSBufs = D == 128 ? 1 : 2;
  static constexpr int kCtasPerSm = D == 128 ? 2 : 1;
  static constexpr int kThreads = 192;
  static constexpr int kTile = 128 * D;                       // codes of K or V
  static constexpr int kStages = 4;                           // of a tile of K or V: K and V in turn
  static constexpr int kColO = 128 * kSBufs, kTmemCols = 256 * kPanels;
  static constexpr int kSmemQ = 0;                            // first codes, second codes; staging of the output
  static constexpr int kSmemRing = 2 * kTile;
  static constexpr int kSmemScales = kSmemRing + kStages * kTile;     // 8 tiles x (4 K scales, 4 exponents of V's)
  static constexpr int kSmemStats = kSmemScales + 8 * 32;     // of a lane: m, l, u
  static constexpr int kSmemRows = kSmemStats + 128 * 16;     // of a row: factor of its logits; where its output goes; by parity of the unit, whether it is marked; NaN tokens of two tiles
  static constexpr int kSmemBars = kSmemRows + 128 * 16 + 32;
  static constexpr int kSmemCum = kSmemBars + 256;            // 136 ints
  static constexpr int kSmem = kSmemCum + 136 * 4 + 1024;
  static_assert(kSmem + 1024 <= (228 * 1024) / kCtasPerSm, "shared memory of an SM");
};

// ------------------------------------------------------------------------------------------------ schedule
// A sequence's tokens and drafted tokens: the last `count` of its n.
struct TreeSeq {
  int n, count;
  __device__ __forceinline__ int base() const { return n - count; }
  __device__ __forceinline__ int tiles() const { return (n + 127) / 128; }
  __device__ __forceinline__ int row_tiles(const CacheTreeParams& p) const { return (count * p.rep + p.row_tile - 1) / p.row_tile; }
};
__device__ __forceinline__ TreeSeq tree_seq(const CacheTreeParams& p, int b) {
  TreeSeq s;
  s.n = cache_length(p.c, b);
  s.count = checked_count(p.c.status, p.counts, b, p.N);
  if (s.count > s.n) {
    report(p.c.status, kStatusBadLength + kInCache);
    s.count = s.n;
  }
  return s;
}
__device__ __forceinline__ int tree_steps(const CacheTreeParams& p, const TreeSeq& s) {
  return s.count > 0 ? (s.tiles() + kTreeCost) * s.row_tiles(p) * p.c.Hk : 0;
}
// Steps before each group of sequences (128 groups, as in dm_cache_sched.cuh), and the workers that share them.  Executed by the whole CTA (at least 128
// threads); `cum`: 129 ints + 4 of scratch.
struct TreeRange {
  int total, workers, chunk;
};
__device__ __forceinline__ TreeRange tree_range(const CacheTreeParams& p, int* cum) {
  const int tid = threadIdx.x, lane = tid & 31, chunk = (p.c.B + 127) / 128;
  int incl = 0;
  if (tid < 128) {
    for (int i = tid * chunk; i < min(p.c.B, (tid + 1) * chunk); ++i) incl += tree_steps(p, tree_seq(p, i));
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += o;
    }
    if (lane == 31) cum[129 + (tid >> 5)] = incl;
  }
  __syncthreads();
  if (tid < 128) {
    for (int w = 0; w < (tid >> 5); ++w) incl += cum[129 + w];
    cum[tid + 1] = incl;
    if (tid == 0) cum[0] = 0;
  }
  __syncthreads();
  const int total = cum[128];
  return TreeRange{total, min(p.grid, total), chunk};         // each has a step at least
}
__device__ __forceinline__ int tree_share(const TreeRange& r, int w) { return static_cast<int>(static_cast<int64_t>(w) * r.total / r.workers); }

// A CTA's piece of a unit: key tiles t0 ... t1 - 1 (none where only steps of the unit's own cost fall to the CTA).
struct TreePiece {
  int b, hk, rt;
  TreeSeq s;
  int begin, f0, f1;                                          // flat: of the unit; of the piece
  int t0, t1;
  __device__ __forceinline__ int end() const { return begin + s.tiles() + kTreeCost; }
  __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == s.tiles(); }
};
__device__ __forceinline__ void tree_cut(TreePiece& x, int f, int f_end) {
  x.f0 = f;
  x.f1 = min(f_end, x.end());
  x.t0 = max(0, f - x.begin - kTreeCost);
  x.t1 = max(0, x.f1 - x.begin - kTreeCost);
}
// The piece that begins at step f < f_end.
__device__ __forceinline__ TreePiece tree_first(const CacheTreeParams& p, const TreeRange& r, const int* cum, int f, int f_end) {
  int lo = 0, hi = 128;                                       // cum[lo] <= f < cum[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (cum[mid] <= f) lo = mid; else hi = mid;
  }
  TreePiece x;
  int off = f - cum[lo];
  for (x.b = lo * r.chunk;; ++x.b) {
    x.s = tree_seq(p, x.b);
    const int steps = tree_steps(p, x.s);
    if (off < steps) break;
    off -= steps;
  }
  const int unit_steps = x.s.tiles() + kTreeCost, unit = off / unit_steps, row_tiles = x.s.row_tiles(p);
  x.hk = unit / row_tiles;
  x.rt = unit - x.hk * row_tiles;
  x.begin = f - (off - unit * unit_steps);
  tree_cut(x, f, f_end);
  return x;
}
__device__ __forceinline__ bool tree_next(const CacheTreeParams& p, TreePiece& x, int f_end) {
  if (x.f1 >= f_end) return false;
  x.begin = x.f1;
  if (++x.rt >= x.s.row_tiles(p)) {
    x.rt = 0;
    if (++x.hk == p.c.Hk) {
      x.hk = 0;
      do {
        x.s = tree_seq(p, ++x.b);
      } while (x.s.count == 0);
    }
  }
  tree_cut(x, x.begin, f_end);
  return true;
}

// The nodes that node i sees, of word w: earlier ones and itself, whatever the bits behind it say.
__device__ __forceinline__ uint32_t seen_word(const uint32_t* seen, int i, int w) {
  if (w > i >> 5) return 0u;
  const uint32_t x = __ldg(seen + w);
  if (w < i >> 5) return x;
  const uint32_t self = 1u << (i & 31);
  return (x & (self - 1u)) | self;
}
// Which of 32 keys from `rel` (behind the first drafted token; negative: before it) node i sees.
__device__ __forceinline__ uint32_t seen_keys(const uint32_t* seen, int i, int rel) {
  const int w = rel >> 5;                                     // floor
  const uint32_t a = w < 0 ? 0xffffffffu : seen_word(seen, i, w), b = w + 1 < 0 ? 0xffffffffu : seen_word(seen, i, w + 1);
  return __funnelshift_r(a, b, rel & 31);
}

// ------------------------------------------------------------------------------------------------ one row
// Row (b, i, head) by one warp and from the definition: a key after the other, the logits' differences exact whatever their size.  For rows that the
// kernel below marks.
template <int D>
__device__ __noinline__ void tree_row(const CacheTreeParams& p, int b, int i, int head) {
  constexpr int kVecs = D / 128;
  const int lane = threadIdx.x & 31, bpp = p.c.page / 32, hk = head / p.rep;
  const TreeSeq t = tree_seq(p, b);
  const uint32_t* seen = p.seen + b * p.s_sb + i * p.s_sn;
  const __nv_bfloat162* q = reinterpret_cast<const __nv_bfloat162*>(p.q + b * p.q_sb + i * p.q_sn + head * p.q_sh) + 2 * lane;
  float4 qv[kVecs], acc[kVecs] = {};
#pragma unroll
  for (int x = 0; x < kVecs; ++x) {
    const float2 a = __bfloat1622float2(q[64 * x]), c = __bfloat1622float2(q[64 * x + 1]);
    qv[x] = make_float4(a.x, a.y, c.x, c.y);
  }
  float m = kNone;
  double l = 0.0;                                             // thousands of terms of one size, one after the other
  const float factor = p.scale * kLog2e;
  for (int j = 0; j <= t.base() + i; ++j) {
    if (j >= t.base()) {
      const int node = j - t.base();
      if (!((seen_word(seen, i, node >> 5) >> (node & 31)) & 1u)) continue;
    }
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
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s = __fmul_rn(s, __fmul_rn(factor, __ldg(p.c.ks + scale)));
    const float m_new = fmaxf(m, s), keep = exp2f(m - m_new), w = exp2f(s - m_new);
    m = m_new;
    l = l * keep + w;
#pragma unroll
    for (int x = 0; x < kVecs; ++x)
      acc[x] = make_float4(fmaf(acc[x].x, keep, w * v[x].x), fmaf(acc[x].y, keep, w * v[x].y), fmaf(acc[x].z, keep, w * v[x].z), fmaf(acc[x].w, keep, w * v[x].w));
  }
  __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(p.o + ((static_cast<int64_t>(b) * p.N + i) * p.H + head) * D) + 2 * lane;
  const float sum = static_cast<float>(l);
#pragma unroll
  for (int x = 0; x < kVecs; ++x) {
    o[64 * x] = __floats2bfloat162_rn(acc[x].x / sum, acc[x].y / sum);
    o[64 * x + 1] = __floats2bfloat162_rn(acc[x].z / sum, acc[x].w / sum);
  }
  if (lane == 0) p.lse[(static_cast<int64_t>(b) * p.H + head) * p.N + i] = (m + log2f(sum)) * kLn2;
}

// ------------------------------------------------------------------------------------------------ instructions
// Two floats -> two e5m2 codes (RNE, saturating): lo in bits 0-7, hi in bits 8-15.
__device__ __forceinline__ uint32_t cvt_e5m2x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Four values up to 448 -> four e4m3 codes, and the codes of what these leave.
__device__ __forceinline__ void split4(float2 x, float2 y, uint32_t& first, uint32_t& second) {
  asm("{\n\t.reg .b16 a, b;\n\t.reg .b32 h, g, u, v;\n\t"
      "cvt.rn.f16x2.f32 h, %3, %2;\n\tcvt.rn.f16x2.f32 g, %5, %4;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 a, h;\n\tcvt.rn.satfinite.e4m3x2.f16x2 b, g;\n\t"
      "mov.b32 %0, {a, b};\n\t"
      "cvt.rn.f16x2.e4m3x2 u, a;\n\tcvt.rn.f16x2.e4m3x2 v, b;\n\t"
      "sub.rn.f16x2 h, h, u;\n\tsub.rn.f16x2 g, g, v;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 a, h;\n\tcvt.rn.satfinite.e4m3x2.f16x2 b, g;\n\t"
      "mov.b32 %1, {a, b};\n\t}"
      : "=r"(first), "=r"(second) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
               "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}

// Whether `x` holds for all threads of a named barrier, which they meet at.
__device__ __forceinline__ bool all_of(int id, int nthreads, bool x) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %3, 0;\n\tbar.red.and.pred b, %1, %2, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
               : "=r"(r) : "r"(id), "r"(nthreads), "r"(x ? 1u : 0u) : "memory");
  return r != 0;
}

enum TreeBar : int {
  kFull = 0, kEmpty = 4,                    // of the ring
  kQ = 8,                                   // queries of the unit written
  kS = 9, kP = 11, kPv = 13,                // by S buffer: S computed, P written, P V done
  kScales = 15,                             // of running tile g: entry g % 8
  kTreeBars = 23,                           // behind them the TMEM slot and the abort flag
};

// ------------------------------------------------------------------------------------------------ main kernel
template <int kD, int kCopies>
__global__ void __launch_bounds__(TreeCfg<kD>::kThreads, TreeCfg<kD>::kCtasPerSm)
cache_tree_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ CacheTreeParams p) {
  using C = TreeCfg<kD>;
  constexpr int D = C::D, kRows = 128 / kCopies;              // rows of a unit
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023) & ~1023u) - raw);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kSmemBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kTreeBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kTreeBars + 1);
  int* cum = reinterpret_cast<int*>(smem + C::kSmemCum);
  float* scales = reinterpret_cast<float*>(smem + C::kSmemScales);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(bars + kFull + i, 1);
      mbar_init(bars + kEmpty + i, 1);
    }
    mbar_init(bars + kQ, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + kS + i, 1);
      mbar_init(bars + kP + i, 4);
      mbar_init(bars + kPv + i, 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(bars + kScales + i, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
    tc_fence_before();
  }
  grid_dep_wait();
  const TreeRange range = tree_range(p, cum);                 // its barriers publish the mbarriers and the TMEM slot too
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int worker = blockIdx.x;
  auto bar = [&](int i) { return smem_u32(bars + i); };
  // of running tile g: its S buffer, and the parity of that buffer's barriers
  auto buf_of = [&](int g) { return C::kSBufs == 2 ? g & 1 : 0; };
  auto parity_of = [&](int g) { return static_cast<uint32_t>(C::kSBufs == 2 ? g >> 1 : g) & 1u; };
  bool ok = true;

  if (worker < range.workers) {
    const int f_begin = tree_share(range, worker), f_end = tree_share(range, worker + 1);
    TreePiece x = tree_first(p, range, cum, f_begin, f_end);
    if (warp == 4) {
      // ---------------------------------------------------------------------------------------- TMA: code tiles and their scales
      // Lane i < 4 looks after block i of a tile.  A tile's pages are asked for two tiles ahead of its loads and its scales one tile ahead.
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
          more = tree_next(p, x, f_end);
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
      int j = 0;                                              // running stage
      Ahead now = look_up(), next = look_up();
      ask_scales(now);
      for (int g = 0; now.live && ok; ++g) {
        const Ahead after = look_up();
        ask_scales(next);
        if (lane < 4) {
          scales[(g & 7) * 8 + lane] = now.ks;                // zero where there is no block
          scales[(g & 7) * 8 + 4 + lane] = static_cast<float>(static_cast<int>(scale_to_sb(now.vs)) - 127);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + kScales + (g & 7));
        const int boxes = __popc(__ballot_sync(0xffffffffu, now.held)) * C::kPanels;
#pragma unroll 1
        for (int kv = 0; kv < 2 && ok; ++kv, ++j) {
          const int st = j % C::kStages;
          if (j >= C::kStages && !(ok = wait_warp(bar(kEmpty + st), (j / C::kStages - 1) & 1, abort_flag))) break;
          if (lane == 0) mbar_expect_tx(bars + kFull + st, boxes * 4096);
          __syncwarp();
          if (now.held) {
#pragma unroll
            for (int c = 0; c < C::kPanels; ++c)
              tma_load_4d(sbase + C::kSmemRing + st * C::kTile + c * 16384 + lane * 4096, kv ? &tv : &tk, bar(kFull + st), 128 * c, now.sub * 32, now.hk, now.page);
          }
        }
        now = next;
        next = after;
      }
      if (!ok) {
        if (lane == 0) raise_abort(abort_flag, p.c.status, kStatusTimeoutProducer + kInCache);
        // what is in flight lands before the shared memory goes
        for (int k = 1; k <= C::kStages; ++k)
          if (j >= k) wait_or_abort(bar(kFull + (j - k) % C::kStages), ((j - k) / C::kStages) & 1, abort_flag);
      }
    } else if (warp == 5) {
      // ---------------------------------------------------------------------------------------- MMA
      if (elect_one()) {
        constexpr uint32_t kIdescFirst = idesc_f8(128, 128, false, false), kIdescSecond = kIdescFirst | (1u << 7);     // A: e4m3; e5m2
        const uint32_t q_lo = desc_lo(sbase + C::kSmemQ), ring_lo = desc_lo(sbase + C::kSmemRing);
        int g = 0, units = 0;                                 // running tile
        // S of running tile h, behind all that read its buffer
        auto issue_s = [&](int h) -> bool {
          const int st = 2 * h % C::kStages;
          if (!wait_or_abort(bar(kFull + st), (2 * h / C::kStages) & 1, abort_flag)) return false;
          if (h >= C::kSBufs && !wait_or_abort(bar(kPv + buf_of(h)), parity_of(h - C::kSBufs), abort_flag)) return false;
          tc_fence_after();
          const uint32_t k_lo = ring_lo + st * (C::kTile >> 4), d = tmem + 128 * buf_of(h);
#pragma unroll
          for (int k = 0; k < D / 32; ++k) {
            const uint32_t off = (k >> 2) * (16384 >> 4) + (k & 3) * 2;
            mma_f8_ss(d, q_lo + off, k_lo + off, kIdescFirst, k > 0);
            mma_f8_ss(d, q_lo + (C::kTile >> 4) + off, k_lo + off, kIdescSecond, true);
          }
          tc_commit(bars + kS + buf_of(h));
          tc_commit(bars + kEmpty + st);
          return true;
        };
        do {
          if (x.t0 >= x.t1) continue;
          const int n = x.t1 - x.t0;
          if (!(ok = wait_or_abort(bar(kQ), units++ & 1, abort_flag))) break;
          if (!(ok = issue_s(g))) break;
          for (int i = 0; i < n && ok; ++i, ++g) {
            if (C::kSBufs == 2 && i + 1 < n && !(ok = issue_s(g + 1))) break;       // the next S, while the softmax is at this one
            const int st = (2 * g + 1) % C::kStages, held = min(4, (x.s.n - 128 * (x.t0 + i) + 31) / 32);        // blocks of the tile
            if (!(ok = wait_or_abort(bar(kP + buf_of(g)), parity_of(g), abort_flag) && wait_or_abort(bar(kFull + st), ((2 * g + 1) / C::kStages) & 1, abort_flag))) break;
            tc_fence_after();
            const uint32_t v_lo = ring_lo + st * (C::kTile >> 4), s = tmem + 128 * buf_of(g);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (k >= held) break;                           // P is zero there and V is not loaded
#pragma unroll
              for (int c = 0; c < C::kPanels; ++c) {
                mma_mxf8_ts(tmem + C::kColO + 128 * c, s + 32 * k, v_lo + c * (16384 >> 4) + k * (4096 >> 4), idesc_mxf8(128, 128, false, true, k, k), s + 16, s + 20,
                            i > 0 || k > 0);
                mma_mxf8_ts(tmem + C::kColO + 128 * c, s + 32 * k + 8, v_lo + c * (16384 >> 4) + k * (4096 >> 4), idesc_mxf8(128, 128, false, true, k, k), s + 16, s + 20,
                            true);
              }
            }
            tc_commit(bars + kEmpty + st);
            tc_commit(bars + kPv + buf_of(g));
            if (C::kSBufs == 1 && i + 1 < n && !(ok = issue_s(g + 1))) break;
          }
        } while (ok && tree_next(p, x, f_end));
        if (!ok) raise_abort(abort_flag, p.c.status, kStatusTimeoutMma + kInCache);
      }
    } else {
      // ---------------------------------------------------------------------------------------- queries, softmax, output
      const int row = tid & (kRows - 1);                      // of the unit
      const int copy = tid / kRows;                           // looks after blocks copy * 4 / kCopies ... of a tile
      constexpr int kBlocks = 4 / kCopies;
      const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
      float4* stats = reinterpret_cast<float4*>(smem + C::kSmemStats);
      float* factors = reinterpret_cast<float*>(smem + C::kSmemRows);
      int* out_rows = reinterpret_cast<int*>(smem + C::kSmemRows) + 128;
      volatile uint32_t* nan_tokens = reinterpret_cast<volatile uint32_t*>(smem + C::kSmemRows) + 512;      // of a tile, by its parity
      int g = 0, units = 0;                                   // running tile, running unit
      do {
        if (x.t0 >= x.t1) continue;
        // (by parity: a warp may be at the next unit's queries while another looks at this one's marks)
        volatile int* marks = reinterpret_cast<volatile int*>(smem + C::kSmemRows) + 256 + 128 * (units++ & 1);
        // Queries, two codes an element, in the layout of the 128-byte swizzle.  A row's lanes take eight elements each.
        {
          constexpr int kLanes = D / 8, kPer = 32 / kLanes, kOwn = kRows / 4, kBatch = kOwn / kPer < 4 ? kOwn / kPer : 4;
          const int l = lane % kLanes;
#pragma unroll 1
          for (int r0 = 0; r0 < kOwn; r0 += kBatch * kPer) {
            uint4 w[kBatch];
            int at_row[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
              const int r = warp * kOwn + r0 + k * kPer + lane / kLanes, unit_row = x.rt * kRows + r, i = unit_row / p.rep, head = x.hk * p.rep + unit_row - i * p.rep;
              w[k] = make_uint4(0, 0, 0, 0);
              at_row[k] = -1;
              if (i < x.s.count) {
                w[k] = __ldg(reinterpret_cast<const uint4*>(p.q + x.b * p.q_sb + i * p.q_sn + head * p.q_sh) + l);
                at_row[k] = (x.b * p.N + i) * p.H + head;
              }
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
              const int r = warp * kOwn + r0 + k * kPer + lane / kLanes;
              const uint32_t v[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
              // the largest size, as bits: NaN and infinities are above all others
              uint32_t top = __vmaxu2(__vmaxu2(v[0] & 0x7FFF7FFFu, v[1] & 0x7FFF7FFFu), __vmaxu2(v[2] & 0x7FFF7FFFu, v[3] & 0x7FFF7FFFu));
              top = max(top & 0xFFFFu, top >> 16);
#pragma unroll
              for (int o = kLanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
              const uint32_t eb = min(254u, max(14u, top >> 7));
              const float up = sb_to_scale(261u - eb);        // largest element to [2^7, 2^8)
              uint32_t first[2], second[2];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float a = __uint_as_float(v[e] << 16) * up, b = __uint_as_float(v[e] & 0xFFFF0000u) * up;
                const uint32_t code = cvt_e4m3x2(a, b);
                const float2 back = f16x2_to_float2(e4m3_lo_f16x2(code));
                const uint32_t rest = cvt_e5m2x2(a - back.x, b - back.y);
                first[e >> 1] = (e & 1) ? first[e >> 1] | code << 16 : code;
                second[e >> 1] = (e & 1) ? second[e >> 1] | rest << 16 : rest;
              }
#pragma unroll
              for (int c = 0; c < kCopies; ++c) {
                const uint32_t at = sbase + C::kSmemQ + (l >> 4) * 16384 + (r + c * kRows) * 128 + ((((l & 15) >> 1) ^ (r & 7)) << 4) + (l & 1) * 8;
                sts_f2(at, __uint_as_float(first[0]), __uint_as_float(first[1]));
                sts_f2(at + C::kTile, __uint_as_float(second[0]), __uint_as_float(second[1]));
              }
              if (l == 0) {                                   // of a row of NaN or infinities the factor is NaN
                factors[r] = top >= 0x7F80u ? CUDART_NAN_F : sb_to_scale(eb - 7u) * p.scale * kLog2e;
                out_rows[r] = at_row[k];
                marks[r] = 0;
              }
            }
          }
          fence_async_smem();
          bar_sync(1, 128);
          if (lane == 0) mbar_arrive(bars + kQ);
        }
        const int unit_row = x.rt * kRows + row, node = unit_row / p.rep;
        const bool real = node < x.s.count;
        const bool idle = !__any_sync(0xffffffffu, real);     // a warp of rows that are none
        const uint32_t* seen = p.seen + x.b * p.s_sb + static_cast<int64_t>(min(node, x.s.count - 1)) * p.s_sn;
        const float f = factors[row];
        // Of the row, whole numbers: m, the reference of the sum l; u, that of the products of a probability and its V scale, in which O counts.  They
        // move only when a row's logits exceed them by more than 2^kReach.
        float m = kNone, u = kNone, l = 0.f;
        bool marked = false;
        // One key tile.  kCut: some row does not see all its keys (a compile-time variant: no select per element elsewhere).
        auto tile = [&](int t, auto cut_tag) -> bool {
          constexpr bool kCut = decltype(cut_tag)::value;
          const uint32_t entry = sbase + C::kSmemScales + (g & 7) * 32, t_s = tmem + lanes + 128 * buf_of(g);
          const int c0 = kCopies == 1 ? 0 : copy * kBlocks;
          uint32_t s_buf[2][32];
          tmem_ld32(t_s + 32 * c0, s_buf[0]);
          float kb[kBlocks], ev[kBlocks], sums[kBlocks];
#pragma unroll
          for (int c = 0; c < kBlocks; ++c) {
            const float fc = f * lds_f(entry + 4 * (c0 + c));
            ev[c] = lds_f(entry + 16 + 4 * (c0 + c));
            tmem_wait_ld();
            if (c < kBlocks - 1) tmem_ld32(t_s + 32 * (c0 + c + 1), s_buf[(c + 1) & 1]);
            uint32_t (&s)[32] = s_buf[c & 1];
            uint32_t sees = 0xffffffffu;
            if (kCut) {
              sees = real ? seen_keys(seen, node, 128 * t + 32 * (c0 + c) - x.s.base()) : 0u;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((sees >> e) & 1u)) s[e] = 0xff800000u;
              marked |= (sees & nan_tokens[4 * (g & 1) + c0 + c]) != 0u;
            }
            float2 s2[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) s2[e] = make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
            const float top = max32(s2);
            kb[c] = kCut && sees == 0u ? kNone : fmaxf(ceilf(top * fc), kNone);
            const float2 f2 = splat2(fc), off = splat2(8.f - kb[c]);
            float2 sum = make_float2(0.f, 0.f);
            uint32_t w[16];                                   // first codes, second codes
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              float2 y[2];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                y[k] = fma2(s2[e + k], f2, off);
                if (kCut) {                                   // (zero times infinity is none)
                  if (!((sees >> (2 * (e + k))) & 1u)) y[k].x = -CUDART_INF_F;
                  if (!((sees >> (2 * (e + k) + 1)) & 1u)) y[k].y = -CUDART_INF_F;
                }
                y[k] = ex2_2(y[k]);
                sum = add2(sum, y[k]);
              }
              split4(y[0], y[1], w[e / 2], w[8 + e / 2]);
            }
            sums[c] = sum.x + sum.y;
            tmem_st16(t_s + 32 * (c0 + c), w);                // over columns that have been read
          }
          if (kCopies > 1) {                                  // other copies' blocks
            const uint32_t zeros[16] = {};
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (c < c0 || c >= c0 + kBlocks) tmem_st16(t_s + 32 * c, zeros);
          }
          float top = kb[0], top_u = kb[0] + ev[0];
#pragma unroll
          for (int c = 1; c < kBlocks; ++c) {
            top = fmaxf(top, kb[c]);
            top_u = fmaxf(top_u, kb[c] + ev[c]);
          }
          marked |= fabsf(top) > kExact && top > kNone;
          const bool moves = top > m + kReach || top_u > u + kReach;
          if (__any_sync(0xffffffffu, moves)) {
            float keep = 1.f;
            if (moves) {
              l *= ex2_approx(m - top);
              keep = ex2_approx(u - top_u);
              m = top;
              u = top_u;
            }
            if (t > x.t0) {
              if (C::kSBufs == 2) {                           // (with one buffer this S came behind those products)
                if (!wait_warp(bar(kPv + buf_of(g - 1)), parity_of(g - 1), abort_flag)) return false;
                tc_fence_after();
              }
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(tmem + lanes + C::kColO + 32 * c, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                tmem_st32(tmem + lanes + C::kColO + 32 * c, o);
              }
            }
          }
          uint32_t word = 0x7F7F7F7Fu;                        // scale bytes of P's codes, 2^(kb + ev - u - 8)
#pragma unroll
          for (int c = 0; c < kBlocks; ++c) {
            l = fmaf(sums[c], ex2_approx(kb[c] - m - 8.f), l);
            const uint32_t sb = static_cast<uint32_t>(fminf(fmaxf(kb[c] + ev[c] - u + 119.f, 0.f), 254.f));
            if (kCopies == 1) word = c == 0 ? sb : word | sb << (8 * c);
            else word = (word & ~(0xFFu << (8 * (c0 + c)))) | sb << (8 * (c0 + c));
          }
          const uint32_t words[8] = {word, word, word, word, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu};
          tmem_st8(t_s + 16, words);
          return true;
        };
        for (int t = x.t0; t < x.t1; ++t, ++g) {
          ok = wait_warp(bar(kScales + (g & 7)), (g >> 3) & 1, abort_flag) && wait_warp(bar(kS + buf_of(g)), parity_of(g), abort_flag);
          if (!ok) break;
          tc_fence_after();
          const bool cut = 128 * (t + 1) > x.s.base();
          if (cut) {
            // V's slots behind the length hold anything, and a drafted token may be NaN, which only the rows that see it are to meet: zeros in the place of both, or
            // they would come through the products with P's zeros.  Which tokens were NaN is left to the rows.  A thread a token.
            const int st = (2 * g + 1) % C::kStages, j = 128 * t + tid;
            ok = wait_warp(bar(kFull + st), ((2 * g + 1) / C::kStages) & 1, abort_flag);
            bool nan = false;
            if (ok && j >= x.s.base() && 128 * t + warp * 32 < x.s.n) {         // in a block that is there
              const uint32_t at = sbase + C::kSmemRing + st * C::kTile + tid * 128;
              auto piece = [&](int y) { return at + (y >> 3) * 16384 + (((y ^ lane) & 7) << 4); };      // lanes on different banks
              uint32_t found = 0;
#pragma unroll
              for (int y = 0; y < 8 * C::kPanels; ++y) {
                const float4 w = lds_f4(piece(y));
                found |= nan_codes(__float_as_uint(w.x)) | nan_codes(__float_as_uint(w.y)) | nan_codes(__float_as_uint(w.z)) | nan_codes(__float_as_uint(w.w));
              }
              if (found != 0 || j >= x.s.n) {
#pragma unroll 1
                for (int y = 0; y < 8 * C::kPanels; ++y) sts_u4(piece(y), 0u, 0u, 0u, 0u);
                fence_async_smem();
              }
              nan = found != 0 && j < x.s.n;
            }
            const uint32_t nans = __ballot_sync(0xffffffffu, nan);
            if (lane == 0) nan_tokens[4 * (g & 1) + warp] = nans;
            if (!(ok = all_of(1, 128, ok))) break;
          }
          if (!idle && !(ok = cut ? tile(t, std::true_type{}) : tile(t, std::false_type{}))) break;
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + kP + buf_of(g));
        }
        // (the four warps give up together: barriers follow)
        if (ok) ok = wait_warp(bar(kPv + buf_of(g - 1)), parity_of(g - 1), abort_flag);
        if (!(ok = all_of(1, 128, ok))) break;
        tc_fence_after();
        // Output.  Over the copies of a row: the largest references, the sum; each lane's values count w of it.
        const bool whole = x.whole();
        stats[tid] = make_float4(m, l, u, 0.f);
        if (kCopies > 1) bar_sync(1, 128);
        float m_all = m, u_all = u, l_all = l, w = 1.f;
        if (kCopies > 1) {
          float4 st[kCopies];
#pragma unroll
          for (int c = 0; c < kCopies; ++c) {
            st[c] = stats[row + c * kRows];
            m_all = fmaxf(m_all, st[c].x);
            u_all = fmaxf(u_all, st[c].z);
          }
          l_all = 0.f;
#pragma unroll
          for (int c = 0; c < kCopies; ++c) l_all = fmaf(st[c].y, ex2_approx(st[c].x - m_all), l_all);
          w = ex2_approx(u - u_all);
        }
        // (in two factors: what V's scales leave may be beyond either's range)
        const float d_all = u_all - m_all, d1 = fminf(fmaxf(d_all, -100.f), 100.f);
        const float w1 = whole ? w * exp2f(d1) : w, w2 = whole ? exp2f(d_all - d1) / l_all : 1.f;
        const int slot = 2 * worker + (x.f0 == f_begin ? 0 : 1);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          const uint32_t stage = sbase + C::kSmemQ + (c & 1) * 16384;         // 128 lanes x 128 bytes, 16-byte pieces XORed with the lane
          uint32_t o[32];
          tmem_ld32(tmem + lanes + C::kColO + 32 * c, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float4 y = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
            y = make_float4(y.x * w1 * w2, y.y * w1 * w2, y.z * w1 * w2, y.w * w1 * w2);
            sts_u4(stage + tid * 128 + ((e ^ (lane & 7)) << 4), __float_as_uint(y.x), __float_as_uint(y.y), __float_as_uint(y.z), __float_as_uint(y.w));
          }
          if (kCopies > 1) bar_sync(1, 128);
          else __syncwarp();
          // eight lanes a row, four rows a warp at a time
#pragma unroll
          for (int k = 0; k < 8 / kCopies; ++k) {
            const int r = (kCopies == 1 ? warp * 32 : warp * (kRows / 4)) + 4 * k + (lane >> 3), piece = lane & 7;
            float4 y = lds_f4(stage + r * 128 + ((piece ^ (r & 7)) << 4));
#pragma unroll
            for (int cc = 1; cc < kCopies; ++cc) {
              const float4 z = lds_f4(stage + (r + cc * kRows) * 128 + ((piece ^ (r & 7)) << 4));
              y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
            }
            const int at = out_rows[r];
            if (at < 0) continue;
            if (whole) {
              const __nv_bfloat162 a = __floats2bfloat162_rn(y.x, y.y), b = __floats2bfloat162_rn(y.z, y.w);
              *reinterpret_cast<uint2*>(p.o + static_cast<int64_t>(at) * D + 32 * c + 4 * piece) =
                  make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
            } else {
              *reinterpret_cast<float4*>(p.part_o + (static_cast<int64_t>(slot) * kRows + r) * D + 32 * c + 4 * piece) = y;
            }
          }
        }
        if (real && marked) marks[row] = 1;
        bar_sync(1, 128);                                     // marks are seen; and the staging has been read: the next queries may come
        const bool mine = copy == 0 && real;
        const bool again = mine && marks[row] != 0;
        if (whole) {
          const int head = x.hk * p.rep + unit_row - node * p.rep;
          if (mine) p.lse[(static_cast<int64_t>(x.b) * p.H + head) * p.N + node] = (m_all + log2f(l_all)) * kLn2;
          for (uint32_t left = __ballot_sync(0xffffffffu, again); left != 0; left &= left - 1) {
            const int from = __ffs(left) - 1;
            __syncwarp();
            tree_row<D>(p, x.b, __shfl_sync(0xffffffffu, node, from), __shfl_sync(0xffffffffu, head, from));
          }
        } else if (mine) {
          p.part_ml[static_cast<int64_t>(slot) * kRows + row] = make_float4(m_all, l_all, u_all, again ? 1.f : 0.f);
        }
        tc_fence_before();
      } while (tree_next(p, x, f_end));
      if (!ok && lane == 0) raise_abort(abort_flag, p.c.status, kStatusTimeoutCompute + kInCache);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// ------------------------------------------------------------------------------------------------ join
// The pieces of cut units: where worker j of the main kernel goes on with a unit that worker j - 1 began, the CTAs (j, ...) join it, a warp a row; and the
// rows behind the counts.
constexpr int kJoinParts = 8;

template <int D>
__global__ void __launch_bounds__(128) cache_tree_join_kernel(const __grid_constant__ CacheTreeParams p) {
  constexpr int kVecs = D / 128;
  __shared__ int cum[136];
  grid_dep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // rows behind the counts: zeros
  for (int b = blockIdx.x; b < p.c.B; b += gridDim.x)
    for (int i = tree_seq(p, b).count + blockIdx.y; i < p.N; i += kJoinParts) {
      uint4* o = reinterpret_cast<uint4*>(p.o + (static_cast<int64_t>(b) * p.N + i) * p.H * D);
      for (int z = threadIdx.x; z < p.H * D / 8; z += 128) o[z] = make_uint4(0, 0, 0, 0);
      for (int z = threadIdx.x; z < p.H; z += 128) p.lse[(static_cast<int64_t>(b) * p.H + z) * p.N + i] = -CUDART_INF_F;
    }
  const TreeRange range = tree_range(p, cum);
  const int j = blockIdx.x;
  if (j == 0 || j >= range.workers) return;
  const int f = tree_share(range, j);
  const TreePiece x = tree_first(p, range, cum, f, f + 1);
  if (x.begin >= f || tree_share(range, j - 1) > x.begin) return;        // no cut, or not the unit's first
  auto worker_at = [&](int step) {                            // whose share it is: share(lo) <= step < share(hi)
    int lo = j - 1, hi = range.workers;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (tree_share(range, mid) <= step) lo = mid; else hi = mid;
    }
    return lo;
  };
  // of the tiles; workers before them have steps of the unit's own cost alone and no piece
  const int first = worker_at(x.begin + kTreeCost), last = worker_at(x.end() - 1);
  if (first == last) return;                                  // whole: written by that worker
  auto slot_of = [&](int w) { return 2 * w + (w == j - 1 && tree_share(range, w) < x.begin ? 1 : 0); };
  for (int r = blockIdx.y * 4 + warp; r < p.row_tile; r += 4 * kJoinParts) {
    const int unit_row = x.rt * p.row_tile + r, node = unit_row / p.rep, head = x.hk * p.rep + unit_row - node * p.rep;
    if (node >= x.s.count) break;
    float top = kNone, u_top = kNone, sum = 0.f;
    float4 acc[kVecs] = {};
    bool marked = false;
    // 32 results at a time, a lane each: their maxima and sums together, then the values of those that count
    for (int w0 = first; w0 <= last; w0 += 32) {
      const int w = w0 + lane;
      const bool there = w <= last;                           // each has a tile at least
      const int64_t at = there ? static_cast<int64_t>(slot_of(w)) * p.row_tile + r : 0;
      const float4 ml = there ? p.part_ml[at] : make_float4(kNone, 0.f, kNone, 0.f);
      marked |= __any_sync(0xffffffffu, ml.w != 0.f);
      float top_new = ml.x, u_new = ml.z;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        top_new = fmaxf(top_new, __shfl_xor_sync(0xffffffffu, top_new, o));
        u_new = fmaxf(u_new, __shfl_xor_sync(0xffffffffu, u_new, o));
      }
      top_new = fmaxf(top, top_new);
      u_new = fmaxf(u_top, u_new);
      float l = ml.y * ex2_approx(ml.x - top_new);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      sum = sum * ex2_approx(top - top_new) + l;
      const float a = ex2_approx(u_top - u_new), wgt = ex2_approx(ml.z - u_new);
      top = top_new;
      u_top = u_new;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) acc[v] = make_float4(acc[v].x * a, acc[v].y * a, acc[v].z * a, acc[v].w * a);
      const uint32_t counts = __ballot_sync(0xffffffffu, there && ml.x > kNone);          // kNone: the row sees nothing of the piece
#pragma unroll 4
      for (int k = 0; k < min(32, last - w0 + 1); ++k) {
        const float w_k = __shfl_sync(0xffffffffu, wgt, k);
        const int64_t at_k = __shfl_sync(0xffffffffu, at, k);
        if (!((counts >> k) & 1)) continue;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          const float4 y = reinterpret_cast<const float4*>(p.part_o + at_k * D)[32 * v + lane];
          acc[v] = make_float4(fmaf(y.x, w_k, acc[v].x), fmaf(y.y, w_k, acc[v].y), fmaf(y.z, w_k, acc[v].z), fmaf(y.w, w_k, acc[v].w));
        }
      }
    }
    if (marked) {
      tree_row<D>(p, x.b, node, head);
      continue;
    }
    const float d_all = u_top - top, d1 = fminf(fmaxf(d_all, -100.f), 100.f);
    const float w1 = exp2f(d1), w2 = exp2f(d_all - d1) / sum;
    __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(p.o + ((static_cast<int64_t>(x.b) * p.N + node) * p.H + head) * D) + 2 * lane;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      o[64 * v] = __floats2bfloat162_rn(acc[v].x * w1 * w2, acc[v].y * w1 * w2);
      o[64 * v + 1] = __floats2bfloat162_rn(acc[v].z * w1 * w2, acc[v].w * w1 * w2);
    }
    if (lane == 0) p.lse[(static_cast<int64_t>(x.b) * p.H + head) * p.N + node] = (top + log2f(sum)) * kLn2;
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

template <int D, int kCopies>
cudaError_t launch_tree(const CUtensorMap& tk, const CUtensorMap& tv, const CacheTreeParams& p, cudaStream_t stream) {
  using C = TreeCfg<D>;
  cudaError_t e = allow_smem<cache_tree_kernel<D, kCopies>>(C::kSmem);
  if (e != cudaSuccess) return e;
  count_launch();
  e = launch_chained(cache_tree_kernel<D, kCopies>, dim3(p.grid), C::kThreads, C::kSmem, stream, tk, tv, p);
  if (e != cudaSuccess) return e;
  count_launch();
  return launch_chained(cache_tree_join_kernel<D>, dim3(p.grid, kJoinParts), 128, 0, stream, p);
}

}  // namespace

CacheTreePlan plan_cache_tree(int B, int N, int H, int Hk, int D, int T, int page) {
  CacheTreePlan x;
  const int64_t R = static_cast<int64_t>(N) * (H / Hk);
  x.row_tile = R <= 32 ? 32 : R <= 64 ? 64 : 128;
  const int64_t wave = static_cast<int64_t>(sm_count()) * (D == 128 ? TreeCfg<128>::kCtasPerSm : TreeCfg<256>::kCtasPerSm);
  const int64_t tiles = static_cast<int64_t>(B) * Hk * ((R + x.row_tile - 1) / x.row_tile) * ((static_cast<int64_t>(T) * page + 127) / 128);
  x.grid = static_cast<int>(tiles < wave ? tiles : wave);      // one wave, and no more workers than there can be tiles
  x.part_o_bytes = 2ll * x.grid * x.row_tile * D * 4;
  x.part_ml_bytes = 2ll * x.grid * x.row_tile * 16;
  return x;
}

cudaError_t launch_cache_tree(int D, const CUtensorMap& tk, const CUtensorMap& tv, const CacheTreeParams& p, cudaStream_t stream) {
  if (D == 128)
    return p.row_tile == 32 ? launch_tree<128, 4>(tk, tv, p, stream) : p.row_tile == 64 ? launch_tree<128, 2>(tk, tv, p, stream) : launch_tree<128, 1>(tk, tv, p, stream);
  return p.row_tile == 32 ? launch_tree<256, 4>(tk, tv, p, stream) : p.row_tile == 64 ? launch_tree<256, 2>(tk, tv, p, stream) : launch_tree<256, 1>(tk, tv, p, stream);
}

}  // namespace dm
