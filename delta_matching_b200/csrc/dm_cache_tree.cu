// Attention of a tree of drafted tokens over the 8-bit cache.
//
//   s_rj = scale q_r . (ks code_j);  o_r = sum_j exp(s_rj - m_r) vs code_j / sum_j exp(s_rj - m_r)  over the keys j that row r sees:
//   all tokens held before the drafted ones, and of these its node's own ancestors and itself
//
// Rows are (drafted token, head of the kv head's group); a unit is (sequence, kv head, up to 128 rows).  The codes of K and V go to the tensor cores as
// they lie in the pages, no code is ever converted: S = Q K^T is the sum of two kind::f8f6f4 chains with q in two codes, e4m3 and what that leaves in e5m2
// (4 and 3 significant bits, of bf16's 8 with the signs: exact down to 2^-13 of the row's largest element, 2^-21 of that off below), and O += P V the sum
// of two block-scaled chains with P in two e4m3 codes relative to the largest of its 32 keys (off by 2^-9 of itself at most, what bf16 would keep of it, and 2^-16 of that largest
// one where it is small).  The power-of-two scale of V's block goes into P's scale byte and that of K's block into the factor of the logits.
//
// The key tiles of 128 tokens of all units are one flat range, divided evenly over the CTAs of one wave; pieces of cut units are joined by a second kernel.  Where units
// have few tiles a cluster takes each, and joins it itself.
// One CTA an SM.  Three teams of four softmax warps (thread = TMEM lane; two teams at head_dim 256) take the tiles of a unit in turn, each with an S buffer in TMEM;
// P's codes and scale bytes lie over the S that they come from.  Of the last four warps two load the code tiles of K and of V from the pages by TMA and two issue the MMAs.
// The power of two that a row of O counts in is fixed by the unit's first blocks: fp32 has room for what may follow (rows for which it has not are marked and made by
// themselves when the tiles are done with), and no team waits for another's maximum.
//
// kCopies: where a unit has at most 64 or 32 rows, they stand twice or four times in the 128 lanes, and copy c looks after its share of a tile's blocks of 32
// keys (P is zero in the others), with a reference, a sum and an accumulator of its own, which the CTA adds up at the end: the softmax of a tile is as much
// shorter, and the tensor cores, which take 128 rows whatever is in them, have no more to do.
//
// Measured (H 32, Hk 8, head_dim 128 but for the last two): 4 sequences of 4000 tokens with 16 drafts 19.4 us; 64 of 4096 with 8 drafts 130 us, 4.1 TB/s of codes, with 25 183 us;
// one of 65536 with 60 drafts of 64 heads 164 us; 8 of 6144 with 33 drafts of 16 heads of 256 101 us, 4.0 TB/s.  What bounds it: with few rows the chain softmax, P V, next S
// of a buffer (2100 cycles behind a tile's 1000; the products of a tile alone take 1024) and 7000 cycles from a unit's last tile to the next one's first; with 128 rows the softmax (1350 cycles a
// tile at saturation, of about 2250).  Above a hundred us the chip is at its power limit (1.4 - 1.7 GHz).  Small calls: 5000 cycles to the first S, 9000 from the last
// tile to the end of the cluster's join, of 32000.
#include <cooperative_groups.h>
#include <type_traits>
#include "dm_cache.cuh"
#include "dm_drafts.h"
#include "dm_kernels.h"

namespace dm {

namespace {

namespace cg = cooperative_groups;

constexpr int kMaxCluster = 8;

// Key tiles that a unit's queries and output are worth (8 instead: as fast to 2 % in calls of 4 x 8000 to 64 x 4096 tokens; 2: 5 % slower in the first).
constexpr int kTreeCost = 4;
// Marks of a row: channels of it become NaN; it is made by itself.
constexpr int kNanChannels = 1, kByItself = 2;
constexpr float kExact = 4194304.f;         // logits (log2) up to this size: whole numbers beside them are exact
constexpr float kReach = 40.f;              // what a row's logits may exceed the reference of its sum by, in powers of two: fp32 has room for it
constexpr int kUnitLift = 40;               // of the reference of the products, above those it was taken from
// What a V scale counts for that, at least: a block of zeros (padding at a sequence's head) has 2^-126, and the products behind it may be of any size.  80 above such a block's products
// still leaves them 2^-29 to the right.
constexpr float kLeastScale = -86.f;

template <int kD>
struct TreeCfg {
  static constexpr int D = kD;
  static constexpr int kPanels = D / 128;                     // of 128 bytes, of a row of codes
  static constexpr int kTeams = D == 128 ? 3 : 2;             // of four softmax warps, each with an S buffer: a tile goes to the next team
  static constexpr int kThreads = 128 * (kTeams + 1);
  static constexpr int kRegsSoftmax = 144, kRegsOther = 80;   // of 128 at launch (head_dim 128)
  static_assert(D != 128 || kTeams * kRegsSoftmax + kRegsOther <= (kTeams + 1) * 128, "a split above the launch's own registers would wait for ever");
  static constexpr int kTile = 128 * D;                       // codes of K or V
  static constexpr int kStages = D == 128 ? 10 : 4;           // of a tile of K or V: K and V in turn
  static constexpr int kColO = 128 * kTeams;                  // TMEM: S buffers, then O
  static constexpr int kSmemQ = 0;                            // first codes, second codes
  static constexpr int kSmemRing = 2 * kTile;
  static constexpr int kSmemOut = kSmemRing + kStages * kTile;        // staging of the output, 128 lanes x 64 bytes a team
  static constexpr int kSmemStats = kSmemOut + kTeams * 8192; // by team and lane: m, l
  static constexpr int kSmemU = kSmemStats + kTeams * 1024;   // by parity of the unit and lane: u
  static constexpr int kSmemRows = kSmemU + 1024;              // by parity of the unit and row: factor of its logits; where its output goes; whether it is marked
  static constexpr int kSmemScales = kSmemRows + 2 * 128 * 12;        // 8 tiles x (4 K scales, 4 exponents of V's)
  static constexpr int kSmemNan = kSmemScales + 8 * 32;       // by S buffer: which tokens of a tile are NaN
  static constexpr int kSmemSums = kSmemNan + 64;             // of a row, for the cluster: m, l, u, marked
  static constexpr int kSmemBars = kSmemSums + 2048;
  static constexpr int kSmem = kSmemBars + 528 + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
};

// ------------------------------------------------------------------------------------------------ schedule
// A sequence's tokens and drafted tokens: the last `count` of its n.
struct TreeSeq {
  int n, count;
  __device__ __forceinline__ int base() const { return n - count; }
  __device__ __forceinline__ int tiles() const { return (n + 127) / 128; }
  __device__ __forceinline__ int row_tiles(const CacheTreeParams& p) const { return (count * p.rep + p.row_tile - 1) >> p.row_shift; }
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
// Rows -> drafted token: r / rep.
__device__ __forceinline__ int node_of(const CacheTreeParams& p, int r) { return p.rep == 1 ? r : p.rep_magic != 0 ? static_cast<int>(__umulhi(r, p.rep_magic)) : r / p.rep; }

// The steps of all sequences, which the workers share evenly.  Each warp reckons for itself, a lane a group of sequences.
struct TreeRange {
  int total, workers, quot, rest;
  __device__ __forceinline__ int share(int w) const { return w * quot + static_cast<int>(static_cast<unsigned>(w) * static_cast<unsigned>(rest) / static_cast<unsigned>(workers)); }
};
__device__ __forceinline__ int warp_scan(int x) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, x, off);
    if ((threadIdx.x & 31) >= off) x += o;
  }
  return x;
}
// Steps before and in sequences a ... of lane's group, for groups of `size` sequences from `from`, none behind `to`: the inclusive sums.
__device__ __forceinline__ int tree_sums(const CacheTreeParams& p, int from, int to, int size) {
  int x = 0;
  const int first = from + (threadIdx.x & 31) * size, last = min(to, first + size);
  for (int b = first; b < last; ++b) x += tree_steps(p, tree_seq(p, b));
  return warp_scan(x);
}
__device__ __forceinline__ TreeRange tree_range(const CacheTreeParams& p, int& sums) {
  sums = tree_sums(p, 0, p.c.B, (p.c.B + 31) / 32);
  TreeRange r;
  r.total = __shfl_sync(0xffffffffu, sums, 31);
  r.workers = max(1, min(p.grid, r.total));                   // each has a step at least (where there are any)
  r.quot = r.total / r.workers;
  r.rest = r.total - r.quot * r.workers;
  return r;
}

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
// The piece that begins at step f < f_end.  `sums`: of tree_range.
__device__ __forceinline__ TreePiece tree_first(const CacheTreeParams& p, int sums, int f, int f_end) {
  TreePiece x;
  int off = f, size = (p.c.B + 31) / 32, from = 0, to = p.c.B;
  for (;;) {
    const int lane = __ffs(__ballot_sync(0xffffffffu, sums > off)) - 1, before = __shfl_sync(0xffffffffu, sums, max(0, lane - 1));
    if (lane > 0) off -= before;
    from += lane * size;
    to = min(to, from + size);
    if (size == 1) break;
    size = (size + 31) / 32;
    sums = tree_sums(p, from, to, size);
  }
  x.b = from;
  x.s = tree_seq(p, x.b);
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
// Rows that the kernels below mark are seen to by one warp each, always when the tiles are done with: nothing that waits with a limit may wait for it.
//
// Row (b, i, head) from the definition: a key after the other, the logits' differences exact whatever their size.  About 0.6 us a key.
template <int D>
__device__ __forceinline__ void tree_row(const CacheTreeParams& p, int b, int i, int head) {
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

// NaN in the channels of row (b, i, head) in which a drafted token that it sees has NaN values, where the tiles had zeros in their place.  (Keys that are NaN need nothing of the kind: their
// logits are.)  64 sequences of 1000 tokens with 25 drafts take 0.25 ms instead of 0.09 where one of them has such a token, 19 where its rows were made by themselves instead.
template <int D>
__device__ __forceinline__ void nan_channels(const CacheTreeParams& p, int b, int i, int head) {
  const int lane = threadIdx.x & 31, bpp = p.c.page / 32, hk = head / p.rep, base = tree_seq(p, b).base();
  const uint32_t* seen = p.seen + b * p.s_sb + i * p.s_sn;
  uint16_t* o = reinterpret_cast<uint16_t*>(p.o + ((static_cast<int64_t>(b) * p.N + i) * p.H + head) * D) + 4 * lane;
  __syncwarp();                                               // the row stands, by whichever lanes
#pragma unroll 1
  for (int node = 0; node <= i; ++node) {
    if (!((seen_word(seen, i, node >> 5) >> (node & 31)) & 1u)) continue;
    const int j = base + node, blk = j / 32, page = max(0, checked_page(p.c, __ldg(p.c.table + b * p.c.t_row + blk / bpp)));
    const uint8_t* code = p.c.v8 + page * p.c.c_page + hk * p.c.c_head + (blk % bpp * 32 + j % 32) * p.c.c_slot + 4 * lane;
#pragma unroll 1
    for (int x = 0; x < D; x += 128) {
      const uint32_t bad = nan_codes(__ldg(reinterpret_cast<const uint32_t*>(code + x)));
      for (int e = 0; e < 4; ++e)
        if ((bad >> (8 * e)) & 1u) o[x + e] = 0x7FFF;
    }
  }
}

// A marked row, whose output stands.  (Two bits of state where the kernels mark, and one call here: as one number 19.3 us for 4 sequences of 4000 tokens became 20.4.)
template <int D>
__device__ __noinline__ void marked_row(const CacheTreeParams& p, int b, int i, int head, int mark) {
  if (mark == kByItself) tree_row<D>(p, b, i, head);
  else nan_channels<D>(p, b, i, head);
}

// ------------------------------------------------------------------------------------------------ instructions
// Two floats -> two e5m2 codes (RNE, saturating): lo in bits 0-7, hi in bits 8-15.
__device__ __forceinline__ uint32_t cvt_e5m2x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Four values of 0 ... 256 -> four e4m3 codes of them, rounded to four significant bits, and the codes of what that leaves, of either sign and 2^(e - 4) at most for a value of
// 2^e ... 2^(e + 1): together off by 2^(e - 9), half a step of the second code; NaN becomes that of the second code.  (Rounded as integers, ties up: 32 exponentials and their codes take a warp alone 510 cycles and three warps
// of a scheduler 335 each; 450 and 324 with the first code cut off, 580 and 341 where what a rounded one left is known by converting it back.  Measured, 64 sequences of 4096 tokens with 25 drafts: first four bits cut off, 2^-8, 178 us; rounded 183; a third code, 2^-12, 201, and 146 instead of
// 130 with 8 drafts.  Two codes keep what bf16 weights would, and o is rounded to bf16 in any case: its error against 64 bits is 0.00083 there, of which that rounding is 0.00076;
// with the bits cut off it was 0.00122.)
__device__ __forceinline__ void split4(float2 x, float2 y, uint32_t& first, uint32_t& second) {
  auto four_bits = [](float v) { return __uint_as_float((__float_as_uint(v) + 0x80000u) & 0xFFF00000u); };
  const float2 a = make_float2(four_bits(x.x), four_bits(x.y)), b = make_float2(four_bits(y.x), four_bits(y.y));
  first = cvt_e4m3x4(a.x, a.y, b.x, b.y);
  const float2 u = add2(x, make_float2(-a.x, -a.y)), v = add2(y, make_float2(-b.x, -b.y));
  second = cvt_e4m3x4(u.x, u.y, v.x, v.y);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
               "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
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
  kFull = 0, kEmpty = 10,                   // of the ring
  kQ = 20, kOut = 22,                       // by parity of the unit: queries written; output read from TMEM
  kS = 24, kP = 27, kPv = 30,               // by S buffer: S computed, P written, P V done
  kU = 33,                                  // by quarter of the lanes: the unit's u stands
  kScales = 37,                             // of running tile g: entry g % 8
  kCut = 45,                                // by team: a cut tile's values have been looked at
  kPHalf = 48,                              // as kP, of the first half of a tile's keys (one copy)
  kTreeBars = 51,                           // behind them the TMEM slot, the abort flag and whether a row of a whole unit is marked
};

// What the join needs of a cut unit, left by the worker that goes on with it first: its rows, and the workers that have tiles of it.
struct TreeCut {
  int b, hk, rt, count;                     // count 0: nothing to join
  int first, last, slot, pad;               // slot of the first piece; worker w's behind it: 2 w
};
// Of worker j, whose share begins at step f with piece x.
__device__ __forceinline__ TreeCut tree_cut_at(const TreeRange& range, const TreePiece& x, int j, int f) {
  TreeCut y{};
  if (j == 0 || x.begin >= f || range.share(j - 1) > x.begin) return y;      // no cut, or not the unit's first
  auto worker_at = [&](int step) {                            // whose share it is: share(lo) <= step < share(hi)
    int lo = j - 1, hi = range.workers;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (range.share(mid) <= step) lo = mid; else hi = mid;
    }
    return lo;
  };
  // of the tiles; workers before them have steps of the unit's own cost alone and no piece
  y.first = worker_at(x.begin + kTreeCost);
  y.last = worker_at(x.end() - 1);
  y.slot = 2 * y.first + (y.first == j - 1 && range.share(j - 1) < x.begin ? 1 : 0);
  y.b = x.b;
  y.hk = x.hk;
  y.rt = x.rt;
  y.count = y.first == y.last ? 0 : x.s.count;                // whole: written by that worker
  return y;
}

// 2^e, e a whole number, in two factors: values may be as far above 1 as it is below fp32's smallest.
__device__ __forceinline__ float2 two_factors(float e) {
  e = fminf(fmaxf(e, -250.f), 250.f);
  const float h = truncf(0.5f * e);
  return make_float2(ex2_approx(h), ex2_approx(e - h));
}
__device__ __forceinline__ float4 add_scaled(float4 acc, float4 y, float2 w) {
  return make_float4(fmaf(y.x * w.x, w.y, acc.x), fmaf(y.y * w.x, w.y, acc.y), fmaf(y.z * w.x, w.y, acc.z), fmaf(y.w * w.x, w.y, acc.w));
}

// CTA `rank` of a cluster writes its share of a unit's rows: the CTAs have left it their sums of them (m, l, u, marked) and their values, a CTA's behind the other's, in
// shared memory (its own: reading others' took 4000 cycles a row; writing to others, at 16 bytes a cycle, is what bounds the exchange, so the copies are added up before),
// 16-byte pieces XORed with the row.  Half a warp a row, over the CTAs in order; rows behind the sequence's count are zeros.
__device__ __forceinline__ int value_at(int row, int piece) { return piece ^ (row & 31); }
template <int D, int kRows, int kWarps>
__device__ __forceinline__ void join_cluster(const CacheTreeParams& p, const TreePiece& x, int rank, const uint8_t* values, const float4* sums) {
  constexpr int kVecs = D / 64;
  const int cl = p.cluster, rows = kRows / cl, lane = threadIdx.x & 31, l = lane & 15;
  for (int i0 = (threadIdx.x >> 5) * 2; i0 < rows; i0 += 2 * kWarps) {
    const int i = i0 + (lane >> 4), row = rank * rows + i, unit_row = x.rt * kRows + row, node = node_of(p, unit_row), head = x.hk * p.rep + unit_row - node * p.rep;
    const bool mine = i < rows && node < p.N, real = mine && node < x.s.count;
    float4 acc[kVecs] = {};
    float top = kNone, u_top = kNone, marked = 0.f, sum = 0.f;
    if (real) {
      for (int c = 0; c < cl; ++c) {
        const float4 st = sums[c * rows + i];
        top = fmaxf(top, st.x);
        if (st.x > kNone) u_top = fmaxf(u_top, st.z);
        marked = fmaxf(marked, st.w);
      }
      for (int c = 0; c < cl; ++c) {
        const float4 st = sums[c * rows + i];
        if (!(st.x > kNone)) {                                // the row sees nothing of the CTA's tiles (or it had none); NaN may have been added to its sum
          sum += st.y;
          continue;
        }
        sum = fmaf(st.y, ex2_approx(st.x - top), sum);
        const float2 w = two_factors(st.z - u_top);
        const float4* from = reinterpret_cast<const float4*>(values) + (c * rows + i) * (D / 4);
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          acc[v] = add_scaled(acc[v], from[value_at(row, 16 * v + l)], w);
        }
      }
    }
    if (mine && marked != kByItself) {
      const float d_all = u_top - top, d1 = fminf(fmaxf(d_all, -100.f), 100.f);
      const float w1 = real ? exp2f(d1) : 0.f, w2 = real ? exp2f(d_all - d1) / sum : 0.f;
      uint2* o = reinterpret_cast<uint2*>(p.o + ((static_cast<int64_t>(x.b) * p.N + node) * p.H + head) * D) + l;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(acc[v].x * w1 * w2, acc[v].y * w1 * w2), b = __floats2bfloat162_rn(acc[v].z * w1 * w2, acc[v].w * w1 * w2);
        o[16 * v] = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
      }
      if (l == 0) p.lse[(static_cast<int64_t>(x.b) * p.H + head) * p.N + node] = real ? (top + log2f(sum)) * kLn2 : -CUDART_INF_F;
    }
    // marked rows: by the whole warp
    for (uint32_t left = __ballot_sync(0xffffffffu, real && marked != 0.f && l == 0); left != 0; left &= left - 1) {
      const int from = __ffs(left) - 1, node_from = __shfl_sync(0xffffffffu, node, from), head_from = __shfl_sync(0xffffffffu, head, from);
      marked_row<D>(p, x.b, node_from, head_from, static_cast<int>(__shfl_sync(0xffffffffu, marked, from)));
    }
  }
}

// ------------------------------------------------------------------------------------------------ main kernel
// kCluster: a cluster of CTAs a unit instead of the even division, each an even share of its tiles, joined through distributed shared memory: nothing is left to a
// second kernel.
template <int kD, int kCopies, bool kCluster>
__global__ void __launch_bounds__(TreeCfg<kD>::kThreads, 1)
cache_tree_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ CacheTreeParams p) {
  using C = TreeCfg<kD>;
  constexpr int D = C::D, kTeams = C::kTeams, kRows = 128 / kCopies;      // rows of a unit
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023) & ~1023u) - raw);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kSmemBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kTreeBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kTreeBars + 1);
  volatile int* any_marked = abort_flag + 1;
  float* scales = reinterpret_cast<float*>(smem + C::kSmemScales);
  float* factors = reinterpret_cast<float*>(smem + C::kSmemRows);
  int* out_rows = reinterpret_cast<int*>(smem + C::kSmemRows) + 256;
  volatile int* marks = reinterpret_cast<volatile int*>(smem + C::kSmemRows) + 512;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, role = warp - 4 * kTeams;       // of the last four warps
  if (tid == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(bars + kFull + i, 1);
      mbar_init(bars + kEmpty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + kQ + i, 4 * kTeams);
      mbar_init(bars + kOut + i, 4 * kTeams);
    }
    for (int i = 0; i < kTeams; ++i) {
      mbar_init(bars + kS + i, 1);
      mbar_init(bars + kP + i, 4);
      mbar_init(bars + kPv + i, 1);
      mbar_init(bars + kCut + i, 4);
      mbar_init(bars + kPHalf + i, 4);
    }
    for (int i = 0; i < 4; ++i) mbar_init(bars + kU + i, 1);
    for (int i = 0; i < 8; ++i) mbar_init(bars + kScales + i, 1);
    *abort_flag = 0;
    *any_marked = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (role == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  grid_dep_wait();
  // the worker's share of the steps, and its first piece
  const int worker = blockIdx.x;
  int f_begin = 0, f_end = 0, sums = 0;
  TreePiece x{};
  TreeRange range{};
  const int rank = kCluster ? worker % p.cluster : 0, rows_each = kCluster ? kRows / p.cluster : kRows;      // of the cluster; rows that each CTA of it writes
  bool met = false;                                           // the cluster's CTAs are done with their tiles
  if constexpr (kCluster) {
    const int unit = worker / p.cluster, row_tiles = (p.N * p.rep + kRows - 1) / kRows;
    x.b = unit / (p.c.Hk * row_tiles);
    const int in_sequence = unit - x.b * p.c.Hk * row_tiles;
    x.hk = in_sequence / row_tiles;
    x.rt = in_sequence - x.hk * row_tiles;
    x.s = tree_seq(p, x.b);
    if (x.rt < x.s.row_tiles(p)) {
      x.t0 = x.s.tiles() * rank / p.cluster;
      x.t1 = x.s.tiles() * (rank + 1) / p.cluster;
    }
  } else {
    range = tree_range(p, sums);
    if (worker < range.workers && range.total > 0) {
      f_begin = range.share(worker);
      f_end = range.share(worker + 1);
      x = tree_first(p, sums, f_begin, f_end);
    }
  }
  __syncthreads();                                            // the mbarriers and the TMEM slot are there
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto bar = [&](int i) { return smem_u32(bars + i); };
  // running tile g goes to team and S buffer g % kTeams, whose barriers' phase it is
  auto phase_of = [&](int g) { return static_cast<uint32_t>(g / kTeams) & 1u; };
  bool ok = true;

  if (kCluster || f_begin < f_end) {
    if (role >= 0 && D == 128) reg_dec<C::kRegsOther>();
    if (role == 0 || role == 3) {
      // ---------------------------------------------------------------------------------------- TMA: K tiles and the scales of both; V tiles
      // (a warp each: the four boxes of a tile take a warp 800 cycles, and one warp for both held up the whole CTA)
      const int kv = role == 3;
      const TreePiece first = x;
      // Eight tiles at a time, a lane a block: a batch's pages are asked for two batches ahead of its loads and its scales one ahead (a tile takes less than the
      // two loads, one behind the other, that lead to its codes).
      struct Batch {
        int tiles;
        bool held;
        int hk, page, sub;
        float ks, vs;
      };
      const int bpp = p.c.page / 32;
      int t = x.t0;
      bool more = true;                                       // (x, t) is the next tile to be looked up
      auto look_up = [&]() {
        Batch a{};
        int b = 0, blk = 0;
        if (more && t + 8 <= x.t1) {                          // all of this piece
          blk = 4 * t + lane;
          a.held = blk * 32 < x.s.n;
          a.hk = x.hk;
          b = x.b;
          a.tiles = 8;
          t += 8;
        }
#pragma unroll 1
        for (; a.tiles < 8; ++a.tiles) {
          while (more && t >= x.t1) {
            more = tree_next(p, x, f_end);
            t = x.t0;
          }
          if (!more) break;
          if (lane >> 2 == a.tiles) {
            blk = 4 * t + (lane & 3);
            a.held = blk * 32 < x.s.n;
            a.hk = x.hk;
            b = x.b;
          }
          ++t;
        }
        if (a.held) {
          const int entry = blk / bpp;
          a.sub = blk - entry * bpp;
          a.page = __ldg(p.c.table + b * p.c.t_row + entry);
        }
        return a;
      };
      auto ask_scales = [&](Batch& a) {
        if (!a.held) return;
        a.page = max(0, checked_page(p.c, a.page));
        if (kv) return;
        const int64_t at = a.page * p.c.s_page + a.hk * p.c.s_head + a.sub;
        a.ks = __ldg(p.c.ks + at);
        a.vs = __ldg(p.c.vs + at);
      };
      int g = 0;                                              // running tile
      Batch now = look_up();
      ask_scales(now);
      Batch next = look_up();
      while (now.tiles > 0 && ok) {
        Batch after{};
        const uint32_t held = __ballot_sync(0xffffffffu, now.held);
#pragma unroll 1
        for (int i = 0; i < now.tiles; ++i, ++g) {
          const int j = 2 * g + kv, st = j % C::kStages, boxes = __popc(held >> (4 * i) & 15u) * C::kPanels;
          const bool mine = lane >> 2 == i;
          if (j >= C::kStages && !(ok = wait_warp(bar(kEmpty + st), (j / C::kStages - 1) & 1, abort_flag))) break;
          if (lane == 0) mbar_expect_tx(bars + kFull + st, boxes * 4096);
          __syncwarp();
          if (mine && now.held) {
#pragma unroll
            for (int c = 0; c < C::kPanels; ++c)
              tma_load_4d(sbase + C::kSmemRing + st * C::kTile + c * 16384 + (lane & 3) * 4096, kv ? &tv : &tk, bar(kFull + st), 128 * c, now.sub * 32, now.hk, now.page);
          }
          if (kv == 0) {
            if (mine) {
              scales[(g & 7) * 8 + (lane & 3)] = now.ks;      // zero where there is no block
              scales[(g & 7) * 8 + 4 + (lane & 3)] = static_cast<float>(static_cast<int>(scale_to_sb(now.vs)) - 127);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + kScales + (g & 7));
          }
          if (i == 0) {                                       // (the first tile is on its way)
            ask_scales(next);
            after = look_up();
          }
        }
        now = next;
        next = after;
      }
      if (!kCluster && kv) {
        const TreeCut y = tree_cut_at(range, first, worker, f_begin);
        if (lane == 0) reinterpret_cast<TreeCut*>(p.cuts)[worker] = y;
      }
      if (!ok && lane == 0) raise_abort(abort_flag, p.c.status, kStatusTimeoutProducer + kInCache);
      // what is in flight lands before the shared memory goes, whichever role gives up
      for (int i = max(0, g - C::kStages / 2); i < g; ++i) wait_or_abort(bar(kFull + (2 * i + kv) % C::kStages), ((2 * i + kv) / C::kStages) & 1, abort_flag);
    } else if (role == 1) {
      // ---------------------------------------------------------------------------------------- MMA: S
      // (an issuing warp for each product: a chain of eight holds its warp until it is nearly done)
      if (elect_one()) {
        constexpr uint32_t kIdescFirst = idesc_f8(128, 128, false, false), kIdescSecond = kIdescFirst | (1u << 7);     // A: e4m3; e5m2
        const uint32_t q_lo = desc_lo(sbase + C::kSmemQ), ring_lo = desc_lo(sbase + C::kSmemRing);
        int g = 0, units = 0;                                 // running tile, running unit
        do {
          if (x.t0 >= x.t1) continue;
          ok = wait_or_abort(bar(kQ + (units & 1)), (units >> 1) & 1, abort_flag);
          for (int t = x.t0; t < x.t1 && ok; ++t, ++g) {
            const int st = 2 * g % C::kStages, buf = g % kTeams;
            // K, and the buffer: behind the products that read P and its scale bytes from it
            if (g >= kTeams && !(ok = wait_or_abort(bar(kPv + buf), phase_of(g - kTeams), abort_flag))) break;
            if (!(ok = wait_or_abort(bar(kFull + st), (2 * g / C::kStages) & 1, abort_flag))) break;
            tc_fence_after();
            const uint32_t k_lo = ring_lo + st * (C::kTile >> 4), d = tmem + 128 * buf;
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
              const uint32_t off = (k >> 2) * (16384 >> 4) + (k & 3) * 2;
              mma_f8_ss(d, q_lo + off, k_lo + off, kIdescFirst, k > 0);
              mma_f8_ss(d, q_lo + (C::kTile >> 4) + off, k_lo + off, kIdescSecond, true);
            }
            tc_commit(bars + kS + buf);
            tc_commit(bars + kEmpty + st);
          }
          ++units;
        } while (ok && tree_next(p, x, f_end));
        if (!ok) raise_abort(abort_flag, p.c.status, kStatusTimeoutMma + kInCache);
      }
    } else if (role == 2) {
      // ---------------------------------------------------------------------------------------- MMA: P V
      if (elect_one()) {
        const uint32_t ring_lo = desc_lo(sbase + C::kSmemRing);
        int g = 0, units = 0;
        do {
          if (x.t0 >= x.t1) continue;
          if (units > 0) ok = wait_or_abort(bar(kOut + ((units - 1) & 1)), ((units - 1) >> 1) & 1, abort_flag);      // O has been read
          for (int t = x.t0; t < x.t1 && ok; ++t, ++g) {
            const int st = (2 * g + 1) % C::kStages, buf = g % kTeams, held = min(4, (x.s.n - 128 * t + 31) / 32);     // blocks of the tile
            const uint32_t v_lo = ring_lo + st * (C::kTile >> 4), s = tmem + 128 * buf;
            // one copy: by halves of the keys, each with scale bytes of its own
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (k == 0 || (k == 2 && kCopies == 1)) {
                if (!(ok = wait_or_abort(bar((k == 0 && kCopies == 1 ? kPHalf : kP) + buf), phase_of(g), abort_flag))) break;
                if (k == 0 && !(ok = wait_or_abort(bar(kFull + st), ((2 * g + 1) / C::kStages) & 1, abort_flag))) break;
                tc_fence_after();
              }
              if (k < held) {                                 // (beyond, P is zero and V is not loaded)
                const uint32_t words = s + (k >= 2 && kCopies == 1 ? 80 : 16);
#pragma unroll
                for (int c = 0; c < C::kPanels; ++c) {
                  mma_mxf8_ts(tmem + C::kColO + 128 * c, s + 32 * k, v_lo + c * (16384 >> 4) + k * (4096 >> 4), idesc_mxf8(128, 128, false, true, k, k), words, words + 4,
                              t > x.t0 || k > 0);
                  mma_mxf8_ts(tmem + C::kColO + 128 * c, s + 32 * k + 8, v_lo + c * (16384 >> 4) + k * (4096 >> 4), idesc_mxf8(128, 128, false, true, k, k), words, words + 4,
                              true);
                }
              }
            }
            if (!ok) break;
            tc_commit(bars + kEmpty + st);
            tc_commit(bars + kPv + buf);
          }
          ++units;
        } while (ok && tree_next(p, x, f_end));
        if (!ok) raise_abort(abort_flag, p.c.status, kStatusTimeoutMma + kInCache);
      }
    } else {
      if (D == 128) reg_inc<C::kRegsSoftmax>();
      // ---------------------------------------------------------------------------------------- softmax, output
      const int team = warp >> 2, quarter = warp & 3, in_tile = tid & 127;
      const int row = in_tile & (kRows - 1);                  // of the unit
      const int copy = in_tile / kRows;                       // looks after blocks copy * 4 / kCopies ... of a tile
      constexpr int kBlocks = 4 / kCopies;
      const int c0 = kCopies == 1 ? 0 : copy * kBlocks;
      const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16, t_s = tmem + lanes + 128 * team, t_o = tmem + lanes + C::kColO;
      float2* stats = reinterpret_cast<float2*>(smem + C::kSmemStats);
      volatile uint32_t* nan_tokens = reinterpret_cast<volatile uint32_t*>(smem + C::kSmemNan) + 4 * team;
      // Queries: two codes an element, in the layout of the 128-byte swizzle.  A row's lanes take eight elements each, the warps of all teams the rows in turn; asked
      // for ahead.
      constexpr int kLanes = D / 8, kPer = 32 / kLanes, kPasses = (kRows / kPer + 4 * kTeams - 1) / (4 * kTeams);
      const int ql = lane % kLanes;
      uint4 asked[kPasses];
      auto ask_queries = [&](const TreePiece& y) {
#pragma unroll
        for (int k = 0; k < kPasses; ++k) {
          const int r = (warp + 4 * kTeams * k) * kPer + lane / kLanes, unit_row = y.rt * kRows + r, i = node_of(p, unit_row), head = y.hk * p.rep + unit_row - i * p.rep;
          asked[k] = make_uint4(0, 0, 0, 0);
          if (r < kRows && i < y.s.count) asked[k] = __ldg(reinterpret_cast<const uint4*>(p.q + y.b * p.q_sb + i * p.q_sn + head * p.q_sh) + ql);
        }
      };
      auto put_queries = [&](const TreePiece& y, int parity) {
#pragma unroll 1
        for (int k = 0; k < kPasses; ++k) {
          const int r = (warp + 4 * kTeams * k) * kPer + lane / kLanes;
          const uint32_t v[4] = {asked[0].x, asked[0].y, asked[0].z, asked[0].w};
#pragma unroll
          for (int z = 1; z < kPasses; ++z) asked[z - 1] = asked[z];
          // the largest size, as bits: NaN and infinities are above all others
          uint32_t top = __vmaxu2(__vmaxu2(v[0] & 0x7FFF7FFFu, v[1] & 0x7FFF7FFFu), __vmaxu2(v[2] & 0x7FFF7FFFu, v[3] & 0x7FFF7FFFu));
          top = max(top & 0xFFFFu, top >> 16);
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          const uint32_t eb = min(254u, max(14u, top >> 7));
          const float up = sb_to_scale(261u - eb);            // largest element to [2^7, 2^8)
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
          if (r < kRows) {
#pragma unroll
            for (int c = 0; c < kCopies; ++c) {
              const uint32_t at = sbase + C::kSmemQ + (ql >> 4) * 16384 + (r + c * kRows) * 128 + ((((ql & 15) >> 1) ^ (r & 7)) << 4) + (ql & 1) * 8;
              sts_f2(at, __uint_as_float(first[0]), __uint_as_float(first[1]));
              sts_f2(at + C::kTile, __uint_as_float(second[0]), __uint_as_float(second[1]));
            }
            if (ql == 0) {                                    // of a row of NaN or infinities the factor is NaN
              const int unit_row = y.rt * kRows + r, i = node_of(p, unit_row);
              factors[128 * parity + r] = top >= 0x7F80u ? CUDART_NAN_F : sb_to_scale(eb - 7u) * p.scale * kLog2e;
              out_rows[128 * parity + r] = i < y.s.count ? (y.b * p.N + i) * p.H + y.hk * p.rep + unit_row - i * p.rep : -1;
              marks[128 * parity + r] = 0;
            }
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + kQ + parity);
      };
      auto to_tiles = [&](TreePiece& y) {                     // on to a piece that has some
        while (y.t0 >= y.t1)
          if (!tree_next(p, y, f_end)) return false;
        return true;
      };
      bool live = to_tiles(x);
      if (live) {
        ask_queries(x);
        put_queries(x, 0);
      }
      int g0 = 0, units = 0, cuts = 0;                        // running tile that the unit begins with, running unit; cut tiles of the team
      while (live) {
        const int parity = units & 1, n_tiles = x.t1 - x.t0;
        volatile int* u_at = reinterpret_cast<volatile int*>(smem + C::kSmemU) + 128 * parity + in_tile;
        ok = wait_warp(bar(kQ + parity), (units >> 1) & 1, abort_flag);
        const int unit_row = x.rt * kRows + row, node = node_of(p, unit_row);
        const bool real = node < x.s.count;
        const bool idle = !__any_sync(0xffffffffu, real);     // a warp of rows that are none
        const uint32_t* seen = p.seen + x.b * p.s_sb + static_cast<int64_t>(min(node, x.s.count - 1)) * p.s_sn;
        const float f = factors[128 * parity + row];
        // Of the row, whole numbers: m, the reference of this team's sum l, which moves where a block's logits exceed it by more than 2^kReach; and u, in which O counts, the same
        // for all teams: kUnitLift above the largest product of a probability and its V scale among the first blocks of the unit, where the row sees any of these.  It does not
        // move: fp32 has room for products 2^95 above it (hi: the largest that this team has met), and a row that has larger ones is marked.
        float m = kNone, l = 0.f, u = 0.f, hi = kNone;
        int u_code = 0;
        bool knows_u = false, marked = false, sees_nan = false;
        // One key tile.  kCut: some row does not see all its keys (a compile-time variant: no select per element elsewhere).
        auto tile = [&](int g, int t, auto cut_tag) -> bool {
          constexpr bool kCut = decltype(cut_tag)::value;
          const uint32_t entry = sbase + C::kSmemScales + (g & 7) * 32;
          auto scale_byte = [&](float ku) { return static_cast<uint32_t>(fminf(fmaxf(ku - u + 119.f, 0.f), 254.f)); };       // of P's codes: 2^(ku - u - 8)
          auto put_words = [&](uint32_t at, uint32_t word) {
            const uint32_t words[8] = {word, word, word, word, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu};
            __syncwarp();
            tmem_st8(at, words);
          };
          // The reference of the unit's products: from its first tile, or what that left.
          auto know_u = [&](float ku0, float ku1) -> bool {
            if (g == g0) {
              auto above = [&](int c) { return fmaxf(0.f, kLeastScale - lds_f(entry + 16 + 4 * (c0 + c))); };
              const float top_u = fmaxf(ku0 + above(0), kBlocks > 1 ? ku1 + above(1) : kNone);
              const bool none = !(top_u > kNone);
              const int code = 2 * (none ? kUnitLift : static_cast<int>(fminf(fmaxf(top_u, -kExact), kExact)) + kUnitLift) + (none ? 1 : 0);
              *u_at = code;
              __syncwarp();
              if (lane == 0) mbar_arrive(bars + kU + quarter);
              u_code = code;
            } else if (!knows_u) {
              if (!wait_warp(bar(kU + quarter), units & 1, abort_flag)) return false;
              u_code = *u_at;
            }
            knows_u = true;
            u = static_cast<float>(u_code >> 1);
            return true;
          };
          float ku[2] = {kNone, kNone};                       // of two blocks, the power of two of their codes with V's scale
          // (not unrolled, here and below: four times as much code had the warps wait for instructions a fifth of the time)
#pragma unroll 1
          for (int c = 0; c < kBlocks; ++c) {
            uint32_t s[32];
            __syncwarp();                                     // (here and below: a TMEM access is the whole warp's, whatever branches came before)
            tmem_ld32(t_s + 32 * (c0 + c), s);
            const float fc = f * lds_f(entry + 4 * (c0 + c));
            const float ev = lds_f(entry + 16 + 4 * (c0 + c));
            uint32_t sees = 0xffffffffu;
            if (kCut) {
              sees = real ? seen_keys(seen, node, 128 * t + 32 * (c0 + c) - x.s.base()) : 0u;
              sees_nan |= (sees & nan_tokens[c0 + c]) != 0u;
              __syncwarp();
            }
            tmem_wait_ld();
            if (kCut) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((sees >> e) & 1u)) s[e] = 0xff800000u;
            }
            float2 s2[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) s2[e] = make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
            const float top = max32(s2);
            const float kb = kCut && sees == 0u ? kNone : fmaxf(ceilf(top * fc), kNone);
            const float2 f2 = splat2(fc), off = splat2(8.f - kb);
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
            tmem_st16(t_s + 32 * (c0 + c), w);                // over columns that have been read
            marked |= fabsf(kb) > kExact && kb > kNone;
            if (kb > m + kReach) {
              l *= ex2_approx(m - kb);
              m = kb;
            }
            l = fmaf(sum.x + sum.y, ex2_approx(kb - m - 8.f), l);
            if (c & 1) ku[1] = kb + ev;
            else ku[0] = kb + ev;
            if (kCopies == 1 && c == 1) {                     // the first half of the keys: the tensor cores may begin
              if (!know_u(ku[0], ku[1])) return false;
              hi = fmaxf(hi, fmaxf(ku[0], ku[1]));
              put_words(t_s + 16, scale_byte(ku[0]) | scale_byte(ku[1]) << 8);
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bars + kPHalf + team);
            }
          }
          if (kCopies > 1) {
            const uint32_t zeros[16] = {};                    // other copies' blocks
            __syncwarp();
#pragma unroll 1
            for (int c = 0; c < 4; ++c)
              if (c < c0 || c >= c0 + kBlocks) tmem_st16(t_s + 32 * c, zeros);
            if (kBlocks == 1) ku[1] = ku[0];
            if (!know_u(ku[0], ku[1])) return false;
          }
          hi = fmaxf(hi, fmaxf(ku[0], ku[1]));
          const uint32_t two = scale_byte(ku[0]) | scale_byte(ku[1]) << 8;
          if (kCopies == 1) put_words(t_s + 80, two << 16);
          else put_words(t_s + 16, kBlocks == 1 ? (two & 0xFFu) << (8 * c0) : two << (8 * c0));
          return true;
        };
        for (int g = g0 + (team + kTeams - g0 % kTeams) % kTeams; ok && g < g0 + n_tiles; g += kTeams) {
          const int t = x.t0 + g - g0;
          ok = wait_warp(bar(kScales + (g & 7)), (g >> 3) & 1, abort_flag) && wait_warp(bar(kS + team), phase_of(g), abort_flag);
          const bool cut = 128 * (t + 1) > x.s.base();
          if (cut) {
            // V's slots behind the length hold anything, and a drafted token may have NaN values, which only the rows that see it are to meet: zeros in the place of both, or
            // they would come through the products with P's zeros.  Which tokens had NaN is left to the rows, which get theirs when they stand.  A thread a token.
            const int st = (2 * g + 1) % C::kStages, j = 128 * t + in_tile;
            if (ok) ok = wait_warp(bar(kFull + st), ((2 * g + 1) / C::kStages) & 1, abort_flag);
            bool nan = false;
            if (ok && j >= x.s.base() && 128 * t + quarter * 32 < x.s.n) {      // in a block that is there
              const uint32_t at = sbase + C::kSmemRing + st * C::kTile + in_tile * 128;
              auto piece = [&](int y) { return at + (y >> 3) * 16384 + (((y ^ lane) & 7) << 4); };      // lanes on different banks
              uint32_t found = 0;
#pragma unroll
              for (int y = 0; y < 8 * C::kPanels; ++y) {
                const float4 w = lds_f4(piece(y));
                found |= nan_codes(__float_as_uint(w.x)) | nan_codes(__float_as_uint(w.y)) | nan_codes(__float_as_uint(w.z)) | nan_codes(__float_as_uint(w.w));
              }
              if (j >= x.s.n) {
#pragma unroll 1
                for (int y = 0; y < 8 * C::kPanels; ++y) sts_u4(piece(y), 0u, 0u, 0u, 0u);
                fence_async_smem();
              } else if (found != 0) {
                auto clean = [](float v) { return __float_as_uint(v) & ~nan_codes(__float_as_uint(v)); };
#pragma unroll 1
                for (int y = 0; y < 8 * C::kPanels; ++y) {
                  const float4 w = lds_f4(piece(y));
                  sts_u4(piece(y), clean(w.x), clean(w.y), clean(w.z), clean(w.w));
                }
                fence_async_smem();
              }
              nan = found != 0 && j < x.s.n;
            }
            const uint32_t nans = __ballot_sync(0xffffffffu, nan);
            if (lane == 0) {
              nan_tokens[quarter] = nans;                     // (the team's last cut tile is done with: its P has arrived)
              mbar_arrive(bars + kCut + team);
            }
            if (ok) ok = wait_warp(bar(kCut + team), cuts & 1, abort_flag);
            ++cuts;
          }
          if (!ok) break;
          tc_fence_after();
          if (idle) {
            if (lane == 0) {
              if (g == g0) mbar_arrive(bars + kU + quarter);
              if (kCopies == 1) mbar_arrive(bars + kPHalf + team);
            }
          } else if (!(ok = cut ? tile(g, t, std::true_type{}) : tile(g, t, std::false_type{}))) {
            break;
          }
          __syncwarp();
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + kP + team);
        }
        g0 += n_tiles;
        TreePiece next = x;
        bool more = tree_next(p, next, f_end);
        if (more) more = to_tiles(next);
        if (more) ask_queries(next);
        // Output, by all teams: over the teams and copies of a row, the largest references and the sum; each lane's values count w of it.
        if (ok) ok = wait_warp(bar(kPv + (g0 - 1) % kTeams), phase_of(g0 - 1), abort_flag);
        stats[128 * team + in_tile] = make_float2(m, l);
        // out of u's range: above; or below where u was not taken from the row's own products
        marked |= hi > u + 95.f || ((u_code & 1) != 0 && hi > kNone && hi < u - 80.f);
        if (real && (marked || sees_nan)) reinterpret_cast<volatile uint8_t*>(marks + 128 * parity + row)[marked ? 1 : 0] = 1;      // (teams and copies may differ)
        if (!(ok = all_of(4, 128 * kTeams, ok))) break;
        tc_fence_after();
        [[maybe_unused]] cg::cluster_group::arrival_token tiles_done;
        if constexpr (kCluster) tiles_done = cg::this_cluster().barrier_arrive();
        if (more) put_queries(next, parity ^ 1);              // all S of this unit have been computed; those of the next run under the output
        const bool whole = !kCluster && x.whole();
        float m_all = kNone, u_all = kNone, l_all = 0.f, m_own = kNone;
        volatile int* unit_u = u_at - in_tile + row;          // of the row's copies
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
          float m_copy = kNone;
#pragma unroll
          for (int y = 0; y < kTeams; ++y) m_copy = fmaxf(m_copy, stats[128 * y + row + c * kRows].x);
          m_all = fmaxf(m_all, m_copy);
          if (c == copy) m_own = m_copy;
          if (m_copy > kNone) u_all = fmaxf(u_all, static_cast<float>(unit_u[c * kRows] >> 1));
        }
#pragma unroll
        for (int c = 0; c < kCopies; ++c)
#pragma unroll
          for (int y = 0; y < kTeams; ++y) {
            const float2 st = stats[128 * y + row + c * kRows];
            l_all = fmaf(st.y, ex2_approx(st.x - m_all), l_all);
          }
        if (!(u_all > kNone)) u_all = static_cast<float>(kUnitLift);        // the row sees nothing here (NaN keys aside)
        // what a value counts: 2^(u - m) / l where the row is whole here, 2^(u - the copies' largest u) else; nothing in a copy that has seen nothing, whose u is anywhere
        const float2 w = two_factors(static_cast<float>(*u_at >> 1) - (whole ? m_all : u_all));
        const float w1 = m_own > kNone ? w.x : 0.f, w2 = whole ? w.y / l_all : w.y;
        const int slot = 2 * worker + (x.f0 == f_begin ? 0 : 1);
        if constexpr (kCluster) {                             // the values go to the CTAs that write their rows, where the ring must be free: all CTAs' tiles are done with
          cg::this_cluster().barrier_wait(std::move(tiles_done));
          met = true;
        }
        // of the row's values, in the CTA that writes it
        auto values_of = [&](int r) {
          const int to = r / rows_each;
          return reinterpret_cast<float4*>(cg::this_cluster().map_shared_rank(smem, to) + C::kSmemRing) + (rank * rows_each + r - to * rows_each) * (D / 4);
        };
        if constexpr (kCopies == 1) {                         // 16 columns at a time, a row a lane
          const int at = out_rows[128 * parity + row];
          float* part = p.part_o + (static_cast<int64_t>(slot) * kRows + row) * D;
          float4* values = nullptr;
          if constexpr (kCluster) values = values_of(row);
#pragma unroll 1
          for (int c = team; c < D / 16; c += kTeams) {
            uint32_t o[16];
            __syncwarp();
            tmem_ld16(t_o + 16 * c, o);
            tmem_wait_ld();
            float y[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = __uint_as_float(o[e]) * w1 * w2;
            if (at < 0) {                                     // a row that is none
            } else if (whole) {
              uint32_t h[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const __nv_bfloat162 b2 = __floats2bfloat162_rn(y[2 * e], y[2 * e + 1]);
                h[e] = *reinterpret_cast<const uint32_t*>(&b2);
              }
              uint4* to_o = reinterpret_cast<uint4*>(p.o + static_cast<int64_t>(at) * D + 16 * c);
              to_o[0] = make_uint4(h[0], h[1], h[2], h[3]);
              to_o[1] = make_uint4(h[4], h[5], h[6], h[7]);
            } else if constexpr (kCluster) {
#pragma unroll
              for (int e = 0; e < 4; ++e) values[value_at(row, 4 * c + e)] = make_float4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) reinterpret_cast<float4*>(part + 16 * c)[e] = make_float4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
            }
          }
        } else {
          // through shared memory: four lanes a row, eight rows a warp at a time; 16-byte pieces XORed with the lane
          const uint32_t stage = sbase + C::kSmemOut + team * 8192;
#pragma unroll 1
          for (int c = team; c < D / 16; c += kTeams) {
            uint32_t o[16];
            __syncwarp();
            tmem_ld16(t_o + 16 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float y[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) y[k] = __uint_as_float(o[4 * e + k]) * w1 * w2;
              sts_u4(stage + in_tile * 64 + ((e ^ ((lane >> 1) & 3)) << 4), __float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
            }
            bar_sync(1 + team, 128);
            const int piece = lane & 3;
#pragma unroll
            for (int k = 0; k < 4 / kCopies; ++k) {
              const int r = quarter * (kRows / 4) + 8 * k + (lane >> 2);
              float4 y = lds_f4(stage + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4));
#pragma unroll
              for (int cc = 1; cc < kCopies; ++cc) {
                const float4 z = lds_f4(stage + (r + cc * kRows) * 64 + ((piece ^ ((r >> 1) & 3)) << 4));
                y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
              }
              const int at = out_rows[128 * parity + r];
              if (at < 0) {
              } else if (kCluster) {
                values_of(r)[value_at(r, 4 * c + piece)] = y;
              } else if (whole) {
                const __nv_bfloat162 a = __floats2bfloat162_rn(y.x, y.y), b = __floats2bfloat162_rn(y.z, y.w);
                *reinterpret_cast<uint2*>(p.o + static_cast<int64_t>(at) * D + 16 * c + 4 * piece) =
                    make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
              } else {
                *reinterpret_cast<float4*>(p.part_o + (static_cast<int64_t>(slot) * kRows + r) * D + 16 * c + 4 * piece) = y;
              }
            }
            __syncwarp();
            bar_sync(1 + team, 128);
          }
        }
        const bool mine = team == 0 && copy == 0 && real;
        const int head = x.hk * p.rep + unit_row - node * p.rep;
        const int said = mine ? marks[128 * parity + row] : 0, mark = said > 1 ? kByItself : said;
        if (mine && whole) {
          const int64_t at = (static_cast<int64_t>(x.b) * p.H + head) * p.N + node;
          p.lse[at] = (m_all + log2f(l_all)) * kLn2;
          p.marks[at] = mark;
          if (mark != 0) *any_marked = 1;
        }
        if constexpr (kCluster) {
          const int to = row / rows_each;
          if (mine)
            reinterpret_cast<float4*>(cg::this_cluster().map_shared_rank(smem, to) + C::kSmemSums)[rank * rows_each + row - to * rows_each] =
                make_float4(m_all, l_all, u_all, mark);
        } else if (mine && !whole) p.part_ml[static_cast<int64_t>(slot) * kRows + row] = make_float4(m_all, l_all, u_all, mark);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + kOut + parity);
        ++units;
        x = next;
        live = more;
      }
      if (!ok && lane == 0) raise_abort(abort_flag, p.c.status, kStatusTimeoutCompute + kInCache);
    }
  } else if (!kCluster && tid == 0) {
    reinterpret_cast<TreeCut*>(p.cuts)[worker] = TreeCut{};
  }
  if constexpr (kCluster) {
    __syncwarp();
    if (!met) {
      cg::this_cluster().sync();
      if (role < 0) {                                         // no tiles (or given up): nothing for the other CTAs' rows
        for (int r = tid; r < kRows; r += 128 * kTeams) {
          const int to = r / rows_each;
          reinterpret_cast<float4*>(cg::this_cluster().map_shared_rank(smem, to) + C::kSmemSums)[rank * rows_each + r - to * rows_each] = make_float4(kNone, 0.f, kNone, 0.f);
        }
      }
    }
    cg::this_cluster().sync();
    if (role < 0) join_cluster<D, kRows, 4 * kTeams>(p, x, rank, smem + C::kSmemRing, reinterpret_cast<const float4*>(smem + C::kSmemSums));
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (role == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if constexpr (!kCluster) {
    // The rows of whole units that were marked, a warp a row: here, where nothing waits for them with a limit.  By the warps of the softmax, which have the registers for it.
    if (role < 0 && *any_marked != 0) {
      x = tree_first(p, sums, f_begin, f_end);
      do {
        if (!x.whole()) continue;
        for (int r = warp; r < kRows; r += 4 * kTeams) {
          const int unit_row = x.rt * kRows + r, node = node_of(p, unit_row), head = x.hk * p.rep + unit_row - node * p.rep;
          const int mark = node < x.s.count ? p.marks[(static_cast<int64_t>(x.b) * p.H + head) * p.N + node] : 0;
          if (mark != 0) marked_row<D>(p, x.b, node, head, mark);
        }
      } while (tree_next(p, x, f_end));
    }
  }
}

// ------------------------------------------------------------------------------------------------ join
// The pieces of cut units, a warp a row, four rows a CTA; and the rows behind the counts.
template <int D>
__global__ void __launch_bounds__(128) cache_tree_join_kernel(const __grid_constant__ CacheTreeParams p) {
  constexpr int kVecs = D / 128;
  grid_dep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TreeCut x = reinterpret_cast<const TreeCut*>(p.cuts)[blockIdx.x];
  // rows behind the counts: zeros
  for (int b = blockIdx.x; b < p.c.B; b += gridDim.x)
    for (int i = tree_seq(p, b).count + blockIdx.y; i < p.N; i += gridDim.y) {
      uint4* o = reinterpret_cast<uint4*>(p.o + (static_cast<int64_t>(b) * p.N + i) * p.H * D);
      for (int z = threadIdx.x; z < p.H * D / 8; z += 128) o[z] = make_uint4(0, 0, 0, 0);
      for (int z = threadIdx.x; z < p.H; z += 128) p.lse[(static_cast<int64_t>(b) * p.H + z) * p.N + i] = -CUDART_INF_F;
    }
  const int r = blockIdx.y * 4 + warp, unit_row = x.rt * p.row_tile + r, node = node_of(p, unit_row), head = x.hk * p.rep + unit_row - node * p.rep;
  if (node >= x.count) return;
  float top = kNone, u_top = kNone, sum = 0.f;
  float4 acc[kVecs] = {};
  float marked = 0.f;
  // 32 results at a time, a lane each: their maxima and sums together, then the values of those that count
  for (int w0 = x.first; w0 <= x.last; w0 += 32) {
    const int w = w0 + lane;
    const bool there = w <= x.last;                           // each has a tile at least
    const int64_t at = there ? static_cast<int64_t>(w == x.first ? x.slot : 2 * w) * p.row_tile + r : 0;
    const float4 ml = there ? p.part_ml[at] : make_float4(kNone, 0.f, kNone, 0.f);
    marked = fmaxf(marked, warp_max(ml.w));
    float top_new = ml.x, u_new = ml.x > kNone ? ml.z : kNone;
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
    const float2 a = two_factors(u_top - u_new);
    const float lift = ml.z - u_new;
    top = top_new;
    u_top = u_new;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) acc[v] = add_scaled(make_float4(0.f, 0.f, 0.f, 0.f), acc[v], a);
    const uint32_t counts = __ballot_sync(0xffffffffu, there && ml.x > kNone);          // kNone: the row sees nothing of the piece
#pragma unroll 8
    for (int k = 0; k < min(32, x.last - w0 + 1); ++k) {
      const float lift_k = __shfl_sync(0xffffffffu, lift, k);
      const int64_t at_k = __shfl_sync(0xffffffffu, at, k);
      if (!((counts >> k) & 1)) continue;
      const float2 w_k = two_factors(lift_k);
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        acc[v] = add_scaled(acc[v], reinterpret_cast<const float4*>(p.part_o + at_k * D)[32 * v + lane], w_k);
      }
    }
  }
  if (marked == kByItself) {
    tree_row<D>(p, x.b, node, head);
    return;
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
  if (marked != 0.f) nan_channels<D>(p, x.b, node, head);
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
  cudaError_t e;
  if (p.cluster > 0) {
    e = allow_smem<cache_tree_kernel<D, kCopies, true>>(C::kSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.grid);
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    count_launch();
    return cudaLaunchKernelEx(&cfg, cache_tree_kernel<D, kCopies, true>, tk, tv, p);
  }
  e = allow_smem<cache_tree_kernel<D, kCopies, false>>(C::kSmem);
  if (e != cudaSuccess) return e;
  count_launch();
  e = launch_chained(cache_tree_kernel<D, kCopies, false>, dim3(p.grid), C::kThreads, C::kSmem, stream, tk, tv, p);
  if (e != cudaSuccess) return e;
  count_launch();
  return launch_chained(cache_tree_join_kernel<D>, dim3(p.grid, p.row_tile / 4), 128, 0, stream, p);
}

// Clusters of 2^log CTAs that the device holds at a time: fewer than its SMs would (of 148, 33 of four and 15 of eight), since a cluster lies within a part of the chip.
int resident_clusters(int log) {
  static int cached[64][4] = {};                              // + 1
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && cached[dev][log] > 0) return cached[dev][log] - 1;
  using C = TreeCfg<128>;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1u << log;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(1u << log);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (allow_smem<cache_tree_kernel<128, 1, true>>(C::kSmem) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, cache_tree_kernel<128, 1, true>, &cfg) != cudaSuccess) {
    cudaGetLastError();                                       // no device: sizes are asked for all the same
    return 0;
  }
  if (dev >= 0 && dev < 64) cached[dev][log] = n + 1;
  return n;
}

// Tiles of a CTA up to which a cluster takes a unit: the lengths may be shorter than the table, which the even division makes good and a cluster does not.
constexpr int kClusterTiles = 12;
// Tiles that a CTA of a cluster may have above its even share: what the join by a second kernel is worth.
constexpr int kClusterGain = 4;
// Tiles that a CTA of the even division has at least, or the join has too many pieces.
constexpr int kWorkerTiles = 4;

}  // namespace

// Measured, in us (GPU time, H 32, Hk 8; a cluster a unit against the even division): one sequence of 8000 tokens with 8 drafts 16.1 and 17.4, four of 1000 with 16 drafts 14.0
// and 17.3, of 4000 19.6 and 22.3; three of 12000 with 8 drafts, 24 tiles a CTA against 15, 30.4 and 27.3; 16 units of 8000 tokens in clusters of 8, of which 15 are resident,
// 30.2 and 20.1 (so clusters of 4: CacheTreePlan).  Pieces of 4 tiles against 2 in a sequence of 16000 tokens with 2 kv heads: 21.0 and 24.7; of 8, one of 12000 with 8 kv
// heads: 21.0 and 19.4.
CacheTreePlan plan_cache_tree(int B, int N, int H, int Hk, int D, int T, int page) {
  CacheTreePlan x;
  const int64_t R = static_cast<int64_t>(N) * (H / Hk), wave = sm_count();
  x.row_tile = R <= 32 ? 32 : R <= 64 ? 64 : 128;             // 8000 tokens, 8 drafts of 4 heads: 16.1 us with 32, 23.1 with 128; 4 x 4000 with 16 drafts: 19.6 with 64, 24.8
  const int64_t unit_tiles = (static_cast<int64_t>(T) * page + 127) / 128, units = static_cast<int64_t>(B) * Hk * ((R + x.row_tile - 1) / x.row_tile);
  const int64_t pieces = units * ((unit_tiles + kWorkerTiles - 1) / kWorkerTiles);
  const int64_t workers = pieces < wave ? pieces : wave;      // one wave
  // A cluster a unit where its CTAs have few tiles each, not many more than their share, and all are resident at a time.
  int log = 0;
  while ((2 << log) <= kMaxCluster && (1 << log) < unit_tiles && units <= resident_clusters(log + 1)) ++log;
  const int64_t tiles = (unit_tiles + (1 << log) - 1) >> log;
  x.cluster = units <= resident_clusters(log) && tiles <= kClusterTiles && tiles <= (units * unit_tiles + workers - 1) / workers + kClusterGain ? 1 << log : 0;
  if (x.cluster > 0) {
    x.grid = static_cast<int>(units) * x.cluster;
    x.part_o_bytes = x.part_ml_bytes = x.mark_bytes = 0;
    x.cut_bytes = 16;
    return x;
  }
  x.grid = static_cast<int>(workers);
  x.mark_bytes = (static_cast<int64_t>(B) * H * N + 15) / 16 * 16;
  x.part_o_bytes = 2ll * x.grid * x.row_tile * D * 4;
  x.part_ml_bytes = 2ll * x.grid * x.row_tile * 16;
  x.cut_bytes = x.grid * static_cast<int64_t>(sizeof(TreeCut));
  return x;
}

cudaError_t launch_cache_tree(int D, const CUtensorMap& tk, const CUtensorMap& tv, const CacheTreeParams& p, cudaStream_t stream) {
  if (D == 128)
    return p.row_tile == 32 ? launch_tree<128, 4>(tk, tv, p, stream) : p.row_tile == 64 ? launch_tree<128, 2>(tk, tv, p, stream) : launch_tree<128, 1>(tk, tv, p, stream);
  return p.row_tile == 32 ? launch_tree<256, 4>(tk, tv, p, stream) : p.row_tile == 64 ? launch_tree<256, 2>(tk, tv, p, stream) : launch_tree<256, 1>(tk, tv, p, stream);
}

}  // namespace dm
