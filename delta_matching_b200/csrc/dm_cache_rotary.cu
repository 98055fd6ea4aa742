// New tokens with their positions' rotation: queries rotated, keys rotated and quantised into the cache, values quantised (the scale rule:
// dm_cache_append.cu).
//
// A pair (a, b) of channels of frequency f at position t becomes (a cos - b sin, b cos + a sin) of the angle t f.  Angles are counted in turns and reduced in 64
// bits (in 32 bits a position of 10^5 would leave them three digits).  Sine and cosine are fp32, of half turns, which need no reduction of their own, and of what rounding these to fp32 leaves to
// first order, so that a channel that all but vanishes keeps its digits too (64 x 20 tokens 11.1 -> 11.36 us, others as before).  Keys go from the fp32 products to their codes with one rounding, queries to bf16.
//
// A CTA is a (sequence, block of 32 slots, group of heads).  The block's sines and cosines are made once, in shared memory, for all its heads; then a warp
// takes a head of k, v or q at a time.  A lane holds eight pairs of a row, so that neither needs another lane's values.
//
// Bound by the bytes of q, k, v and what they become: 4 x 2560 tokens of 32 query and 8 kv heads take 52 us (4.4 TB/s), 4 x 4096 77 us.  Rows of one head lie 256 bytes wide
// and far apart, so bandwidth comes from the rows in flight: with one behind the other's arithmetic it was 67 and 100 us.  One token of 64 sequences: 4.1 us.
#include "dm_cache.cuh"
#include "dm_drafts.h"
#include "dm_kernels.h"
#include "dm_quant_block.cuh"

namespace dm {

namespace {

constexpr int kRotaryWarps = 8;
// From so many tokens on, four passes' rows are in flight instead of two: 52.4 instead of 55.5 us for 4 x 2560 tokens, but 4.7 instead of 4.1 for 64 x 1 (more code, which
// is cold), both sides equal at 2048 and 4096.
constexpr int kManyTokens = 4096;

// cos and sin of so many turns; `rest`: what fp32 leaves of the angle, up to 2^-25 of half a turn (its square is nothing).
__device__ __forceinline__ float2 turn(double turns) {
  const double half_turns = 2.0 * (turns - rint(turns));
  const float near = static_cast<float>(half_turns), rest = static_cast<float>(half_turns - near) * 3.14159265f;
  float s, c;
  sincospif(near, &s, &c);
  return make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
}

// kAhead: passes whose rows are in flight.
template <int D, int kAhead>
__global__ void __launch_bounds__(kRotaryWarps * 32, 3) cache_rotary_kernel(const CacheRotaryParams p, const int blocks, const int group) {
  constexpr int kTpr = D / 16, kRpp = 32 / kTpr;             // lanes a row, rows a pass
  // cos and sin of (row, pair): four float4 of two pairs each for a lane's eight pairs, lane after lane, so that the lanes of a load lie side by side
  extern __shared__ float4 turns[];
  grid_dep_wait();
  const CacheView& c = p.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x / blocks, j = blockIdx.x - b * blocks;
  const int start = cache_length(c, b), cap = c.T * c.page;
  const int asked = checked_count(c.status, p.counts, b, p.N);
  int count = asked;
  if (count > cap - start) {
    report(c.status, kStatusBadLength + kInCache);
    count = cap - start;
  }
  if (j == 0 && blockIdx.y == 0 && threadIdx.x == 0) p.new_lengths[b] = start + count;
  const int blk = start / 32 + j, slot0 = blk * 32;
  const int r_begin = max(0, start - slot0), r_end = min(32, start + count - slot0);       // rows of the block that are written
  const int r_last = min(32, start + p.N - slot0);            // rows of the call: q's beyond the count are zeros
  if (r_last <= r_begin) return;
  const int lanes = p.half / 8;                               // of a row, that hold pairs
  for (int x = threadIdx.x; x < (r_end - r_begin) * p.half; x += blockDim.x) {
    const int r = r_begin + x / p.half, f = x % p.half, i = slot0 + r - start;
    const int64_t t = static_cast<int64_t>(start) + (p.offsets != nullptr ? __ldg(p.offsets + b * p.o_row + i) : i);
    const float2 cs = turn(static_cast<double>(t) * (static_cast<double>(__ldg(p.freqs + f)) * 0.15915494309189535));
    reinterpret_cast<float2*>(turns)[((r * 4 + (f % 8) / 2) * lanes + f / 8) * 2 + f % 2] = cs;
  }
  __syncthreads();
  const int l = lane % kTpr, r0 = lane / kTpr;
  const bool turned = l < lanes;
  // this lane's two vectors of eight channels: pairs between them, or within each
  const int va = p.interleaved || !turned ? (turned ? 2 * l : 2 * lanes + 2 * (l - lanes)) : l, vb = p.interleaved || !turned ? va + 1 : l + lanes;
  // The 16 values of a row, rotated (f[0..7]: the first vector).
  auto rotate = [&](const uint4& a, const uint4& b4, int r, float (&f)[16]) {
    bf16x8_to_float(a, f);
    bf16x8_to_float(b4, f + 8);
    if (!turned) return;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float4 cs = turns[(r * 4 + x) * lanes + l];
      if (p.interleaved) {
        const float a0 = f[4 * x], b0 = f[4 * x + 1], a1 = f[4 * x + 2], b1 = f[4 * x + 3];
        f[4 * x] = a0 * cs.x - b0 * cs.y;
        f[4 * x + 1] = b0 * cs.x + a0 * cs.y;
        f[4 * x + 2] = a1 * cs.z - b1 * cs.w;
        f[4 * x + 3] = b1 * cs.z + a1 * cs.w;
      } else {
        const float a0 = f[2 * x], b0 = f[2 * x + 8], a1 = f[2 * x + 1], b1 = f[2 * x + 9];
        f[2 * x] = a0 * cs.x - b0 * cs.y;
        f[2 * x + 8] = b0 * cs.x + a0 * cs.y;
        f[2 * x + 1] = a1 * cs.z - b1 * cs.w;
        f[2 * x + 9] = b1 * cs.z + a1 * cs.w;
      }
    }
  };
  // Some passes' rows at a time, of those that are written: asked for together (one row behind the other's arithmetic had a third of the bandwidth).
  auto ask = [&](const __nv_bfloat16* x, int64_t sn, int ps, uint4 (&a)[kAhead], uint4 (&b4)[kAhead]) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int r = r0 + (ps + k) * kRpp;
      a[k] = b4[k] = make_uint4(0, 0, 0, 0);
      if (r >= r_begin && r < r_end) {
        const uint4* src = reinterpret_cast<const uint4*>(x + (slot0 + r - start) * sn);
        a[k] = __ldg(src + va);
        b4[k] = __ldg(src + vb);
      }
    }
  };
  const int first = r_begin / (kAhead * kRpp) * kAhead;
  const int heads = 2 * c.Hk + p.H;                           // K, V, Q
  for (int h = blockIdx.y * group + warp; h < min(heads, (static_cast<int>(blockIdx.y) + 1) * group); h += kRotaryWarps) {
    if (h >= 2 * c.Hk) {
      const int hq = h - 2 * c.Hk;
      const __nv_bfloat16* x = p.q + b * p.q_sb + hq * p.q_sh;
      __nv_bfloat16* out = p.q_out + (static_cast<int64_t>(b) * p.N * p.H + hq) * D;
#pragma unroll 1
      for (int ps = first; ps * kRpp < r_last; ps += kAhead) {
        uint4 a[kAhead], b4[kAhead];
        ask(x, p.q_sn, ps, a, b4);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int r = r0 + (ps + k) * kRpp;
          if (r < r_begin || r >= r_last) continue;
          uint4 wa = make_uint4(0, 0, 0, 0), wb = wa;
          if (r < r_end) {
            float f[16];
            rotate(a[k], b4[k], r, f);
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const __nv_bfloat162 v2 = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
              w[e] = *reinterpret_cast<const uint32_t*>(&v2);
            }
            wa = make_uint4(w[0], w[1], w[2], w[3]);
            wb = make_uint4(w[4], w[5], w[6], w[7]);
          }
          uint4* to = reinterpret_cast<uint4*>(out + static_cast<int64_t>(slot0 + r - start) * p.H * D);
          to[va] = wa;
          to[vb] = wb;
        }
      }
      continue;
    }
    if (r_end <= r_begin) continue;
    const bool is_v = h >= c.Hk;
    const int hk = is_v ? h - c.Hk : h, bpp = c.page / 32;
    const int page = checked_page(c, __ldg(c.table + b * c.t_row + blk / bpp));
    if (page < 0) continue;
    const int sub = blk % bpp;
    uint8_t* codes = (is_v ? c.v8 : c.k8) + page * c.c_page + hk * c.c_head + static_cast<int64_t>(sub) * 32 * c.c_slot;
    float* scale_at = (is_v ? c.vs : c.ks) + page * c.s_page + hk * c.s_head + sub;
    const float s_old = (j == 0 && r_begin > 0) ? *scale_at : 0.f;
    const __nv_bfloat16* x = is_v ? p.v + b * p.v_sb + hk * p.v_sh : p.k + b * p.k_sb + hk * p.k_sh;
    const int64_t sn = is_v ? p.v_sn : p.k_sn;
    // The rows twice, once for the maximum, once for the codes: the second time from L1 (held in registers they left room for eight warps an SM).
    auto values = [&](const uint4& a, const uint4& b4, int r, float (&f)[16]) {
      if (is_v) {
        bf16x8_to_float(a, f);
        bf16x8_to_float(b4, f + 8);
      } else {
        rotate(a, b4, r, f);
      }
    };
    float amax = 0.f;                                         // NaN never wins
#pragma unroll 1
    for (int ps = first; ps * kRpp < r_end; ps += kAhead) {
      uint4 a[kAhead], b4[kAhead];
      ask(x, sn, ps, a, b4);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int r = r0 + (ps + k) * kRpp;
        if (r < r_begin || r >= r_end) continue;
        float f[16];
        values(a[k], b4[k], r, f);
#pragma unroll
        for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(f[e]));
      }
    }
    amax = warp_max(amax);
    const float s = fmaxf(sb_to_scale(pow2_sb(amax, 1u)), s_old);
    const float inv = sb_to_inv(scale_to_sb(s));
#pragma unroll 1
    for (int ps = first; ps * kRpp < r_end; ps += kAhead) {
      uint4 a[kAhead], b4[kAhead];
      ask(x, sn, ps, a, b4);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int r = r0 + (ps + k) * kRpp;
        if (r < r_begin || r >= r_end) continue;
        float f[16];
        values(a[k], b4[k], r, f);
        uint2* to = reinterpret_cast<uint2*>(codes + r * c.c_slot);
        to[va] = make_uint2(cvt_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv), cvt_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
        to[vb] = make_uint2(cvt_e4m3x4(f[8] * inv, f[9] * inv, f[10] * inv, f[11] * inv), cvt_e4m3x4(f[12] * inv, f[13] * inv, f[14] * inv, f[15] * inv));
      }
    }
    if (s_old > 0.f && s > s_old) {                           // the block's older rows on the new scale
      const float ratio = s_old * inv;
      for (int r = r0; r < r_begin; r += kRpp) {
        uint4* at = reinterpret_cast<uint4*>(codes + r * c.c_slot) + l;
        const uint4 w = *at;
        *at = make_uint4(requant4(w.x, ratio), requant4(w.y, ratio), requant4(w.z, ratio), requant4(w.w, ratio));
      }
    }
    if (lane == 0) *scale_at = s;
  }
}

}  // namespace

cudaError_t launch_cache_rotary(int D, const CacheRotaryParams& p, cudaStream_t stream) {
  const int blocks = (p.N + 30) / 32 + 1, heads = 2 * p.c.Hk + p.H;      // blocks that N tokens can touch behind any start
  // heads to a CTA: all, which share its sines and cosines, where there are blocks enough for the SMs; otherwise fewer, whole rounds of a head a warp.  (64 x 20 tokens: 11.1
  // us with 8 CTAs an SM wanted, 16.8 with 4; 2 x 2560 at head_dim 256: 63.7 and 61.4; 4 x 4096: 77.7 with 8 and 16, 86.5 with 32.)
  const int64_t all = static_cast<int64_t>(p.c.B) * blocks, want = 8ll * sm_count();
  const int rounds = (heads + kRotaryWarps - 1) / kRotaryWarps;         // of a head a warp
  const int parts = static_cast<int>(all >= want ? 1 : (want + all - 1) / all < rounds ? (want + all - 1) / all : rounds);
  const int group = (rounds + parts - 1) / parts * kRotaryWarps, groups = (heads + group - 1) / group;
  const dim3 grid(static_cast<unsigned>(all), groups);
  const int smem = 32 * p.half * 8;
  count_launch();
  auto launch = [&](auto kernel) { return launch_chained(kernel, grid, kRotaryWarps * 32, smem, stream, p, blocks, group); };
  if (static_cast<int64_t>(p.c.B) * p.N >= kManyTokens) return D == 128 ? launch(cache_rotary_kernel<128, 4>) : launch(cache_rotary_kernel<256, 4>);
  return D == 128 ? launch(cache_rotary_kernel<128, 2>) : launch(cache_rotary_kernel<256, 2>);
}

}  // namespace dm
