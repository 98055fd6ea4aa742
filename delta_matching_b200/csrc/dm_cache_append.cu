// New tokens into the cache: bf16 K and V rows -> e4m3 codes and the scale of each (32-slot block, head) that they touch.
//
// Per touched block and head, over the new rows in it: s_new = smallest power of two with amax <= 448 s_new, at least 2^-126 (which is also
// the scale of zeros: a block that begins with zeros must not fix a coarse scale for what follows).  Where the block holds older tokens,
// s = max(s_old, s_new), and if it grew their codes become e4m3_rne(code * s_old / s); else s = s_new.  New codes: e4m3_rne(x / s).
// Scales are powers of two, so every product is exact and each value is rounded once per change of its block's scale.  Called again with
// the same arguments, the kernel leaves the same cache.
//
// One warp per (sequence, touched block, head, K or V): the block's rows stay in its registers between the maximum and the codes, no
// exchange between warps.  Bound by its bytes (2 read, 1 written per element) for prompts: 10242 tokens of four sequences, 8 heads of 128, 50 MB in
// 12.3 us = 4.1 TB/s (of 6.5; a launch and one round of loads, half the warps of the grid at a time, are 4 us of it).  By the launch for single
// tokens: 5.4 us for 64 sequences.
#include "dm_cache.cuh"
#include "dm_kernels.h"
#include "dm_quant_block.cuh"

namespace dm {

template <int D>
__global__ void __launch_bounds__(128) cache_append_kernel(const CacheAppendParams p, int blocks, int64_t items) {
  constexpr int kTpr = D / 16;            // lanes per row, 16 elements each
  constexpr int kRpp = 32 / kTpr;         // rows per pass
  constexpr int kPass = 32 / kRpp;
  grid_dep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (item >= items) return;
  // heads first, then K and V: neighbouring warps read neighbouring rows of a token
  const CacheView& c = p.c;
  int64_t rest = item;
  const int hk = static_cast<int>(rest % c.Hk);
  rest /= c.Hk;
  const bool is_v = (rest & 1) != 0;
  rest >>= 1;
  const int j = static_cast<int>(rest % blocks), b = static_cast<int>(rest / blocks);

  const int start = cache_length(c, b), cap = c.T * c.page;
  int count = checked_count(c.status, p.counts, b, p.N);
  if (count > cap - start) {
    report(c.status, kStatusBadLength + kInCache);
    count = cap - start;
  }
  if (hk == 0 && !is_v && j == 0 && lane == 0) p.new_lengths[b] = start + count;
  const int blk = start / 32 + j, slot0 = blk * 32;
  const int r_begin = max(0, start - slot0), r_end = min(32, start + count - slot0);     // new rows of the block
  if (r_end <= r_begin) return;
  const int bpp = c.page / 32;
  const int page = checked_page(c, __ldg(c.table + b * c.t_row + blk / bpp));
  if (page < 0) return;
  const int sub = blk % bpp;
  uint8_t* codes = (is_v ? c.v8 : c.k8) + page * c.c_page + hk * c.c_head + static_cast<int64_t>(sub) * 32 * c.c_slot;
  float* scale_at = (is_v ? c.vs : c.ks) + page * c.s_page + hk * c.s_head + sub;
  const float s_old = (j == 0 && r_begin > 0) ? *scale_at : 0.f;

  const int c16 = (lane % kTpr) * 16, r0 = lane / kTpr;
  const __nv_bfloat16* x = is_v ? p.v + b * p.v_sb + hk * p.v_sh : p.k + b * p.k_sb + hk * p.k_sh;
  const int64_t sn = is_v ? p.v_sn : p.k_sn;
  x += static_cast<int64_t>(slot0 - start) * sn + c16;          // row r of the block is token slot0 - start + r of the call
  uint4 y[kPass][2];
#pragma unroll
  for (int ps = 0; ps < kPass; ++ps) {
    const int r = r0 + ps * kRpp;
    y[ps][0] = y[ps][1] = make_uint4(0, 0, 0, 0);
    if (r >= r_begin && r < r_end) {
      const uint4* src = reinterpret_cast<const uint4*>(x + r * sn);
      y[ps][0] = __ldg(src);
      y[ps][1] = __ldg(src + 1);
    }
  }
  // the maximum on pairs of bf16, exact; NaN never wins
  __nv_bfloat162 top = __float2bfloat162_rn(0.f);
#pragma unroll
  for (int ps = 0; ps < kPass; ++ps) {
    const uint32_t w[8] = {y[ps][0].x, y[ps][0].y, y[ps][0].z, y[ps][0].w, y[ps][1].x, y[ps][1].y, y[ps][1].z, y[ps][1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __hmax2(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
  }
  float amax = fmaxf(__low2float(top), __high2float(top));
  amax = warp_max(amax);
  const float s = fmaxf(sb_to_scale(pow2_sb(amax, 1u)), s_old);
  const float inv = sb_to_inv(scale_to_sb(s));
#pragma unroll
  for (int ps = 0; ps < kPass; ++ps) {
    const int r = r0 + ps * kRpp;
    if (r >= r_begin && r < r_end) {
      float f[16];
      bf16x8_to_float(y[ps][0], f);
      bf16x8_to_float(y[ps][1], f + 8);
      uint4 w;
      w.x = cvt_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
      w.y = cvt_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
      w.z = cvt_e4m3x4(f[8] * inv, f[9] * inv, f[10] * inv, f[11] * inv);
      w.w = cvt_e4m3x4(f[12] * inv, f[13] * inv, f[14] * inv, f[15] * inv);
      *reinterpret_cast<uint4*>(codes + r * c.c_slot + c16) = w;
    }
  }
  if (s_old > 0.f && s > s_old) {                               // the block's older rows on the new scale
    const float ratio = s_old * inv;
    for (int r = r0; r < r_begin; r += kRpp) {
      uint4* at = reinterpret_cast<uint4*>(codes + r * c.c_slot + c16);
      uint4 w = *at;
      w.x = requant4(w.x, ratio);
      w.y = requant4(w.y, ratio);
      w.z = requant4(w.z, ratio);
      w.w = requant4(w.w, ratio);
      *at = w;
    }
  }
  if (lane == 0) *scale_at = s;
}

cudaError_t launch_cache_append(int D, const CacheAppendParams& p, cudaStream_t stream) {
  // blocks that N tokens can touch behind any start
  const int blocks = static_cast<int>((static_cast<int64_t>(p.N) + 30) / 32 + 1);
  const int64_t items = static_cast<int64_t>(p.c.B) * blocks * p.c.Hk * 2;
  const dim3 grid(static_cast<unsigned>((items + 3) / 4));
  count_launch();
  return D == 128 ? launch_chained(cache_append_kernel<128>, grid, 128, 0, stream, p, blocks, items)
                  : launch_chained(cache_append_kernel<256>, grid, 128, 0, stream, p, blocks, items);
}

}  // namespace dm
