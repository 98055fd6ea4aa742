// Trees of drafted tokens: what each node sees, and the tokens of one path moved together in the cache.
#include "dm_cache.cuh"
#include "dm_drafts.h"
#include "dm_kernels.h"

namespace dm {

namespace {

// ------------------------------------------------------------------------------------------------ depths and ancestors
// seen_i = {i} united with seen of i's parent; depth_i = |seen_i| - 1.  One CTA a sequence, one thread a node.  A warp's 32 nodes first find their ancestors among
// themselves, by doubling with shuffles (five rounds), and the ancestor behind those; then each node walks from group of 32 to group of 32, at most as many steps as it has words.  Bound by latency: 64 trees
// of up to 509 nodes, each within three nodes of its parent, take 3.5 us of the GPU; 10.9 where each node walked from parent to parent.
__global__ void __launch_bounds__(1024) draft_tree_kernel(const DraftTreeParams p, const int words) {
  extern __shared__ uint32_t sets[];                          // (N, pitch)
  __shared__ uint32_t among[kMaxNodes];                       // of a node, its ancestors in its group and itself
  __shared__ int behind[kMaxNodes];                           // and the nearest ancestor in an earlier group, or -1
  grid_dep_wait();
  const int b = blockIdx.x, i = threadIdx.x, lane = i & 31, N = p.N, pitch = words | 1, count = checked_count(p.status, p.counts, b, N);
  int parent = -1;
  if (i < count) {
    parent = __ldg(p.parents + b * p.row + i);
    if (parent < -1 || parent >= i) {                         // no earlier node
      report(p.status, kStatusBadTree + kInCache);
      parent = -1;
    }
  }
  const int first = i - lane;
  uint32_t mask = i < count ? 1u << lane : 0u;
  int jump = parent >= first ? parent - first : -1, exit = parent >= first ? -1 : parent;
#pragma unroll
  for (int r = 0; r < 5; ++r) {                               // after it, the first 2^(r + 1) ancestors of the group
    const int from = max(jump, 0);
    const uint32_t m = __shfl_sync(0xffffffffu, mask, from);
    const int j = __shfl_sync(0xffffffffu, jump, from), x = __shfl_sync(0xffffffffu, exit, from);
    if (jump >= 0) {
      mask |= m;
      exit = x;
      jump = j;
    }
  }
  among[i] = mask;
  behind[i] = exit;
  for (int x = i; x < N * pitch; x += blockDim.x) sets[x] = 0u;
  __syncthreads();
  if (i < N) {
    int bits = __popc(mask);
    sets[i * pitch + (i >> 5)] = mask;
    for (int at = exit; at >= 0; at = behind[at]) {           // the groups fall
      const uint32_t m = among[at];
      sets[i * pitch + (at >> 5)] = m;
      bits += __popc(m);
    }
    p.depth[static_cast<int64_t>(b) * N + i] = max(0, bits - 1);
  }
  __syncthreads();
  uint32_t* out = p.seen + static_cast<int64_t>(b) * N * words;
  for (int row = i / words, w = i - row * words; row < N;) {
    out[row * words + w] = sets[row * pitch + w];
    const int rows = blockDim.x / words;                      // the CTA's threads are whole rows: 32 a word
    row += rows;
  }
}

// ------------------------------------------------------------------------------------------------ keeping a path
// Token path[i] behind `before` becomes token i behind it.  A CTA is a (sequence, kv head, K or V), a warp a block of 32 tokens that is written: it reads
// the block's older tokens and its tokens of the path, takes the smallest power-of-two scale that holds them (as the eviction does), and rounds the codes
// to it.  A path is strictly increasing, so a token never moves up: what a block takes lies in it or behind it, and the warps of a CTA read all that
// they need before any of them writes; blocks of a later round are behind those.  The path is looked over while the first round's codes are on their way.
//
// Bound by the chain of loads (length, path, page, codes) of a round: 64 sequences of up to 250 drafts of which most are kept take 10.9 us (8 kv heads, 1.5 TB/s), 4 of 16 drafts 3.
// Warps a CTA 4, 6, 8: 11.9, 11.4, 12.8 us there; 8.3, 10.0, 9.9 with 120 drafts; 14.7, 12.0, 13.3 with 250 drafts in each sequence.
constexpr int kKeepWarps = 4;

template <int D>
__global__ void __launch_bounds__(kKeepWarps * 32, D == 128 ? 8 : 4) cache_keep_kernel(const CacheKeepParams p) {
  constexpr int kTpr = D / 16, kRpp = 32 / kTpr, kPass = 32 / kRpp;      // lanes a row, rows a pass, passes
  grid_dep_wait();
  const CacheView& c = p.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int rest = blockIdx.x;
  const bool is_v = (rest & 1) != 0;
  rest >>= 1;
  const int hk = rest % c.Hk, b = rest / c.Hk;
  const int n = cache_length(c, b);
  int start = __ldg(p.before + b), count = checked_count(c.status, p.counts, b, p.M);
  if (start < 0 || start > n) {
    report(c.status, kStatusBadLength + kInCache);
    start = min(max(start, 0), n);
  }
  const int* path = p.path + b * p.p_row;
  bool bad = false;
  for (int i = threadIdx.x; i < count; i += blockDim.x) {
    const int at = __ldg(path + i);
    bad |= at < 0 || at >= n - start || (i > 0 && __ldg(path + i - 1) >= at);
  }
  bool first_round = true;
  uint8_t* codes = (is_v ? c.v8 : c.k8) + hk * c.c_head;
  float* scales = (is_v ? c.vs : c.ks) + hk * c.s_head;
  const int bpp = c.page / 32, first = start / 32, blocks = count > 0 ? (start + count - 1) / 32 - first + 1 : 1;
  const int c16 = (lane % kTpr) * 16, r0 = lane / kTpr;
  for (int j0 = 0; j0 < blocks; j0 += blockDim.x / 32) {
    const int blk = first + j0 + warp, row = blk * 32 + lane; // this lane's row of the block, of 32
    const bool live = j0 + warp < blocks, held = live && row < start + count && (row < start || start < n);
    int64_t at = -1;                                          // its codes
    float s_row = 0.f;
    if (held) {
      // (not known to be a path yet: within the sequence in any case)
      const int from = row < start ? row : start + min(max(__ldg(path + row - start), 0), max(n - start - 1, 0)), entry = from / c.page;
      const int slot = from - entry * c.page, page = checked_page(c, __ldg(c.table + b * c.t_row + entry));
      if (page >= 0) {
        at = page * c.c_page + slot * c.c_slot;
        s_row = scales[page * c.s_page + slot / 32];
      }
    }
    uint4 y[kPass];
    float top = 0.f;                                          // of this lane's rows' codes, times their scales
    float s_of[kPass];
#pragma unroll
    for (int ps = 0; ps < kPass; ++ps) {
      const int r = r0 + ps * kRpp;
      const int64_t at_r = __shfl_sync(0xffffffffu, at, r);
      s_of[ps] = __shfl_sync(0xffffffffu, s_row, r);
      y[ps] = make_uint4(0, 0, 0, 0);
      if (at_r >= 0) y[ps] = *reinterpret_cast<const uint4*>(codes + at_r + c16);
    }
#pragma unroll
    for (int ps = 0; ps < kPass; ++ps) {
      const uint32_t w[4] = {y[ps].x, y[ps].y, y[ps].z, y[ps].w};
      // sizes of codes are in the order of their bytes; one more, so that NaN is the least (as f16 pairs the maximum took half as long again)
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t even = ((w[i] & 0x007F007Fu) + 0x00010001u) & 0x007F007Fu, odd = ((w[i] >> 8 & 0x007F007Fu) + 0x00010001u) & 0x007F007Fu;
        m = __vmaxu2(m, __vmaxu2(even, odd));
      }
      m = max(m & 0xFFFFu, m >> 16);
      top = fmaxf(top, f16x2_to_float2(e4m3_lo_f16x2(m > 0 ? m - 1 : 0)).x * s_of[ps]);
    }
    const uint32_t sb = pow2_sb(warp_max(top), 1u);
    const float s = sb_to_scale(sb);
    // the block's own place
    const int entry = live ? blk / bpp : 0;
    const int to = live && count > 0 && entry < c.T ? checked_page(c, __ldg(c.table + b * c.t_row + entry)) : -1;
    if (first_round) {                                        // not a path: nothing of the sequence is changed
      first_round = false;
      bad = __syncthreads_or(bad) != 0;
      if (bad && threadIdx.x == 0) report(c.status, kStatusBadTree + kInCache);
      if (hk == 0 && !is_v && threadIdx.x == 0) p.new_lengths[b] = start + (bad ? 0 : count);
      if (bad) return;
    } else {
      __syncthreads();
    }
    if (to >= 0) {
      uint8_t* out = codes + to * c.c_page + static_cast<int64_t>(blk - entry * bpp) * 32 * c.c_slot + c16;
#pragma unroll
      for (int ps = 0; ps < kPass; ++ps) {
        const int r = r0 + ps * kRpp;
        if (blk * 32 + r >= start + count) continue;
        // a code that is not zero needs no more than 2^18; zero stays zero
        const int e = static_cast<int>(scale_to_sb(s_of[ps])) - static_cast<int>(sb);
        const float ratio = sb_to_scale(static_cast<uint32_t>(min(18, max(e, -100)) + 127));
        uint4 w = y[ps];
        if (e != 0) w = make_uint4(requant4(w.x, ratio), requant4(w.y, ratio), requant4(w.z, ratio), requant4(w.w, ratio));
        *reinterpret_cast<uint4*>(out + r * c.c_slot) = w;
      }
      if (lane == 0) scales[to * c.s_page + blk - entry * bpp] = s;
    }
  }
}

}  // namespace

cudaError_t launch_draft_tree(const DraftTreeParams& p, cudaStream_t stream) {
  const int words = (p.N + 31) / 32, threads = words * 32, smem = (words | 1) * p.N * 4;
  if (smem > 40 * 1024) {                                     // beyond what a kernel has unasked, its static arrays aside
    static bool allowed[64] = {};                             // once per device: the driver call takes longer than a launch
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !allowed[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(draft_tree_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMaxNodes / 32 + 1) * kMaxNodes * 4);
      if (e != cudaSuccess) return e;
      if (dev >= 0 && dev < 64) allowed[dev] = true;
    }
  }
  count_launch();
  return launch_chained(draft_tree_kernel, dim3(p.B), threads, smem, stream, p, words);
}

cudaError_t launch_cache_keep(int D, const CacheKeepParams& p, cudaStream_t stream) {
  const int blocks = (p.M + 30) / 32 + 1, warps = blocks < kKeepWarps ? blocks : kKeepWarps;       // blocks that a path can touch
  const dim3 grid(static_cast<unsigned>(p.c.B) * p.c.Hk * 2);
  count_launch();
  return D == 128 ? launch_chained(cache_keep_kernel<128>, grid, warps * 32, 0, stream, p) : launch_chained(cache_keep_kernel<256>, grid, warps * 32, 0, stream, p);
}

}  // namespace dm
