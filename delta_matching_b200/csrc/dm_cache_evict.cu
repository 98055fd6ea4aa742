// Eviction by accumulated attention weight: which tokens of each (sequence, kv head) stay, then their codes into the pages of a new table.
//
// A sequence of n <= budget tokens keeps all.  Otherwise the last `recent` tokens stay, and of the others the budget - recent of greatest
// weight (equal weights: the lowest positions; NaN counts as the least), in their order.  Kept tokens of several old blocks share a new
// block of 32, so their codes move to the new block's scale: the smallest power of two s with amax <= 448 s over the values they stand for.
// The new pages are others than the old ones: an old page may be shared by several sequences, and every block can be written at once.
#include <cooperative_groups.h>
#include "dm_cache.cuh"
#include "dm_kernels.h"

namespace dm {

namespace {

namespace cg = cooperative_groups;

constexpr int kSelThreads = 512;
constexpr int kBins = 2048;

// Unsigned integers that order like the weights.
__device__ __forceinline__ uint32_t weight_key(float w) {
  w = w != w ? -CUDART_INF_F : w + 0.f;                       // -0 and +0 are equal
  const uint32_t u = __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive scan over the block of one value a thread; `total` for all.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t& total) {
  const int tid = threadIdx.x, lane = tid & 31;
  uint32_t incl = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += o;
  }
  __syncthreads();                                            // the sums of the scan before have been read
  if (lane == 31) warp_sums[tid >> 5] = incl;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) {
    if (w < (tid >> 5)) before += warp_sums[w];
    total += warp_sums[w];
  }
  return before + incl - v;
}

// One cluster per (sequence, kv head), each CTA a contiguous slice of the candidates.  The k-th greatest key by three digits of 11, 11 and 10
// bits, histograms added over the cluster; then the kept positions in order, by scans.
__global__ void __launch_bounds__(kSelThreads) cache_select_kernel(const CacheEvictParams p) {
  __shared__ uint4 hist4[kBins / 4];
  __shared__ uint32_t warp_sums[kSelThreads / 32];
  __shared__ uint32_t found[2];
  __shared__ uint32_t counts[2];
  uint32_t* hist = reinterpret_cast<uint32_t*>(hist4);
  grid_dep_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank(), tid = threadIdx.x;
  const int row = blockIdx.x / C, b = row / p.c.Hk, hk = row % p.c.Hk;
  const int n = cache_length(p.c, b), left = min(n, p.budget);
  const float* w = p.weights + b * p.w_sb + hk * p.w_sh;
  int* kept = p.kept + static_cast<int64_t>(row) * p.budget;
  const int W2 = p.T2 * p.c.page;
  float* nw = p.new_weights + static_cast<int64_t>(row) * W2;
  const int me = rank * kSelThreads + tid, all = C * kSelThreads;
  if (hk == 0 && me == 0) p.new_lengths[b] = left;
  for (int i = left + me; i < p.budget; i += all) kept[i] = -1;
  for (int i = left + me; i < W2; i += all) nw[i] = 0.f;
  if (n <= p.budget) {
    for (int i = me; i < n; i += all) {
      kept[i] = i;
      nw[i] = w[i];
    }
    return;
  }
  const int late = min(p.recent, p.budget), k = p.budget - late, cand = n - late;
  for (int i = me; i < late; i += all) {
    kept[k + i] = cand + i;
    nw[k + i] = w[cand + i];
  }
  if (k == 0) return;
  const int per = (cand + C - 1) / C, s0 = min(cand, rank * per), s1 = min(cand, s0 + per);

  uint32_t prefix = 0, mask = 0, want = k;                    // the want-th greatest among the keys that agree with prefix in mask
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digit = pass == 2 ? 1023u : 2047u;
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = s0 + tid; i < s1; i += kSelThreads) {
      const uint32_t key = weight_key(w[i]);
      if ((key & mask) == prefix) atomicAdd(hist + ((key >> shift) & digit), 1u);
    }
    cluster.sync();
    uint32_t h[4] = {0, 0, 0, 0};                             // bins 4 tid ... + 3 over the cluster
    for (int r = 0; r < C; ++r) {
      const uint4 v = *cluster.map_shared_rank(hist4 + tid, r);
      h[0] += v.x; h[1] += v.y; h[2] += v.z; h[3] += v.w;
    }
    uint32_t total;
    const uint32_t below = block_scan(h[0] + h[1] + h[2] + h[3], warp_sums, total);
    uint32_t above = total - below;                           // keys in this bin and the greater ones
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t greater = above - h[i];
      if (greater < want && want <= above) {
        found[0] = 4 * tid + i;
        found[1] = greater;
      }
      above = greater;
    }
    cluster.sync();                                           // found is there, and nobody reads the histograms any more
    prefix |= found[0] << shift;
    mask |= digit << shift;
    want -= found[1];
    __syncthreads();
  }

  // how many of the slices before mine are above the threshold, and equal to it
  uint32_t mine = 0, equal = 0;
  for (int i = s0 + tid; i < s1; i += kSelThreads) {
    const uint32_t key = weight_key(w[i]);
    mine += key > prefix;
    equal += key == prefix;
  }
  uint32_t total_mine, total_equal;
  block_scan(mine, warp_sums, total_mine);
  block_scan(equal, warp_sums, total_equal);
  if (tid == 0) {
    counts[0] = total_mine;
    counts[1] = total_equal;
  }
  cluster.sync();
  uint32_t gt = 0, eq = 0;
  for (int r = 0; r < rank; ++r) {
    gt += *cluster.map_shared_rank(counts, r);
    eq += *cluster.map_shared_rank(counts + 1, r);
  }
  cluster.sync();                                             // a CTA's shared memory stays until all have read it
  for (int at = s0; at < s1; at += kSelThreads * 4) {
    uint32_t flags = 0, ngt = 0, neq = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = at + tid * 4 + i;
      const uint32_t key = j < s1 ? weight_key(w[j]) : 0u;    // no weight has key 0
      if (key > prefix) {
        flags |= 1u << i;
        ++ngt;
      } else if (key == prefix && j < s1) {
        flags |= 16u << i;
        ++neq;
      }
    }
    uint32_t total;
    const uint32_t before = block_scan(ngt | neq << 16, warp_sums, total);
    uint32_t g = gt + (before & 0xFFFFu), e = eq + (before >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = at + tid * 4 + i;
      const bool is_gt = (flags >> i) & 1, is_eq = (flags >> (4 + i)) & 1;
      if (is_gt || (is_eq && e < want)) {
        const uint32_t to = g + min(e, want);
        kept[to] = j;
        nw[to] = w[j];
      }
      g += is_gt;
      e += is_eq;
    }
    gt += total & 0xFFFFu;
    eq += total >> 16;
  }
}

// Largest magnitude of four codes, NaN aside, as a code.
__device__ __forceinline__ uint32_t max_code4(uint32_t w) {
  w &= 0x7F7F7F7Fu;
  return w & ~__vcmpeq4(w, 0x7F7F7F7Fu);
}

// The kept tokens of a new block: one warp per (sequence, kv head, new block, K or V), rows in registers as in the append kernel.
template <int D>
__global__ void __launch_bounds__(128) cache_move_kernel(const CacheEvictParams p, int blocks, int64_t items) {
  constexpr int kTpr = D / 16, kRpp = 32 / kTpr, kPass = 32 / kRpp;
  grid_dep_wait();
  const CacheView& c = p.c;
  const int lane = threadIdx.x & 31;
  int64_t rest = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (rest >= items) return;
  const bool is_v = (rest & 1) != 0;
  rest >>= 1;
  const int j = static_cast<int>(rest % blocks);
  rest /= blocks;
  const int hk = static_cast<int>(rest % c.Hk), b = static_cast<int>(rest / c.Hk);
  const int left = min(cache_length(c, b), p.budget);
  if (j * 32 >= left) return;
  const int bpp = c.page / 32;
  const int to_page = checked_page(c, __ldg(p.new_table + b * p.nt_row + j / bpp));
  if (to_page < 0) return;
  // lane r looks row r up
  const uint8_t* pool = is_v ? c.v8 : c.k8;
  float* scales = is_v ? c.vs : c.ks;
  int64_t src = -1;
  float scale = 0.f;
  if (j * 32 + lane < left) {
    const int token = p.kept[(static_cast<int64_t>(b) * c.Hk + hk) * p.budget + j * 32 + lane];
    const int slot = token % c.page, page = checked_page(c, __ldg(c.table + b * c.t_row + token / c.page));
    if (page >= 0) {
      src = page * c.c_page + hk * c.c_head + slot * c.c_slot;
      scale = __ldg(scales + page * c.s_page + hk * c.s_head + slot / 32);
    }
  }
  const int c16 = (lane % kTpr) * 16, r0 = lane / kTpr;
  uint4 y[kPass];
#pragma unroll
  for (int ps = 0; ps < kPass; ++ps) {
    const int64_t at = __shfl_sync(0xffffffffu, src, r0 + ps * kRpp);
    y[ps] = at >= 0 ? __ldg(reinterpret_cast<const uint4*>(pool + at + c16)) : make_uint4(0, 0, 0, 0);
  }
  float amax = 0.f;
#pragma unroll
  for (int ps = 0; ps < kPass; ++ps) {
    uint32_t m = __vmaxu4(__vmaxu4(max_code4(y[ps].x), max_code4(y[ps].y)), __vmaxu4(max_code4(y[ps].z), max_code4(y[ps].w)));
    m = __vmaxu4(m, m >> 16);
    m = max(m & 0xFFu, (m >> 8) & 0xFFu);
    amax = fmaxf(amax, f16x2_to_float2(e4m3_lo_f16x2(m)).x * __shfl_sync(0xffffffffu, scale, r0 + ps * kRpp));
  }
  amax = warp_max(amax);
  const uint32_t sb = pow2_sb(amax, 1u);
  const float inv = sb_to_inv(sb);
  uint8_t* to = (is_v ? c.v8 : c.k8) + to_page * c.c_page + hk * c.c_head + static_cast<int64_t>(j % bpp) * 32 * c.c_slot + c16;
#pragma unroll
  for (int ps = 0; ps < kPass; ++ps) {
    const int r = r0 + ps * kRpp;
    // codes other than zero need at most 2^18; more would make zero times infinity of a zero row on a coarse scale
    const float ratio = fminf(__shfl_sync(0xffffffffu, scale, r) * inv, 1.099511627776e12f);
    uint4 v = y[ps];
    if (ratio != 1.f) {
      v.x = requant4(v.x, ratio);
      v.y = requant4(v.y, ratio);
      v.z = requant4(v.z, ratio);
      v.w = requant4(v.w, ratio);
    }
    *reinterpret_cast<uint4*>(to + r * c.c_slot) = v;
  }
  if (lane == 0) scales[to_page * c.s_page + hk * c.s_head + j % bpp] = sb_to_scale(sb);
}

}  // namespace

cudaError_t launch_cache_evict(int D, const CacheEvictParams& p, cudaStream_t stream) {
  // a CTA of the cluster takes 4096 tokens or more
  const int64_t most = static_cast<int64_t>(p.c.T) * p.c.page;
  int C = 1;
  while (C < 8 && most > 4096ll * C) C *= 2;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.c.B) * p.c.Hk * C);
  cfg.blockDim = dim3(kSelThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  count_launch();
  cudaError_t e = cudaLaunchKernelEx(&cfg, cache_select_kernel, p);
  if (e != cudaSuccess) return e;
  const int64_t kept = most < p.budget ? most : p.budget;
  const int blocks = static_cast<int>((kept + 31) / 32);
  const int64_t items = static_cast<int64_t>(p.c.B) * p.c.Hk * blocks * 2;
  const dim3 grid(static_cast<unsigned>((items + 3) / 4));
  count_launch();
  return D == 128 ? launch_chained(cache_move_kernel<128>, grid, 128, 0, stream, p, blocks, items)
                  : launch_chained(cache_move_kernel<256>, grid, 128, 0, stream, p, blocks, items);
}

}  // namespace dm
