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
constexpr int kBins = 4096;
constexpr int kSelKeys = 40960;             // keys of a CTA's slice that shared memory holds; longer slices are read again in each pass
constexpr int kSelSmem = kSelKeys * 4;
constexpr int kMaxCluster = 8;

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
  uint32_t sums = lane < kSelThreads / 32 ? warp_sums[lane] : 0;        // every warp scans the warps' sums
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, sums, off);
    if (lane >= off) sums += o;
  }
  total = __shfl_sync(0xffffffffu, sums, 31);
  const uint32_t before = __shfl_sync(0xffffffffu, sums, (tid >> 5) > 0 ? (tid >> 5) - 1 : 0);
  return ((tid >> 5) > 0 ? before : 0) + incl - v;
}

// One cluster per (sequence, kv head), each CTA a contiguous slice of the candidates, whose keys it keeps in shared memory.  The k-th greatest
// key by three digits of 12, 10 and 10 bits (the first is sign, exponent and three bits: weights of one size spread over many bins),
// histograms added over the cluster; then the kept positions in order, by scans.  Bound by the latency of its barriers: a barrier of eight CTAs
// takes 1200 - 3500 cycles, so of each other's histograms the CTAs read 32 sums and then the 32nd of the bins that matters.  Eight rows of
// 131071 tokens, 32768 kept: 19 us; 32 rows of 3001 - 4096: 8.
__global__ void __launch_bounds__(kSelThreads) cache_select_kernel(const CacheEvictParams p) {
  extern __shared__ uint4 keys4[];
  __shared__ uint4 hist4[kBins / 4];
  __shared__ uint32_t warp_sums[kSelThreads / 32];
  __shared__ uint32_t found[3];                               // bin, keys in greater ones, keys in it
  __shared__ uint32_t counts[2], sums[32];                    // sums: of the 32nds of the histogram
  uint32_t* keys = reinterpret_cast<uint32_t*>(keys4);
  uint32_t* hist = reinterpret_cast<uint32_t*>(hist4);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank(), tid = threadIdx.x, lane = tid & 31;
  for (int i = tid; i < kBins / 4; i += kSelThreads) hist4[i] = make_uint4(0, 0, 0, 0);
  grid_dep_wait();
  const auto sync_all = [&]() {
    if (C > 1) cluster.sync(); else __syncthreads();
  };
  const int row = blockIdx.x / C, b = row / p.c.Hk, hk = row - b * p.c.Hk;
  const int n = cache_length(p.c, b), left = min(n, p.budget);
  const float* w_row = p.weights + b * p.w_sb + hk * p.w_sh;
  int* kept = p.kept + static_cast<int64_t>(row) * p.budget;
  const int W2 = p.T2 * p.c.page;
  float* nw = p.new_weights + static_cast<int64_t>(row) * W2;
  const int me = rank * kSelThreads + tid, all = C * kSelThreads;
  const int late = n > p.budget ? min(p.recent, p.budget) : n, k = left - late, cand = n - late;      // k of the first cand, and the late ones
  if (k > 0) {
    const int per = ((cand + C - 1) / C + 3) & ~3, s0 = min(cand, rank * per), len = min(cand, s0 + per) - s0;
    const bool held = per <= kSelKeys;
    const float* w = w_row + s0;
    auto key_at = [&](int i) { return held ? keys[i] : weight_key(__ldg(w + i)); };
    __syncthreads();

    uint32_t prefix = 0, mask = 0, want = k;                  // the want-th greatest among the keys that agree with prefix in mask
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 20 : pass == 1 ? 10 : 0, quads = (pass == 0 ? kBins : 1024) / 4;
      if (pass == 0) {
        const int loads = (reinterpret_cast<uintptr_t>(w) & 15) == 0 ? len / 4 : 0;
#pragma unroll 4
        for (int i = tid; i < loads; i += kSelThreads) {
          const float4 x = __ldg(reinterpret_cast<const float4*>(w) + i);
          const uint4 key = make_uint4(weight_key(x.x), weight_key(x.y), weight_key(x.z), weight_key(x.w));
          if (held) keys4[i] = key;
          atomicAdd(hist + (key.x >> 20), 1u);
          atomicAdd(hist + (key.y >> 20), 1u);
          atomicAdd(hist + (key.z >> 20), 1u);
          atomicAdd(hist + (key.w >> 20), 1u);
        }
        for (int i = 4 * loads + tid; i < len; i += kSelThreads) {
          const uint32_t key = weight_key(__ldg(w + i));
          if (held) keys[i] = key;
          atomicAdd(hist + (key >> 20), 1u);
        }
      } else {
        const auto take = [&](uint32_t key) {
          if ((key & mask) == prefix) atomicAdd(hist + ((key >> shift) & 1023u), 1u);
        };
        const int loads = held ? len / 4 : 0;
#pragma unroll 2
        for (int i = tid; i < loads; i += kSelThreads) {
          const uint4 key = keys4[i];
          take(key.x);
          take(key.y);
          take(key.z);
          take(key.w);
        }
        for (int i = 4 * loads + tid; i < len; i += kSelThreads) take(key_at(i));
      }
      __syncthreads();
      // which 32nd of the bins holds the want-th key: from the CTAs' sums
      const int part = quads / 32;                            // quads of a 32nd: a warp's, or those of eight lanes
      for (int i = tid; i < quads; i += kSelThreads) {
        const uint4 v = hist4[i];
        uint32_t sum = v.x + v.y + v.z + v.w;
        for (int o = part / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if ((i & (part - 1)) == 0) sums[i / part] = sum;
      }
      sync_all();
      if (tid < 32) {
        uint32_t sum = C == 1 ? sums[lane] : 0;
        if (C > 1) {
#pragma unroll
          for (int r = 0; r < kMaxCluster; ++r) sum += r < C ? *cluster.map_shared_rank(sums + lane, r) : 0;      // all on their way together
        }
        uint32_t from = sum;                                  // keys in this 32nd and the greater ones
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t x = __shfl_down_sync(0xffffffffu, from, o);
          if (lane + o < 32) from += x;
        }
        const int which = __ffs(__ballot_sync(0xffffffffu, from - sum < want && want <= from)) - 1;
        const uint32_t above = __shfl_sync(0xffffffffu, from, which);         // keys in its bins and the greater ones
        // its bins over the cluster
        uint32_t h[4] = {0, 0, 0, 0};
        if (lane < part) {
          const uint4* mine = hist4 + which * part + lane;
          uint4 v[kMaxCluster];
          v[0] = C > 1 ? *cluster.map_shared_rank(mine, 0) : *mine;
#pragma unroll
          for (int r = 1; r < kMaxCluster; ++r) v[r] = r < C ? *cluster.map_shared_rank(mine, r) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < kMaxCluster; ++r) {
            h[0] += v[r].x; h[1] += v[r].y; h[2] += v[r].z; h[3] += v[r].w;
          }
        }
        const uint32_t four = h[0] + h[1] + h[2] + h[3];
        uint32_t incl = four;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += x;
        }
        uint32_t at = above - (incl - four);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t greater = at - h[i];
          if (greater < want && want <= at) {
            found[0] = 4 * (which * part + lane) + i;
            found[1] = greater;
            found[2] = h[i];
          }
          at = greater;
        }
      }
      sync_all();                                             // found is there, and nobody reads the histograms any more
      prefix |= found[0] << shift;
      mask |= (pass == 0 ? 4095u : 1023u) << shift;
      want -= found[1];
      if (found[2] == want && prefix > 0) {                   // all of the bin are taken: what is above its lower end, and none that is equal to that
        --prefix;
        want = 0;
        break;
      }
      if (pass < 2) {
        for (int i = tid; i < 1024 / 4; i += kSelThreads) hist4[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
      }
    }

    // Adjacent tokens a thread takes at a time, and a slice that is taken at once: above the threshold, equal to it, as bits.  (Eight at a time in any
    // case, and the numbers for the cluster counted on their own, took 14000 cycles of a slice of 16384; a slice of 4096 by 32 at a time leaves
    // most threads idle.)
    const int take = per > 8 * kSelThreads ? 32 : 8;
    const bool once = per <= take * kSelThreads;
    uint32_t above = 0, equal = 0, before = 0, total = 0;
    const auto look = [&](int j0) {
      above = equal = 0;
      for (int i = 0; i < take / 4; ++i) {
        const int q = take == 32 ? 4 * ((i + lane) & 7) : 4 * i, j = j0 + q;        // (lanes on different banks)
        if (j >= len) continue;
        uint32_t key[4];
        if (held) {                                           // a slice's keys are whole quads
          const uint4 v = keys4[j / 4];
          key[0] = v.x; key[1] = v.y; key[2] = v.z; key[3] = v.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) key[e] = weight_key(__ldg(w + min(j + e, len - 1)));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (j + e >= len) break;
          above |= (key[e] > prefix ? 1u : 0u) << (q + e);
          equal |= (key[e] == prefix ? 1u : 0u) << (q + e);
        }
      }
      before = block_scan(__popc(above) | __popc(equal) << 16, warp_sums, total);
    };
    if (once) look(tid * take);
    uint32_t gt = 0, eq = 0;                                  // of the slices before mine
    if (C > 1) {
      if (!once) {
        uint32_t mine = 0, same = 0;
        for (int i = tid; i < len; i += kSelThreads) {
          const uint32_t key = key_at(i);
          mine += key > prefix;
          same += key == prefix;
        }
        mine = __reduce_add_sync(0xffffffffu, mine);
        same = __reduce_add_sync(0xffffffffu, same);
        if (tid < 2) counts[tid] = 0;
        __syncthreads();
        if (lane == 0) {
          atomicAdd(counts, mine);
          atomicAdd(counts + 1, same);
        }
      } else if (tid == 0) {
        counts[0] = total & 0xFFFFu;
        counts[1] = total >> 16;
      }
      cluster.sync();
      gt = __reduce_add_sync(0xffffffffu, lane < rank ? *cluster.map_shared_rank(counts, lane) : 0u);       // a lane per CTA before this one
      eq = __reduce_add_sync(0xffffffffu, lane < rank ? *cluster.map_shared_rank(counts + 1, lane) : 0u);
    }
    for (int at = 0; at < len; at += kSelThreads * take) {
      const int j0 = at + tid * take;
      if (!once) look(j0);
      const uint32_t g = gt + (before & 0xFFFFu), e = eq + (before >> 16);
      // of mine that are equal to the threshold, the first ones until there are `want`
      uint32_t picks = above, equals = equal;
      for (uint32_t room = e < want ? want - e : 0; equals != 0 && room > 0; --room) {
        picks |= equals & -equals;
        equals &= equals - 1;
      }
      // a list of the picked ones over the keys that have been read (behind the scan's barriers), written out by adjacent threads
      uint32_t* list = held ? keys + at : keys;
      const uint32_t first = gt + min(eq, want);
      for (uint32_t to = g + min(e, want) - first; picks != 0; ++to) {
        list[to] = j0 + __ffs(picks) - 1;
        picks &= picks - 1;
      }
      gt += total & 0xFFFFu;
      eq += total >> 16;
      __syncthreads();
      const int picked = gt + min(eq, want) - first;
#pragma unroll 4
      for (int i = tid; i < picked; i += kSelThreads) {
        const int j = list[i];
        kept[first + i] = s0 + j;
        nw[first + i] = __ldg(w + j);
      }
    }
  }
  // the late ones (all, within the budget), and what lies behind
  for (int i = me; i < late; i += all) {
    kept[k + i] = cand + i;
    nw[k + i] = __ldg(w_row + cand + i);
  }
  for (int i = left + me; i < p.budget; i += all) kept[i] = -1;
  for (int i = left + me; i < W2; i += all) nw[i] = 0.f;
  if (hk == 0 && me == 0) p.new_lengths[b] = left;
  if (C > 1) cluster.sync();                                  // a CTA's counts stay until all have read them
}

// Two f16 values, as words: largest magnitudes (NaN aside), product, e4m3 codes (round to nearest even).
__device__ __forceinline__ uint32_t h2_max_abs(uint32_t a, uint32_t b) {
  const __half2 m = __hmax2(__habs2(*reinterpret_cast<const __half2*>(&a)), __habs2(*reinterpret_cast<const __half2*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t h2_scaled_codes(uint32_t a, uint32_t b, __half2 by) {
  const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&a), by), y = __hmul2(*reinterpret_cast<const __half2*>(&b), by);
  uint32_t w;
  asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f16x2 lo, %1;\n\tcvt.rn.satfinite.e4m3x2.f16x2 hi, %2;\n\tmov.b32 %0, {lo, hi};\n\t}"
      : "=r"(w) : "r"(*reinterpret_cast<const uint32_t*>(&x)), "r"(*reinterpret_cast<const uint32_t*>(&y)));
  return w;
}

// The kept tokens of a new block: one warp per (sequence, kv head, new block, K or V), rows in registers as in the append kernel.
// Registers are held down (the f16 values of the maximum are made again for the codes): what hides the loads is many warps.
template <int D>
__global__ void __launch_bounds__(128, D == 128 ? 7 : 4) cache_move_kernel(const CacheEvictParams p, int blocks, int64_t items) {
  constexpr int kTpr = D / 16, kRpp = 32 / kTpr, kPass = 32 / kRpp;
  const CacheView& c = p.c;
  const int lane = threadIdx.x & 31;
  int64_t rest = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (rest >= items) {
    grid_dep_wait();
    return;
  }
  const bool is_v = (rest & 1) != 0;
  rest >>= 1;
  const int j = static_cast<int>(rest % blocks);
  rest /= blocks;
  const int hk = static_cast<int>(rest % c.Hk), b = static_cast<int>(rest / c.Hk);
  // what the caller gave, before the wait for the selection (which has itself waited for all kernels before it)
  const int left = min(cache_length(c, b), p.budget), bpp = c.page / 32;
  const int to_page = j * 32 < left ? checked_page(c, __ldg(p.new_table + b * p.nt_row + j / bpp)) : -1;
  grid_dep_wait();
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
    uint32_t m = 0;
    const uint32_t v[4] = {y[ps].x, y[ps].y, y[ps].z, y[ps].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = h2_max_abs(m, h2_max_abs(e4m3_lo_f16x2(v[i]), e4m3_hi_f16x2(v[i])));
    const float2 top = f16x2_to_float2(m);
    amax = fmaxf(amax, fmaxf(top.x, top.y) * __shfl_sync(0xffffffffu, scale, r0 + ps * kRpp));
  }
  amax = warp_max(amax);
  const uint32_t sb = pow2_sb(amax, 1u);
  const float ratio = scale * sb_to_inv(sb);                  // of this lane's row
  uint8_t* to = (is_v ? c.v8 : c.k8) + to_page * c.c_page + hk * c.c_head + static_cast<int64_t>(j % bpp) * 32 * c.c_slot + c16;
  if (__all_sync(0xffffffffu, ratio == 1.f || src < 0)) {     // all from blocks of the new scale: as they are
#pragma unroll
    for (int ps = 0; ps < kPass; ++ps) *reinterpret_cast<uint4*>(to + (r0 + ps * kRpp) * c.c_slot) = y[ps];
  } else if (__all_sync(0xffffffffu, ratio <= 32768.f)) {
    // in f16: what its subnormals round away is far below half of e4m3's smallest step
#pragma unroll
    for (int ps = 0; ps < kPass; ++ps) {
      const __half2 by = __float2half2_rn(__shfl_sync(0xffffffffu, ratio, r0 + ps * kRpp));
      uint4 v = y[ps];
      asm volatile("" : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w));      // not the f16 values from above, kept in registers
      v.x = h2_scaled_codes(e4m3_lo_f16x2(v.x), e4m3_hi_f16x2(v.x), by);
      v.y = h2_scaled_codes(e4m3_lo_f16x2(v.y), e4m3_hi_f16x2(v.y), by);
      v.z = h2_scaled_codes(e4m3_lo_f16x2(v.z), e4m3_hi_f16x2(v.z), by);
      v.w = h2_scaled_codes(e4m3_lo_f16x2(v.w), e4m3_hi_f16x2(v.w), by);
      *reinterpret_cast<uint4*>(to + (r0 + ps * kRpp) * c.c_slot) = v;
    }
  } else {
#pragma unroll 1
    for (int r = r0; r < 32; r += kRpp) {
      // codes other than zero need at most 2^18; more would make zero times infinity of a zero row on a coarse scale
      const float by = fminf(__shfl_sync(0xffffffffu, ratio, r), 1.099511627776e12f);
      const int64_t at = __shfl_sync(0xffffffffu, src, r);
      uint4 v = at >= 0 ? __ldg(reinterpret_cast<const uint4*>(pool + at + c16)) : make_uint4(0, 0, 0, 0);
      v.x = requant4(v.x, by);
      v.y = requant4(v.y, by);
      v.z = requant4(v.z, by);
      v.w = requant4(v.w, by);
      *reinterpret_cast<uint4*>(to + r * c.c_slot) = v;
    }
  }
  if (lane == 0) scales[to_page * c.s_page + hk * c.s_head + j % bpp] = sb_to_scale(sb);
}

}  // namespace

cudaError_t launch_cache_evict(int D, const CacheEvictParams& p, cudaStream_t stream) {
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(cache_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  // A CTA of the cluster takes 4096 tokens or more.  us of a call with 2048, 4096 and 8192: 32 rows of 3001 - 4096 tokens 16.2, 13.6 and 13.6, 128 rows of
  // 2500 - 4096 47.0, 37.5 and 37.5, 16 rows of 16384 23.2, 15.9 and 17.8, 8 rows of 32768 17.6, 17.6 and 19.5.  (Clusters of 16: few are resident
  // at a time; eight rows of 131072 tokens took 75 against 33.)
  const int64_t most = static_cast<int64_t>(p.c.T) * p.c.page;
  int C = 1;
  while (C < kMaxCluster && most > 4096ll * C) C *= 2;
  const int64_t slice = ((most + C - 1) / C + 3) / 4 * 4;
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
  cfg.dynamicSmemBytes = (slice <= kSelKeys ? slice : kSelKeys) * 4;
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
