// Attention of a tree of drafted tokens over the 8-bit cache.
//
//   s_rj = scale q_r . (ks code_j);  o_r = sum_j exp(s_rj - m_r) vs code_j / sum_j exp(s_rj - m_r)  over the keys j that row r sees:
//   all tokens held before the drafted ones, and of these its node's own ancestors and itself
//
// A warp a row, a key after the other.
#include "dm_cache.cuh"
#include "dm_drafts.h"
#include "dm_kernels.h"

namespace dm {

namespace {

// A sequence's tokens and drafted tokens: the last `count` of its n.
struct TreeSeq {
  int n, count;
  __device__ __forceinline__ int base() const { return n - count; }
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
// The nodes that node i sees, of word w: earlier ones and itself, whatever the bits behind it say.
__device__ __forceinline__ uint32_t seen_word(const uint32_t* seen, int i, int w) {
  if (w > i >> 5) return 0u;
  const uint32_t x = __ldg(seen + w);
  if (w < i >> 5) return x;
  const uint32_t self = 1u << (i & 31);
  return (x & (self - 1u)) | self;
}

template <int D>
__global__ void __launch_bounds__(128) cache_tree_rows_kernel(const CacheTreeParams p) {
  constexpr int kVecs = D / 128;
  grid_dep_wait();
  const int lane = threadIdx.x & 31, bpp = p.c.page / 32;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<int64_t>(p.c.B) * p.N * p.H) return;
  const int head = static_cast<int>(row % p.H), i = static_cast<int>(row / p.H % p.N), b = static_cast<int>(row / p.H / p.N), hk = head / p.rep;
  const TreeSeq t = tree_seq(p, b);
  __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(p.o + row * D) + 2 * lane;
  float* lse = p.lse + (static_cast<int64_t>(b) * p.H + head) * p.N + i;
  if (i >= t.count) {
#pragma unroll
    for (int x = 0; x < kVecs; ++x) o[64 * x] = o[64 * x + 1] = __floats2bfloat162_rn(0.f, 0.f);
    if (lane == 0) *lse = -CUDART_INF_F;
    return;
  }
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
  const float sum = static_cast<float>(l);
#pragma unroll
  for (int x = 0; x < kVecs; ++x) {
    o[64 * x] = __floats2bfloat162_rn(acc[x].x / sum, acc[x].y / sum);
    o[64 * x + 1] = __floats2bfloat162_rn(acc[x].z / sum, acc[x].w / sum);
  }
  if (lane == 0) *lse = (m + log2f(sum)) * kLn2;
}

}  // namespace

cudaError_t launch_cache_tree(int D, const CacheTreeParams& p, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(p.c.B) * p.N * p.H + 3) / 4));
  count_launch();
  return D == 128 ? launch_chained(cache_tree_rows_kernel<128>, grid, 128, 0, stream, p) : launch_chained(cache_tree_rows_kernel<256>, grid, 128, 0, stream, p);
}

}  // namespace dm
