// C-ABI layer of the functions for drafted tokens: argument validation, launches (see dm_abi.cu for the conventions).
#include <cfloat>

#include "dm_cache_abi.h"
#include "dm_drafts.h"

using namespace dm::abi;

namespace {

int check_nodes(const char* what, int B, int N) {
  if (B <= 0 || N <= 0) return fail(DM_ERR_ARG, "delta_matching: empty tensor (B=%d N=%d)", B, N);
  if (N > dm::kMaxNodes) return fail(DM_ERR_ARG, "delta_matching: %s of at most %d drafted tokens (got %d)", what, dm::kMaxNodes, N);
  return 0;
}

int check_pointer(const void* p, const char* name) {
  return p != nullptr ? 0 : fail(DM_ERR_ARG, "delta_matching: %s is NULL (every tensor must be a CUDA buffer)", name);
}

int check_tree_shape(int B, int N, int H, int Hk, int D, int T, int page) {
  DM_TRY(check_nodes("a tree", B, N));
  if (D != 128 && D != 256) return fail(DM_ERR_ARG, "delta_matching: head_dim must be 128 or 256 (got %d)", D);
  if (H <= 0 || Hk <= 0 || T <= 0) return fail(DM_ERR_ARG, "delta_matching: empty tensor (B=%d N=%d H=%d Hk=%d)", B, N, H, Hk);
  if (page <= 0 || page % 32) return fail(DM_ERR_ARG, "delta_matching: page size must be a positive multiple of 32 (got %d)", page);
  if (H % Hk) return fail(DM_ERR_ARG, "delta_matching: nheads (%d) must be a multiple of nheads_k (%d)", H, Hk);
  if (static_cast<int64_t>(B) * H > 65535) return fail(DM_ERR_ARG, "delta_matching: batch * nheads must be at most 65535");
  // steps of the division of the work are ints: of 128 rows x 128 tokens, and a few a unit
  const int64_t row_tiles = (static_cast<int64_t>(N) * (H / Hk) + 127) / 128;
  if (static_cast<int64_t>(T) * page / 128 + 8 > (1ll << 30) / (static_cast<int64_t>(B) * Hk * row_tiles))
    return fail(DM_ERR_ARG, "delta_matching: too much work for one call (%d sequences with room for %lld tokens, %lld rows)", B,
                static_cast<long long>(T) * page, static_cast<long long>(N) * H);
  return 0;
}

}  // namespace

extern "C" {

int dm_draft_tree(const int* parents, int64_t parents_row, const int* counts, int B, int N, int* depth, int* seen, int* status, void* stream) {
  DM_TRY(check_nodes("a tree", B, N));
  DM_TRY(check_pointer(parents, "parents"));
  DM_TRY(check_pointer(depth, "depth"));
  DM_TRY(check_pointer(seen, "seen"));
  if (parents_row < 0) return fail(DM_ERR_ARG, "delta_matching: rows of parents are %lld apart", static_cast<long long>(parents_row));
  DM_TRY(check_sm100());
  dm::DraftTreeParams p{};
  p.parents = parents; p.row = parents_row; p.counts = counts;
  p.B = B; p.N = N;
  p.depth = depth;
  p.seen = reinterpret_cast<uint32_t*>(seen);
  p.status = status;
  const cudaError_t e = dm::launch_draft_tree(p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : cuda_fail(e, "draft tree launch");
}

int dm_cache_append_rotary(const dm_kv_cache* cache, const void* q, int64_t q_sb, int64_t q_sn, int64_t q_sh,
                           const void* k, int64_t k_sb, int64_t k_sn, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_sn, int64_t v_sh,
                           int B, int N, int H, const float* freqs, int n_freqs, int interleaved,
                           const int* table, int64_t table_row, int T, const int* lengths, const int* offsets, int64_t offsets_row, const int* counts,
                           void* q_out, int* new_lengths, int* status, void* stream) {
  DM_TRY(check_cache(cache));
  DM_TRY(check_table(cache, table, table_row, T, lengths, B, "block table"));
  if (N <= 0 || H <= 0) return fail(DM_ERR_ARG, "delta_matching: empty tensor (N=%d H=%d)", N, H);
  if (H % cache->heads) return fail(DM_ERR_ARG, "delta_matching: nheads (%d) must be a multiple of nheads_k (%d)", H, cache->heads);
  DM_TRY(check_rows("q", q, q_sb, q_sn, q_sh));
  DM_TRY(check_rows("k", k, k_sb, k_sn, k_sh));
  DM_TRY(check_rows("v", v, v_sb, v_sn, v_sh));
  DM_TRY(check_address(q_out, "rotated q"));
  DM_TRY(check_pointer(freqs, "freqs"));
  DM_TRY(check_pointer(new_lengths, "new lengths"));
  if (n_freqs <= 0 || n_freqs % 8 || 2 * n_freqs > cache->head_dim)
    return fail(DM_ERR_ARG, "delta_matching: freqs must be a multiple of 8 frequencies, for at most the %d channels of a head (got %d)", cache->head_dim, n_freqs);
  if (offsets != nullptr && offsets_row < 0) return fail(DM_ERR_ARG, "delta_matching: rows of offsets are %lld apart", static_cast<long long>(offsets_row));
  if (N > (1 << 28) || (static_cast<int64_t>(N) + 30) / 32 + 1 > (1ll << 31) / B - 1 || static_cast<int64_t>(B) * H > 65535)
    return fail(DM_ERR_ARG, "delta_matching: too many tokens in one call (%d x %d, %d heads)", B, N, H);
  DM_TRY(check_new_lengths(new_lengths, B, {{lengths, 1, 1, "lengths"}, {counts, 1, 1, "counts"}, {offsets, offsets_row, N, "offsets"}, {table, table_row, T, "block table"}}));
  DM_TRY(check_sm100());
  dm::CacheRotaryParams p{};
  p.c = view_of(cache, table, table_row, T, lengths, B, status);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.q_sb = q_sb; p.q_sn = q_sn; p.q_sh = q_sh;
  p.k_sb = k_sb; p.k_sn = k_sn; p.k_sh = k_sh;
  p.v_sb = v_sb; p.v_sn = v_sn; p.v_sh = v_sh;
  p.freqs = freqs; p.half = n_freqs; p.interleaved = interleaved ? 1 : 0;
  p.offsets = offsets; p.o_row = offsets_row;
  p.counts = counts;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.new_lengths = new_lengths;
  p.N = N; p.H = H;
  const cudaError_t e = dm::launch_cache_rotary(cache->head_dim, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : cuda_fail(e, "cache append with rotation launch");
}

int64_t dm_cache_attn_tree_workspace_bytes(int B, int N, int H, int Hk, int D, int T, int page_size) {
  if (check_tree_shape(B, N, H, Hk, D, T, page_size) != 0) return 0;
  return dm::plan_cache_tree(B, N, H, Hk, D, T, page_size).bytes();
}

int dm_dbg_cache_tree_plan(int B, int N, int H, int Hk, int D, int T, int page_size, int what) {
  DM_TRY(check_tree_shape(B, N, H, Hk, D, T, page_size));
  const dm::CacheTreePlan x = dm::plan_cache_tree(B, N, H, Hk, D, T, page_size);
  switch (what) {
    case 0: return x.cluster;
    case 1: return x.grid;
    case 2: return x.row_tile;
    case 3: return static_cast<int>(x.part_o_bytes + x.part_ml_bytes);        // (of 148 CTAs at most: 80 MB)
  }
  return fail(DM_ERR_ARG, "delta_matching: what must be 0 ... 3 (got %d)", what);
}

int dm_cache_attn_tree(const dm_kv_cache* cache, const void* q, int64_t q_sb, int64_t q_sn, int64_t q_sh, int B, int N, int H,
                       const int* table, int64_t table_row, int T, const int* lengths, const int* counts, const int* seen, int64_t seen_sb, int64_t seen_sn,
                       float softmax_scale, void* o, float* lse, void* workspace, int64_t workspace_bytes, int* status, void* stream) {
  DM_TRY(check_cache(cache));
  DM_TRY(check_table(cache, table, table_row, T, lengths, B, "block table"));
  DM_TRY(check_tree_shape(B, N, H, cache->heads, cache->head_dim, T, cache->page_size));
  DM_TRY(check_rows("q", q, q_sb, q_sn, q_sh));
  DM_TRY(check_addresses({{o, "o"}, {lse, "lse"}, {workspace, "workspace"}}));
  DM_TRY(check_pointer(seen, "seen"));
  if (seen_sb < 0 || seen_sn < 0) return fail(DM_ERR_ARG, "delta_matching: strides of seen must not be negative");
  if (!(softmax_scale > 0.f && softmax_scale <= FLT_MAX)) return fail(DM_ERR_ARG, "delta_matching: softmax_scale must be positive and finite in 32 bits (got %g)", softmax_scale);
  const dm::CacheTreePlan x = dm::plan_cache_tree(B, N, H, cache->heads, cache->head_dim, T, cache->page_size);
  const int64_t need = x.bytes();
  if (workspace_bytes < need)
    return fail(DM_ERR_ARG, "delta_matching: workspace of %lld bytes given, %lld needed", static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  DM_TRY(check_sm100());
  dm::CacheTreeParams p{};
  p.c = view_of(cache, table, table_row, T, lengths, B, status);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_sb = q_sb; p.q_sn = q_sn; p.q_sh = q_sh;
  p.counts = counts;
  p.seen = reinterpret_cast<const uint32_t*>(seen);
  p.s_sb = seen_sb; p.s_sn = seen_sn;
  p.N = N; p.H = H; p.rep = H / cache->heads;
  p.scale = softmax_scale;
  p.o = static_cast<__nv_bfloat16*>(o);
  p.lse = lse;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float4*>(static_cast<uint8_t*>(workspace) + x.part_o_bytes);
  p.marks = static_cast<uint8_t*>(workspace) + x.part_o_bytes + x.part_ml_bytes;
  p.cuts = static_cast<uint8_t*>(workspace) + x.part_o_bytes + x.part_ml_bytes + x.mark_bytes;
  p.grid = x.grid;
  p.cluster = x.cluster;
  p.row_tile = x.row_tile;
  for (p.row_shift = 0; 1 << p.row_shift < x.row_tile;) ++p.row_shift;
  // exact up to r < 2^32 / rep
  if (p.rep > 1 && (static_cast<int64_t>(N) * p.rep + x.row_tile) * p.rep < (1ll << 32)) p.rep_magic = static_cast<uint32_t>(((1ll << 32) + p.rep - 1) / p.rep);
  CUtensorMap tk, tv;
  DM_TRY(pool_map(&tk, cache, cache->k8));
  DM_TRY(pool_map(&tv, cache, cache->v8));
  const cudaError_t e = dm::launch_cache_tree(cache->head_dim, tk, tv, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : cuda_fail(e, "cache tree attention launch");
}

int dm_cache_keep(const dm_kv_cache* cache, int B, const int* table, int64_t table_row, int T, const int* before, const int* lengths,
                  const int* path, int64_t path_row, int M, const int* counts, int* new_lengths, int* status, void* stream) {
  DM_TRY(check_cache(cache));
  DM_TRY(check_table(cache, table, table_row, T, lengths, B, "block table"));
  DM_TRY(check_nodes("a path", B, M));
  DM_TRY(check_pointer(before, "before"));
  DM_TRY(check_pointer(path, "path"));
  DM_TRY(check_pointer(counts, "counts"));
  DM_TRY(check_pointer(new_lengths, "new lengths"));
  if (path_row < 0) return fail(DM_ERR_ARG, "delta_matching: rows of path are %lld apart", static_cast<long long>(path_row));
  DM_TRY(check_new_lengths(new_lengths, B, {{before, 1, 1, "before"}, {lengths, 1, 1, "lengths"}, {counts, 1, 1, "counts"}, {path, path_row, M, "path"}, {table, table_row, T, "block table"}}));
  DM_TRY(check_sm100());
  dm::CacheKeepParams p{};
  p.c = view_of(cache, table, table_row, T, lengths, B, status);
  p.before = before;
  p.path = path; p.p_row = path_row; p.M = M;
  p.counts = counts;
  p.new_lengths = new_lengths;
  const cudaError_t e = dm::launch_cache_keep(cache->head_dim, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : cuda_fail(e, "cache keep launch");
}

}  // extern "C"
