// C-ABI layer of the 8-bit key / value cache: argument validation, tensor maps of the pools, launches (see dm_abi.cu for the conventions).
#include <cfloat>

#include "dm_cache_abi.h"

using namespace dm::abi;

extern "C" {

int dm_cache_append(const dm_kv_cache* cache, const void* k, int64_t k_sb, int64_t k_sn, int64_t k_sh,
                    const void* v, int64_t v_sb, int64_t v_sn, int64_t v_sh, int B, int N,
                    const int* table, int64_t table_row, int T, const int* lengths, const int* counts, int* new_lengths,
                    int* status, void* stream) {
  DM_TRY(check_cache(cache));
  DM_TRY(check_table(cache, table, table_row, T, lengths, B, "block table"));
  if (N <= 0) return fail(DM_ERR_ARG, "delta_matching: empty tensor (N=%d)", N);
  DM_TRY(check_rows("k", k, k_sb, k_sn, k_sh));
  DM_TRY(check_rows("v", v, v_sb, v_sn, v_sh));
  if (new_lengths == nullptr) return fail(DM_ERR_ARG, "delta_matching: new lengths is NULL (every tensor must be a CUDA buffer)");
  if ((static_cast<int64_t>(N) + 30) / 32 + 1 > (1ll << 32) / (static_cast<int64_t>(B) * cache->heads * 2))
    return fail(DM_ERR_ARG, "delta_matching: too many tokens in one call (%d x %d)", B, N);
  DM_TRY(check_new_lengths(new_lengths, B, {{lengths, 1, 1, "lengths"}, {counts, 1, 1, "counts"}, {table, table_row, T, "block table"}}));
  DM_TRY(check_sm100());
  dm::CacheAppendParams p{};
  p.c = view_of(cache, table, table_row, T, lengths, B, status);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.k_sb = k_sb; p.k_sn = k_sn; p.k_sh = k_sh;
  p.v_sb = v_sb; p.v_sn = v_sn; p.v_sh = v_sh;
  p.counts = counts;
  p.new_lengths = new_lengths;
  p.N = N;
  const cudaError_t e = dm::launch_cache_append(cache->head_dim, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : cuda_fail(e, "cache append launch");
}

static int check_attn_shape(int B, int Nq, int H, int Hk, int D, int T, int page) {
  if (D != 128 && D != 256) return fail(DM_ERR_ARG, "delta_matching: head_dim must be 128 or 256 (got %d)", D);
  if (B <= 0 || Nq <= 0 || H <= 0 || Hk <= 0 || T <= 0) return fail(DM_ERR_ARG, "delta_matching: empty tensor (B=%d N=%d H=%d Hk=%d)", B, Nq, H, Hk);
  if (page <= 0 || page % 32) return fail(DM_ERR_ARG, "delta_matching: page size must be a positive multiple of 32 (got %d)", page);
  if (H % Hk) return fail(DM_ERR_ARG, "delta_matching: nheads (%d) must be a multiple of nheads_k (%d)", H, Hk);
  if (static_cast<int64_t>(B) * H > 65535) return fail(DM_ERR_ARG, "delta_matching: batch * nheads must be at most 65535");
  if (Nq > (1 << 20) || static_cast<int64_t>(B) * H * Nq > (1ll << 30))
    return fail(DM_ERR_ARG, "delta_matching: too many query rows (%d sequences, %d heads, %d tokens)", B, H, Nq);
  // Steps of the division of the work are ints: of 8 rows x 32 tokens at least, for many rows of 128 x 128.
  const int64_t rows = static_cast<int64_t>(Nq) * (H / Hk), row_tiles = (rows + 7) / 8, most = rows >= dm::cache_chunk_from(D) ? 1ll << 34 : 1ll << 30;
  if (static_cast<int64_t>(T) * page / 32 + 4 > most / (static_cast<int64_t>(B) * Hk * row_tiles))
    return fail(DM_ERR_ARG, "delta_matching: too much work for one call (%d sequences with room for %lld tokens, %lld rows)", B,
                static_cast<long long>(T) * page, static_cast<long long>(Nq) * H);
  return 0;
}

int64_t dm_cache_attn_workspace_bytes(int B, int Nq, int H, int Hk, int D, int T, int page_size, int with_weights) {
  if (check_attn_shape(B, Nq, H, Hk, D, T, page_size) != 0) return 0;
  const dm::CacheAttnPlan x = dm::plan_cache_attn(B, Nq, H, Hk, D, T, page_size, with_weights != 0);
  return x.bytes();
}

int dm_cache_attn(const dm_kv_cache* cache, const void* q, int64_t q_sb, int64_t q_sn, int64_t q_sh, int B, int Nq, int H,
                  const int* table, int64_t table_row, int T, const int* lengths, const int* q_counts, int causal, float softmax_scale,
                  void* o, float* lse, float* weights, int64_t w_sb, int64_t w_sh, int W, int accumulate,
                  void* workspace, int64_t workspace_bytes, int* status, void* stream) {
  DM_TRY(check_cache(cache));
  DM_TRY(check_table(cache, table, table_row, T, lengths, B, "block table"));
  DM_TRY(check_attn_shape(B, Nq, H, cache->heads, cache->head_dim, T, cache->page_size));
  DM_TRY(check_rows("q", q, q_sb, q_sn, q_sh));
  DM_TRY(check_addresses({{o, "o"}, {lse, "lse"}, {workspace, "workspace"}}));
  if (!(softmax_scale > 0.f && softmax_scale <= FLT_MAX)) return fail(DM_ERR_ARG, "delta_matching: softmax_scale must be positive and finite in 32 bits (got %g)", softmax_scale);
  if (weights != nullptr && W < T * cache->page_size)
    return fail(DM_ERR_ARG, "delta_matching: weights must have room for the %d tokens of a row of the block table (got %d)", T * cache->page_size, W);
  const dm::CacheAttnPlan x = dm::plan_cache_attn(B, Nq, H, cache->heads, cache->head_dim, T, cache->page_size, weights != nullptr);
  const int64_t need = x.bytes();
  if (workspace_bytes < need)
    return fail(DM_ERR_ARG, "delta_matching: workspace of %lld bytes given, %lld needed", static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  DM_TRY(check_sm100());
  dm::CacheAttnParams p{};
  p.c = view_of(cache, table, table_row, T, lengths, B, status);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_sb = q_sb; p.q_sn = q_sn; p.q_sh = q_sh;
  p.counts = q_counts;
  p.Nq = Nq; p.H = H; p.rep = H / cache->heads;
  p.causal = causal ? 1 : 0;
  p.scale = softmax_scale;
  p.o = static_cast<__nv_bfloat16*>(o);
  p.lse = lse;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  auto take = [&ws](int64_t bytes) {                          // every part is a multiple of 8 bytes, those up to the factors of 16
    uint8_t* at = ws;
    ws += bytes;
    return at;
  };
  p.part_o = reinterpret_cast<float*>(take(x.part_o_bytes));
  p.logits = x.logit_bytes > 0 ? reinterpret_cast<float*>(take(x.logit_bytes)) : nullptr;
  p.logit_rows = x.logit_rows;
  p.q16 = reinterpret_cast<__half*>(take(x.q16_bytes));
  p.part_ml = reinterpret_cast<float4*>(take(x.part_ml_bytes));
  p.marked = reinterpret_cast<int*>(take(x.mark_bytes));
  p.factors = reinterpret_cast<float*>(take(x.factor_bytes));
  p.row_ml = weights != nullptr ? reinterpret_cast<float2*>(take(x.row_ml_bytes)) : nullptr;
  p.starts = take(x.start_bytes);
  p.unit_slots = reinterpret_cast<int2*>(take(x.unit_bytes));
  p.weights = weights;
  p.w_sb = w_sb; p.w_sh = w_sh; p.W = W; p.accumulate = accumulate ? 1 : 0;
  p.grid = x.grid;
  p.cluster = x.cluster;
  for (p.unit_shift = 0; x.chunk && 1 << p.unit_shift < x.row_tile;) ++p.unit_shift;
  CUtensorMap tk, tv, tq{};
  DM_TRY(pool_map(&tk, cache, cache->k8));
  DM_TRY(pool_map(&tv, cache, cache->v8));
  if (x.chunk) {                                              // f16 rows as bytes: boxes of 64 values x 128 rows
    const cuuint64_t row = 2ull * cache->head_dim, dims[2] = {row, static_cast<cuuint64_t>(x.q16_bytes) / row}, strides[1] = {row};
    const cuuint32_t box[2] = {128, 128};
    DM_TRY(encode_byte_map(&tq, p.q16, 2, dims, strides, box));
  }
  const cudaError_t e = dm::launch_cache_attn(cache->head_dim, tk, tv, tq, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : cuda_fail(e, "cache attention launch");
}

int dm_dbg_cache_join_slots(int many_rows, int x, int y, int grid, int i) {
  if (grid <= 0) return fail(DM_ERR_ARG, "delta_matching: grid must be positive (got %d)", grid);
  const dm::JoinSlots s = many_rows ? dm::join_slots_of_ctas(make_int2(x, y), grid) : dm::join_slots_of_warps(make_int2(x, y), grid);
  if (i < 0) return s.count;
  if (i >= s.count) return fail(DM_ERR_ARG, "delta_matching: piece %d of %d", i, s.count);
  return s.slot(i);
}

int dm_cache_evict(const dm_kv_cache* cache, int B, const int* table, int64_t table_row, int T, const int* lengths,
                   const float* weights, int64_t w_sb, int64_t w_sh, const int* new_table, int64_t new_table_row, int new_T,
                   int budget, int recent, int* new_lengths, int* kept, float* new_weights, int* status, void* stream) {
  DM_TRY(check_cache(cache));
  DM_TRY(check_table(cache, table, table_row, T, lengths, B, "block table"));
  DM_TRY(check_table(cache, new_table, new_table_row, new_T, lengths, B, "new block table"));
  if (budget <= 0 || budget > new_T * cache->page_size)
    return fail(DM_ERR_ARG, "delta_matching: budget must be between 1 and the %d tokens of a row of the new block table (got %d)",
                new_T * cache->page_size, budget);
  if (recent < 0 || recent > budget) return fail(DM_ERR_ARG, "delta_matching: recent must be between 0 and the budget (got %d)", recent);
  for (const NamedPtr& x : {NamedPtr{weights, "weights"}, {new_lengths, "new lengths"}, {kept, "kept"}, {new_weights, "new weights"}})
    if (x.p == nullptr) return fail(DM_ERR_ARG, "delta_matching: %s is NULL (every tensor must be a CUDA buffer)", x.name);
  DM_TRY(check_new_lengths(new_lengths, B, {{lengths, 1, 1, "lengths"}, {table, table_row, T, "block table"}, {new_table, new_table_row, new_T, "new block table"}}));
  DM_TRY(check_sm100());
  dm::CacheEvictParams p{};
  p.c = view_of(cache, table, table_row, T, lengths, B, status);
  p.new_table = new_table; p.nt_row = new_table_row; p.T2 = new_T;
  p.weights = weights; p.w_sb = w_sb; p.w_sh = w_sh;
  p.budget = budget; p.recent = recent;
  p.new_lengths = new_lengths; p.kept = kept; p.new_weights = new_weights;
  const cudaError_t e = dm::launch_cache_evict(cache->head_dim, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : cuda_fail(e, "cache eviction launch");
}

}  // extern "C"
