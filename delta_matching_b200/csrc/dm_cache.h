// Internal launch interface of the 8-bit key / value cache (append, attention, eviction) between its C-ABI layer (dm_cache_abi.cu) and the
// kernel translation units.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace dm {

// Pools of pages and one block table over them.  Token j of sequence b is slot j % page of page table[b, j / page]; a slot's row of D codes
// is contiguous; 32 slots of a page and head share a scale.
struct CacheView {
  uint8_t* k8;
  uint8_t* v8;
  float* ks;
  float* vs;
  int64_t c_page, c_head, c_slot;   // byte strides of k8 and v8
  int64_t s_page, s_head;           // element strides of ks and vs (the page / 32 scales of a head are adjacent)
  int pages, Hk, page;
  const int* table;                 // (B, T), rows t_row entries apart
  int64_t t_row;
  int T;
  const int* lengths;               // (B)
  int B;
  int* status;
};

struct CacheAppendParams {
  CacheView c;
  const __nv_bfloat16* k;           // (B, N, Hk, D) by element strides, rows 16-byte aligned
  const __nv_bfloat16* v;
  int64_t k_sb, k_sn, k_sh, v_sb, v_sn, v_sh;
  const int* counts;                // (B) or null: N each
  int* new_lengths;                 // (B)
  int N;
};

struct CacheAttnParams {
  CacheView c;
  const __nv_bfloat16* q;           // (B, Nq, H, D) by element strides, rows 16-byte aligned
  int64_t q_sb, q_sn, q_sh;
  const int* counts;                // (B) or null: Nq each
  int Nq, H, rep;
  int causal;
  float scale;                      // softmax scale
  __nv_bfloat16* o;                 // (B, Nq, H, D) contiguous
  float* lse;                       // (B, H, Nq)
  float* part_o;                    // partial results: 2 slots a warp of (row tile, D) fp32, and of their rows (m, l, v, -): the sum is l 2^m, the values
  float4* part_ml;                  // count in 2^(m + v) (and a constant of the form)
  __half* q16;                      // many rows: the queries in f16 and the order of the row tiles, and the factors of their logits
  float* factors;                   // (negative: a row marked for the join to make by itself)
  int* marked;                      // whether any is
  void* starts;                     // and what each CTA begins with
  int2* unit_slots;                 // per unit (B, Hk, row tiles), where its pieces are: slot of the first (-1: whole); the last worker (for the
                                    // small form twice that, plus one where its piece lies in a slot of its own)
  float2* row_ml;                   // (B, Hk, Nq * rep): maximum (log2 domain) and 1 / sum of each row, for the weights; may be null.  Of the form
                                    // for many rows: factor of the logits and log2 of the sum, rows of a head filled up to whole tiles
  float* logits;                    // (B, Hk, T * page, logit_rows), log2 domain, masked: for the weights of up to 16 rows; or null
  int logit_rows;                   // a token's, a multiple of four
  float* weights;                   // (B, Hk, W) or null
  int64_t w_sb, w_sh;
  int W;
  int accumulate;
  int grid;                         // CTAs of the main kernel
  int cluster;                      // of a unit, or 0: the even division
  int unit_shift;                   // of the form for many rows: log2 of a unit's; otherwise 0
};

struct CacheEvictParams {
  CacheView c;                      // the pages read
  const int* new_table;             // (B, T2): the pages written
  int64_t nt_row;
  int T2;
  const float* weights;             // (B, Hk, >= T * page)
  int64_t w_sb, w_sh;
  int budget, recent;
  int* new_lengths;                 // (B)
  int* kept;                        // (B, Hk, budget), -1 beyond what is kept
  float* new_weights;               // (B, Hk, T2 * page), 0 beyond
};

// Where the join finds the pieces of a cut unit, from its entry of unit_slots.  A main kernel that gave up has left entries as the workspace came, so
// that any value may be met: none() where the entry does not stand for slots that a grid of this size has.
struct JoinSlots {
  int first, count;                 // slot of the first piece; pieces, at most the grid's CTAs and one
  int next, step;                   // slots of the pieces between: next, next + step, ...
  int last;                         // slot of the last piece
  __host__ __device__ bool none() const { return count == 0; }
  __host__ __device__ int slot(int i) const { return i == 0 ? first : i == count - 1 ? last : next + (i - 1) * step; }
};
// dm_cache_attn.cu, four warps a CTA, two slots a warp: after the first piece the joined ones of the CTAs behind it, then the last warp's own where that
// went on with another unit.
__host__ __device__ inline JoinSlots join_slots_of_warps(int2 unit, int grid) {
  const int end = unit.y >> 1;      // the last warp that has a piece
  if (unit.x < 0 || unit.y < 0 || unit.x / 2 > end || end / 4 >= grid) return JoinSlots{};
  const int cta0 = unit.x / 8, cta1 = end / 4, own = unit.y & 1;
  JoinSlots x;
  x.first = unit.x;
  x.count = 1 + cta1 - cta0 - (own && cta1 > cta0 && end == 4 * cta1 ? 1 : 0) + own;
  x.next = 8 * (cta0 + 1);
  x.step = 8;
  x.last = own ? 2 * end : 8 * cta1;
  return x;
}
// dm_cache_chunk.cu, two slots a CTA: the pieces behind the first one are the first ones of their CTAs.
__host__ __device__ inline JoinSlots join_slots_of_ctas(int2 unit, int grid) {
  if (unit.x < 0 || unit.x / 2 > unit.y || unit.y >= grid) return JoinSlots{};
  const int cta0 = unit.x / 2;
  return JoinSlots{unit.x, 1 + unit.y - cta0, 2 * (cta0 + 1), 2, 2 * unit.y};
}

// Slots of partial results and their sizes for a call of dm_cache_attn.
struct CacheAttnPlan {
  bool chunk;                       // dm_cache_chunk.cu: many rows
  int row_tile;                     // query rows (new tokens x heads of a group) a CTA keeps
  int row_tiles;
  int grid;
  int cluster;                      // CTAs a unit, or 0: the even division
  int logit_rows;
  int64_t part_o_bytes, part_ml_bytes, q16_bytes, mark_bytes, factor_bytes, start_bytes, unit_bytes, row_ml_bytes, logit_bytes;
  int64_t bytes() const { return part_o_bytes + part_ml_bytes + q16_bytes + mark_bytes + factor_bytes + start_bytes + unit_bytes + row_ml_bytes + logit_bytes; }
};
int cache_chunk_from(int D);         // rows of a head from which the form for many rows is taken
CacheAttnPlan plan_cache_attn(int B, int Nq, int H, int Hk, int D, int T, int page, bool weights);

cudaError_t launch_cache_append(int D, const CacheAppendParams& p, cudaStream_t stream);
// tq: p.q16 as 64 x 128 boxes, for the form for many rows.
cudaError_t launch_cache_attn(int D, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tq, const CacheAttnParams& p, cudaStream_t stream);
// The form for many rows (its partial results: 2 slots a CTA), and what a row tile of it holds.
cudaError_t launch_cache_chunk(int D, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tq, const CacheAttnParams& p, cudaStream_t stream);
int cache_chunk_rows(int D);
int64_t cache_chunk_start_bytes();                           // of a CTA's start
int64_t cache_chunk_query_rows(int B, int Hk, int R);         // rows of D f16 values
cudaError_t launch_cache_evict(int D, const CacheEvictParams& p, cudaStream_t stream);

}  // namespace dm
