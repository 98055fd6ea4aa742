// Internal launch interface of the functions for drafted tokens (trees, rotation with append, attention of a tree, keeping a path) between their
// C-ABI layer (dm_drafts_abi.cu) and the kernel translation units.
#pragma once
#include "dm_cache.h"

namespace dm {

constexpr int kMaxNodes = 1024;     // of a tree

struct DraftTreeParams {
  const int* parents;               // (B, N), rows `row` entries apart
  int64_t row;
  const int* counts;                // (B) or null: N each
  int B, N;
  int* depth;                       // (B, N)
  uint32_t* seen;                   // (B, N, words)
  int* status;
};

struct CacheRotaryParams {
  CacheView c;
  const __nv_bfloat16* q;           // (B, N, H, D), k, v (B, N, Hk, D) by element strides, rows 16-byte aligned
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t q_sb, q_sn, q_sh, k_sb, k_sn, k_sh, v_sb, v_sn, v_sh;
  const float* freqs;               // (half)
  int half;                         // pairs of channels that are rotated, a multiple of 8
  int interleaved;                  // pairs (2 j, 2 j + 1), else (j, j + half)
  const int* offsets;               // (B, N) or null: positions behind lengths[b]; rows o_row entries apart
  int64_t o_row;
  const int* counts;                // (B) or null: N each
  __nv_bfloat16* q_out;             // (B, N, H, D) contiguous
  int* new_lengths;                 // (B)
  int N, H;
};

struct CacheTreeParams {
  CacheView c;
  const __nv_bfloat16* q;           // (B, N, H, D) by element strides, rows 16-byte aligned
  int64_t q_sb, q_sn, q_sh;
  const int* counts;                // (B) or null: N each
  const uint32_t* seen;             // (B, N, words): bit j % 32 of word j / 32 of node i: node i sees node j; by element strides, words adjacent
  int64_t s_sb, s_sn;
  int N, H, rep;
  float scale;                      // softmax scale
  __nv_bfloat16* o;                 // (B, N, H, D) contiguous
  float* lse;                       // (B, H, N)
  float* part_o;                    // partial results: 2 slots a CTA, of row_tile rows of D fp32 each, and of their rows (m, l, u, marked): the sum is
  float4* part_ml;                  // l 2^m, the values count in 2^u
  uint8_t* marks;                   // (B, H, N): of a row of a whole unit, its mark
  void* cuts;                       // and what the join needs of each cut unit
  int grid;                         // CTAs of the main kernel
  int cluster;                      // of a unit, or 0: the even division
  int row_tile, row_shift;          // rows (drafted tokens x heads of a group) of a unit, a power of two
  uint32_t rep_magic;               // r / rep is the upper half of r times it (0: divide)
};

// How a call of dm_cache_attn_tree is laid out, and its workspace.
struct CacheTreePlan {
  int row_tile, grid, cluster;
  int64_t part_o_bytes, part_ml_bytes, mark_bytes, cut_bytes;
  int64_t bytes() const { return part_o_bytes + part_ml_bytes + mark_bytes + cut_bytes; }
};
CacheTreePlan plan_cache_tree(int B, int N, int H, int Hk, int D, int T, int page);

struct CacheKeepParams {
  CacheView c;                      // lengths: with the drafted tokens
  const int* before;                // (B): without them
  const int* path;                  // (B, M), rows p_row entries apart
  int64_t p_row;
  int M;
  const int* counts;                // (B): entries of the path
  int* new_lengths;                 // (B)
};

cudaError_t launch_draft_tree(const DraftTreeParams& p, cudaStream_t stream);
cudaError_t launch_cache_rotary(int D, const CacheRotaryParams& p, cudaStream_t stream);
cudaError_t launch_cache_tree(int D, const CUtensorMap& tk, const CUtensorMap& tv, const CacheTreeParams& p, cudaStream_t stream);
cudaError_t launch_cache_keep(int D, const CacheKeepParams& p, cudaStream_t stream);

}  // namespace dm
