// What the C-ABI layers of the cache's functions share: checks of a cache, its tables and rows, the kernels' view of it, tensor maps of the pools.
#pragma once
#include "dm_abi_util.h"
#include "dm_cache.h"

namespace dm {
namespace abi {

inline int check_cache(const dm_kv_cache* c) {
  if (c == nullptr) return fail(DM_ERR_ARG, "delta_matching: cache is NULL");
  DM_TRY(check_addresses({{c->k8, "k8"}, {c->v8, "v8"}}));
  if (c->ks == nullptr || c->vs == nullptr) return fail(DM_ERR_ARG, "delta_matching: %s is NULL (every tensor must be a CUDA buffer)", c->ks == nullptr ? "ks" : "vs");
  if (c->head_dim != 128 && c->head_dim != 256) return fail(DM_ERR_ARG, "delta_matching: head_dim must be 128 or 256 (got %d)", c->head_dim);
  if (c->pages <= 0 || c->heads <= 0) return fail(DM_ERR_ARG, "delta_matching: empty cache (%d pages, %d heads)", c->pages, c->heads);
  if (c->page_size <= 0 || c->page_size % 32) return fail(DM_ERR_ARG, "delta_matching: page size must be a positive multiple of 32 (got %d)", c->page_size);
  for (const int64_t s : {c->code_page, c->code_head, c->code_slot})
    if (s <= 0 || s % 16 || s >= (1ll << 40))
      return fail(DM_ERR_ARG, "delta_matching: code strides must be positive multiples of 16 bytes (got %lld)", static_cast<long long>(s));
  return 0;
}

inline int check_table(const dm_kv_cache* c, const int* table, int64_t row, int T, const int* lengths, int B, const char* name) {
  if (table == nullptr) return fail(DM_ERR_ARG, "delta_matching: %s is NULL (every tensor must be a CUDA buffer)", name);
  if (lengths == nullptr) return fail(DM_ERR_ARG, "delta_matching: lengths is NULL (every tensor must be a CUDA buffer)");
  if (B <= 0 || T <= 0) return fail(DM_ERR_ARG, "delta_matching: empty %s (%d sequences, %d pages each)", name, B, T);
  if (row < 0) return fail(DM_ERR_ARG, "delta_matching: rows of %s are %lld apart", name, static_cast<long long>(row));
  if (static_cast<int64_t>(B) * c->heads > 65535) return fail(DM_ERR_ARG, "delta_matching: batch * nheads_k must be at most 65535");
  if (static_cast<int64_t>(T) * c->page_size > (1ll << 30))
    return fail(DM_ERR_ARG, "delta_matching: a sequence has room for at most 2^30 tokens (got %d pages of %d)", T, c->page_size);
  return 0;
}

inline dm::CacheView view_of(const dm_kv_cache* c, const int* table, int64_t row, int T, const int* lengths, int B, int* status) {
  dm::CacheView v{};
  v.k8 = static_cast<uint8_t*>(c->k8);
  v.v8 = static_cast<uint8_t*>(c->v8);
  v.ks = c->ks;
  v.vs = c->vs;
  v.c_page = c->code_page; v.c_head = c->code_head; v.c_slot = c->code_slot;
  v.s_page = c->scale_page; v.s_head = c->scale_head;
  v.pages = c->pages; v.Hk = c->heads; v.page = c->page_size;
  v.table = table; v.t_row = row; v.T = T;
  v.lengths = lengths; v.B = B; v.status = status;
  return v;
}

// The pool as (D, slot, head, page) bytes: boxes of one block of 32 slots x 128 bytes.
inline int pool_map(CUtensorMap* m, const dm_kv_cache* c, const void* base) {
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c->head_dim), static_cast<cuuint64_t>(c->page_size), static_cast<cuuint64_t>(c->heads),
                              static_cast<cuuint64_t>(c->pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(c->code_slot), static_cast<cuuint64_t>(c->code_head), static_cast<cuuint64_t>(c->code_page)};
  const cuuint32_t box[4] = {128, 32, 1, 1};
  return encode_byte_map(m, base, 4, dims, strides, box);
}

inline int check_rows(const char* name, const void* p, int64_t a, int64_t b, int64_t c) {
  DM_TRY(check_address(p, name));
  if ((a % 8) || (b % 8) || (c % 8))
    return fail(DM_ERR_ARG, "delta_matching: %s strides must be multiples of 8 elements (16-byte aligned rows)", name);
  return 0;
}

// B rows of n int32 each that a kernel reads, `row` entries apart.
struct IntRows {
  const int* p;
  int64_t row, n;
  const char* name;
};
// The kernels' CTAs read these while one of them writes new_lengths.  (Between two rows it may lie.)
inline int check_new_lengths(const int* out, int B, std::initializer_list<IntRows> in) {
  for (const IntRows& x : in) {
    if (x.p == nullptr) continue;
    const int64_t at = (static_cast<int64_t>(reinterpret_cast<uintptr_t>(out)) - static_cast<int64_t>(reinterpret_cast<uintptr_t>(x.p))) / 4;      // behind the first row's begin
    const int64_t b = at < x.n ? 0 : x.row > 0 ? (at - x.n) / x.row + 1 : B;          // first row that ends behind it
    if (b < B && b * x.row < at + B) return fail(DM_ERR_ARG, "delta_matching: new lengths must not share memory with %s (a buffer of their own)", x.name);
  }
  return 0;
}

}  // namespace abi
}  // namespace dm
