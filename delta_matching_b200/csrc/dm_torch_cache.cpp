// The eager route of the cache functions in C++, beside that of the attention (dm_torch.cpp): a decoding step's kernels take a few microseconds,
// the Python route's checks and ctypes calls 30 - 40.  Each method makes the checks of cache.py and returns None for whatever does not pass
// them, so that the Python route raises the exception, or serves the call.
#include "dm_torch_cache.h"

namespace {

using at::Tensor;

struct Lib {
  decltype(&dm_cache_append) append = nullptr;
  decltype(&dm_cache_attn) attn = nullptr;
  decltype(&dm_cache_attn_workspace_bytes) attn_workspace_bytes = nullptr;
  decltype(&dm_cache_evict) evict = nullptr;
} g_lib;

}  // namespace

namespace dm_native {

// cache_append(cache, k, v, block_table, lengths, counts) -> new lengths, or None
PyObject* cache_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Cache cache;
  const Tensor *kp, *vp;
  if (n != 6 || elsewhere() || !cache.read(args[0]) || !cache.written_apart() || !read_rows(args[1], cache, cache.c.heads, kp) || !read_rows(args[2], cache, cache.c.heads, vp) ||
      kp->sizes() != vp->sizes() || !sm100(cache.dev))
    Py_RETURN_NONE;
  const int64_t B = kp->size(0), N = kp->size(1);
  Table table;
  const int *lengths, *counts;
  if (!table.read(args[3], cache, B) || !read_lengths(args[4], cache, B, lengths) || !read_counts(args[5], cache, B, counts)) Py_RETURN_NONE;
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(cache.dev);
    int* status = status_of(cache.dev.index());
    const Tensor k = rows(*kp), v = rows(*vp);
    out = empty({B}, at::kInt, cache.dev);
    check(g_lib.append(&cache.c, k.const_data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.const_data_ptr(), v.stride(0), v.stride(1), v.stride(2),
                       static_cast<int>(B), static_cast<int>(N), table.p, table.row, table.T, lengths, counts, static_cast<int*>(out.mutable_data_ptr()), status,
                       stream_of(cache.dev)));
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// cache_attn(q, cache, block_table, lengths, q_counts, causal, softmax_scale, weights, accumulate, return_lse) -> o, or (o, lse), or None
PyObject* cache_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Cache cache;
  const Tensor* qp;
  if (n != 10 || elsewhere() || !cache.read(args[1]) || !read_rows(args[0], cache, 0, qp) || !sm100(cache.dev)) Py_RETURN_NONE;
  const int64_t B = qp->size(0), N = qp->size(1), H = qp->size(2), D = qp->size(3);
  if (H % cache.c.heads) Py_RETURN_NONE;
  Table table;
  const int *lengths, *counts;
  if (!table.read(args[2], cache, B) || !read_lengths(args[3], cache, B, lengths) || !read_counts(args[4], cache, B, counts)) Py_RETURN_NONE;
  const int causal = PyObject_IsTrue(args[5]), accumulate = PyObject_IsTrue(args[8]), with_lse = PyObject_IsTrue(args[9]);
  if (causal < 0 || accumulate < 0 || with_lse < 0) return nullptr;
  double scale = 1.0 / std::sqrt(static_cast<double>(D));
  if (args[6] != Py_None) {
    scale = PyFloat_AsDouble(args[6]);
    if (scale == -1.0 && PyErr_Occurred()) PyErr_Clear();
    if (!(static_cast<float>(scale) > 0.f && std::isfinite(static_cast<float>(scale)))) Py_RETURN_NONE;
  }
  const Tensor* w = nullptr;
  if (args[7] == Py_None ? accumulate != 0 : !(read_weights(args[7], cache, B, table.room(cache), w) && !overlaps(*w))) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(cache.dev);                // the plan is the cache's device's
  const int64_t ws_bytes = g_lib.attn_workspace_bytes(static_cast<int>(B), static_cast<int>(N), static_cast<int>(H), cache.c.heads, cache.c.head_dim, table.T,
                                                      cache.c.page_size, w != nullptr);
  if (ws_bytes <= 0) Py_RETURN_NONE;
  Tensor o, lse;
  {
    pybind11::gil_scoped_release no_gil;
    int* status = status_of(cache.dev.index());
    const Tensor q = rows(*qp);
    o = empty({B, N, H, D}, at::kBFloat16, cache.dev);
    // the LSE behind the workspace where the caller does not keep it
    const int64_t lse_at = (ws_bytes + 255) & ~int64_t(255);
    if (with_lse) lse = empty({B, H, N}, at::kFloat, cache.dev);
    Tensor ws = empty({with_lse ? ws_bytes : lse_at + 4 * B * H * N}, at::kByte, cache.dev);
    uint8_t* p = static_cast<uint8_t*>(ws.mutable_data_ptr());
    float* lse_p = with_lse ? static_cast<float*>(lse.mutable_data_ptr()) : reinterpret_cast<float*>(p + lse_at);
    check(g_lib.attn(&cache.c, q.const_data_ptr(), q.stride(0), q.stride(1), q.stride(2), static_cast<int>(B), static_cast<int>(N), static_cast<int>(H), table.p,
                     table.row, table.T, lengths, counts, causal, static_cast<float>(scale), o.mutable_data_ptr(), lse_p,
                     w != nullptr ? static_cast<float*>(w->mutable_data_ptr()) : nullptr, w != nullptr ? w->stride(0) : 0, w != nullptr ? w->stride(1) : 0,
                     w != nullptr ? static_cast<int>(w->size(2)) : 0, accumulate, p, ws_bytes, status, stream_of(cache.dev)));
  }
  if (!with_lse) return THPVariable_Wrap(std::move(o));
  PyObject* both = PyTuple_New(2);
  if (both == nullptr) return nullptr;
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(o)));
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(lse)));
  return both;
  END_HANDLE_TH_ERRORS
}

// cache_evict(cache, block_table, lengths, weights, new_block_table, budget, recent) -> (new lengths, kept, new weights), or None
PyObject* cache_evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Cache cache;
  const Tensor* len;
  if (n != 7 || elsewhere() || !cache.read(args[0]) || !cache.written_apart() || !sm100(cache.dev) || !plain_cuda(args[2], len) || len->dim() != 1 || len->size(0) <= 0) Py_RETURN_NONE;
  const int64_t B = len->size(0);
  Table table, to;
  const int* lengths;
  const Tensor* w;
  long long budget, recent;
  if (!table.read(args[1], cache, B) || !read_lengths(args[2], cache, B, lengths) || !read_weights(args[3], cache, B, table.room(cache), w) ||
      !to.read(args[4], cache, B) || !read_int(args[5], budget) || !read_int(args[6], recent))
    Py_RETURN_NONE;
  if (budget <= 0 || budget > to.room(cache) || budget > INT32_MAX || recent < 0 || recent > budget) Py_RETURN_NONE;
  Tensor out, kept, nw;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(cache.dev);
    int* status = status_of(cache.dev.index());
    out = empty({B}, at::kInt, cache.dev);
    kept = empty({B, cache.c.heads, static_cast<int64_t>(budget)}, at::kInt, cache.dev);
    nw = empty({B, cache.c.heads, to.room(cache)}, at::kFloat, cache.dev);
    check(g_lib.evict(&cache.c, static_cast<int>(B), table.p, table.row, table.T, lengths, static_cast<const float*>(w->const_data_ptr()), w->stride(0),
                      w->stride(1), to.p, to.row, to.T, static_cast<int>(budget), static_cast<int>(recent), static_cast<int*>(out.mutable_data_ptr()),
                      static_cast<int*>(kept.mutable_data_ptr()), static_cast<float*>(nw.mutable_data_ptr()), status, stream_of(cache.dev)));
  }
  PyObject* all = PyTuple_New(3);
  if (all == nullptr) return nullptr;
  PyTuple_SET_ITEM(all, 0, THPVariable_Wrap(std::move(out)));
  PyTuple_SET_ITEM(all, 1, THPVariable_Wrap(std::move(kept)));
  PyTuple_SET_ITEM(all, 2, THPVariable_Wrap(std::move(nw)));
  return all;
  END_HANDLE_TH_ERRORS
}

// bind_cache(append, attn, attn_workspace_bytes, evict): addresses of the entry points
PyObject* bind_cache(PyObject*, PyObject* args) {
  unsigned long long a[4];
  if (!PyArg_ParseTuple(args, "KKKK", &a[0], &a[1], &a[2], &a[3])) return nullptr;
  g_lib.append = reinterpret_cast<decltype(&dm_cache_append)>(a[0]);
  g_lib.attn = reinterpret_cast<decltype(&dm_cache_attn)>(a[1]);
  g_lib.attn_workspace_bytes = reinterpret_cast<decltype(&dm_cache_attn_workspace_bytes)>(a[2]);
  g_lib.evict = reinterpret_cast<decltype(&dm_cache_evict)>(a[3]);
  Py_RETURN_NONE;
}

}  // namespace dm_native
