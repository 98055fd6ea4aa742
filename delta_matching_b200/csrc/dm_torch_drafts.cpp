// The eager route of the functions for drafted tokens in C++ (see dm_torch_cache.cpp).  Each method makes the checks of drafts.py and returns None for
// whatever does not pass them, so that the Python route raises the exception, or serves the call.
#include "dm_torch_cache.h"

namespace {

using at::Tensor;

constexpr int64_t kMaxNodes = 1024;

struct Lib {
  decltype(&dm_draft_tree) tree = nullptr;
  decltype(&dm_cache_append_rotary) append = nullptr;
  decltype(&dm_cache_attn_tree) attn = nullptr;
  decltype(&dm_cache_attn_tree_workspace_bytes) attn_workspace_bytes = nullptr;
  decltype(&dm_cache_keep) keep = nullptr;
} g_lib;

// An int32 matrix whose rows' entries are adjacent; B, N: wanted, or -1.
struct Ints {
  const Tensor* t;
  const int* p;
  int64_t row;
  bool read(PyObject* o, int64_t B, int64_t N, const at::Device* dev) {
    if (!dm_native::plain_cuda(o, t) || t->scalar_type() != at::kInt || t->dim() != 2 || t->numel() == 0 || (B >= 0 && t->size(0) != B) ||
        (N >= 0 && t->size(1) != N) || (dev != nullptr && t->device() != *dev) || (t->size(1) > 1 && t->stride(1) != 1) || t->size(0) > INT32_MAX)
      return false;
    p = static_cast<const int*>(t->const_data_ptr());
    row = t->size(0) > 1 ? t->stride(0) : t->size(1);
    return true;
  }
};

// What two results are returned as.
PyObject* pair(Tensor a, Tensor b) {
  PyObject* both = PyTuple_New(2);
  if (both == nullptr) return nullptr;
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(a)));
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(b)));
  return both;
}

}  // namespace

namespace dm_native {

// draft_tree(parents, counts) -> (depth, seen), or None
PyObject* draft_tree(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Ints parents;
  if (n != 2 || elsewhere() || !parents.read(args[0], -1, -1, nullptr)) Py_RETURN_NONE;
  const int64_t B = parents.t->size(0), N = parents.t->size(1);
  Cache at_device;                                            // whose device the counts are held to
  at_device.dev = parents.t->device();
  const int* counts;
  if (N > kMaxNodes || at_device.dev.index() >= kMaxDevices || !sm100(at_device.dev) || !read_counts(args[1], at_device, B, counts)) Py_RETURN_NONE;
  Tensor depth, seen;
  {
    pybind11::gil_scoped_release no_gil;
    const at::Device dev = at_device.dev;
    const c10::cuda::CUDAGuard guard(dev);
    int* status = status_of(dev.index());
    depth = empty({B, N}, at::kInt, dev);
    seen = empty({B, N, (N + 31) / 32}, at::kInt, dev);
    check(g_lib.tree(parents.p, parents.row, counts, static_cast<int>(B), static_cast<int>(N), static_cast<int*>(depth.mutable_data_ptr()),
                     static_cast<int*>(seen.mutable_data_ptr()), status, stream_of(dev)));
  }
  return pair(std::move(depth), std::move(seen));
  END_HANDLE_TH_ERRORS
}

// cache_append_rotary(cache, q, k, v, block_table, lengths, freqs, offsets, counts, interleaved) -> (q, new lengths), or None
PyObject* cache_append_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Cache cache;
  const Tensor *qp, *kp, *vp, *freqs;
  if (n != 10 || elsewhere() || !cache.read(args[0]) || !cache.written_apart() || !read_rows(args[1], cache, 0, qp) || !read_rows(args[2], cache, cache.c.heads, kp) ||
      !read_rows(args[3], cache, cache.c.heads, vp) || kp->sizes() != vp->sizes() || !sm100(cache.dev))
    Py_RETURN_NONE;
  const int64_t B = qp->size(0), N = qp->size(1), H = qp->size(2), D = qp->size(3);
  if (kp->size(0) != B || kp->size(1) != N || H % cache.c.heads) Py_RETURN_NONE;
  if (!plain_cuda(args[6], freqs) || freqs->scalar_type() != at::kFloat || freqs->dim() != 1 || freqs->size(0) <= 0 || freqs->size(0) % 8 ||
      2 * freqs->size(0) > D || freqs->device() != cache.dev || !freqs->is_contiguous())
    Py_RETURN_NONE;
  Table table;
  Ints offsets{};
  const int *lengths, *counts;
  if (!table.read(args[4], cache, B) || !read_lengths(args[5], cache, B, lengths) || (args[7] != Py_None && !offsets.read(args[7], B, N, &cache.dev)) ||
      !read_counts(args[8], cache, B, counts))
    Py_RETURN_NONE;
  const int interleaved = PyObject_IsTrue(args[9]);
  if (interleaved < 0) return nullptr;
  Tensor out, lens;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(cache.dev);
    int* status = status_of(cache.dev.index());
    const Tensor q = rows(*qp), k = rows(*kp), v = rows(*vp);
    out = empty({B, N, H, D}, at::kBFloat16, cache.dev);
    lens = empty({B}, at::kInt, cache.dev);
    check(g_lib.append(&cache.c, q.const_data_ptr(), q.stride(0), q.stride(1), q.stride(2), k.const_data_ptr(), k.stride(0), k.stride(1), k.stride(2),
                       v.const_data_ptr(), v.stride(0), v.stride(1), v.stride(2), static_cast<int>(B), static_cast<int>(N), static_cast<int>(H),
                       static_cast<const float*>(freqs->const_data_ptr()), static_cast<int>(freqs->size(0)), interleaved, table.p, table.row, table.T, lengths,
                       offsets.p, offsets.row, counts, out.mutable_data_ptr(), static_cast<int*>(lens.mutable_data_ptr()), status, stream_of(cache.dev)));
  }
  return pair(std::move(out), std::move(lens));
  END_HANDLE_TH_ERRORS
}

// cache_attn_tree(q, cache, block_table, lengths, tree, softmax_scale, return_lse) -> o, or (o, lse), or None
PyObject* cache_attn_tree(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Cache cache;
  const Tensor *qp, *depth, *seen;
  if (n != 7 || elsewhere() || !cache.read(args[1]) || !read_rows(args[0], cache, 0, qp) || !sm100(cache.dev)) Py_RETURN_NONE;
  const int64_t B = qp->size(0), N = qp->size(1), H = qp->size(2), D = qp->size(3);
  if (H % cache.c.heads || N > kMaxNodes) Py_RETURN_NONE;
  Table table;
  const int *lengths, *counts;
  PyObject* tree = args[4];                                   // a DraftTree, no plain tuple
  if (!PyTuple_Check(tree) || PyTuple_CheckExact(tree) || PyTuple_GET_SIZE(tree) != 3 || !plain_cuda(PyTuple_GET_ITEM(tree, 0), depth) ||
      !plain_cuda(PyTuple_GET_ITEM(tree, 1), seen) || seen->scalar_type() != at::kInt || seen->dim() != 3 || seen->size(0) != B || seen->size(1) != N ||
      seen->size(2) != (N + 31) / 32 || seen->device() != cache.dev || (seen->size(2) > 1 && seen->stride(2) != 1))
    Py_RETURN_NONE;
  if (!table.read(args[2], cache, B) || !read_lengths(args[3], cache, B, lengths) || !read_counts(PyTuple_GET_ITEM(tree, 2), cache, B, counts)) Py_RETURN_NONE;
  const int with_lse = PyObject_IsTrue(args[6]);
  if (with_lse < 0) return nullptr;
  double scale = 1.0 / std::sqrt(static_cast<double>(D));
  if (args[5] != Py_None) {
    scale = PyFloat_AsDouble(args[5]);
    if (scale == -1.0 && PyErr_Occurred()) PyErr_Clear();
    if (!(static_cast<float>(scale) > 0.f && std::isfinite(static_cast<float>(scale)))) Py_RETURN_NONE;
  }
  const c10::cuda::CUDAGuard guard(cache.dev);                // the plan is the cache's device's
  const int64_t ws_bytes = g_lib.attn_workspace_bytes(static_cast<int>(B), static_cast<int>(N), static_cast<int>(H), cache.c.heads, cache.c.head_dim, table.T,
                                                      cache.c.page_size);
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
                     table.row, table.T, lengths, counts, static_cast<const int*>(seen->const_data_ptr()), seen->stride(0), seen->stride(1),
                     static_cast<float>(scale), o.mutable_data_ptr(), lse_p, p, ws_bytes, status, stream_of(cache.dev)));
  }
  if (!with_lse) return THPVariable_Wrap(std::move(o));
  return pair(std::move(o), std::move(lse));
  END_HANDLE_TH_ERRORS
}

// cache_keep(cache, block_table, before, lengths, path, counts) -> new lengths, or None
PyObject* cache_keep(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Cache cache;
  Ints path;
  if (n != 6 || elsewhere() || !cache.read(args[0]) || !cache.written_apart() || !sm100(cache.dev) || !path.read(args[4], -1, -1, &cache.dev)) Py_RETURN_NONE;
  const int64_t B = path.t->size(0), M = path.t->size(1);
  Table table;
  const int *before, *lengths, *counts;
  if (M > kMaxNodes || !table.read(args[1], cache, B) || !read_lengths(args[2], cache, B, before) || !read_lengths(args[3], cache, B, lengths) ||
      !read_lengths(args[5], cache, B, counts))
    Py_RETURN_NONE;
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(cache.dev);
    int* status = status_of(cache.dev.index());
    out = empty({B}, at::kInt, cache.dev);
    check(g_lib.keep(&cache.c, static_cast<int>(B), table.p, table.row, table.T, before, lengths, path.p, path.row, static_cast<int>(M), counts,
                     static_cast<int*>(out.mutable_data_ptr()), status, stream_of(cache.dev)));
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// bind_drafts(tree, append, attn, attn_workspace_bytes, keep): addresses of the entry points
PyObject* bind_drafts(PyObject*, PyObject* args) {
  unsigned long long a[5];
  if (!PyArg_ParseTuple(args, "KKKKK", &a[0], &a[1], &a[2], &a[3], &a[4])) return nullptr;
  g_lib.tree = reinterpret_cast<decltype(&dm_draft_tree)>(a[0]);
  g_lib.append = reinterpret_cast<decltype(&dm_cache_append_rotary)>(a[1]);
  g_lib.attn = reinterpret_cast<decltype(&dm_cache_attn_tree)>(a[2]);
  g_lib.attn_workspace_bytes = reinterpret_cast<decltype(&dm_cache_attn_tree_workspace_bytes)>(a[3]);
  g_lib.keep = reinterpret_cast<decltype(&dm_cache_keep)>(a[4]);
  Py_RETURN_NONE;
}

}  // namespace dm_native
