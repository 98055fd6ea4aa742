// What the native eager routes of the cache's functions share (dm_torch_cache.cpp, dm_torch_drafts.cpp): a call's arguments as the checks of
// cache.py take them.
#pragma once
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/utils/wrap_outputs.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>

#include "../../include/dm_b200.h"
#include "dm_torch.h"

namespace dm_native {

using at::Tensor;

constexpr int64_t kBlk = 32;

// Whether two elements of `t` may share an address: a dimension's stride is below what the dimensions of smaller strides span.
inline bool overlaps(const Tensor& t) {
  int64_t reach = 1;                                          // elements that the dimensions looked at so far span
  bool done[4] = {};
  for (int64_t k = 0; k < t.dim(); ++k) {
    int64_t least = -1;
    for (int64_t d = 0; d < t.dim(); ++d)
      if (!done[d] && (least < 0 || t.stride(d) < t.stride(least))) least = d;
    done[least] = true;
    if (t.size(least) == 1) continue;
    if (t.stride(least) < reach) return true;
    reach += (t.size(least) - 1) * t.stride(least);
  }
  return false;
}

inline bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }

// The pools of a KVCache8 (a tuple of four), as cache.py's _check_cache takes them.
struct Cache {
  const Tensor *k8, *v8, *ks, *vs;
  dm_kv_cache c;
  at::Device dev{at::kCUDA};
  bool written_apart() const { return !overlaps(*k8) && !overlaps(*ks); }        // V's strides are K's
  bool read(PyObject* o) {
    if (!PyTuple_Check(o) || PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 4) return false;     // a KVCache8, no plain tuple
    const Tensor** t[4] = {&k8, &v8, &ks, &vs};
    for (int i = 0; i < 4; ++i)
      if (!plain_cuda(PyTuple_GET_ITEM(o, i), *t[i])) return false;
    if (k8->dim() != 4 || ks->dim() != 3 || k8->scalar_type() != at::kFloat8_e4m3fn || v8->scalar_type() != at::kFloat8_e4m3fn ||
        ks->scalar_type() != at::kFloat || vs->scalar_type() != at::kFloat || k8->sizes() != v8->sizes() || ks->sizes() != vs->sizes() ||
        k8->strides() != v8->strides() || ks->strides() != vs->strides())
      return false;
    const int64_t pages = k8->size(0), heads = k8->size(1), page = k8->size(2), D = k8->size(3);
    if ((D != 128 && D != 256) || page <= 0 || page % kBlk || pages <= 0 || heads <= 0 || pages > INT32_MAX || heads > INT32_MAX || page > INT32_MAX) return false;
    if (ks->size(0) != pages || ks->size(1) != heads || ks->size(2) != page / kBlk || (page > kBlk && ks->stride(2) != 1)) return false;
    if (k8->stride(3) != 1 || k8->stride(0) % 16 || k8->stride(1) % 16 || k8->stride(2) % 16 || !aligned16(*k8) || !aligned16(*v8)) return false;
    dev = k8->device();
    if (v8->device() != dev || ks->device() != dev || vs->device() != dev || dev.index() >= kMaxDevices) return false;
    c.k8 = const_cast<void*>(k8->const_data_ptr());
    c.v8 = const_cast<void*>(v8->const_data_ptr());
    c.ks = static_cast<float*>(const_cast<void*>(ks->const_data_ptr()));
    c.vs = static_cast<float*>(const_cast<void*>(vs->const_data_ptr()));
    c.code_page = pages > 1 ? k8->stride(0) : 16;
    c.code_head = heads > 1 ? k8->stride(1) : 16;
    c.code_slot = k8->stride(2);
    c.scale_page = ks->stride(0);
    c.scale_head = ks->stride(1);
    c.pages = static_cast<int>(pages);
    c.heads = static_cast<int>(heads);
    c.page_size = static_cast<int>(page);
    c.head_dim = static_cast<int>(D);
    return true;
  }
};

// Calls that the Python route serves or refuses: tracing, dispatch modes.
inline bool elsewhere() { return c10::impl::TorchDispatchModeTLS::any_modes_set() || torch::jit::tracer::isTracing(); }

inline bool read_rows(PyObject* o, const Cache& cache, int64_t heads, const Tensor*& t) {
  return plain_cuda(o, t) && t->dim() == 4 && t->scalar_type() == at::kBFloat16 && t->device() == cache.dev && t->numel() > 0 &&
         (heads == 0 || t->size(2) == heads) && t->size(3) == cache.c.head_dim && t->size(0) <= INT32_MAX && t->size(1) <= INT32_MAX && t->size(2) <= INT32_MAX;
}
inline bool read_lengths(PyObject* o, const Cache& cache, int64_t B, const int*& p) {
  const Tensor* t;
  if (!plain_cuda(o, t) || t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != B || t->device() != cache.dev || !t->is_contiguous()) return false;
  p = static_cast<const int*>(t->const_data_ptr());
  return true;
}
inline bool read_counts(PyObject* o, const Cache& cache, int64_t B, const int*& p) {
  p = nullptr;
  return o == Py_None || read_lengths(o, cache, B, p);
}
struct Table {
  const int* p;
  int64_t row;
  int T;
  bool read(PyObject* o, const Cache& cache, int64_t B) {
    const Tensor* t;
    if (!plain_cuda(o, t) || t->scalar_type() != at::kInt || t->dim() != 2 || t->size(0) != B || t->size(1) <= 0 || t->size(1) > INT32_MAX ||
        t->device() != cache.dev || (t->size(1) > 1 && t->stride(1) != 1))
      return false;
    p = static_cast<const int*>(t->const_data_ptr());
    T = static_cast<int>(t->size(1));
    row = B > 1 ? t->stride(0) : T;
    return true;
  }
  int64_t room(const Cache& cache) const { return static_cast<int64_t>(T) * cache.c.page_size; }
};
inline bool read_weights(PyObject* o, const Cache& cache, int64_t B, int64_t room, const Tensor*& t) {
  return plain_cuda(o, t) && t->scalar_type() == at::kFloat && t->dim() == 3 && t->size(0) == B && t->size(1) == cache.c.heads && t->size(2) >= room &&
         t->size(2) <= INT32_MAX && t->device() == cache.dev && (t->size(2) == 1 || t->stride(2) == 1);
}
// An int (or what converts to one without an error); false sends the call to the Python route.
inline bool read_int(PyObject* o, long long& v) {
  v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

inline Tensor empty(at::IntArrayRef size, at::ScalarType type, const at::Device& dev) {
  return Tensor(at::detail::empty_cuda(size, type, dev, std::nullopt));
}
inline void* stream_of(const at::Device& dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }
inline bool sm100(const at::Device& dev) { return at::cuda::getDeviceProperties(dev.index())->major == 10; }

}  // namespace dm_native
