// What the translation units of the native eager route share (defined in dm_torch.cpp).
#pragma once
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/core/PythonFallbackKernel.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

namespace dm_native {

// Throw with the kernel library's message for a non-zero return code.
void check(int rc);
// The device's status word, raising first if a kernel has set it.
int* status_of(int dev);
// `t` with rows that the kernels can read: as it is, or copied.
at::Tensor rows(const at::Tensor& t);

constexpr int kMaxDevices = 64;

// A CUDA tensor that nothing wraps: no subclass, function transform or forward-mode tangent.
inline bool plain_cuda(PyObject* o, const at::Tensor*& t) {
  if (!THPVariable_CheckExact(o)) return false;
  t = &THPVariable_Unpack(o);
  constexpr c10::DispatchKeySet kWrapped({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::Functionalize,
                                          c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Conjugate, c10::DispatchKey::Negative});
  return t->is_cuda() && t->layout() == at::kStrided && !t->unsafeGetTensorImpl()->key_set().has_any(kWrapped) && !t->_fw_grad(0).defined();
}

// The methods of dm_torch_cache.cpp.
PyObject* cache_append(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* cache_attn(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* cache_evict(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* bind_cache(PyObject*, PyObject* args);

}  // namespace dm_native
