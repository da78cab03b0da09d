// What the host modules of the plain calls share (decode_calls.cpp, layer_calls.cpp): looking torch
// tensors over, and what a backward pass has to watch. Each module includes it once; nothing here is exported.
#pragma once
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/object_ptr.h>

#include <ATen/ATen.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include "dan_tree_attn.h"

namespace {

using at::Tensor;
using torch::autograd::variable_list;

inline int code_of(at::ScalarType t) {  // DanDtype, or -1
  switch (t) {
    case at::kBFloat16: return DAN_DTYPE_BF16;
    case at::kHalf: return DAN_DTYPE_F16;
    case at::kFloat: return DAN_DTYPE_F32;
    case at::kFloat8_e4m3fn: return DAN_DTYPE_E4M3;
    default: return -1;
  }
}
inline bool is16(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }

using LastError = const char *(*)(void);
inline void check(int rc, const char *name, LastError last_error) {
  TORCH_CHECK_WITH(Error, rc == DAN_OK, name, " failed (status ", rc, "): ", last_error());
}

// A plain tensor on device `index`: nothing wraps it, and it carries no tangent.
inline bool plain(const Tensor &t, int index) {
  return t.defined() && t.is_cuda() && t.get_device() == index && t.layout() == at::kStrided && !at::isTensorSubclassLike(t) &&
         !t.is_neg() && !t._is_zerotensor() && !t._fw_grad(0).defined();
}
inline bool aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }
inline void *at_of(const Tensor &t) { return t.defined() ? const_cast<void *>(t.const_data_ptr()) : nullptr; }  // read, or new

// Rows that the kernels read in place: unit stride, 16-byte aligned.
inline bool rows_ok(const Tensor &t) {
  const int64_t es = t.element_size(), n = t.dim();
  if (t.stride(n - 1) != 1 || !aligned(t.const_data_ptr())) return false;
  for (int64_t i = 0; i + 1 < n; ++i)
    if (t.stride(i) * es % 16) return false;
  return true;
}
inline bool index_ok(const Tensor &t, int64_t n, int index) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && (n <= 1 || t.stride(0) == 1) && plain(t, index);
}
inline bool fits(int64_t x) { return x >= 0 && x <= INT32_MAX; }

// A Python argument as a tensor: undefined for None; false for anything else.
inline bool tensor_of(PyObject *o, Tensor &t) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  t = THPVariable_Unpack(o);
  return true;
}
inline bool grads_of(std::initializer_list<const Tensor *> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// A backward in a stream capture whose result goes to a node that lives on a stream outside of it, as the
// accumulator of a leaf does while an eager graph of the same leaf is alive: the engine would make that
// stream wait for the capture, which ends the process where it is the default one.
inline bool leaves_capture(int index) {
  const auto node = torch::autograd::get_current_node();
  if (!node) return false;
  const c10::hip::HIPStream here = c10::hip::getCurrentHIPStream(index);
  auto captures = [](hipStream_t s) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    return s && hipStreamIsCapturing(s, &status) == hipSuccess && status != hipStreamCaptureStatusNone;  // never the default one
  };
  for (const auto &edge : node->next_edges()) {
    if (!edge.function) continue;
    const auto to = edge.function->stream();
    if (!to || to->device_index() != index || to->id() == here.id()) continue;
    const c10::hip::HIPStream there(c10::Stream(c10::Stream::UNSAFE, here.unwrap().device(), to->id()));
    if (captures(here.stream()) && !captures(there.stream())) return true;
  }
  return false;
}

inline void check_capture(int index, const char *name = "token_logprobs") {
  TORCH_CHECK(!leaves_capture(index), name, ": a captured backward whose inputs were first used outside of the capture; "
              "drop every earlier result that holds their graph before the capture");
}
// A gradient whose own derivative is an error where it is taken, not before (`again`: one is being recorded).
inline Tensor differentiable_once(Tensor grad, bool again, const char *message) {
  if (!again || !grad.defined()) return grad;
  torch::autograd::DelayedError twice(message, 1);
  return twice.apply({grad.set_requires_grad(true)})[0];
}

}  // namespace
