// What the source files of the module `attention_cuda` share: types, dense and fresh tensors, errors, the mirror of the
// status word, and which calls the C++ autograd functions take.
#pragma once

#include <torch/extension.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/FuncTorchTLS.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <atomic>
#include <cstdio>
#include <initializer_list>
#include <mutex>
#include <vector>

#include "attn_b200.h"

namespace ext {

inline int dtype_code(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return ATTN_F16;
    case at::kBFloat16: return ATTN_BF16;
    case at::kFloat: return ATTN_F32;
    default: TORCH_CHECK(false, "V7 requires fp16, bf16 or fp32, got ", t.scalar_type());
  }
  return -1;
}

// Contiguous, and re-materialised if a view starts at an address TMA cannot use.
inline torch::Tensor dense(const torch::Tensor& t) {
  torch::Tensor c = t.contiguous();
  if (reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 != 0) c = c.clone();
  return c;
}

// New tensors of a contiguous shape on t's device, straight from the caching allocator: the
// dispatcher's factory functions take twice as long, and a call makes three to five tensors.  A tracer
// has to see where its tensors come from.
inline torch::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const torch::Tensor& t) {
  if (torch::jit::tracer::isTracing()) return torch::empty(sizes, t.options().dtype(type));
  return at::detail::empty_cuda(sizes, type, t.device(), c10::nullopt);
}
inline torch::Tensor fresh_like(const torch::Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t); }

inline void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == ATTN_OK, what, " failed (", rc, "): ", attn_b200_last_error());
}

// A kernel that gives up on a bounded wait stores a code in the device's status word and returns;
// its outputs are then meaningless.  This module registers one page-locked host word per device
// as a mirror of that status word (the failing kernel writes its code there too) and looks at it
// at the start of every call: a time-out of an earlier call is reported as an exception of the
// first call that starts after it, and the good path costs one read of host memory.
inline uint32_t* status_mirror(int device) {
  static torch::Tensor words[64];
  static std::atomic<uint32_t*> known[64];
  static std::mutex mu;
  TORCH_CHECK(device >= 0 && device < 64, "device index out of range");
  if (uint32_t* w = known[device].load(std::memory_order_acquire)) return w;
  std::lock_guard<std::mutex> lock(mu);
  if (!words[device].defined()) {
    words[device] = torch::zeros({1}, torch::dtype(torch::kInt32).pinned_memory(true));
    check_rc(attn_b200_set_status_mirror(reinterpret_cast<uint32_t*>(words[device].data_ptr<int32_t>())),
             "attn_b200_set_status_mirror");
  }
  uint32_t* w = reinterpret_cast<uint32_t*>(words[device].data_ptr<int32_t>());
  known[device].store(w, std::memory_order_release);
  return w;
}

inline void raise_if_earlier_call_timed_out(int device) {
  volatile uint32_t* w = status_mirror(device);
  if (*w == 0u) return;
  *w = 0u;
  uint32_t code = 0;
  int rc = attn_b200_device_status(&code);     // synchronises, reads and clears the device word
  char hex[16];
  snprintf(hex, sizeof(hex), "0x%x", code);
  TORCH_CHECK(rc == ATTN_OK && code == 0u, "an earlier attention kernel on this device gave up on a bounded wait (status ",
              hex, "); its outputs are invalid");
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline bool has_tangent(std::initializer_list<const torch::Tensor*> inputs) {
  for (const torch::Tensor* t : inputs)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined()) return true;
  return false;
}

// A call for the Python autograd functions: torch.jit.trace records them, and they refuse a tangent,
// which kernels called directly would drop.  Under a functorch transform neither kind of function has
// a rule: refused here, whether or not gradients are asked for.
inline bool leave_to_python(std::initializer_list<const torch::Tensor*> inputs) {
  if (const auto& functorch = at::functorch::functorchTLSAccessor()) functorch->checkSupportsCppAutogradFunction();
  return torch::jit::tracer::isTracing() || has_tangent(inputs);
}

// For operators without a Python form: what a C++ autograd function cannot do is refused.
inline void refuse_transforms(std::initializer_list<const torch::Tensor*> inputs, const char* what) {
  if (const auto& functorch = at::functorch::functorchTLSAccessor()) functorch->checkSupportsCppAutogradFunction();
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " cannot be traced");
  TORCH_CHECK(!has_tangent(inputs), what, " has no forward-mode derivative");
}

inline bool wants_graph(std::initializer_list<const torch::Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const torch::Tensor* t : inputs)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

void register_packed(pybind11::module& m);
void register_loss(pybind11::module& m);

}  // namespace ext

std::vector<torch::Tensor> v7_double_backward_cuda(torch::Tensor g_dQ, torch::Tensor g_dK, torch::Tensor g_dV,
                                                   torch::Tensor dO, torch::Tensor Q, torch::Tensor K,
                                                   torch::Tensor V, torch::Tensor O, torch::Tensor L,
                                                   int window_size, int chunk_id, int mask_mode, int impl);
