// What the autograd functions of the module built against torch share (torch_norm.cpp, torch_tokens.cpp, torch_training.cpp).
#pragma once
#include <ATen/ATen.h>
#include <torch/csrc/utils/pybind.h>

#include <atomic>

namespace ccf_torch {

inline std::atomic<long long> g_launches{0};   // kernels that the module has launched

inline void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed with code ", rc); }

// as the kernels read it: contiguous and on a 16-byte boundary (a view may begin anywhere)
inline at::Tensor packed(const at::Tensor& t) {
  const at::Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

void add_token_ops(py::module_& m);
void add_training_ops(py::module_& m);

}  // namespace ccf_torch
