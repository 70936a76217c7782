// Graph nodes in C++ around the library's kernels (torch_tokens.cpp, torch_training.cpp).
#pragma once
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>

#include "torch_ops.h"

namespace ccf_torch {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = std::optional<at::Tensor>;

inline int type_code(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 0 : t.scalar_type() == at::kHalf ? 1 : 2; }
inline void* current_stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// A node of the graph with members of its own for what it keeps: an autograd::Function around it all (with its dictionary of boxed values) took the
// host 3 us more on either side of a pass.
struct TokenNode : torch::autograd::Node {
  std::vector<SavedVariable> saved;
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable& v : saved) v.reset_data();
  }
  void keep(const at::Tensor& t) { saved.emplace_back(t, false); }
  // the i-th kept tensor: hooks on saved tensors may hand it back in memory of their own, with other strides
  at::Tensor kept(int i) { return saved[i].unpack(shared_from_this()); }
  at::Tensor kept_contiguous(int i) {
    const at::Tensor t = kept(i);
    return t.defined() ? t.contiguous() : t;
  }
  variable_list apply(variable_list&& grads) final {
    const bool again = at::GradMode::is_enabled();   // the gradient is to be differentiated in its turn
    TORCH_CHECK(!again || twice, "ccfuser_b200: this operator's gradient cannot be differentiated again (create_graph=True)");
    const std::lock_guard<std::mutex> lock(mutex_);
    return again ? torch_gradients(grads) : gradients(grads);
  }
  virtual variable_list gradients(const variable_list& grads) = 0;
  // the same by operations of torch, which record a graph; for nodes with `twice`: those that models make
  virtual variable_list torch_gradients(const variable_list&) { return {}; }
  bool twice = false;
};
template <typename T, typename... Inputs>
std::shared_ptr<T> make_node(const Inputs&... inputs) {
  std::shared_ptr<T> node(new T(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}
// whether a graph is being built; forward-mode derivatives are refused
template <typename... Inputs>
bool builds_graph(const Inputs&... inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!((inputs.defined() && inputs._fw_grad(0).defined()) || ...), "ccfuser_b200: this operator has no forward-mode derivative");
  return at::GradMode::is_enabled() && ((inputs.defined() && inputs.requires_grad()) || ...);
}
inline const at::Tensor& or_none(const OptTensor& t) {
  static const at::Tensor none;
  return t.has_value() ? *t : none;
}

}  // namespace ccf_torch
