// What a training step of a mixture of experts needs around its products: the nodes of the graph around expert_sort.cu, and the lists of tensors of adamw.cu,
// with the checks of their arguments. ops/expert_sort.py and ops/optim.py hold both in Python as well, for where this module is missing, a graph is being
// traced or the tensors are not on a GPU.
#include <c10/cuda/CUDAGuard.h>

#include <torch/csrc/autograd/python_variable.h>

#include <unordered_set>

#include "adamw.h"
#include "expert_sort.h"
#include "torch_nodes.h"

namespace {

using namespace ccf_torch;

bool kernel_type(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat;
}

// ---- tokens sorted by expert -------------------------------------------------------------------------------------------
struct Order {
  at::Tensor slot_row, row_slot, counts, base;
};

void check_idx(const at::Tensor& idx, int64_t experts, const std::optional<int64_t>& capacity, int64_t align) {
  TORCH_CHECK_TYPE(idx.scalar_type() == at::kLong || idx.scalar_type() == at::kInt, "idx is int64 or int32, not ", idx.scalar_type());
  TORCH_CHECK_VALUE(idx.dim() >= 1, "idx: [..., top_k], got ", idx.sizes());
  TORCH_CHECK_VALUE(1 <= experts && experts <= CCF_SORT_MAX_EXPERTS, "num_experts: 1 to ", CCF_SORT_MAX_EXPERTS, ", got ", experts);
  TORCH_CHECK_VALUE(!capacity.has_value() || *capacity >= 1, "capacity: at least 1, got ", capacity.value_or(0));
  TORCH_CHECK_VALUE(1 <= align && align <= CCF_SORT_MAX_ALIGN, "align: 1 to ", CCF_SORT_MAX_ALIGN, ", got ", align);
  TORCH_CHECK_VALUE(idx.numel() <= CCF_SORT_MAX_SLOTS, idx.numel(), " slots: at most 2^30 in one call");
}

// a tensor of its own in the memory of another; without the dispatcher, which takes longer than the launches of a small call
at::Tensor part_of(const at::Tensor& t, int64_t first, at::IntArrayRef sizes) {
  at::Tensor r = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
  r.unsafeGetTensorImpl()->set_storage_offset(first);
  r.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return r;
}

// Memory for the order of idx, contiguous, and the arguments of its kernels.
Order new_order(CcfOrder& o, const at::Tensor& idx, int64_t experts, const std::optional<int64_t>& capacity, int64_t align) {
  o.idx = idx.data_ptr();
  o.slots = idx.numel();
  o.capacity = capacity.value_or(o.slots);
  o.experts = static_cast<int>(experts);
  o.align = static_cast<int>(align);
  o.wide = idx.scalar_type() == at::kLong;
  o.rows = ccf_order_rows(o.slots, o.experts, o.capacity, o.align);
  TORCH_CHECK_VALUE(o.rows >= 0, "at most 2^31 - 1 rows in one call");
  const auto up = [](int64_t n) { return (n + 3) / 4 * 4; };      // each on 16 bytes
  const int64_t at_base = up(experts), at_slots = at_base + up(experts + 1), at_rows = at_slots + up(o.slots), at_scratch = at_rows + up(o.rows);
  const at::Tensor all = at::empty({at_scratch + ccf_order_scratch(o.slots, o.experts) / 4}, at::TensorOptions(idx.device()).dtype(at::kInt));
  const Order r = {part_of(all, at_slots, idx.sizes()), part_of(all, at_rows, {o.rows}), part_of(all, 0, {experts}), part_of(all, at_base, {experts + 1})};
  o.slot_row = r.slot_row.data_ptr<int>();
  o.row_slot = r.row_slot.data_ptr<int>();
  o.counts = r.counts.data_ptr<int>();
  o.base = r.base.data_ptr<int>();
  o.scratch = all.data_ptr<int>() + at_scratch;
  return r;
}

// tokens as the kernels read them: rows with any distance, their elements next to each other
at::Tensor token_rows(const at::Tensor& x, int64_t tokens, int64_t d) {
  const at::Tensor r = x.dim() == 2 ? x : x.reshape({tokens, d});
  return r.stride(1) == 1 && (tokens == 1 || r.stride(0) >= d) ? r : r.contiguous();
}

CcfRows rows_args(const at::Tensor& slot_row, int64_t rows, int64_t d, const at::Tensor& typed) {
  CcfRows a{};
  a.slot_row = slot_row.data_ptr<int>();
  a.top_k = static_cast<int>(slot_row.size(-1));
  a.tokens = slot_row.numel() / a.top_k;
  a.rows = rows;
  a.d = static_cast<int>(d);
  a.ld = d;
  a.type = type_code(typed);
  return a;
}

// The rows of an order; with `o` the order is made as well, of what lies in `o`.
at::Tensor run_sort(const at::Tensor& x_, const at::Tensor& slot_row, const at::Tensor& row_slot, const CcfOrder* o) {
  const int64_t d = x_.size(-1);
  CcfRows a = rows_args(slot_row, row_slot.numel(), d, x_);
  const at::Tensor x = token_rows(x_, a.tokens, d);
  const at::Tensor rows = at::empty({a.rows, d}, x.options().requires_grad(false));
  a.tokens_in = x.data_ptr();
  if (a.tokens > 1) a.ld = x.stride(0);
  a.row_slot = row_slot.data_ptr<int>();
  a.rows_out = rows.data_ptr();
  if (o == nullptr) {
    check(ccf_sort_rows(&a, 0, current_stream()), "ccf_sort_rows");
    ++g_launches;
  } else {
    const int launches = ccf_sort_by_expert(o, &a, current_stream());
    TORCH_CHECK(launches > 0, "ccf_sort_by_expert failed with code ", launches);
    g_launches += launches;
  }
  return rows;
}

at::Tensor run_return(const at::Tensor& rows_, const at::Tensor& slot_row, const at::Tensor& weights) {
  const at::Tensor rows = rows_.contiguous();
  const int64_t d = rows.size(1);
  CcfRows a = rows_args(slot_row, rows.size(0), d, rows);
  at::DimVector shape(slot_row.sizes().slice(0, slot_row.dim() - 1));
  shape.push_back(d);
  const at::Tensor y = at::empty(shape, rows.options().requires_grad(false));
  a.rows_in = rows.data_ptr();
  a.tokens_out = y.data_ptr();
  if (weights.defined()) {
    a.weights = weights.data_ptr();
    a.weight_type = type_code(weights);
  }
  check(ccf_return_rows(&a, current_stream()), "ccf_return_rows");
  ++g_launches;
  return y;
}

// where a number is none of `count`: what the kernels leave out, and torch's operations must not see
at::Tensor outside(const at::Tensor& numbers, int64_t count) { return numbers.lt(0).logical_or(numbers.ge(count)); }

// by torch's operations, which record a graph: each slot's row, zeros where it has none: [tokens, top_k, d]
at::Tensor torch_slots(const at::Tensor& rows, const at::Tensor& slot_row) {
  const int64_t k = slot_row.size(-1), tokens = slot_row.numel() / k;
  const at::Tensor at = slot_row.reshape({tokens, k}), none = outside(at, rows.size(0));
  return rows.to(at::kFloat).index_select(0, at.masked_fill(none, 0).reshape({-1}).to(at::kLong)).reshape({tokens, k, rows.size(1)}).masked_fill(none.unsqueeze(2), 0);
}

struct SortNode : TokenNode {
  std::vector<int64_t> shape;
  SortNode() { twice = true; }
  std::string name() const override { return "CcfSortRowsBackward"; }
  variable_list gradients(const variable_list& grads) override {
    variable_list out(1);
    if (!grads[0].defined()) return out;
    const c10::cuda::CUDAGuard guard(grads[0].device());
    out[0] = run_return(grads[0], kept_contiguous(0), at::Tensor()).view(shape);
    return out;
  }
  variable_list torch_gradients(const variable_list& grads) override {
    variable_list out(1);
    if (grads[0].defined()) out[0] = torch_slots(grads[0], kept(0)).sum(1).to(grads[0].scalar_type()).reshape(shape);
    return out;
  }
};

struct ReturnNode : TokenNode {
  int64_t rows;
  std::vector<int64_t> weight_shape;
  ReturnNode() { twice = true; }
  std::string name() const override { return "CcfReturnRowsBackward"; }
  variable_list gradients(const variable_list& grads) override {
    variable_list out(2);
    if (!grads[0].defined()) return out;
    const at::Tensor slot_row = kept_contiguous(0), row_slot = kept_contiguous(1), weights = kept_contiguous(2), values = kept_contiguous(3);
    const c10::cuda::CUDAGuard guard(grads[0].device());
    const int64_t d = grads[0].size(-1);
    CcfRows a = rows_args(slot_row, rows, d, grads[0]);
    const at::Tensor dy = token_rows(grads[0], a.tokens, d);
    a.tokens_in = dy.data_ptr();
    if (a.tokens > 1) a.ld = dy.stride(0);
    a.row_slot = row_slot.data_ptr<int>();
    if (weights.defined()) {
      a.weights = weights.data_ptr();
      a.weight_type = type_code(weights);
    }
    if (task_should_compute_output(0)) {
      out[0] = at::empty({rows, d}, dy.options());
      a.rows_out = out[0].data_ptr();
    }
    if (weights.defined() && values.defined() && task_should_compute_output(1)) {
      out[1] = at::empty(weight_shape, weights.options());
      a.d_weights = out[1].data_ptr();
      a.rows_in = values.data_ptr();
    }
    check(ccf_return_rows_bwd(&a, current_stream()), "ccf_return_rows_bwd");
    ++g_launches;
    return out;
  }
  variable_list torch_gradients(const variable_list& grads) override {
    variable_list out(2);
    if (!grads[0].defined()) return out;
    const at::Tensor slot_row = kept(0), row_slot = kept(1), weights = kept(2), values = kept(3);
    const int64_t k = slot_row.size(-1), tokens = slot_row.numel() / k, d = grads[0].size(-1);
    const at::Tensor dy = grads[0].reshape({tokens, d}).to(at::kFloat), none = outside(row_slot, tokens * k), slot = row_slot.masked_fill(none, 0).to(at::kLong);
    if (task_should_compute_output(0)) {
      at::Tensor g = dy.index_select(0, at::floor_divide(slot, k));
      if (weights.defined()) g = g * weights.reshape({-1}).to(at::kFloat).index_select(0, slot).masked_fill(none, 0).unsqueeze(1);
      out[0] = g.masked_fill(none.unsqueeze(1), 0).to(grads[0].scalar_type());
    }
    if (weights.defined() && values.defined() && task_should_compute_output(1))
      out[1] = (torch_slots(values, slot_row) * dy.unsqueeze(1)).sum(2).to(weights.scalar_type()).reshape(weight_shape);
    return out;
  }
};

void check_tokens(const at::Tensor& x, const at::Tensor& idx) {
  TORCH_CHECK_VALUE(x.dim() == idx.dim() && x.dim() >= 1 && x.sizes().slice(0, x.dim() - 1) == idx.sizes().slice(0, idx.dim() - 1),
                    "x: [..., d] with the tokens of the experts' ids, [..., top_k], got ", x.sizes(), " and ", idx.sizes());
  TORCH_CHECK_VALUE(x.device() == idx.device(), "x is on ", x.device(), ", the tensor beside it on ", idx.device());
  TORCH_CHECK_TYPE(kernel_type(x), "on a GPU bf16, fp16 or fp32, not ", x.scalar_type());
  TORCH_CHECK_VALUE(x.size(-1) <= CCF_SORT_MAX_D, "at most 2^24 columns, got ", x.size(-1));
}
void check_order(const at::Tensor& slot_row, const at::Tensor& row_slot) {
  TORCH_CHECK_TYPE(slot_row.scalar_type() == at::kInt && row_slot.scalar_type() == at::kInt, "an order's numbers are int32, not ", slot_row.scalar_type(), " and ",
                   row_slot.scalar_type());
  TORCH_CHECK_VALUE(slot_row.dim() >= 1 && row_slot.dim() == 1 && slot_row.device() == row_slot.device(), "an order: slot_row [..., top_k] and row_slot [rows] on one device, got ",
                    slot_row.sizes(), " on ", slot_row.device(), " and ", row_slot.sizes(), " on ", row_slot.device());
  TORCH_CHECK_VALUE(slot_row.numel() <= CCF_SORT_MAX_SLOTS && row_slot.numel() <= 0x7fffffff, "at most 2^30 slots and 2^31 - 1 rows in one call");
}

at::Tensor sorted(const at::Tensor& x, const at::Tensor& slot_row, const at::Tensor& row_slot, const CcfOrder* o, bool training) {
  const at::Tensor rows = run_sort(x, slot_row, row_slot, o);
  if (training) {
    const auto node = make_node<SortNode>(x);
    node->keep(slot_row);
    node->shape = x.sizes().vec();
    torch::autograd::set_history(rows, node);
  }
  return rows;
}

variable_list expert_order(const at::Tensor& idx, int64_t experts, const std::optional<int64_t>& capacity, int64_t align) {
  check_idx(idx, experts, capacity, align);
  const c10::cuda::CUDAGuard guard(idx.device());
  CcfOrder a{};
  const at::Tensor packed_idx = idx.contiguous();
  const Order o = new_order(a, packed_idx, experts, capacity, align);
  const int launches = ccf_order(&a, current_stream());
  TORCH_CHECK(launches > 0, "ccf_order failed with code ", launches);
  g_launches += launches;
  return {o.slot_row, o.row_slot, o.counts, o.base};
}

variable_list sort_by_expert(const at::Tensor& x, const at::Tensor& idx, int64_t experts, const std::optional<int64_t>& capacity, int64_t align) {
  check_idx(idx, experts, capacity, align);
  check_tokens(x, idx);
  const c10::cuda::CUDAGuard guard(x.device());
  const bool training = builds_graph(x);
  const at::NoGradGuard no_graph;   // views still share their base's version: a change before the backward pass is noticed
  CcfOrder a{};
  const at::Tensor packed_idx = idx.contiguous();
  const Order o = new_order(a, packed_idx, experts, capacity, align);
  return {sorted(x, o.slot_row, o.row_slot, &a, training), o.slot_row, o.row_slot, o.counts, o.base};
}

at::Tensor sort_rows(const at::Tensor& x, const at::Tensor& slot_row, const at::Tensor& row_slot) {
  check_order(slot_row, row_slot);
  check_tokens(x, slot_row);
  const c10::cuda::CUDAGuard guard(x.device());
  const bool training = builds_graph(x);
  const at::NoGradGuard no_graph;
  return sorted(x, slot_row.contiguous(), row_slot.contiguous(), nullptr, training);
}

at::Tensor return_rows(const at::Tensor& rows, const at::Tensor& slot_row_, const at::Tensor& row_slot_, const OptTensor& weights_) {
  const at::Tensor& weights = or_none(weights_);
  check_order(slot_row_, row_slot_);
  TORCH_CHECK_VALUE(rows.dim() == 2 && rows.size(0) == row_slot_.size(0) && rows.device() == slot_row_.device(), "rows: [", row_slot_.size(0), ", d] on ",
                    slot_row_.device(), ", got ", rows.sizes(), " on ", rows.device());
  TORCH_CHECK_TYPE(kernel_type(rows), "on a GPU bf16, fp16 or fp32, not ", rows.scalar_type());
  TORCH_CHECK_VALUE(rows.size(1) <= CCF_SORT_MAX_D, "at most 2^24 columns, got ", rows.size(1));
  TORCH_CHECK_VALUE(!weights.defined() || (weights.sizes() == slot_row_.sizes() && weights.device() == rows.device()), "weights: ", slot_row_.sizes(), " on ", rows.device(),
                    ", got ", weights.defined() ? weights.sizes() : rows.sizes());
  TORCH_CHECK_TYPE(!weights.defined() || kernel_type(weights), "weights are bf16, fp16 or fp32");
  const c10::cuda::CUDAGuard guard(rows.device());
  const bool training = builds_graph(rows, weights);
  const at::NoGradGuard no_graph;
  const at::Tensor slot_row = slot_row_.contiguous(), row_slot = row_slot_.contiguous();
  const at::Tensor y = run_return(rows, slot_row, weights.defined() ? weights.contiguous() : weights);
  if (training) {
    const auto node = make_node<ReturnNode>(rows, weights);
    node->keep(slot_row);
    node->keep(row_slot);
    node->keep(weights);
    node->keep(weights.defined() && weights.requires_grad() ? rows : at::Tensor());   // only the weights' gradient reads the rows
    node->rows = rows.size(0);
    if (weights.defined()) node->weight_shape = weights.sizes().vec();
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------
struct AdamwCall {
  c10::Device device;
  int type;
  std::vector<CcfAdamwTensor> tensors;
};

// The tensors of a list or tuple, without a count of references for each (a step of 60 tensors took the host 34 us with
// std::vector<at::Tensor>, 19 so).
// The interpreter's lock is held as long as they are used.
struct TensorList {
  py::object fast;      // keeps the items
  std::vector<const at::Tensor*> items;
  TensorList(const py::object& list, const char* name) {
    fast = py::reinterpret_steal<py::object>(PySequence_Fast(list.ptr(), name));
    if (!fast) throw py::error_already_set();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast.ptr());
    PyObject** const from = PySequence_Fast_ITEMS(fast.ptr());
    items.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      TORCH_CHECK_TYPE(THPVariable_Check(from[i]), name, ": element ", i, " is no tensor");
      items.push_back(&THPVariable_Unpack(from[i]));
    }
  }
  size_t size() const { return items.size(); }
  const at::Tensor& operator[](size_t i) const { return *items[i]; }
};

void check_state(const at::Tensor& p, const at::Tensor& g, const at::Tensor& m, const at::Tensor& v, const at::Tensor* e, size_t i) {
  TORCH_CHECK_TYPE(g.layout() == at::kStrided && g.scalar_type() == p.scalar_type(), "grads: tensor ", i, " is ", g.layout(), " of ", g.scalar_type(), ", its parameter ",
                   p.scalar_type());
  const auto type = e != nullptr ? at::kByte : at::kFloat;
  TORCH_CHECK_TYPE(m.scalar_type() == type && v.scalar_type() == type && (e == nullptr || e->scalar_type() == at::kByte), "moments of tensor ", i, " are ", type, ", not ",
                   m.scalar_type(), " and ", v.scalar_type());
  TORCH_CHECK_VALUE(g.sizes() == p.sizes() && m.sizes() == p.sizes() && v.sizes() == p.sizes(), "tensor ", i, ": ", p.sizes(), ", its gradient and moments ", g.sizes(), ", ",
                    m.sizes(), " and ", v.sizes());
  TORCH_CHECK_VALUE(g.device() == p.device() && m.device() == p.device() && v.device() == p.device() && (e == nullptr || e->device() == p.device()), "tensor ", i,
                    " and what belongs to it lie on several devices");
  if (e == nullptr) return;
  const int64_t rows = e->dim() == 3 ? e->size(0) : 0;
  TORCH_CHECK_VALUE(rows >= 1 && p.numel() % rows == 0 && e->size(1) == (p.numel() / rows + CCF_ADAMW_BLOCK - 1) / CCF_ADAMW_BLOCK && e->size(2) == 2,
                    "exponents of tensor ", i, ": [rows, blocks of a row, 2] for ", p.numel(), " weights, got ", e->sizes());
}

// One step; false, with nothing changed, where a tensor is not one for the kernels (another type or device, not contiguous).
bool adamw_step(const py::object& params_, const py::object& grads_, const py::object& first_, const py::object& second_, const py::object& exponents_, double lr, double beta1,
                double beta2, double eps, double weight_decay, int64_t seed, int64_t step, const OptTensor& counter, const OptTensor& device_lr,
                const std::optional<std::vector<int64_t>>& numbers) {
  const TensorList params(params_, "params"), grads(grads_, "grads"), first(first_, "exp_avgs"), second(second_, "exp_avg_sqs");
  const bool eight = !exponents_.is_none();
  const TensorList exponents(eight ? exponents_ : py::object(py::list()), "exponents");
  const size_t n = params.size();
  TORCH_CHECK_VALUE(grads.size() == n && first.size() == n && second.size() == n && (!eight || exponents.size() == n) && (!numbers.has_value() || numbers->size() == n), n,
                    " params need as many gradients, moments, exponents and numbers");
  std::vector<at::Tensor> packed_grads;      // lives until the launches
  std::vector<AdamwCall> calls;
  std::unordered_set<const void*> seen;
  seen.reserve(n);
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor &p = params[i], &g = grads[i], &m = first[i], &v = second[i];
    const at::Tensor* const e = eight ? &exponents[i] : nullptr;
    if (!p.is_cuda() || !kernel_type(p) || !p.is_contiguous() || !m.is_contiguous() || !v.is_contiguous() || (e != nullptr && !e->is_contiguous())) return false;
    check_state(p, g, m, v, e, i);
    if (p.numel() == 0) continue;
    TORCH_CHECK_VALUE(seen.insert(p.data_ptr()).second, "params: tensor ", i, " is there twice");
    const int type = type_code(p);
    AdamwCall* call = nullptr;
    for (AdamwCall& c : calls)
      if (c.device == p.device() && c.type == type) call = &c;
    if (call == nullptr) {
      calls.push_back({p.device(), type, {}});
      call = &calls.back();
      call->tensors.reserve(n);
    }
    if (!g.is_contiguous()) packed_grads.push_back(g.contiguous());
    CcfAdamwTensor t{};
    t.p = p.data_ptr();
    t.g = g.is_contiguous() ? g.data_ptr() : packed_grads.back().data_ptr();
    t.m = m.data_ptr();
    t.v = v.data_ptr();
    t.n = p.numel();
    t.rows = 1;
    t.number = numbers.has_value() ? (*numbers)[i] : static_cast<int64_t>(i);
    if (e != nullptr) {
      t.e = e->data_ptr<uint8_t>();
      t.rows = e->size(0);
    }
    call->tensors.push_back(t);
  }
  CcfAdamw a{};
  a.lr = lr;
  a.beta1 = beta1;
  a.beta2 = beta2;
  a.eps = eps;
  a.weight_decay = weight_decay;
  a.seed = static_cast<unsigned long long>(seed);
  a.step = step;
  at::Tensor scalars;
  if (counter.has_value()) {
    for (const AdamwCall& c : calls)
      TORCH_CHECK_VALUE(c.device == counter->device(), "counter: on ", counter->device(), ", the tensors beside it on ", c.device);
    const c10::cuda::CUDAGuard guard(counter->device());
    scalars = at::empty({CCF_ADAMW_SCALARS}, counter->options().dtype(at::kByte));
    check(ccf_adamw_scalars(&a, reinterpret_cast<long long*>(counter->data_ptr<int64_t>()), device_lr.has_value() ? device_lr->data_ptr<float>() : nullptr,
                            scalars.data_ptr(), current_stream()),
          "ccf_adamw_scalars");
    ++g_launches;
    a.scalars = scalars.data_ptr();
  }
  for (const AdamwCall& c : calls) {
    const c10::cuda::CUDAGuard guard(c.device);
    a.tensors = c.tensors.data();
    a.count = static_cast<int>(c.tensors.size());
    a.type = c.type;
    const int launches = ccf_adamw(&a, current_stream());
    TORCH_CHECK(launches > 0, "ccf_adamw failed with code ", launches);
    g_launches += launches;
  }
  const auto changed = [](const at::Tensor& t) {      // as by an operation in place
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  };
  for (size_t i = 0; i < n; ++i) {
    changed(params[i]);
    changed(first[i]);
    changed(second[i]);
    if (eight) changed(exponents[i]);
  }
  if (counter.has_value()) changed(*counter);
  return true;
}

at::Tensor state_values(const at::Tensor& codes_, const at::Tensor& exponents_, bool second, int64_t type) {
  const at::Tensor codes = codes_.contiguous(), exponents = exponents_.contiguous();
  const c10::cuda::CUDAGuard guard(codes.device());
  const at::Tensor out = at::empty(codes.sizes(), codes.options().dtype(type == 0 ? at::kBFloat16 : type == 1 ? at::kHalf : at::kFloat));
  check(ccf_state_values(codes.data_ptr(), exponents.data_ptr<uint8_t>(), out.data_ptr(), codes.numel(), exponents.dim() == 3 ? exponents.size(0) : 1, second,
                         static_cast<int>(type), current_stream()),
        "ccf_state_values");
  ++g_launches;
  return out;
}

}  // namespace

void ccf_torch::add_training_ops(py::module_& m) {
  const auto free = py::call_guard<py::gil_scoped_release>();
  m.def("expert_order", &expert_order, free);
  m.def("sort_by_expert", &sort_by_expert, free);
  m.def("sort_rows", &sort_rows, free);
  m.def("return_rows", &return_rows, free);
  m.def("adamw_step", &adamw_step);
  m.def("state_values", &state_values, free);
}
