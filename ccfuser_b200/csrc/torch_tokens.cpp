// The autograd functions around embedding.cu, logprobs.cu and dropout.cu. ops/embedding.py, ops/logprobs.py and ops/dropout.py check the
// arguments, and hold the same functions in Python for where this module is missing or a graph is being traced.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>

#include "dropout.h"
#include "embedding.h"
#include "logprobs.h"
#include "torch_ops.h"

namespace {

using ccf_torch::check;
using ccf_torch::g_launches;
using ccf_torch::packed;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<at::Tensor>;

int type_code(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 0 : t.scalar_type() == at::kHalf ? 1 : 2; }
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
void once() { TORCH_CHECK(!at::GradMode::is_enabled(), "ccfuser_b200: this operator's gradient cannot be differentiated again (create_graph=True)"); }

// ---- embedding ---------------------------------------------------------------------------------------------------------
// A table as the kernels read it: rows with any distance, their elements next to each other.
at::Tensor table_of(const at::Tensor& w) { return w.stride(1) == 1 && w.stride(0) >= w.size(1) ? w : w.contiguous(); }

void add_table(CcfEmbed& e, const at::Tensor& ids, int64_t rows, double scale, int64_t skip) {
  CcfEmbedTable& t = e.table[e.tables++];
  t.rows = rows;
  t.scale = static_cast<float>(scale);
  t.skip = skip;
  if (ids.defined()) {
    t.ids = ids.data_ptr();
    t.wide = ids.scalar_type() == at::kLong;
  }
}

// One gradient launch for up to three tables: grads[k] [rows, d] from dy [tokens, d].
void run_grad(CcfEmbed& e, const at::Tensor& dy, const std::vector<at::Tensor>& grads, const at::Tensor& status) {
  int64_t at[3] = {}, bytes = 0;
  for (int k = 0; k < e.tables; ++k) {
    at[k] = bytes;
    bytes += ccf_embedding_scratch(e.tokens, e.seq, e.table[k].rows, e.d, e.table[k].ids != nullptr);   // a multiple of 16
  }
  const at::Tensor scratch = at::empty({bytes}, dy.options().dtype(at::kByte));
  for (int k = 0; k < e.tables; ++k) {
    e.table[k].scratch = static_cast<uint8_t*>(scratch.data_ptr()) + at[k];
    e.table[k].grad = grads[k].data_ptr();
  }
  const int launches = ccf_embedding_bwd(&e, dy.data_ptr(), status.data_ptr<int>(), stream());
  TORCH_CHECK(launches > 0, "ccf_embedding_bwd failed with code ", launches);
  g_launches += launches;
}

// The sum of the lookups; `index`: the ids as the kernels read them.
at::Tensor run_embedding(const at::Tensor& ids, const at::Tensor& weight, const OptTensor& position, const OptTensor& position_ids,
                         const OptTensor& type, const OptTensor& type_ids, double scale, const at::Tensor& status, at::Tensor (&index)[3]) {
  const c10::cuda::CUDAGuard guard(weight.device());
  const at::Tensor tables[3] = {table_of(weight), position.has_value() ? table_of(*position) : at::Tensor(),
                                type.has_value() ? table_of(*type) : at::Tensor()};
  index[0] = ids.contiguous();
  if (position_ids.has_value()) index[1] = position_ids->contiguous();
  if (type_ids.has_value()) index[2] = type_ids->contiguous();
  CcfEmbed e{};
  e.tokens = ids.numel();
  e.seq = ids.dim() > 0 ? ids.size(-1) : 1;
  e.d = static_cast<int>(weight.size(1));
  e.type = type_code(weight);
  for (int k = 0; k < 3; ++k) {
    if (!tables[k].defined()) continue;
    add_table(e, index[k], tables[k].size(0), k == 0 ? scale : 1.0, -1);
    e.table[e.tables - 1].weight = tables[k].data_ptr();
    e.table[e.tables - 1].ld = tables[k].size(0) > 1 ? tables[k].stride(0) : e.d;
  }
  at::DimVector shape(ids.sizes());
  shape.push_back(e.d);
  const at::Tensor y = at::empty(shape, weight.options().requires_grad(false));
  check(ccf_embedding_fwd(&e, y.data_ptr(), status.data_ptr<int>(), stream()), "ccf_embedding_fwd");
  ++g_launches;
  return y;
}

struct EmbeddingFn : torch::autograd::Function<EmbeddingFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& ids, const at::Tensor& weight, const OptTensor& position,
                            const OptTensor& position_ids, const OptTensor& type, const OptTensor& type_ids, double scale, int64_t skip,
                            const at::Tensor& status) {
    at::Tensor index[3];
    const at::Tensor y = run_embedding(ids, weight, position, position_ids, type, type_ids, scale, status, index);
    ctx->save_for_backward({index[0], index[1], index[2]});
    ctx->saved_data["rows"] = std::vector<int64_t>{weight.size(0), position.has_value() ? position->size(0) : 0, type.has_value() ? type->size(0) : 0};
    // autograd counts the tensors that are there: ids, weight, position, its ids, type
    ctx->saved_data["edges"] = std::vector<int64_t>{1, 2, 2 + position.has_value() + position_ids.has_value()};
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["skip"] = skip;
    ctx->saved_data["status"] = status;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    variable_list out(9);
    if (!grads[0].defined()) return out;
    const auto index = ctx->get_saved_variables();
    const auto rows = ctx->saved_data["rows"].toIntVector();
    const c10::cuda::CUDAGuard guard(grads[0].device());
    const at::Tensor dy = packed(grads[0]);
    CcfEmbed e{};
    e.tokens = index[0].numel();
    e.seq = index[0].dim() > 0 ? index[0].size(-1) : 1;
    e.d = static_cast<int>(dy.size(-1));
    e.type = type_code(dy);
    constexpr int kInput[3] = {1, 2, 4};
    const auto edges = ctx->saved_data["edges"].toIntVector();
    std::vector<at::Tensor> dw;
    for (int k = 0; k < 3; ++k) {
      if (rows[k] == 0 || !ctx->needs_input_grad(edges[k])) continue;
      add_table(e, index[k], rows[k], k == 0 ? ctx->saved_data["scale"].toDouble() : 1.0, k == 0 ? ctx->saved_data["skip"].toInt() : -1);
      dw.push_back(at::empty({rows[k], e.d}, dy.options()));
      out[kInput[k]] = dw.back();
    }
    if (e.tables > 0) run_grad(e, dy, dw, ctx->saved_data["status"].toTensor());
    return out;
  }
};

at::Tensor embedding_grad(const at::Tensor& grad, const at::Tensor& ids, int64_t rows, double scale, int64_t skip, const at::Tensor& status) {
  const c10::cuda::CUDAGuard guard(grad.device());
  const at::Tensor dy = packed(grad), index = ids.contiguous();
  CcfEmbed e{};
  e.tokens = index.numel();
  e.seq = 1;
  e.d = static_cast<int>(dy.size(-1));
  e.type = type_code(dy);
  add_table(e, index, rows, scale, skip);
  const at::Tensor dw = at::empty({rows, e.d}, dy.options());
  run_grad(e, dy, {dw}, status);
  return dw;
}

// ---- log probabilities -------------------------------------------------------------------------------------------------
// A call over the logits' rows as the kernels read them.
struct Scored {
  at::Tensor x, targets, logprobs, entropy, top, top_ids, stats;
  int64_t ld;
};
Scored run_logprobs(const at::Tensor& logits, const at::Tensor& targets, int64_t top_k, double temperature, int64_t vocab, int64_t ignore,
                    const at::Tensor& status, bool training) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t width = logits.size(-1), rows = targets.numel();
  Scored r;
  r.x = logits.dim() == 2 ? logits : logits.reshape({rows, width});
  if (r.x.stride(1) != 1 || (rows > 1 && r.x.stride(0) < width)) r.x = r.x.contiguous();
  if (reinterpret_cast<uintptr_t>(r.x.data_ptr()) % 16 != 0) r.x = r.x.clone(at::MemoryFormat::Contiguous);
  r.targets = targets.contiguous();
  r.ld = rows > 1 ? r.x.stride(0) : width;
  const auto f32 = at::TensorOptions(logits.device()).dtype(at::kFloat);
  r.logprobs = at::empty(targets.sizes(), f32);
  r.entropy = at::empty(targets.sizes(), f32);
  CcfLogprobs a{};
  a.x = r.x.data_ptr();
  a.targets = r.targets.data_ptr();
  a.wide = r.targets.scalar_type() == at::kLong;
  a.logprobs = r.logprobs.data_ptr<float>();
  a.entropy = r.entropy.data_ptr<float>();
  a.status = status.data_ptr<int>();
  a.rows = rows;
  a.ld = r.ld;
  a.ignore = ignore;
  a.vocab = static_cast<int>(vocab);
  a.width = static_cast<int>(width);
  a.top_k = static_cast<int>(top_k);
  a.type = type_code(r.x);
  a.inv_t = static_cast<float>(1.0 / temperature);
  if (top_k > 0) {
    at::DimVector wide(targets.sizes());
    wide.push_back(top_k);
    r.top = at::empty(wide, f32);
    r.top_ids = at::empty(wide, f32.dtype(at::kLong));
    a.top_logprobs = r.top.data_ptr<float>();
    a.top_ids = reinterpret_cast<long long*>(r.top_ids.data_ptr<int64_t>());
  }
  if (training) {
    r.stats = at::empty({rows, 3}, f32);
    a.stats = r.stats.data_ptr<float>();
  }
  check(ccf_logprobs_fwd(&a, stream()), "ccf_logprobs_fwd");
  ++g_launches;
  return r;
}

struct LogprobsFn : torch::autograd::Function<LogprobsFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& targets, int64_t top_k, double temperature,
                               int64_t vocab, int64_t ignore, const at::Tensor& status) {
    const Scored r = run_logprobs(logits, targets, top_k, temperature, vocab, ignore, status, true);
    ctx->save_for_backward({r.x, r.targets, r.stats, r.top_ids});
    ctx->saved_data["args"] = std::vector<int64_t>{top_k, vocab, ignore, r.ld};
    ctx->saved_data["inv_t"] = 1.0 / temperature;
    ctx->saved_data["shape"] = logits.sizes();
    ctx->set_materialize_grads(false);
    if (top_k == 0) return {r.logprobs, r.entropy};
    ctx->mark_non_differentiable({r.top_ids});
    return {r.logprobs, r.entropy, r.top, r.top_ids};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    variable_list out(7);
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &t = saved[1], &stats = saved[2];
    const auto args = ctx->saved_data["args"].toIntVector();
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t rows = x.size(0), width = x.size(1), ld = args[3];
    at::Tensor g[3];
    for (int i = 0; i < 3 && i < static_cast<int>(grads.size()); ++i)
      if (grads[i].defined()) g[i] = grads[i].contiguous();
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return out;
    const at::Tensor whole = at::empty({rows, ld}, x.options());   // rows lie as those of the logits do
    CcfLogprobs a{};
    a.x = x.data_ptr();
    a.targets = t.data_ptr();
    a.wide = t.scalar_type() == at::kLong;
    a.stats = stats.data_ptr<float>();
    a.top_ids = args[0] > 0 ? reinterpret_cast<long long*>(saved[3].data_ptr<int64_t>()) : nullptr;
    a.d_logprobs = g[0].defined() ? g[0].data_ptr<float>() : nullptr;
    a.d_entropy = g[1].defined() ? g[1].data_ptr<float>() : nullptr;
    a.d_top = g[2].defined() ? g[2].data_ptr<float>() : nullptr;
    a.dx = whole.data_ptr();
    a.rows = rows;
    a.ld = ld;
    a.top_k = static_cast<int>(args[0]);
    a.vocab = static_cast<int>(args[1]);
    a.ignore = args[2];
    a.width = static_cast<int>(width);
    a.type = type_code(x);
    a.inv_t = static_cast<float>(ctx->saved_data["inv_t"].toDouble());
    check(ccf_logprobs_bwd(&a, stream()), "ccf_logprobs_bwd");
    ++g_launches;
    out[0] = whole.narrow(1, 0, width).view(ctx->saved_data["shape"].toIntVector());
    return out;
  }
};

// ---- dropout -----------------------------------------------------------------------------------------------------------
at::Tensor run_dropout(const at::Tensor& x, const at::Tensor& residual, const long long* state, long long* copy, int64_t call, int64_t drop) {
  const at::Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  check(ccf_dropout(x.data_ptr(), residual.defined() ? residual.data_ptr() : nullptr, y.data_ptr(), state, copy, static_cast<unsigned>(call),
                    static_cast<unsigned>(drop), x.numel(), type_code(x), stream()),
        "ccf_dropout");
  ++g_launches;
  return y;
}

struct DropoutFn : torch::autograd::Function<DropoutFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& residual, const at::Tensor& state, int64_t call, int64_t drop) {
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor used = at::empty({2}, state.options());   // the seed and step of this pass: the state may move on before the backward pass
    const at::Tensor y = run_dropout(packed(x), residual.has_value() ? packed(*residual) : at::Tensor(),
                                     reinterpret_cast<const long long*>(state.data_ptr<int64_t>()),
                                     reinterpret_cast<long long*>(used.data_ptr<int64_t>()), call, drop);
    ctx->save_for_backward({used});
    ctx->saved_data["call"] = call;
    ctx->saved_data["drop"] = drop;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    variable_list out(5);
    const c10::cuda::CUDAGuard guard(grads[0].device());
    if (ctx->needs_input_grad(1)) out[1] = grads[0];
    if (ctx->needs_input_grad(0)) {
      const at::Tensor used = ctx->get_saved_variables()[0];
      out[0] = run_dropout(packed(grads[0]), at::Tensor(), reinterpret_cast<const long long*>(used.data_ptr<int64_t>()), nullptr,
                           ctx->saved_data["call"].toInt(), ctx->saved_data["drop"].toInt());
    }
    return out;
  }
};

// Without a graph to build, the kernels alone: the function around them costs the host about 2 us.
// A forward-mode tangent goes to the function as well, which refuses it.
bool needs_graph(const at::Tensor& t) { return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined(); }

}  // namespace

void ccf_torch::add_token_ops(py::module_& m) {
  m.def(
      "embedding",
      [](const at::Tensor& ids, const at::Tensor& weight, const OptTensor& position, const OptTensor& position_ids, const OptTensor& type,
         const OptTensor& type_ids, double scale, int64_t skip, const at::Tensor& status) {
        if (needs_graph(weight) || (position.has_value() && needs_graph(*position)) || (type.has_value() && needs_graph(*type)))
          return EmbeddingFn::apply(ids, weight, position, position_ids, type, type_ids, scale, skip, status);
        const at::AutoDispatchBelowADInplaceOrView below;
        at::Tensor index[3];
        return run_embedding(ids, weight, position, position_ids, type, type_ids, scale, status, index);
      },
      py::call_guard<py::gil_scoped_release>());
  m.def("embedding_grad", &embedding_grad, py::call_guard<py::gil_scoped_release>());
  m.def(
      "token_logprobs",
      [](const at::Tensor& logits, const at::Tensor& targets, int64_t top_k, double temperature, int64_t vocab, int64_t ignore,
         const at::Tensor& status) -> variable_list {
        if (needs_graph(logits)) return LogprobsFn::apply(logits, targets, top_k, temperature, vocab, ignore, status);
        const at::AutoDispatchBelowADInplaceOrView below;
        const Scored r = run_logprobs(logits, targets, top_k, temperature, vocab, ignore, status, false);
        if (top_k == 0) return {r.logprobs, r.entropy};
        return {r.logprobs, r.entropy, r.top, r.top_ids};
      },
      py::call_guard<py::gil_scoped_release>());
  m.def(
      "dropout",
      [](const at::Tensor& x, const OptTensor& residual, const at::Tensor& state, int64_t call, int64_t drop) {
        if (needs_graph(x) || (residual.has_value() && needs_graph(*residual))) return DropoutFn::apply(x, residual, state, call, drop);
        const c10::cuda::CUDAGuard guard(x.device());
        const at::AutoDispatchBelowADInplaceOrView below;
        return run_dropout(packed(x), residual.has_value() ? packed(*residual) : at::Tensor(),
                           reinterpret_cast<const long long*>(state.data_ptr<int64_t>()), nullptr, call, drop);
      },
      py::call_guard<py::gil_scoped_release>());
}
