// The autograd functions around embedding.cu, logprobs.cu and dropout.cu, with the checks of their arguments (in Python they took 2 of a small call's 9 us).
// ops/embedding.py, ops/logprobs.py and ops/dropout.py hold both in Python as well, for where this module is missing, a graph is being traced or
// the tensors are not on a GPU.
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>

#include "dropout.h"
#include "embedding.h"
#include "logprobs.h"
#include "torch_nodes.h"

namespace {

using namespace ccf_torch;

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

// The gradients of up to three tables from dy [tokens, d].
void run_grad(CcfEmbed& e, const at::Tensor& dy, const at::Tensor& status) {
  int64_t at[3] = {}, bytes = 0;
  for (int k = 0; k < e.tables; ++k) {
    at[k] = bytes;
    bytes += ccf_embedding_scratch(e.tokens, e.seq, e.table[k].rows, e.d, e.table[k].ids != nullptr);   // a multiple of 16
  }
  at::Tensor scratch;
  if (bytes > 0) {
    scratch = at::empty({bytes}, dy.options().dtype(at::kByte));
    for (int k = 0; k < e.tables; ++k) e.table[k].scratch = static_cast<uint8_t*>(scratch.data_ptr()) + at[k];
  }
  const int launches = ccf_embedding_bwd(&e, dy.data_ptr(), status.data_ptr<int>(), current_stream());
  TORCH_CHECK(launches > 0, "ccf_embedding_bwd failed with code ", launches);
  g_launches += launches;
}

// The sum of the lookups; `index`: the ids as the kernels read them.
at::Tensor run_embedding(const at::Tensor& ids, const at::Tensor& weight, const at::Tensor& position, const at::Tensor& position_ids,
                         const at::Tensor& type, const at::Tensor& type_ids, double scale, const at::Tensor& status, at::Tensor (&index)[3]) {
  const at::Tensor tables[3] = {table_of(weight), position.defined() ? table_of(position) : at::Tensor(),
                                type.defined() ? table_of(type) : at::Tensor()};
  index[0] = ids.contiguous();
  if (position_ids.defined()) index[1] = position_ids.contiguous();
  if (type_ids.defined()) index[2] = type_ids.contiguous();
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
  check(ccf_embedding_fwd(&e, y.data_ptr(), status.data_ptr<int>(), current_stream()), "ccf_embedding_fwd");
  ++g_launches;
  return y;
}

struct EmbeddingNode : TokenNode {
  int64_t rows[3], skip;
  double scale;
  at::Tensor status;
  std::string name() const override { return "CcfEmbeddingBackward"; }
  variable_list gradients(const variable_list& grads) override {
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const at::Tensor index[3] = {kept_contiguous(0), kept_contiguous(1), kept_contiguous(2)};
    const c10::cuda::CUDAGuard guard(grads[0].device());
    const at::Tensor dy = packed(grads[0]);
    CcfEmbed e{};
    e.tokens = index[0].numel();
    e.seq = index[0].dim() > 0 ? index[0].size(-1) : 1;
    e.d = static_cast<int>(dy.size(-1));
    e.type = type_code(dy);
    for (int k = 0; k < 3; ++k) {
      if (rows[k] == 0 || !task_should_compute_output(k)) continue;
      add_table(e, index[k], rows[k], k == 0 ? scale : 1.0, k == 0 ? skip : -1);
      out[k] = at::empty({rows[k], e.d}, dy.options());
      e.table[e.tables - 1].grad = out[k].data_ptr();
    }
    if (e.tables > 0) run_grad(e, dy, status);
    return out;
  }
  variable_list torch_gradients(const variable_list& grads) override {
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const at::Tensor index[3] = {kept(0), kept(1), kept(2)};
    const int64_t tokens = index[0].numel(), seq = index[0].dim() > 0 ? index[0].size(-1) : 1;
    const at::Tensor dy = grads[0].reshape({tokens, grads[0].size(-1)}).to(at::kFloat);
    for (int k = 0; k < 3; ++k) {
      if (rows[k] == 0 || !task_should_compute_output(k)) continue;
      const at::Tensor ids =
          index[k].defined() ? index[k].reshape({tokens}).to(at::kLong) : at::arange(tokens, index[0].options().dtype(at::kLong)).remainder(seq);
      at::Tensor off = ids.lt(0).logical_or(ids.ge(rows[k]));   // adds nothing
      if (k == 0) off = off.logical_or(ids.eq(skip));
      const at::Tensor g = at::embedding_dense_backward(dy.masked_fill(off.unsqueeze(1), 0), ids.masked_fill(off, 0), rows[k], -1, false);
      out[k] = g.mul(k == 0 ? scale : 1.0).to(grads[0].scalar_type());
    }
    return out;
  }
};

void check_index(const char* name, const at::Tensor& ids, const at::Tensor& of) {
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, name, " are int64 or int32, not ", ids.scalar_type());
  TORCH_CHECK_VALUE(ids.device() == of.device(), name, " are on ", ids.device(), ", the tensor beside them on ", of.device());
}
void check_table(const char* name, const at::Tensor& t, const at::Tensor& w) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) > 0 && t.size(1) == w.size(1) && t.scalar_type() == w.scalar_type() && t.device() == w.device(), name, ": [rows, ",
                    w.size(1), "] of ", w.scalar_type(), " on ", w.device(), ", got ", t.sizes(), " of ", t.scalar_type(), " on ", t.device());
}
// what the kernels count in 32 bits
void check_size(const at::Tensor& w) {
  TORCH_CHECK_VALUE(w.size(0) <= 0x7fffffff && w.size(1) <= CCF_EMBED_MAX_D, "a table of at most 2^31 - 1 rows and 2^24 columns, got ", w.sizes());
}
void check_type(const at::Tensor& t) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat,
                   "on a GPU bf16, fp16 or fp32, not ", t.scalar_type());
}
int64_t skipped(const std::optional<int64_t>& padding, int64_t rows) {
  if (!padding.has_value()) return -1;
  TORCH_CHECK_VALUE(-rows <= *padding && *padding < rows, "padding_idx ", *padding, " lies outside the table's ", rows, " rows");
  return *padding < 0 ? *padding + rows : *padding;
}
void check_count(int64_t tokens) { TORCH_CHECK_VALUE(tokens <= CCF_EMBED_MAX_TOKENS, tokens, " tokens: at most 2^26 in one call"); }
// as many as the ids
OptTensor spread(const OptTensor& t, const at::Tensor& ids) {
  return !t.has_value() || t->sizes() == ids.sizes() ? t : OptTensor(t->expand(ids.sizes()));
}

at::Tensor embedding(const at::Tensor& ids, const at::Tensor& weight, const OptTensor& position_, const OptTensor& position_ids_, const OptTensor& type_,
                     const OptTensor& type_ids_, double scale, const std::optional<int64_t>& padding, const at::Tensor& status, bool twice) {
  const at::Tensor &position = or_none(position_), &type = or_none(type_);
  TORCH_CHECK_VALUE(weight.dim() == 2, "weight: [rows, d], got ", weight.sizes());
  check_type(weight);
  check_size(weight);
  check_index("ids", ids, weight);
  check_count(ids.numel());
  const int64_t skip = skipped(padding, weight.size(0));
  if (position.defined()) {
    check_table("position_weight", position, weight);
    check_size(position);
    if (position_ids_.has_value()) check_index("position_ids", *position_ids_, weight);
    const int64_t seq = ids.dim() > 0 ? ids.size(-1) : 1;
    TORCH_CHECK_VALUE(position_ids_.has_value() || seq <= position.size(0), seq, " positions, and ", position.size(0), " rows in position_weight");
  } else {
    TORCH_CHECK_VALUE(!position_ids_.has_value(), "position_ids without position_weight");
  }
  TORCH_CHECK_VALUE(type.defined() == type_ids_.has_value(), "type_weight and type_ids go together");
  if (type.defined()) {
    check_table("type_weight", type, weight);
    check_size(type);
    check_index("type_ids", *type_ids_, weight);
  }
  const OptTensor position_ids = spread(position_ids_, ids), type_ids = spread(type_ids_, ids);
  const c10::cuda::CUDAGuard guard(weight.device());
  at::Tensor index[3], y;
  {
    const at::NoGradGuard no_graph;   // views still share their base's version: a change before the backward pass is noticed
    y = run_embedding(ids, weight, position, or_none(position_ids), type, or_none(type_ids), scale, status, index);
  }
  if (builds_graph(weight, position, type)) {
    const auto node = make_node<EmbeddingNode>(weight, position, type);
    for (const at::Tensor& t : index) node->keep(t);
    node->rows[0] = weight.size(0);
    node->rows[1] = position.defined() ? position.size(0) : 0;
    node->rows[2] = type.defined() ? type.size(0) : 0;
    node->scale = scale;
    node->skip = skip;
    node->status = status;
    node->twice = twice;
    torch::autograd::set_history(y, node);
  }
  return y;
}

at::Tensor embedding_grad(const at::Tensor& grad, const at::Tensor& ids, int64_t rows, double scale, const std::optional<int64_t>& padding,
                          const at::Tensor& status) {
  check_index("ids", ids, grad);
  check_type(grad);
  check_count(ids.numel());
  TORCH_CHECK_VALUE(rows >= 1 && rows <= 0x7fffffff && grad.dim() == ids.dim() + 1 && grad.sizes().slice(0, ids.dim()) == ids.sizes() &&
                        grad.size(-1) <= CCF_EMBED_MAX_D,
                    "grad: ", ids.sizes(), " + [d], 1 to 2^31 - 1 rows and at most 2^24 columns, got ", grad.sizes(), " and ", rows, " rows");
  const int64_t skip = skipped(padding, rows);
  const c10::cuda::CUDAGuard guard(grad.device());
  const at::Tensor dy = packed(grad), index = ids.contiguous();
  CcfEmbed e{};
  e.tokens = index.numel();
  e.seq = 1;
  e.d = static_cast<int>(dy.size(-1));
  e.type = type_code(dy);
  add_table(e, index, rows, scale, skip);
  const at::Tensor dw = at::empty({rows, e.d}, dy.options().requires_grad(false));
  e.table[0].grad = dw.data_ptr();
  run_grad(e, dy, status);
  return dw;
}

// ---- log probabilities -------------------------------------------------------------------------------------------------
// The logits as the kernels read them: rows with any distance, the first on a 16-byte boundary, their elements next to each other.
at::Tensor rows_of(const at::Tensor& logits, int64_t rows, int64_t width) {
  at::Tensor x = logits.dim() == 2 ? logits : logits.reshape({rows, width});
  if (x.stride(1) != 1 || (rows > 1 && x.stride(0) < width)) x = x.contiguous();
  if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0) x = x.clone(at::MemoryFormat::Contiguous);
  return x;
}
int64_t distance_of(const at::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

// A call over the logits' rows.
struct Scored {
  at::Tensor x, targets, logprobs, entropy, top, top_ids, stats;
};
Scored run_logprobs(const at::Tensor& logits, const at::Tensor& targets, int64_t top_k, double temperature, int64_t vocab, int64_t ignore,
                    const at::Tensor& status, bool training) {
  const int64_t width = logits.size(-1), rows = targets.numel();
  Scored r;
  r.x = rows_of(logits, rows, width);
  r.targets = targets.contiguous();
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
  a.ld = distance_of(r.x);
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
  check(ccf_logprobs_fwd(&a, current_stream()), "ccf_logprobs_fwd");
  ++g_launches;
  return r;
}

struct LogprobsNode : TokenNode {
  int64_t top_k, vocab, ignore;
  double inv_t;
  std::vector<int64_t> shape;
  std::string name() const override { return "CcfTokenLogprobsBackward"; }
  variable_list gradients(const variable_list& grads) override {
    variable_list out(1);
    const at::Tensor logits = kept(0), t = kept_contiguous(1), stats = kept_contiguous(2), top_ids = kept_contiguous(3);
    const c10::cuda::CUDAGuard guard(logits.device());
    const int64_t rows = t.numel(), width = shape.back();
    const at::Tensor x = rows_of(logits, rows, width);
    const int64_t ld = distance_of(x);
    at::Tensor g[3];
    bool any = false;
    for (int i = 0; i < static_cast<int>(grads.size()); ++i) {
      if (!grads[i].defined()) continue;
      g[i] = grads[i].contiguous();
      any = true;
    }
    if (!any) return out;
    const int64_t dx_ld = width + (ld - width) % (type_code(x) == 2 ? 4 : 8);   // rows begin where those of the logits do in their 16 bytes
    const at::Tensor whole = at::empty({rows, dx_ld}, x.options());
    CcfLogprobs a{};
    a.x = x.data_ptr();
    a.targets = t.data_ptr();
    a.wide = t.scalar_type() == at::kLong;
    a.stats = stats.data_ptr<float>();
    a.top_ids = top_k > 0 ? reinterpret_cast<long long*>(top_ids.data_ptr<int64_t>()) : nullptr;
    a.d_logprobs = g[0].defined() ? g[0].data_ptr<float>() : nullptr;
    a.d_entropy = g[1].defined() ? g[1].data_ptr<float>() : nullptr;
    a.d_top = g[2].defined() ? g[2].data_ptr<float>() : nullptr;
    a.dx = whole.data_ptr();
    a.rows = rows;
    a.ld = ld;
    a.dx_ld = dx_ld;
    a.top_k = static_cast<int>(top_k);
    a.vocab = static_cast<int>(vocab);
    a.ignore = ignore;
    a.width = static_cast<int>(width);
    a.type = type_code(x);
    a.inv_t = static_cast<float>(inv_t);
    check(ccf_logprobs_bwd(&a, current_stream()), "ccf_logprobs_bwd");
    ++g_launches;
    out[0] = (dx_ld == width ? whole : whole.narrow(1, 0, width)).view(shape);
    return out;
  }
  // of the log probabilities alone
  variable_list torch_gradients(const variable_list& grads) override {
    variable_list out(1);
    TORCH_CHECK(top_k == 0 && !grads[1].defined(), "ccfuser_b200: only the gradient of the log probabilities can be differentiated again");
    if (!grads[0].defined()) return out;
    const at::Tensor logits = kept(0), t = kept(1).reshape({-1}).to(at::kLong);
    const int64_t rows = t.numel(), width = shape.back();
    const at::Tensor z = logits.reshape({rows, width}).narrow(1, 0, vocab).to(at::kFloat).mul(inv_t);
    const at::Tensor none = z.detach().isneginf().all(1, true);
    const at::Tensor p = at::softmax(z.masked_fill(none, 0), 1);
    const at::Tensor off = t.eq(ignore).logical_or(t.lt(0)).logical_or(t.ge(vocab)).logical_or(none.squeeze(1));
    const at::Tensor g = grads[0].reshape({rows}).masked_fill(off, 0).unsqueeze(1);
    const at::Tensor d = p.mul(g.neg()).scatter_add(1, t.masked_fill(off, 0).unsqueeze(1), g).mul(inv_t);
    out[0] = at::constant_pad_nd(d, {0, width - vocab}).to(logits.scalar_type()).reshape(shape);
    return out;
  }
};

variable_list token_logprobs(const at::Tensor& logits, const at::Tensor& targets, int64_t top_k, double temperature,
                             const std::optional<int64_t>& vocab_size, int64_t ignore, const at::Tensor& status, bool twice) {
  TORCH_CHECK_VALUE(logits.dim() >= 1 && targets.sizes() == logits.sizes().slice(0, logits.dim() - 1), "targets: one per row of the logits, ",
                    logits.sizes(), ", got ", targets.sizes());
  check_type(logits);
  check_index("targets", targets, logits);
  const int64_t width = logits.size(-1), vocab = vocab_size.value_or(width);
  TORCH_CHECK_VALUE(1 <= vocab && vocab <= width, "vocab_size: 1 to the ", width, " columns of the logits, got ", vocab);
  const int64_t most = std::min<int64_t>(CCF_LOGPROBS_MAX_TOP, vocab);
  TORCH_CHECK_VALUE(0 <= top_k && top_k <= most, "top_k: 0 to ", most, ", got ", top_k);
  TORCH_CHECK_VALUE(1e-37 <= temperature && temperature <= 1e37, "temperature: a positive number that fp32 holds, got ", temperature);
  TORCH_CHECK_VALUE(width <= (1 << 30) && targets.numel() < (1 << 28), "at most 2^30 columns and 2^28 - 1 rows in one call");
  const c10::cuda::CUDAGuard guard(logits.device());
  const bool training = builds_graph(logits);
  Scored r;
  {
    const at::NoGradGuard no_graph;   // views still share their base's version: a change before the backward pass is noticed
    r = run_logprobs(logits, targets, top_k, temperature, vocab, ignore, status, training);
  }
  if (training) {
    const auto node = make_node<LogprobsNode>(logits);
    for (const at::Tensor& t : {twice ? logits : r.x, r.targets, r.stats, r.top_ids}) node->keep(t);   // r.x has no history
    node->twice = twice;
    node->top_k = top_k;
    node->vocab = vocab;
    node->ignore = ignore;
    node->inv_t = 1.0 / temperature;
    node->shape = logits.sizes().vec();
    torch::autograd::set_history(r.logprobs, node);
    torch::autograd::set_history(r.entropy, node);
    if (top_k > 0) torch::autograd::set_history(r.top, node);
  }
  if (top_k == 0) return {r.logprobs, r.entropy};
  return {r.logprobs, r.entropy, r.top, r.top_ids};
}

// ---- dropout -----------------------------------------------------------------------------------------------------------
at::Tensor run_dropout(const at::Tensor& x, const at::Tensor& residual, const long long* state, long long* copy, int64_t call, int64_t drop) {
  const at::Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  check(ccf_dropout(x.data_ptr(), residual.defined() ? residual.data_ptr() : nullptr, y.data_ptr(), state, copy, static_cast<unsigned>(call),
                    static_cast<unsigned>(drop), x.numel(), type_code(x), current_stream()),
        "ccf_dropout");
  ++g_launches;
  return y;
}

struct DropoutNode : TokenNode {
  int64_t call, drop;
  std::string name() const override { return "CcfDropoutBackward"; }
  variable_list gradients(const variable_list& grads) override {
    variable_list out(2);
    if (!grads[0].defined()) return out;
    const c10::cuda::CUDAGuard guard(grads[0].device());
    out[1] = grads[0];
    if (task_should_compute_output(0)) {
      const at::Tensor used = kept_contiguous(0);
      out[0] = run_dropout(packed(grads[0]), at::Tensor(), reinterpret_cast<const long long*>(used.data_ptr<int64_t>()), nullptr, call, drop);
    }
    return out;
  }
};

at::Tensor dropout(const at::Tensor& x, const OptTensor& residual_, const at::Tensor& state, int64_t call, double p) {
  const at::Tensor& residual = or_none(residual_);
  TORCH_CHECK_VALUE(0.0 <= p && p <= 1.0, "p: 0 to 1, got ", p);
  TORCH_CHECK_VALUE(0 <= call && call <= 0xffffffffll, "call: 0 to 2^32 - 1, got ", call);
  TORCH_CHECK_VALUE(state.scalar_type() == at::kLong && state.dim() == 1 && state.size(0) == 2 && state.device() == x.device() && state.is_contiguous(),
                    "state: two int64 next to each other on ", x.device(), ", got ", state.sizes(), " of ", state.scalar_type(), " on ", state.device());
  check_type(x);
  TORCH_CHECK_VALUE(!residual.defined() || (residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type() && residual.device() == x.device()),
                    "residual: ", x.sizes(), " of ", x.scalar_type(), " on ", x.device(), ", got ", residual.defined() ? residual.sizes() : x.sizes());
  const int64_t drop = std::llrint(p * 65536.0);   // to even, as Python's round
  const c10::cuda::CUDAGuard guard(x.device());
  const bool training = builds_graph(x, residual);
  at::Tensor y, used;
  {
    const at::NoGradGuard no_graph;   // views still share their base's version: a change before the backward pass is noticed
    if (training) used = at::empty({2}, state.options());   // the seed and step of this pass: the state may move on before the backward pass
    y = run_dropout(packed(x), residual.defined() ? packed(residual) : at::Tensor(), reinterpret_cast<const long long*>(state.data_ptr<int64_t>()),
                    training ? reinterpret_cast<long long*>(used.data_ptr<int64_t>()) : nullptr, call, drop);
  }
  if (training) {
    const auto node = make_node<DropoutNode>(x, residual);
    node->keep(used);
    node->call = call;
    node->drop = drop;
    torch::autograd::set_history(y, node);
  }
  return y;
}

}  // namespace

void ccf_torch::add_token_ops(py::module_& m) {
  const auto free = py::call_guard<py::gil_scoped_release>();
  m.def("embedding", &embedding, free);
  m.def("embedding_grad", &embedding_grad, free);
  m.def("token_logprobs", &token_logprobs, free);
  m.def("dropout", &dropout, free);
}
