// Host path of the operators at a model's two ends: rows of a token table with their gradient, and the losses over the vocabulary.  Each call checks what it is
// given, allocates its results and calls the C ABI; each is an autograd node of its own.
#include <mutex>

#include "torch_checks.h"

namespace {

// int64 numbers one after another (int32 is converted)
Tensor whole_numbers(const char* op, const Tensor& t, const char* name) {
  check_plain(op, t, name);
  if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)
    refuse(op, std::string(name) + " has type " + c10::toString(t.scalar_type()) + "; int64 and int32 are served");
  return t.to(at::kLong).contiguous();
}
bool needs_gradient(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
void* p256(const Tensor& t) { return t.data_ptr(); }      // (the allocator's blocks begin on 512 bytes)

// What came back of a tensor that was saved: hooks may hand out another one, laid out otherwise, but its values have to be the same
struct Saved {
  SavedVariable v;
  std::vector<int64_t> sizes;
  at::ScalarType type = at::kFloat;
  c10::Device device = at::kCPU;
  void operator=(const Tensor& t) { v = save(t), sizes = t.sizes().vec(), type = t.scalar_type(), device = t.device(); }
  Tensor unpack(const char* node, const char* name) const {
    const Tensor t = v.unpack();
    if (t.defined() && (t.sizes() != at::IntArrayRef(sizes) || t.scalar_type() != type || t.device() != device || t.layout() != at::kStrided))
      refuse(node, std::string("a hook on saved tensors gave ") + name + " back with shape " + shape_of(t) + " and type " + c10::toString(t.scalar_type()) + " on " +
             t.device().str() + "; it was saved with another");
    return t;
  }
};

// ------------------------------------------------------------------------------------------------ rows of a table
struct TokenRowsNode : public Node {
  Saved ids;
  std::vector<int64_t> table;
  at::ScalarType type = at::kFloat;
  c10::TensorOptions options;
  double scale = 1;
  int64_t padding = -1;
  bool released = false;
  std::string name() const override { return "TokenRowsBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    ids.v.reset_data();
    released = true;
  }
  variable_list apply(variable_list&& grads) override {
    return as_backward([&] { return backward(grads); });
  }
  variable_list backward(const variable_list& grads) {
    std::lock_guard<std::mutex> lock(mutex_);
    TORCH_CHECK(!released, "Trying to backward through the graph a second time (the saved tensors have been freed)");
    variable_list out(1);
    if (!grads[0].defined() || !task_should_compute_output(0)) return out;
    const Tensor i = ids.unpack("TokenRowsBackward", "ids").contiguous();      // (a hook may have spread them out)
    const int64_t V = table[0], N = table[1];
    c10::cuda::CUDAGuard guard(i.device());
    if (recorded()) {                    // by torch operators: the gradient of what arrives is part of a graph
      OutsideAutocast outside;
      const Tensor flat = i.reshape({-1}), none = flat.lt(0).logical_or(flat.ge(V)).logical_or(flat.eq(padding));
      const Tensor g = grads[0].to(at::kFloat).reshape({-1, N}).masked_fill(none.unsqueeze(1), 0.);
      out[0] = at::zeros({V, N}, options.dtype(at::kFloat)).index_add(0, flat.masked_fill(none, 0), g * scale).to(type);
      return out;
    }
    Tensor g = grads[0];
    if (!stream_type(g.scalar_type())) g = g.to(at::kFloat);
    const Rows rows(g);
    const int64_t T = rows.M;
    Tensor dw = at::empty({V, N}, options.dtype(type));
    const Tensor ws = at::empty({std::max<int64_t>(1, spion_token_rows_workspace_bytes(T, V, N))}, options.dtype(at::kByte));
    check(spion_token_rows_backward((const long long*)p(i), p(rows.t), rows.ld, type_code(g.scalar_type()), p(dw), type_code(type), (float)scale, padding, T, V, N,
                                    p256(ws), stream_of(i)), "spion_token_rows_backward");
    out[0] = dw;
    return out;
  }
};

Tensor token_rows(const Tensor& ids, const Tensor& w, double scale, const optional<int64_t>& padding, const optional<at::ScalarType>& out_type) {
  const char* op = "embed_tokens";
  check_plain(op, w, "weight");
  if (w.dim() != 2 || w.size(1) < 1 || !stream_type(w.scalar_type()))
    refuse(op, "weight has shape " + shape_of(w) + " and type " + c10::toString(w.scalar_type()) + ": a table [rows, features] in fp32, bf16 or fp16 is needed");
  const int64_t V = w.size(0), N = w.size(1);
  const at::ScalarType type = out_type.value_or(w.scalar_type());
  if (!stream_type(type)) refuse(op, std::string("an output of type ") + c10::toString(type) + "; fp32, bf16 and fp16 are served");
  int64_t pad = -1;
  if (padding.has_value()) {
    if (*padding < -V || *padding >= V) refuse(op, "padding_idx is " + std::to_string(*padding) + ", the table has " + std::to_string(V) + " rows");
    pad = *padding < 0 ? *padding + V : *padding;
  }
  c10::cuda::CUDAGuard guard(w.device());
  const bool need = needs_gradient({w});
  Tensor i, y;
  {
    Below below;
    i = whole_numbers(op, ids, "ids");
    same_device(op, i, w, "ids");
    if (i.numel() > 0x7fffffff - 4096) refuse(op, std::to_string(i.numel()) + " ids");
    if (V > 0x7fffffff - 4096) refuse(op, "weight has shape " + shape_of(w));
    Rows rows(w);
    if (V > 1 && rows.ld < N) rows = Rows(w.contiguous());
    auto sizes = ids.sizes().vec();
    sizes.push_back(N);
    y = made(op, at::empty(sizes, w.options().dtype(type)));
    check(spion_token_rows_forward((const long long*)p(i), p(rows.t), std::max(rows.ld, N), type_code(w.scalar_type()), p(y), type_code(type), (float)scale, i.numel(), V, N,
                                   stream_of(w)), "spion_token_rows_forward");
  }
  if (need) {
    auto node = std::shared_ptr<TokenRowsNode>(new TokenRowsNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(w));
    node->table = {V, N};
    node->type = w.scalar_type();
    node->options = w.options().requires_grad(false);
    node->scale = scale;
    node->padding = pad;
    torch::autograd::set_history(y, node);
    node->ids = i;
  }
  return y;
}

// ------------------------------------------------------------------------------------------------ losses
struct Problem {
  Tensor x, w, bias, labels, teacher;    // teacher undefined: labels
  int64_t ignore = -100;
  int reduction = 1;
  double tau = 1;
  int layout = 0;                        // how the forward read its operands
};
// The operands as the kernels read them, and what keeps their memory
struct Operands {
  Rows x, w;
  Tensor bias, teacher;
  spion_vocab_problem c;
  explicit Operands(const Problem& a) : x(a.x), w(a.w) {
    if (w.M > 1 && w.ld < w.N) w = Rows(a.w.contiguous());
    if (a.bias.defined()) bias = a.bias.contiguous();
    if (a.teacher.defined()) teacher = a.teacher.contiguous();
    c = {};
    c.x = p(x.t), c.w = p(w.t), c.bias = p(bias), c.teacher = p(teacher), c.labels = (const long long*)p(a.labels);
    c.ldx = x.ld, c.ldw = std::max(w.ld, w.N), c.T = x.M, c.K = x.N, c.V = w.M;
    c.k = teacher.defined() ? teacher.size(-1) : 1;
    c.ignore_index = a.ignore;
    c.type = type_code(a.x.scalar_type());
    c.bias_type = bias.defined() ? type_code(bias.scalar_type()) : SPION_F32;
    c.teacher_type = teacher.defined() ? type_code(teacher.scalar_type()) : SPION_F32;
    c.reduction = a.reduction;
    c.temperature = (float)a.tau;
    c.layout = a.layout;
  }
};

struct VocabLossNode : public Node {
  Saved x, w, bias, labels, teacher;
  Tensor keep;
  Problem rest;                          // without its tensors
  bool released = false;
  std::string name() const override { return "VocabLossBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (Saved* s : {&x, &w, &bias, &labels, &teacher}) s->v.reset_data();
    keep.reset();
    released = true;
  }
  variable_list apply(variable_list&& grads) override {
    return as_backward([&] { return backward(grads); });
  }
  // inputs: x, w[, bias]
  variable_list backward(const variable_list& grads) {
    std::lock_guard<std::mutex> lock(mutex_);
    TORCH_CHECK(!released, "Trying to backward through the graph a second time (the saved tensors have been freed)");
    variable_list out(num_outputs());
    const bool want_x = task_should_compute_output(0), want_w = task_should_compute_output(1), want_b = num_outputs() > 2 && task_should_compute_output(2);
    if (!grads[0].defined() || !(want_x || want_w || want_b)) return out;
    Problem a = rest;
    const char* me = "VocabLossBackward";
    a.x = x.unpack(me, "x"), a.w = w.unpack(me, "weight"), a.bias = bias.unpack(me, "bias"), a.labels = labels.unpack(me, "labels"), a.teacher = teacher.unpack(me, "teacher_logits");
    c10::cuda::CUDAGuard guard(a.x.device());
    if (recorded()) return by_operators(a, grads[0], want_x, want_w, want_b);
    if (a.x.numel() == 0) {
      if (want_x) out[0] = at::zeros_like(a.x);
      if (want_w) out[1] = at::zeros_like(a.w);
      if (want_b) out[2] = at::zeros_like(a.bias);
      return out;
    }
    const Operands o(a);
    const Tensor g = grads[0].to(at::kFloat).contiguous();
    if (want_x) out[0] = at::empty(a.x.sizes(), a.x.options().requires_grad(false));
    if (want_w) out[1] = at::empty(a.w.sizes(), a.w.options().requires_grad(false));
    if (want_b) out[2] = at::empty(a.bias.sizes(), a.bias.options().requires_grad(false));
    long long bytes = 0;
    check(spion_vocab_sizes(&o.c, nullptr, nullptr, &bytes), "spion_vocab_sizes");
    const Tensor ws = at::empty({(int64_t)bytes}, a.x.options().dtype(at::kByte).requires_grad(false));
    check(spion_vocab_loss_backward(&o.c, pf(g), p(keep), want_x ? p(out[0]) : nullptr, want_w ? p(out[1]) : nullptr, want_b ? p(out[2]) : nullptr,
                                    want_b ? type_code(a.bias.scalar_type()) : SPION_F32, p256(ws), stream_of(a.x)), "spion_vocab_loss_backward");
    return out;
  }
  // From tensors that are part of a graph (create_graph), with the logits in memory
  variable_list by_operators(const Problem& a, const Tensor& given, bool want_x, bool want_w, bool want_b) {
    OutsideAutocast outside;
    variable_list out(num_outputs());
    const int64_t K = a.x.size(-1), V = a.w.size(0), k = a.teacher.defined() ? a.teacher.size(-1) : 1;
    const Tensor X = a.x.to(at::kFloat).reshape({-1, K}), W = a.w.to(at::kFloat);
    const Tensor idx = a.labels.reshape({-1, k});
    Tensor there, q;
    if (a.teacher.defined()) {
      const Tensor t = a.teacher.to(at::kFloat).reshape({-1, k});
      there = idx.ne(-1).logical_and(t.ne(-INFINITY));
      const Tensor left = t.masked_fill(there.logical_not(), -INFINITY);
      q = at::softmax((left - left.amax(1, true)) / a.tau, 1).masked_fill(there.logical_not(), 0.);
    } else {
      there = idx.ne(a.ignore);
      q = there.to(at::kFloat);
    }
    const Tensor counts = there.any(1, true), rows = X.masked_fill(counts.logical_not(), 0.);
    const Tensor bad = there.logical_and(idx.lt(0).logical_or(idx.ge(V))).any(1, true);
    Tensor z = at::matmul(rows, W.t());
    if (a.bias.defined()) z = z + a.bias.to(at::kFloat);
    Tensor G = at::softmax(z / a.tau, 1).scatter_add(1, idx.clamp(0, V - 1), q.neg());
    Tensor c = given.to(at::kFloat);
    c = a.reduction == 0 ? c.reshape({-1, 1}) : a.reduction == 1 ? c / counts.sum().clamp_min(1) : c;
    G = (G * (c / a.tau)).masked_fill(counts.logical_not(), 0.).masked_fill(bad, NAN);
    if (want_x) out[0] = at::matmul(G, W).masked_fill(counts.logical_not(), 0.).to(a.x.scalar_type()).reshape(a.x.sizes());
    if (want_w) out[1] = at::matmul(G.t(), rows).to(a.w.scalar_type());
    if (want_b) out[2] = G.sum(0).to(a.bias.scalar_type());
    return out;
  }
};

void no_gradient(const char* op, const Tensor& t, const char* name) {
  if (at::GradMode::is_enabled() && t.requires_grad()) refuse(op, std::string(name) + " requires a gradient, which this loss has not: detach it");
}

Tensor vocab_loss(const char* op, const Tensor& x, const Tensor& w, const Tensor& labels, const optional<Tensor>& teacher, const optional<Tensor>& bias, int64_t ignore,
                  int reduction, double tau) {
  check_rows(op, x, "x");
  check_plain(op, w, "weight");
  if (w.dim() != 2 || w.size(0) < 1 || w.size(1) != x.size(-1) || w.scalar_type() != x.scalar_type())
    refuse(op, "weight has shape " + shape_of(w) + " and type " + c10::toString(w.scalar_type()) + ", x has " + shape_of(x) + " and " + c10::toString(x.scalar_type()) +
           ": [vocabulary, features] of x's type is needed");
  same_device(op, w, x, "weight");
  if (!(tau > 0) || !std::isfinite(tau)) refuse(op, "the temperature is " + std::to_string(tau));
  auto shape = x.sizes().vec();
  shape.pop_back();
  if (teacher.has_value()) {
    check_plain(op, *teacher, "teacher_logits");
    same_device(op, *teacher, x, "teacher_logits");
    no_gradient(op, *teacher, "teacher_logits");
    if (!stream_type(teacher->scalar_type()) || teacher->dim() != x.dim() || teacher->sizes().slice(0, shape.size()) != at::IntArrayRef(shape) || teacher->size(-1) < 1 ||
        teacher->size(-1) > 128)
      refuse(op, "teacher_logits has shape " + shape_of(*teacher) + " and type " + c10::toString(teacher->scalar_type()) + ", x has " + shape_of(x) +
             ": 1 to 128 fp32, bf16 or fp16 logits a row are needed");
    if (labels.sizes() != teacher->sizes()) refuse(op, "indices has shape " + shape_of(labels) + ", teacher_logits has " + shape_of(*teacher));
  } else if (labels.sizes() != at::IntArrayRef(shape)) {
    refuse(op, "labels has shape " + shape_of(labels) + ", x has " + shape_of(x));
  }
  if (bias.has_value()) {
    check_plain(op, *bias, "bias");
    if (bias->dim() != 1 || bias->size(0) != w.size(0) || !stream_type(bias->scalar_type()))
      refuse(op, "bias has shape " + shape_of(*bias) + " and type " + c10::toString(bias->scalar_type()) + ", weight has " + shape_of(w));
    same_device(op, *bias, x, "bias");
  }
  c10::cuda::CUDAGuard guard(x.device());
  const bool need = needs_gradient({x, w, bias.value_or(Tensor())});
  Problem a;
  a.x = x, a.w = w, a.bias = bias.value_or(Tensor()), a.teacher = teacher.value_or(Tensor());
  a.ignore = ignore, a.reduction = reduction, a.tau = tau;
  Tensor loss, keep;
  {
    Below below;
    a.labels = whole_numbers(op, labels, teacher.has_value() ? "indices" : "labels");
    same_device(op, a.labels, x, teacher.has_value() ? "indices" : "labels");
    loss = made(op, reduction == 0 ? at::empty(shape, x.options().dtype(at::kFloat)) : at::empty({}, x.options().dtype(at::kFloat)));
    if (x.numel() == 0) {
      if (reduction > 0) loss.fill_(reduction == 1 ? NAN : 0.);
    } else {
      const Operands o(a);
      long long keeps = 0, bytes = 0;
      const int rc = spion_vocab_sizes(&o.c, &keeps, &bytes, nullptr);
      if (rc == SPION_ERR_SHAPE) refuse(op, "x has shape " + shape_of(x) + ", weight " + shape_of(w) + ": too large");
      check(rc, "spion_vocab_sizes");
      a.layout = spion_vocab_layout(&o.c);
      check(std::min(a.layout, 0), "spion_vocab_layout");
      keep = at::empty({(int64_t)keeps}, x.options().dtype(at::kByte));
      const Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
      check(spion_vocab_loss_forward(&o.c, (float*)p(loss), p256(keep), p256(ws), stream_of(x)), "spion_vocab_loss_forward");
    }
  }
  if (need) {
    auto node = std::shared_ptr<VocabLossNode>(new VocabLossNode(), torch::autograd::deleteNode);
    node->set_next_edges(bias.has_value() ? torch::autograd::collect_next_edges(x, w, *bias) : torch::autograd::collect_next_edges(x, w));
    torch::autograd::set_history(loss, node);
    node->rest.ignore = ignore, node->rest.reduction = reduction, node->rest.tau = tau, node->rest.layout = a.layout;
    node->keep = keep;
    node->x = x, node->w = w, node->labels = a.labels;
    if (bias.has_value()) node->bias = *bias;
    if (teacher.has_value()) node->teacher = *teacher;
  }
  return loss;
}

int reduction_of(const char* op, const std::string& name) {
  if (name == "none") return 0;
  if (name == "mean") return 1;
  if (name == "sum") return 2;
  refuse(op, "reduction is '" + name + "': 'mean', 'sum' and 'none' are served");
}

}  // namespace

namespace spion_torch {

void add_vocab_ops(py::module_& m) {
  m.def("token_rows", [](const Tensor& ids, const Tensor& w, double scale, const optional<int64_t>& padding, const optional<at::ScalarType>& type) {
    py::gil_scoped_release nogil;
    return token_rows(ids, w, scale, padding, type);
  });
  m.def("linear_cross_entropy", [](const Tensor& x, const Tensor& w, const Tensor& labels, const optional<Tensor>& bias, int64_t ignore, const std::string& reduction) {
    py::gil_scoped_release nogil;
    return vocab_loss("linear_cross_entropy", x, w, labels, {}, bias, ignore, reduction_of("linear_cross_entropy", reduction), 1.0);
  });
  m.def("distill_top_logits", [](const Tensor& x, const Tensor& w, const Tensor& indices, const Tensor& teacher, const optional<Tensor>& bias, double tau,
                                 const std::string& reduction) {
    py::gil_scoped_release nogil;
    return vocab_loss("distill_top_logits", x, w, indices, teacher, bias, 0, reduction_of("distill_top_logits", reduction), tau);
  });
}

}  // namespace spion_torch
