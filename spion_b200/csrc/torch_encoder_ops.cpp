// Host path of the encoder's operators around the attention call: root-mean-square norm, rows in e4m3.  Each call checks what it is given, allocates
// its results and calls the C ABI; the norm is an autograd node of its own.
#include <cmath>
#include <mutex>

#include "torch_common.h"

namespace {

// ------------------------------------------------------------------------------------------------ checks
[[noreturn]] void refuse(const char* op, const std::string& why) { throw Failure(std::string(op) + ": " + why); }
std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SPION_F32;
    case at::kBFloat16: return SPION_BF16;
    case at::kHalf: return SPION_F16;
    case at::kFloat8_e4m3fn: return SPION_E4M3;
    default: return -1;
  }
}
bool stream_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }

// The kernels work on memory that tracers, function transforms and forward-mode tangents would not see.
void check_plain(const char* op, const Tensor& t, const char* name) {
  if (!t.is_cuda()) refuse(op, std::string(name) + " is not a CUDA tensor (there is no CPU path)");
  if (t.layout() != at::kStrided || torch::jit::tracer::isTracing() || !plain(t))
    refuse(op, std::string(name) + " is not an ordinary tensor of an ordinary call (tracing, function transforms, forward-mode tangents, tensor subclasses "
           "and sparse layouts are not served)");
}
// ... nor do dispatch modes that hand out tensors without memory
Tensor made(const char* op, Tensor t) {
  if (!plain(t)) refuse(op, "a dispatch mode without real tensors is active");
  return t;
}
void same_device(const char* op, const Tensor& t, const Tensor& like, const char* name) {
  if (t.device() != like.device()) refuse(op, std::string(name) + " is on " + t.device().str() + ", the rows are on " + like.device().str());
}

// A tensor's rows over its last dimension as the kernels read them: rows a constant step apart, elements next to one another.
struct Rows {
  Tensor t;                              // [M, N]
  int64_t M = 0, N = 0, ld = 0;
  explicit Rows(const Tensor& x) {
    N = x.size(-1);
    M = N ? x.numel() / N : 0;
    t = x.reshape({M, N});               // a view where the strides allow it
    if (N > 1 && t.stride(1) != 1) t = t.contiguous();
    ld = M > 1 ? t.stride(0) : N;
  }
};

void check_rows(const char* op, const Tensor& x, const char* name) {
  check_plain(op, x, name);
  if (!stream_type(x.scalar_type())) refuse(op, std::string(name) + " has type " + c10::toString(x.scalar_type()) + "; fp32, bf16 and fp16 are served");
  if (x.dim() < 1 || x.size(-1) < 1) refuse(op, std::string(name) + " has shape " + shape_of(x) + ": it needs a last dimension of one element or more");
  if (x.size(-1) > 0x7fffffff / 2) refuse(op, std::string(name) + " has rows of " + std::to_string(x.size(-1)) + " elements");
}
void check_norm(const char* op, const Tensor& x, const Tensor& w, const optional<Tensor>& res) {
  check_rows(op, x, "x");
  check_plain(op, w, "weight");
  if (w.dim() != 1 || w.size(0) != x.size(-1) || !stream_type(w.scalar_type()))
    refuse(op, "weight has shape " + shape_of(w) + " and type " + c10::toString(w.scalar_type()) + ", rows have " + std::to_string(x.size(-1)) + " elements");
  same_device(op, w, x, "weight");
  if (!res.has_value()) return;
  check_rows(op, *res, "res");
  same_device(op, *res, x, "res");
  if (res->sizes() != x.sizes()) refuse(op, "res has shape " + shape_of(*res) + ", x has " + shape_of(x));
  if (res->scalar_type() != x.scalar_type() && x.scalar_type() != at::kFloat)
    refuse(op, std::string("res has type ") + c10::toString(res->scalar_type()) + " beside a stream of " + c10::toString(x.scalar_type()) +
           ": it has the stream's type, or 16 bits beside fp32");
}
struct Below {                           // what happens inside is not recorded
  at::AutoDispatchBelowADInplaceOrView below;
  c10::impl::ExcludeDispatchKeyGuard no_autocast{c10::autocast_dispatch_keyset};
};
// Rows of bytes that start on 16: [.., N] of a buffer [M, N rounded up]
Tensor empty_rows8(const Tensor& x, int64_t M, int64_t N) {
  const int64_t ld = (N + 15) / 16 * 16;
  Tensor t = at::empty({M, ld}, x.options().dtype(at::kFloat8_e4m3fn));
  return ld == N ? t : t.narrow(1, 0, N);
}

// ------------------------------------------------------------------------------------------------ root-mean-square norm
struct RmsNode : public Node {
  SavedVariable s, w, rho;               // s: the sum (the node's own first output), or x
  bool added = false, released = false;
  double eps = 0;
  at::ScalarType x_type, r_type, y_type;
  std::string name() const override { return "RootMeanSquareNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    s.reset_data(); w.reset_data(); rho.reset_data();
    released = true;
  }
  variable_list apply(variable_list&& grads) override {
    return as_backward([&] { return backward(grads); });
  }
  // inputs: x, weight[, res]; outputs: [sum,] y
  variable_list backward(const variable_list& grads) {
    std::lock_guard<std::mutex> lock(mutex_);
    TORCH_CHECK(!released, "Trying to backward through the graph a second time (the saved tensors have been freed)");
    variable_list out(added ? 3 : 2);
    const Tensor& ds = added ? grads[0] : Tensor();
    const Tensor& dy = grads[added ? 1 : 0];
    if (!dy.defined()) {                 // the normalised rows were not used
      if (!ds.defined()) return out;
      if (task_should_compute_output(0)) out[0] = ds.to(x_type);
      if (task_should_compute_output(2)) out[2] = ds.to(r_type);
      return out;
    }
    const Tensor S = s.unpack(added ? shared_from_this() : nullptr), W = w.unpack();
    const bool want_x = task_should_compute_output(0) || (added && task_should_compute_output(2)), want_w = task_should_compute_output(1);
    c10::cuda::CUDAGuard guard(S.device());
    if (recorded()) {                    // by torch operators, from tensors that are part of the graph
      OutsideAutocast outside;
      const Tensor t = S.to(at::kFloat), n = t * at::rsqrt((t * t).mean(-1, true) + eps), g = dy.to(at::kFloat) * W.to(at::kFloat);
      if (want_x) {
        Tensor dx = (g - n * (g * n).mean(-1, true)) * at::rsqrt((t * t).mean(-1, true) + eps);
        if (ds.defined()) dx = dx + ds.to(at::kFloat);
        if (task_should_compute_output(0)) out[0] = dx.to(x_type);
        if (added && task_should_compute_output(2)) out[2] = dx.to(r_type);
      }
      if (want_w) out[1] = (dy.to(at::kFloat) * n).reshape({-1, W.size(0)}).sum(0).to(W.scalar_type());
      return out;
    }
    const Rows rows(S);
    const Tensor d = dy.to(y_type).contiguous(), k = ds.defined() ? ds.to(x_type).contiguous() : Tensor(), r = rho.unpack();
    const Tensor wc = W.contiguous();
    Tensor dx, dr, dw, ws;
    const bool two = added && r_type != x_type;
    const bool want_dx = task_should_compute_output(0) || (added && !two && task_should_compute_output(2));
    if (want_dx) dx = at::empty(S.sizes(), d.options().dtype(x_type));
    if (two && task_should_compute_output(2)) dr = at::empty(S.sizes(), d.options().dtype(r_type));
    if (want_w) {
      dw = at::empty(W.sizes(), wc.options());
      ws = at::empty({(int64_t)spion_rmsnorm_workspace_floats(rows.M, (int)rows.N)}, d.options().dtype(at::kFloat));
    }
    check(spion_rmsnorm_backward(p(rows.t), rows.ld, type_code(x_type), p(d), type_code(y_type), p(k), p(wc), type_code(wc.scalar_type()), pf(r), p(dx), p(dr),
                                 two ? type_code(r_type) : SPION_F32, p(dw), (float*)p(ws), rows.M, (int)rows.N, stream_of(S)), "spion_rmsnorm_backward");
    if (task_should_compute_output(0)) out[0] = dx;
    if (added && task_should_compute_output(2)) out[2] = two ? dr : dx;
    out[1] = dw;
    return out;
  }
};

// -> (sum or undefined, y)
std::pair<Tensor, Tensor> rms_norm(const Tensor& x, const Tensor& w, double eps, const optional<Tensor>& res, const optional<at::ScalarType>& out_type) {
  const char* op = "rms_norm";
  check_norm(op, x, w, res);
  const at::ScalarType type = out_type.value_or(x.scalar_type());
  if (!stream_type(type) || (type != x.scalar_type() && x.scalar_type() != at::kFloat))
    refuse(op, std::string("an output of type ") + c10::toString(type) + " from a stream of " + c10::toString(x.scalar_type()) +
           ": it has the stream's type, or 16 bits beside fp32");
  c10::cuda::CUDAGuard guard(x.device());
  const bool need = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (res.has_value() && res->requires_grad()));
  Tensor s, y, rho;
  {
    Below below;
    const Rows rx(x.detach());
    const Tensor wc = w.detach().contiguous();
    y = made(op, at::empty(x.sizes(), x.options().dtype(type)));
    if (need) rho = at::empty({rx.M}, x.options().dtype(at::kFloat));
    if (res.has_value()) {
      const Rows rr(res->detach());
      s = at::empty(x.sizes(), x.options());
      check(spion_rmsnorm_forward(p(rx.t), rx.ld, type_code(x.scalar_type()), p(rr.t), rr.ld, type_code(res->scalar_type()), p(wc), type_code(wc.scalar_type()),
                                  p(s), p(y), rx.N, type_code(type), nullptr, (float*)p(rho), rx.M, (int)rx.N, (float)eps, 1, stream_of(x)),
            "spion_rmsnorm_forward");
    } else {
      check(spion_rmsnorm_forward(p(rx.t), rx.ld, type_code(x.scalar_type()), nullptr, 0, 0, p(wc), type_code(wc.scalar_type()), nullptr, p(y), rx.N,
                                  type_code(type), nullptr, (float*)p(rho), rx.M, (int)rx.N, (float)eps, 1, stream_of(x)), "spion_rmsnorm_forward");
    }
  }
  if (need) {
    auto node = std::shared_ptr<RmsNode>(new RmsNode(), torch::autograd::deleteNode);
    node->set_next_edges(res.has_value() ? torch::autograd::collect_next_edges(x, w, *res) : torch::autograd::collect_next_edges(x, w));
    node->added = res.has_value();
    node->eps = eps;
    node->x_type = x.scalar_type(); node->y_type = type;
    node->r_type = res.has_value() ? res->scalar_type() : type;
    if (s.defined()) torch::autograd::set_history(s, node);
    torch::autograd::set_history(y, node);
    node->s = s.defined() ? SavedVariable(s, true) : save(x);
    node->w = save(w);
    node->rho = save(rho);
  }
  return {s, y};
}

void no_gradient(const char* op, const Tensor& t) {
  if (at::GradMode::is_enabled() && t.requires_grad()) refuse(op, "8-bit rows have no gradient: call it under torch.no_grad() or with detached tensors");
}

struct Rows8 { Tensor values, scales; };
Rows8 empty_result(const char* op, const Tensor& x, const Rows& r) {
  auto sizes = x.sizes().vec();
  Tensor values = made(op, empty_rows8(x, r.M, r.N));
  if (x.dim() != 2) values = x.numel() ? values.view(sizes) : at::empty(sizes, values.options());
  sizes.pop_back();
  return {values, at::empty(sizes, x.options().dtype(at::kFloat))};
}

// -> (sum or undefined, values, scales)
std::tuple<Tensor, Tensor, Tensor> rms_norm_e4m3(const Tensor& x, const Tensor& w, double eps, const optional<Tensor>& res) {
  const char* op = "rms_norm_e4m3";
  check_norm(op, x, w, res);
  no_gradient(op, x); no_gradient(op, w);
  if (res.has_value()) no_gradient(op, *res);
  c10::cuda::CUDAGuard guard(x.device());
  Below below;
  const Rows rx(x.detach());
  const Tensor wc = w.detach().contiguous();
  const Rows8 q = empty_result(op, x, rx);
  Tensor s;
  const int64_t ld = (rx.N + 15) / 16 * 16;
  if (res.has_value()) {
    const Rows rr(res->detach());
    s = at::empty(x.sizes(), x.options());
    check(spion_rmsnorm_forward(p(rx.t), rx.ld, type_code(x.scalar_type()), p(rr.t), rr.ld, type_code(res->scalar_type()), p(wc), type_code(wc.scalar_type()), p(s),
                                p(q.values), ld, SPION_E4M3, (float*)p(q.scales), nullptr, rx.M, (int)rx.N, (float)eps, 1, stream_of(x)),
          "spion_rmsnorm_forward");
  } else {
    check(spion_rmsnorm_forward(p(rx.t), rx.ld, type_code(x.scalar_type()), nullptr, 0, 0, p(wc), type_code(wc.scalar_type()), nullptr, p(q.values), ld,
                                SPION_E4M3, (float*)p(q.scales), nullptr, rx.M, (int)rx.N, (float)eps, 1, stream_of(x)), "spion_rmsnorm_forward");
  }
  return {s, q.values, q.scales};
}

Rows8 quantize_rows(const Tensor& x) {
  const char* op = "quantize_rows";
  check_rows(op, x, "x");
  no_gradient(op, x);
  c10::cuda::CUDAGuard guard(x.device());
  Below below;
  const Rows rx(x.detach());
  const Rows8 q = empty_result(op, x, rx);
  check(spion_rmsnorm_forward(p(rx.t), rx.ld, type_code(x.scalar_type()), nullptr, 0, 0, nullptr, 0, nullptr, p(q.values), (rx.N + 15) / 16 * 16, SPION_E4M3,
                              (float*)p(q.scales), nullptr, rx.M, (int)rx.N, 0.f, 0, stream_of(x)), "spion_rmsnorm_forward");
  return q;
}

py::object or_none(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }

}  // namespace

namespace spion_torch {

void add_encoder_ops(py::module_& m) {
  m.def("rms_norm", [](const Tensor& x, const Tensor& w, double eps, const optional<Tensor>& res, const optional<at::ScalarType>& type) {
    std::pair<Tensor, Tensor> r;
    {
      py::gil_scoped_release nogil;
      r = rms_norm(x, w, eps, res, type);
    }
    return py::make_tuple(or_none(r.first), r.second);
  });
  m.def("rms_norm_e4m3", [](const Tensor& x, const Tensor& w, double eps, const optional<Tensor>& res) {
    std::tuple<Tensor, Tensor, Tensor> r;
    {
      py::gil_scoped_release nogil;
      r = rms_norm_e4m3(x, w, eps, res);
    }
    return py::make_tuple(or_none(std::get<0>(r)), std::get<1>(r), std::get<2>(r));
  });
  m.def("quantize_rows", [](const Tensor& x) {
    Rows8 r;
    {
      py::gil_scoped_release nogil;
      r = quantize_rows(x);
    }
    return py::make_tuple(r.values, r.scales);
  });
}

}  // namespace spion_torch
