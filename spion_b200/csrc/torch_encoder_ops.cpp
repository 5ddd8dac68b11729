// Host path of the encoder's operators around the attention call: root-mean-square norm, rows in e4m3, linear layer on them, optimizer.  Each call checks
// what it is given, allocates its results and calls the C ABI; the norm is an autograd node of its own.
#include <algorithm>
#include <mutex>

#include "torch_checks.h"

namespace {

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
// Rows of bytes start on 32, a sector of memory: tensor maps ask for 16, which costs them every box's rows a sector more (65536 x 272 to 256: 20.0 us, 65536 x
// 288: 17.2; 112 and 96 14.7, 11.8).
int64_t row8_stride(int64_t N) { return (N + 31) / 32 * 32; }
// [.., N] of a buffer [M, N rounded up]
Tensor empty_rows8(const Tensor& x, int64_t M, int64_t N) {
  const int64_t ld = row8_stride(N);
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
    const Rows rx(x);
    const Tensor wc = w.contiguous();
    y = made(op, at::empty(x.sizes(), x.options().dtype(type)));
    if (need) rho = at::empty({rx.M}, x.options().dtype(at::kFloat));
    if (res.has_value()) {
      const Rows rr(*res);
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
  const Rows rx(x);
  const Tensor wc = w.contiguous();
  const Rows8 q = empty_result(op, x, rx);
  Tensor s;
  const int64_t ld = row8_stride(rx.N);
  if (res.has_value()) {
    const Rows rr(*res);
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
  const Rows rx(x);
  const Rows8 q = empty_result(op, x, rx);
  check(spion_rmsnorm_forward(p(rx.t), rx.ld, type_code(x.scalar_type()), nullptr, 0, 0, nullptr, 0, nullptr, p(q.values), row8_stride(rx.N), SPION_E4M3,
                              (float*)p(q.scales), nullptr, rx.M, (int)rx.N, 0.f, 0, stream_of(x)), "spion_rmsnorm_forward");
  return q;
}

// ------------------------------------------------------------------------------------------------ linear layer on 8-bit rows
// Rows of bytes as the products read them: on 16-byte boundaries (a copy where they lie otherwise), scales one after another.
struct Operand8 {
  Tensor values, scales;                 // what keeps the memory
  const void* p8 = nullptr;
  const float* ps = nullptr;
  int64_t M = 0, N = 0, ld = 0;
  Operand8(const char* op, const Tensor& v, const Tensor& s, const char* name) {
    check_plain(op, v, name);
    check_plain(op, s, "a tensor of scales");
    if (v.scalar_type() != at::kFloat8_e4m3fn || v.dim() < 1 || v.size(-1) < 1 || v.size(-1) > 0x7fffffff / 2)
      refuse(op, std::string(name) + " has shape " + shape_of(v) + " and type " + c10::toString(v.scalar_type()) + ": rows of e4m3 are needed");
    if (s.scalar_type() != at::kFloat || s.sizes() != v.sizes().slice(0, v.dim() - 1))
      refuse(op, std::string(name) + " has shape " + shape_of(v) + ", its scales have " + shape_of(s) + " and type " + c10::toString(s.scalar_type()) +
             ": an fp32 scale per row is needed");
    same_device(op, s, v, "a tensor of scales");
    const Rows r(v);
    M = r.M; N = r.N;
    values = r.t;
    ld = M > 1 ? r.ld : row8_stride(N);
    if (M > 0 && (((uintptr_t)values.data_ptr() | (uintptr_t)ld) % 16 != 0 || ld < N)) {
      ld = row8_stride(N);
      Tensor copy = empty_rows8(v, M, N);
      copy.copy_(values.view({M, N}));
      values = copy;
    }
    scales = s.contiguous();
    p8 = p(values);
    ps = pf(scales);
  }
  // rows in floating point, quantised here: scales and values in one piece of memory
  Operand8(const char* op, const Tensor& x) {
    check_rows(op, x, "x");
    const Rows r(x);
    M = r.M; N = r.N;
    ld = row8_stride(N);
    const int64_t at = (4 * M + 31) / 32 * 32;
    values = made(op, at::empty({at + M * ld}, x.options().dtype(at::kByte)));
    char* const base = (char*)p(values);
    ps = (const float*)base;
    p8 = base + at;
    check(spion_rmsnorm_forward(p(r.t), r.ld, type_code(x.scalar_type()), nullptr, 0, 0, nullptr, 0, nullptr, base + at, ld, SPION_E4M3, (float*)base, nullptr, M, (int)N,
                                0.f, 0, stream_of(x)), "spion_rmsnorm_forward");
  }
};

// x_scales undefined: x in floating point, its rows are quantised first
Tensor linear_e4m3(const Tensor& x, const Tensor& x_scales, const Tensor& w, const Tensor& w_scales, const optional<Tensor>& bias,
                   const optional<at::ScalarType>& out_type) {
  const char* op = "linear_e4m3";
  check_plain(op, x, "x");
  if (x.dim() < 1) refuse(op, "x has no dimension");
  no_gradient(op, x); no_gradient(op, w); no_gradient(op, w_scales);
  if (x_scales.defined()) no_gradient(op, x_scales);
  const at::ScalarType type = out_type.value_or(x_scales.defined() ? at::kBFloat16 : x.scalar_type());
  if (!stream_type(type)) refuse(op, std::string("an output of type ") + c10::toString(type) + "; fp32, bf16 and fp16 are served");
  if (w.dim() != 2) refuse(op, "the weights have shape " + shape_of(w) + ": [features out, features in] is needed");
  if (w.size(0) < 1 || w.size(0) > 0x7fffffff / 2) refuse(op, "w has shape " + shape_of(w));
  c10::cuda::CUDAGuard guard(x.device());
  Below below;
  const Operand8 b(op, w, w_scales, "w");
  same_device(op, w, x, "w");
  if (x.size(-1) != b.N) refuse(op, "x has rows of " + std::to_string(x.size(-1)) + " features, w of " + std::to_string(b.N));
  if (x.numel() / x.size(-1) > 0x7fffffff / 2) refuse(op, "x has shape " + shape_of(x));
  Tensor bc;
  if (bias.has_value()) {
    no_gradient(op, *bias);
    check_plain(op, *bias, "bias");
    if (bias->dim() != 1 || bias->size(0) != b.M || !stream_type(bias->scalar_type()))
      refuse(op, "bias has shape " + shape_of(*bias) + " and type " + c10::toString(bias->scalar_type()) + ", w has " + shape_of(w));
    same_device(op, *bias, x, "bias");
    bc = bias->contiguous();
  }
  const Operand8 a = x_scales.defined() ? Operand8(op, x, x_scales, "x") : Operand8(op, x);
  auto sizes = x.sizes().vec();
  sizes.back() = b.M;
  Tensor y = made(op, at::empty(sizes, x.options().dtype(type)));
  check(spion_linear_e4m3(a.p8, a.ld, a.ps, b.p8, b.ld, b.ps, p(bc), bc.defined() ? type_code(bc.scalar_type()) : SPION_F32, p(y), b.M, type_code(type), a.M,
                          (int)a.N, (int)b.M, stream_of(x)), "spion_linear_e4m3");
  return y;
}

// ------------------------------------------------------------------------------------------------ AdamW
struct Hyper { double lr, b1, b2, eps, wd, clip; unsigned seed; };

// What one step changes is known to autograd's checks of saved tensors
void changed(const Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void check_flat(const char* op, const Tensor& t, const char* name, at::ScalarType type, int64_t least, const Tensor& like) {
  check_plain(op, t, name);
  same_device(op, t, like, name);
  if (t.scalar_type() != type || !t.is_contiguous() || t.numel() < least)
    refuse(op, std::string(name) + " has shape " + shape_of(t) + " and type " + c10::toString(t.scalar_type()) + ": " + std::to_string(least) +
           " contiguous values of type " + c10::toString(type) + " are needed");
}
bool overlap(std::vector<std::pair<const char*, const char*>>& spans) {      // [begin, end)
  if (!std::is_sorted(spans.begin(), spans.end())) std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) return true;
  return false;
}

// grads: undefined where a tensor has none (it is left alone); copies: empty, or undefined where a tensor has none
void adamw_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const Tensor& m, const Tensor& v, const Tensor& steps, const Tensor& m_scale,
                const Tensor& v_scale, const Tensor& lr_dev, const std::vector<Tensor>& copies, const Hyper& h) {
  const char* op = "adamw_step";
  if (grads.size() != params.size()) refuse(op, std::to_string(params.size()) + " parameters and " + std::to_string(grads.size()) + " gradients");
  if (!copies.empty() && copies.size() != params.size()) refuse(op, std::to_string(params.size()) + " parameters and " + std::to_string(copies.size()) + " copies");
  if (params.empty()) return;
  if (!(h.lr >= 0) && !lr_dev.defined()) refuse(op, "lr is " + std::to_string(h.lr));
  if (!(h.b1 >= 0 && h.b1 < 1 && h.b2 >= 0 && h.b2 < 1)) refuse(op, "betas are " + std::to_string(h.b1) + ", " + std::to_string(h.b2));
  if (!(h.eps >= 0) || !(h.wd >= 0)) refuse(op, "eps is " + std::to_string(h.eps) + ", weight_decay is " + std::to_string(h.wd));
  const at::ScalarType type = params[0].scalar_type();
  const Tensor& like = params[0];
  check_plain(op, like, "a parameter");
  if (!stream_type(type)) refuse(op, std::string("parameters have type ") + c10::toString(type) + "; fp32, bf16 and fp16 are served");
  c10::cuda::CUDAGuard guard(like.device());
  at::NoGradGuard no_grad;
  std::vector<spion_adamw_tensor> table;
  std::vector<Tensor> held;                                // gradients that had to be copied
  std::vector<std::pair<const char*, const char*>> written;
  table.reserve(params.size());
  written.reserve(params.size() + 8);
  int64_t at = 0;
  int copy_type = -1;
  for (size_t i = 0; i < params.size(); ++i) {
    const Tensor& t = params[i];
    check_plain(op, t, "a parameter");
    if (t.scalar_type() != type || t.device() != like.device() || !t.is_contiguous())
      refuse(op, "parameter " + std::to_string(i) + " has type " + c10::toString(t.scalar_type()) + " on " + t.device().str() + " and strides that are " +
             (t.is_contiguous() ? "" : "not ") + "contiguous; all are contiguous, of one type and on one device");
    const int64_t n = t.numel(), begin = at;
    at += (n + 255) / 256 * 256;
    if (!grads[i].defined()) continue;
    Tensor g = grads[i];
    check_plain(op, g, "a gradient");
    if (g.scalar_type() != type || g.device() != t.device() || g.sizes() != t.sizes())
      refuse(op, "gradient " + std::to_string(i) + " has shape " + shape_of(g) + " and type " + c10::toString(g.scalar_type()) + " on " + g.device().str() +
             ", its parameter " + shape_of(t) + ", " + c10::toString(type) + ", " + t.device().str());
    if (!g.is_contiguous()) held.push_back(g = g.contiguous());
    spion_adamw_tensor e = {t.data_ptr(), g.data_ptr(), nullptr, n, begin, (int)i};
    if (!copies.empty() && copies[i].defined()) {
      const Tensor& c = copies[i];
      check_plain(op, c, "a copy");
      if ((c.scalar_type() != at::kBFloat16 && c.scalar_type() != at::kHalf) || !c.is_contiguous() || c.sizes() != t.sizes() || c.device() != t.device())
        refuse(op, "copy " + std::to_string(i) + " has shape " + shape_of(c) + " and type " + c10::toString(c.scalar_type()) +
               ": contiguous, in 16 bits and of its parameter's shape and device is served");
      const int ct = type_code(c.scalar_type());
      if (copy_type >= 0 && ct != copy_type) refuse(op, "copies of two types");
      copy_type = ct;
      e.copy = c.data_ptr();
      if (n) written.push_back({(const char*)e.copy, (const char*)e.copy + 2 * n});
    }
    if (n) written.push_back({(const char*)e.p, (const char*)e.p + n * t.element_size()});
    table.push_back(e);
  }
  const bool bits8 = m_scale.defined();
  if (bits8 != v_scale.defined()) refuse(op, "scales of one of the two moments are missing");
  check_flat(op, m, "exp_avg", bits8 ? at::kFloat8_e4m3fn : at::kFloat, at, like);
  check_flat(op, v, "exp_avg_sq", bits8 ? at::kFloat8_e5m2 : at::kFloat, at, like);
  check_flat(op, steps, "steps", at::kFloat, (int64_t)params.size(), like);
  if (bits8) {
    check_flat(op, m_scale, "the scales of exp_avg", at::kFloat, at / 256, like);
    check_flat(op, v_scale, "the scales of exp_avg_sq", at::kFloat, at / 256, like);
  }
  if (lr_dev.defined()) check_flat(op, lr_dev, "lr", at::kFloat, 1, like);
  if (table.empty()) return;
  for (const Tensor* t : {&m, &v, &steps, &m_scale, &v_scale})
    if (t->defined() && t->numel()) written.push_back({(const char*)t->data_ptr(), (const char*)t->data_ptr() + t->numel() * t->element_size()});
  if (overlap(written)) refuse(op, "two of the tensors that the step writes share memory");
  const Tensor ws = made(op, at::empty({4 * (int64_t)std::min<size_t>(table.size(), 256)}, like.options().dtype(at::kFloat)));
  check(spion_adamw_step(table.data(), (int)table.size(), type_code(type), bits8 ? 8 : 32, p(m), p(v), (float*)p(m_scale), (float*)p(v_scale), (float*)p(steps),
                         pf(lr_dev), h.lr, h.b1, h.b2, h.eps, h.wd, h.clip, h.seed, copy_type, p(ws), stream_of(like)),
        "spion_adamw_step");
  for (const Tensor* t : {&m, &v, &steps, &m_scale, &v_scale}) changed(*t);
  for (size_t i = 0; i < params.size(); ++i)
    if (grads[i].defined()) {
      changed(params[i]);
      if (!copies.empty()) changed(copies[i]);
    }
}

// A sequence of tensors and None, without the cost of a general conversion
std::vector<Tensor> tensors(const py::object& list, const char* name) {
  std::vector<Tensor> out;
  if (list.is_none()) return out;
  py::object fast = py::reinterpret_steal<py::object>(PySequence_Fast(list.ptr(), "a sequence of tensors is needed"));
  if (!fast) throw py::error_already_set();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast.ptr());
  out.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PySequence_Fast_GET_ITEM(fast.ptr(), i);
    if (o == Py_None) out.emplace_back();
    else if (THPVariable_Check(o)) out.push_back(THPVariable_Unpack(o));
    else throw Failure(std::string("adamw_step: ") + name + " " + std::to_string(i) + " is not a tensor");
  }
  return out;
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
  m.def("linear_e4m3", [](const Tensor& x, const optional<Tensor>& x_scales, const Tensor& w, const Tensor& w_scales, const optional<Tensor>& bias,
                          const optional<at::ScalarType>& type) {
    py::gil_scoped_release nogil;
    return linear_e4m3(x, x_scales.value_or(Tensor()), w, w_scales, bias, type);
  });
  m.def("adamw_step", [](const py::object& params, const py::object& grads, const Tensor& exp_avg, const Tensor& exp_avg_sq, const Tensor& steps,
                         const optional<Tensor>& m_scale, const optional<Tensor>& v_scale, const optional<Tensor>& lr_dev, const py::object& copies, double lr,
                         double b1, double b2, double eps, double wd, double clip, uint64_t seed) {
    const auto ps = tensors(params, "parameter"), gs = tensors(grads, "gradient"), cs = tensors(copies, "copy");
    for (const Tensor& t : ps)
      if (!t.defined()) throw Failure("adamw_step: a parameter is None");
    adamw_step(ps, gs, exp_avg, exp_avg_sq, steps, m_scale.value_or(Tensor()), v_scale.value_or(Tensor()), lr_dev.value_or(Tensor()), cs,
               Hyper{lr, b1, b2, eps, wd, clip, (unsigned)seed});
  });
}

}  // namespace spion_torch
