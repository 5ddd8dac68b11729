// What the operators' host paths check and how they see a tensor's rows (torch_encoder_ops.cpp, torch_vocab_ops.cpp).
#pragma once
#include "torch_common.h"

namespace {

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
  Tensor t;
  int64_t M = 0, N = 0, ld = 0;
  explicit Rows(const Tensor& x) {
    N = x.size(-1);
    M = N ? x.numel() / N : 0;
    ld = N;
    if (x.is_contiguous()) {
      t = x;
      return;
    }
    t = x.reshape({M, N});               // a view where the strides allow it
    if (N > 1 && t.stride(1) != 1) t = t.contiguous();
    if (M > 1) ld = t.stride(0);
  }
};

void check_rows(const char* op, const Tensor& x, const char* name) {
  check_plain(op, x, name);
  if (!stream_type(x.scalar_type())) refuse(op, std::string(name) + " has type " + c10::toString(x.scalar_type()) + "; fp32, bf16 and fp16 are served");
  if (x.dim() < 1 || x.size(-1) < 1) refuse(op, std::string(name) + " has shape " + shape_of(x) + ": it needs a last dimension of one element or more");
  if (x.size(-1) > 0x7fffffff / 2) refuse(op, std::string(name) + " has rows of " + std::to_string(x.size(-1)) + " elements");
}
struct Below {                           // what happens inside is not recorded
  at::AutoDispatchBelowADInplaceOrView below;
  c10::impl::ExcludeDispatchKeyGuard no_autocast{c10::autocast_dispatch_keyset};
};

}  // namespace
