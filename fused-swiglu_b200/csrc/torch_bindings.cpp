// Operator boundary: the same Python module (`fused_mlp_module`) and dispatcher library
// (`ASMLLM`) as the reference's csrc/torch_bindings.cpp:27-50, with the same two ops
//
//   fused_swiglu_bf16(Tensor X, Tensor W1W3) -> Tensor
//   swiglu_fwd_bf16(int m, int n, int k, Tensor A, int ldA, Tensor B, int ldB, Tensor C, int ldC) -> ()
//
// plus the split-weight and whole-MLP ops the reference lacks.  This file is the only one
// that sees torch types: it validates tensors, takes the current device / stream and hands
// raw pointers to the C ABI in include/fswiglu.h.  A non-zero status becomes a c10::Error
// (RuntimeError in Python), like the reference's TORCH_CHECKs (csrc/SwiGLU/swiglu.cu:475-480).
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <optional>
#include <tuple>
#include <vector>

#include "fswiglu.h"

namespace {

void check_status(int rc, const char* where) {
  TORCH_CHECK(rc == FSWIGLU_OK, where, ": ", fswiglu_status_string(rc), " (status ", rc, ")");
}

// A fake tensor says that it is a CUDA tensor, and as its address gives its offset from nothing.  Plain tensors are told by their
// keys: calls over many small ones pass here for each.
void check_data(const at::Tensor& t, const char* name) {
  constexpr c10::DispatchKeySet wrapped({c10::DispatchKey::Python, c10::DispatchKey::Functionalize});
  if (C10_LIKELY(!t.key_set().has_any(wrapped))) return;
  TORCH_CHECK(t.numel() == 0 || (t.has_storage() && t.storage().data() != nullptr), name,
              " has no data: traced tensors go through torch.ops.ASMLLM");
}

void check_bf16_cuda(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be a bfloat16 tensor");
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  check_data(t, name);
}

int64_t row_pitch(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 2, name, " must be 2-D");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " must have unit stride along its last dimension");
  return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.stride(0), t.size(1));
}

void* current_stream(const at::Tensor& t) {
  return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

}  // namespace

// Raw launcher, reference semantics (csrc/SwiGLU/swiglu.cu:397-525): leading dimensions in elements,
// B holds up rows at even and gate rows at odd indices, the [m, n/2] result is written into C with
// row stride ldC/2.
void swiglu_fwd_bf16(int64_t m, int64_t n, int64_t k, at::Tensor const& A, int64_t ldA, at::Tensor const& B,
                     int64_t ldB, at::Tensor const& C, int64_t ldC) {
  check_bf16_cuda(A, "A");
  check_bf16_cuda(B, "B");
  check_bf16_cuda(C, "C");
  TORCH_CHECK(n % 2 == 0 && ldC % 2 == 0, "n and ldC must be even (up/gate rows are interleaved)");
  const c10::cuda::OptionalCUDAGuard guard(device_of(A));
  check_status(fswiglu_gateup_bf16(A.data_ptr(), ldA, B.data_ptr(), ldB, nullptr, C.data_ptr(), ldC / 2, m, n / 2,
                                   k, 1, current_stream(A)),
               "swiglu_fwd_bf16");
}

// Convenience wrapper, reference semantics (csrc/SwiGLU/swiglu.cu:538-553): allocates [M, N/2].
at::Tensor fused_swiglu_bf16(at::Tensor const& X, at::Tensor const& W1W3) {
  check_bf16_cuda(X, "X");
  check_bf16_cuda(W1W3, "W1W3");
  const int64_t M = X.size(0), N = W1W3.size(0), K = X.size(1);
  at::Tensor out = at::empty({M, N / 2}, X.options());
  swiglu_fwd_bf16(M, N, K, X, row_pitch(X, "X"), W1W3, row_pitch(W1W3, "W1W3"), out, N);
  return out;
}

// In-place form of the raw launcher with the mutation of C declared in its schema (Tensor(a!)), so that
// graph capture (torch.compile, export) keeps the call and orders it.  The reference's schema
// (csrc/torch_bindings.cpp:42) declares no mutation, which is why the op of that name is registered
// here without a shape-only kernel: like the reference's, it cannot be traced, instead of being
// traced wrongly.
void swiglu_fwd_bf16_out(int64_t m, int64_t n, int64_t k, at::Tensor const& A, int64_t ldA, at::Tensor const& B,
                         int64_t ldB, at::Tensor& C, int64_t ldC) {
  swiglu_fwd_bf16(m, n, k, A, ldA, B, ldB, C, ldC);
}

const float* optional_row_scale(const std::optional<at::Tensor>& row_scale, const at::Tensor& x) {
  if (!row_scale.has_value() || !row_scale->defined()) return nullptr;
  TORCH_CHECK(row_scale->scalar_type() == at::kFloat && row_scale->is_cuda() && row_scale->is_contiguous() &&
                  row_scale->numel() == x.size(0),
              "row_scale must be a contiguous float32 CUDA tensor with one entry per row of x");
  return row_scale->data_ptr<float>();
}

const void* optional_residual(const std::optional<at::Tensor>& residual, int64_t M, int64_t d, int64_t* ldr) {
  *ldr = 0;
  if (!residual.has_value() || !residual->defined()) return nullptr;
  check_bf16_cuda(*residual, "residual");
  TORCH_CHECK(residual->dim() == 2 && residual->size(0) == M && residual->size(1) == d, "residual must be [M, d]");
  *ldr = row_pitch(*residual, "residual");
  return residual->data_ptr();
}

// scale[r] = rsqrt(mean(x[r]^2) + eps): the RMSNorm statistic, consumed as `row_scale` below.
at::Tensor rms_scale(at::Tensor const& x, double eps) {
  check_bf16_cuda(x, "x");
  at::Tensor scale = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
  const c10::cuda::OptionalCUDAGuard guard(device_of(x));
  check_status(fswiglu_rms_scale_f32(x.data_ptr(), row_pitch(x, "x"), x.size(0), x.size(1), static_cast<float>(eps),
                                     scale.data_ptr<float>(), current_stream(x)),
               "rms_scale");
  return scale;
}

at::Tensor fused_swiglu_gateup_bf16(at::Tensor const& x, at::Tensor const& W_gate, at::Tensor const& W_up,
                                    std::optional<at::Tensor> const& row_scale) {
  check_bf16_cuda(x, "x");
  check_bf16_cuda(W_gate, "W_gate");
  check_bf16_cuda(W_up, "W_up");
  const int64_t M = x.size(0), d = x.size(1), F = W_gate.size(0);
  TORCH_CHECK(W_up.sizes() == W_gate.sizes() && W_gate.size(1) == d, "W_gate and W_up must both be [F, d]");
  const int64_t ldw = row_pitch(W_gate, "W_gate");
  TORCH_CHECK(row_pitch(W_up, "W_up") == ldw, "W_gate and W_up must share one leading dimension");
  at::Tensor h = at::empty({M, F}, x.options());
  const c10::cuda::OptionalCUDAGuard guard(device_of(x));
  check_status(fswiglu_gateup_bf16_ex(x.data_ptr(), row_pitch(x, "x"), W_gate.data_ptr(), ldw, W_up.data_ptr(),
                                      h.data_ptr(), F, M, F, d, 0, optional_row_scale(row_scale, x), nullptr, 0,
                                      current_stream(x)),
               "fused_swiglu_gateup_bf16");
  return h;
}

at::Tensor swiglu_down_bf16(at::Tensor const& h, at::Tensor const& W_down, bool fp32_out,
                            std::optional<at::Tensor> const& residual) {
  check_bf16_cuda(h, "h");
  check_bf16_cuda(W_down, "W_down");
  const int64_t M = h.size(0), F = h.size(1), d = W_down.size(0);
  TORCH_CHECK(W_down.size(1) == F, "W_down must be [d, F]");
  at::Tensor out = at::empty({M, d}, h.options().dtype(fp32_out ? at::kFloat : at::kBFloat16));
  const c10::cuda::OptionalCUDAGuard guard(device_of(h));
  int64_t ldr = 0;
  const void* res = optional_residual(residual, M, d, &ldr);
  check_status(fswiglu_down_bf16_ex(h.data_ptr(), row_pitch(h, "h"), W_down.data_ptr(), row_pitch(W_down, "W_down"),
                                    out.data_ptr(), d, M, d, F, fp32_out ? FSWIGLU_OUT_F32 : FSWIGLU_OUT_BF16, res,
                                    ldr, nullptr, 0, current_stream(h)),
               "swiglu_down_bf16");
  return out;
}

// residual / row_scale: the fusions either side of the MLP (see include/fswiglu.h); fp32_out is the
// switch the reference makes at compile time (csrc/constants.cuh:9-14).
at::Tensor fused_swiglu_mlp_bf16(at::Tensor const& x, at::Tensor const& W_gate, at::Tensor const& W_up,
                                 at::Tensor const& W_down, std::optional<at::Tensor> const& residual,
                                 std::optional<at::Tensor> const& row_scale, bool fp32_out) {
  check_bf16_cuda(x, "x");
  check_bf16_cuda(W_gate, "W_gate");
  check_bf16_cuda(W_up, "W_up");
  check_bf16_cuda(W_down, "W_down");
  const int64_t M = x.size(0), d = x.size(1), F = W_gate.size(0);
  TORCH_CHECK(W_up.sizes() == W_gate.sizes() && W_gate.size(1) == d && W_down.size(0) == d && W_down.size(1) == F,
              "expected W_gate/W_up [F, d] and W_down [d, F]");
  const int64_t ldw = row_pitch(W_gate, "W_gate");
  TORCH_CHECK(row_pitch(W_up, "W_up") == ldw, "W_gate and W_up must share one leading dimension");
  at::Tensor out = at::empty({M, d}, x.options().dtype(fp32_out ? at::kFloat : at::kBFloat16));
  if (M == 0) return out;
  int64_t ldr = 0;
  const void* res = optional_residual(residual, M, d, &ldr);
  const int64_t ws_bytes = static_cast<int64_t>(fswiglu_workspace_bytes(M, d, F));
  at::Tensor ws = at::empty({std::max<int64_t>(ws_bytes, 256)}, x.options().dtype(at::kByte));
  const c10::cuda::OptionalCUDAGuard guard(device_of(x));
  check_status(fswiglu_mlp_bf16_ex(x.data_ptr(), row_pitch(x, "x"), optional_row_scale(row_scale, x),
                                   W_gate.data_ptr(), W_up.data_ptr(), ldw, W_down.data_ptr(),
                                   row_pitch(W_down, "W_down"), res, ldr, out.data_ptr(), d,
                                   fp32_out ? FSWIGLU_OUT_F32 : FSWIGLU_OUT_BF16, M, d, F, ws.data_ptr(),
                                   static_cast<size_t>(ws.numel()), current_stream(x)),
               "fused_swiglu_mlp_bf16");
  return out;
}

// Shape-only ("Meta") implementations: what fake-tensor tracing (torch.compile, export) needs to see
// through the ops without running them.  The reference registers CUDA kernels only
// (csrc/torch_bindings.cpp:45-50 there), so its ops cannot be traced.
at::Tensor fused_swiglu_bf16_meta(at::Tensor const& X, at::Tensor const& W1W3) {
  return at::empty({X.size(0), W1W3.size(0) / 2}, X.options());
}
void swiglu_fwd_bf16_out_meta(int64_t, int64_t, int64_t, at::Tensor const&, int64_t, at::Tensor const&, int64_t,
                              at::Tensor&, int64_t) {}
at::Tensor rms_scale_meta(at::Tensor const& x, double) { return at::empty({x.size(0)}, x.options().dtype(at::kFloat)); }
at::Tensor fused_swiglu_gateup_bf16_meta(at::Tensor const& x, at::Tensor const& W_gate, at::Tensor const&,
                                         std::optional<at::Tensor> const&) {
  return at::empty({x.size(0), W_gate.size(0)}, x.options());
}
at::Tensor swiglu_down_bf16_meta(at::Tensor const& h, at::Tensor const& W_down, bool fp32_out,
                                 std::optional<at::Tensor> const&) {
  return at::empty({h.size(0), W_down.size(0)}, h.options().dtype(fp32_out ? at::kFloat : at::kBFloat16));
}
at::Tensor fused_swiglu_mlp_bf16_meta(at::Tensor const& x, at::Tensor const&, at::Tensor const&,
                                      at::Tensor const& W_down, std::optional<at::Tensor> const&,
                                      std::optional<at::Tensor> const&, bool fp32_out) {
  return at::empty({x.size(0), W_down.size(0)}, x.options().dtype(fp32_out ? at::kFloat : at::kBFloat16));
}

// ---- training operators: norms with gradients, AdamW over many tensors, clipped gradient norm (include/fswiglu.h) ----

namespace {

int element_type(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, name, " must be a bfloat16 or float32 tensor");
  return t.scalar_type() == at::kFloat ? FSWIGLU_OUT_F32 : FSWIGLU_OUT_BF16;
}

// A [M, d] operand of a norm, of x's type and on its device; its row pitch.
int64_t norm_rows(const at::Tensor& t, const char* name, const at::Tensor& x) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == 2 && t.sizes() == x.sizes(), name, " must be 2-D, of the shape of x");
  TORCH_CHECK(t.scalar_type() == x.scalar_type() && t.device() == x.device(), name, " must have the type and device of x");
  check_data(t, name);
  return row_pitch(t, name);
}

const void* norm_vector(const std::optional<at::Tensor>& v, const char* name, const at::Tensor& x) {
  if (!v.has_value() || !v->defined()) return nullptr;
  TORCH_CHECK(v->dim() == 1 && v->size(0) == x.size(1) && v->is_contiguous() && v->device() == x.device(), name,
              " must be a contiguous vector of x's row length on the device of x");
  check_data(*v, name);
  return v->data_ptr();
}

int norm_vector_type(const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& bias, const at::Tensor& x) {
  const bool w = weight.has_value() && weight->defined(), b = bias.has_value() && bias->defined();
  if (w && b) TORCH_CHECK(weight->scalar_type() == bias->scalar_type(), "weight and bias must have one type");
  return w ? element_type(*weight, "weight") : b ? element_type(*bias, "bias") : element_type(x, "x");
}

const float* norm_statistic(const at::Tensor& t, const char* name, const at::Tensor& x) {
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.device() == x.device() && t.dim() == 1 && t.size(0) == x.size(0) &&
                  t.is_contiguous(),
              name, " must be a contiguous float32 vector with one entry per row of x, on the device of x");
  check_data(t, name);
  return t.data_ptr<float>();
}

// What a call allocates, without the dispatcher's round: these calls may take less time on the GPU than on the host.
at::Tensor empty_beside(const at::Tensor& x, at::IntArrayRef sizes, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, x.device(), std::nullopt));
}

at::Tensor like_rows(const at::Tensor& x) { return empty_beside(x, {x.size(0), x.size(1)}, x.scalar_type()); }

struct NormGradients {
  at::Tensor dx, dweight, dbias;
};

NormGradients norm_backward(bool layer, at::Tensor const& dout, at::Tensor const& x, const at::Tensor* mean,
                            at::Tensor const& rstd, std::optional<at::Tensor> const& weight,
                            std::optional<at::Tensor> const& residual, bool fp32_grads, bool weight_grad, bool bias_grad) {
  const int64_t ldx = norm_rows(x, "x", x), ld_dout = norm_rows(dout, "dout", x);
  const int xt = element_type(x, "x"), wt = norm_vector_type(weight, std::nullopt, x);
  const void* w = norm_vector(weight, "weight", x);
  const bool res = residual.has_value() && residual->defined();
  const int64_t ld_res = res ? norm_rows(*residual, "residual", x) : 0;
  const float* m = layer ? norm_statistic(*mean, "mean", x) : nullptr;
  const float* r = norm_statistic(rstd, "rstd", x);
  const int64_t M = x.size(0), d = x.size(1);
  const c10::cuda::OptionalCUDAGuard guard(device_of(x));
  const int gt = fp32_grads ? FSWIGLU_OUT_F32 : wt;
  const at::ScalarType grads = gt == FSWIGLU_OUT_F32 ? at::kFloat : at::kBFloat16;
  NormGradients g;
  g.dx = like_rows(x);
  if (w != nullptr && weight_grad) g.dweight = empty_beside(x, {d}, grads);
  if (bias_grad) g.dbias = empty_beside(x, {d}, grads);
  at::Tensor ws;
  size_t bytes = 0;
  if ((g.dweight.defined() || g.dbias.defined()) && M > 0) {
    bytes = fswiglu_norm_backward_workspace_bytes(M, d);
    ws = empty_beside(x, {static_cast<int64_t>(bytes)}, at::kByte);
  }
  void* dw = g.dweight.defined() ? g.dweight.data_ptr() : nullptr;
  void* db = g.dbias.defined() ? g.dbias.data_ptr() : nullptr;
  void* wsp = ws.defined() ? ws.data_ptr() : nullptr;
  const void* resp = res ? residual->data_ptr() : nullptr;
  if (layer) {
    check_status(fswiglu_layer_norm_backward(dout.data_ptr(), ld_dout, x.data_ptr(), ldx, m, r, w, resp, ld_res,
                                             g.dx.data_ptr(), d, dw, db, M, d, xt, wt, gt, wsp, bytes, current_stream(x)),
                 "layer_norm_backward");
  } else {
    check_status(fswiglu_rms_norm_backward(dout.data_ptr(), ld_dout, x.data_ptr(), ldx, r, w, resp, ld_res,
                                           g.dx.data_ptr(), d, dw, M, d, xt, wt, gt, wsp, bytes, current_stream(x)),
                 "rms_norm_backward");
  }
  return g;
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_forward(at::Tensor const& x, std::optional<at::Tensor> const& weight,
                                                                  std::optional<at::Tensor> const& bias, double eps) {
  const int64_t ldx = norm_rows(x, "x", x), M = x.size(0), d = x.size(1);
  const int xt = element_type(x, "x"), wt = norm_vector_type(weight, bias, x);
  const void* w = norm_vector(weight, "weight", x);
  const void* b = norm_vector(bias, "bias", x);
  const c10::cuda::OptionalCUDAGuard guard(device_of(x));
  at::Tensor y = like_rows(x), mean = empty_beside(x, {M}, at::kFloat), rstd = empty_beside(x, {M}, at::kFloat);
  check_status(fswiglu_layer_norm_forward(x.data_ptr(), ldx, w, b, y.data_ptr(), d, mean.data_ptr<float>(),
                                          rstd.data_ptr<float>(), M, d, xt, wt, static_cast<float>(eps), current_stream(x)),
               "layer_norm_forward");
  return {y, mean, rstd};
}

std::tuple<at::Tensor, at::Tensor> rms_norm_forward(at::Tensor const& x, std::optional<at::Tensor> const& weight, double eps) {
  const int64_t ldx = norm_rows(x, "x", x), M = x.size(0), d = x.size(1);
  const int xt = element_type(x, "x"), wt = norm_vector_type(weight, std::nullopt, x);
  const void* w = norm_vector(weight, "weight", x);
  const c10::cuda::OptionalCUDAGuard guard(device_of(x));
  at::Tensor y = like_rows(x), rstd = empty_beside(x, {M}, at::kFloat);
  check_status(fswiglu_rms_norm_forward(x.data_ptr(), ldx, w, y.data_ptr(), d, rstd.data_ptr<float>(), M, d, xt, wt,
                                        static_cast<float>(eps), current_stream(x)),
               "rms_norm_forward");
  return {y, rstd};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_backward(at::Tensor const& dout, at::Tensor const& x,
                                                                   at::Tensor const& mean, at::Tensor const& rstd,
                                                                   std::optional<at::Tensor> const& weight, bool bias_grad,
                                                                   std::optional<at::Tensor> const& residual,
                                                                   bool fp32_grads, bool weight_grad) {
  NormGradients g = norm_backward(true, dout, x, &mean, rstd, weight, residual, fp32_grads, weight_grad, bias_grad);
  return {g.dx, g.dweight, g.dbias};
}

std::tuple<at::Tensor, at::Tensor> rms_norm_backward(at::Tensor const& dout, at::Tensor const& x, at::Tensor const& rstd,
                                                     std::optional<at::Tensor> const& weight,
                                                     std::optional<at::Tensor> const& residual, bool fp32_grads,
                                                     bool weight_grad) {
  NormGradients g = norm_backward(false, dout, x, nullptr, rstd, weight, residual, fp32_grads, weight_grad, false);
  return {g.dx, g.dweight};
}

namespace {

// The tensors of a list, by reference: what a step over many of them has to touch one by one.
using Refs = std::vector<const at::Tensor*>;

Refs refs_of(at::TensorList list) {
  Refs r;
  r.reserve(list.size());
  for (const at::Tensor& t : list) r.push_back(&t);
  return r;
}

// The same from a Python list or tuple, which the caller holds.
Refs refs_of(const pybind11::handle& list, const char* name) {
  TORCH_CHECK(PyList_Check(list.ptr()) || PyTuple_Check(list.ptr()), name, " must be a list of tensors");
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(list.ptr());
  PyObject** items = PySequence_Fast_ITEMS(list.ptr());
  Refs r(static_cast<size_t>(n));
  for (Py_ssize_t i = 0; i < n; ++i) {
    TORCH_CHECK(THPVariable_Check(items[i]), name, " must be a list of tensors");
    r[static_cast<size_t>(i)] = &THPVariable_Unpack(items[i]);
  }
  return r;
}

// One list of a step over many tensors: as many entries as parameters, each contiguous, of one type, on one device.
void check_list(const Refs& list, const Refs& params, at::ScalarType type, const char* name) {
  TORCH_CHECK(list.size() == params.size(), name, " must have one tensor for each parameter");
  const auto device = params[0]->device();
  for (const at::Tensor* t : list) {
    TORCH_CHECK(t->scalar_type() == type, name, " must all be ", type, " tensors");
    TORCH_CHECK(t->device() == device, name, " must all be on the device of the parameters");
    TORCH_CHECK(t->is_contiguous(), name, " must all be contiguous");
    check_data(*t, name);
  }
}

const void* scalar_on_device(const std::optional<at::Tensor>& t, at::ScalarType type, const at::Tensor& p, const char* name) {
  if (!t.has_value() || !t->defined()) return nullptr;
  TORCH_CHECK(t->scalar_type() == type && t->numel() == 1 && t->device() == p.device(), name, " must be one ", type,
              " element on the device of the parameters");
  check_data(*t, name);
  return t->data_ptr();
}

void adamw_step_refs(const Refs& params, const Refs& grads, const Refs& exp_avgs, const Refs& exp_avg_sqs, int64_t step,
                     double lr, double beta1, double beta2, double eps, double weight_decay, const Refs& masters,
                     const Refs& exp_avg_scales, const Refs& exp_avg_sq_scales, std::optional<at::Tensor> const& grad_scale,
                     int64_t seed, std::optional<at::Tensor> const& lr_tensor, std::optional<at::Tensor> const& step_tensor) {
  if (params.empty()) {
    TORCH_CHECK(grads.empty() && exp_avgs.empty() && exp_avg_sqs.empty(), "the lists must be of one length");
    return;
  }
  const at::Tensor& p0 = *params[0];
  TORCH_CHECK(p0.is_cuda(), "params must be CUDA tensors");
  TORCH_CHECK(grads.size() == params.size() && exp_avgs.size() == params.size(), "the lists must be of one length");
  const int pt = element_type(p0, "params"), gt = element_type(*grads[0], "grads");
  const bool eight = exp_avgs[0]->scalar_type() == at::kFloat8_e4m3fn;
  check_list(params, params, p0.scalar_type(), "params");
  check_list(grads, params, grads[0]->scalar_type(), "grads");
  check_list(exp_avgs, params, eight ? at::kFloat8_e4m3fn : at::kFloat, "exp_avgs");
  check_list(exp_avg_sqs, params, eight ? at::kFloat8_e5m2 : at::kFloat, "exp_avg_sqs");
  if (!masters.empty()) {
    TORCH_CHECK(pt == FSWIGLU_OUT_BF16, "masters go with bfloat16 params");
    check_list(masters, params, at::kFloat, "masters");
  }
  if (eight) {
    check_list(exp_avg_scales, params, at::kFloat, "exp_avg_scales");
    check_list(exp_avg_sq_scales, params, at::kFloat, "exp_avg_sq_scales");
  } else {
    TORCH_CHECK(exp_avg_scales.empty() && exp_avg_sq_scales.empty(), "scales go with 8-bit moments");
  }
  std::vector<fswiglu_adamw_tensor> table(params.size());
  for (size_t i = 0; i < params.size(); ++i) {
    const int64_t n = params[i]->numel();
    TORCH_CHECK(grads[i]->numel() == n && exp_avgs[i]->numel() == n && exp_avg_sqs[i]->numel() == n &&
                    (masters.empty() || masters[i]->numel() == n),
                "tensor ", i, ": parameter, gradient, moments and master must have as many elements");
    if (eight) {
      TORCH_CHECK(exp_avg_scales[i]->numel() == (n + 255) / 256 && exp_avg_sq_scales[i]->numel() == (n + 255) / 256, "tensor ",
                  i, ": scales must have one element for each 256 of the parameter");
    }
    table[i] = {params[i]->data_ptr(),
                grads[i]->data_ptr(),
                exp_avgs[i]->data_ptr(),
                exp_avg_sqs[i]->data_ptr(),
                masters.empty() ? nullptr : masters[i]->data_ptr<float>(),
                eight ? exp_avg_scales[i]->data_ptr<float>() : nullptr,
                eight ? exp_avg_sq_scales[i]->data_ptr<float>() : nullptr,
                n};
  }
  fswiglu_adamw_options o = {};
  o.lr = lr;
  o.beta1 = beta1;
  o.beta2 = beta2;
  o.eps = eps;
  o.weight_decay = weight_decay;
  o.step = step;
  o.seed = static_cast<uint64_t>(seed);
  o.lr_device = static_cast<const float*>(scalar_on_device(lr_tensor, at::kFloat, p0, "lr_tensor"));
  o.step_device = static_cast<const int64_t*>(scalar_on_device(step_tensor, at::kLong, p0, "step_tensor"));
  o.grad_scale = static_cast<const float*>(scalar_on_device(grad_scale, at::kFloat, p0, "grad_scale"));
  const c10::cuda::OptionalCUDAGuard guard(device_of(p0));
  check_status(fswiglu_adamw_step(table.data(), static_cast<int64_t>(table.size()), pt, gt, eight ? 8 : 32, &o, current_stream(p0)),
               "adamw_step");
  // written through raw pointers: what a graph saved of a parameter is known to be stale
  for (const at::Tensor* p : params) {
    if (!p->is_inference()) p->unsafeGetTensorImpl()->bump_version();
  }
}

at::Tensor grad_norm_clip_refs(const Refs& grads, double max_norm) {
  TORCH_CHECK(!grads.empty(), "grads must not be empty");
  const at::Tensor& g0 = *grads[0];
  std::vector<fswiglu_grad_tensor> table(grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    const at::Tensor& g = *grads[i];
    TORCH_CHECK(g.is_cuda() && g.device() == g0.device(), "grads must all be CUDA tensors of one device");
    TORCH_CHECK(g.is_contiguous(), "grads must all be contiguous");
    check_data(g, "grads");
    table[i] = {g.data_ptr(), g.numel(), element_type(g, "grads")};
  }
  const c10::cuda::OptionalCUDAGuard guard(device_of(g0));
  at::Tensor out = empty_beside(g0, {2}, at::kFloat);
  const size_t bytes = fswiglu_grad_norm_workspace_bytes();
  at::Tensor ws = empty_beside(g0, {static_cast<int64_t>(bytes)}, at::kByte);
  check_status(fswiglu_grad_norm_clip(table.data(), static_cast<int64_t>(table.size()), static_cast<float>(max_norm),
                                      out.data_ptr<float>(), ws.data_ptr(), bytes, current_stream(g0)),
               "grad_norm_clip");
  return out;
}

}  // namespace

void adamw_step(at::TensorList params, at::TensorList grads, at::TensorList exp_avgs, at::TensorList exp_avg_sqs, int64_t step,
                double lr, double beta1, double beta2, double eps, double weight_decay, at::TensorList masters,
                at::TensorList exp_avg_scales, at::TensorList exp_avg_sq_scales, std::optional<at::Tensor> const& grad_scale,
                int64_t seed, std::optional<at::Tensor> const& lr_tensor, std::optional<at::Tensor> const& step_tensor) {
  adamw_step_refs(refs_of(params), refs_of(grads), refs_of(exp_avgs), refs_of(exp_avg_sqs), step, lr, beta1, beta2, eps,
                  weight_decay, refs_of(masters), refs_of(exp_avg_scales), refs_of(exp_avg_sq_scales), grad_scale, seed,
                  lr_tensor, step_tensor);
}

// [norm, factor]: the 2-norm over all gradients, and min(1, max_norm / (norm + 1e-6)) for adamw_step's grad_scale.
at::Tensor grad_norm_clip(at::TensorList grads, double max_norm) { return grad_norm_clip_refs(refs_of(grads), max_norm); }

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_forward_meta(at::Tensor const& x, std::optional<at::Tensor> const&,
                                                                       std::optional<at::Tensor> const&, double) {
  const auto f32 = x.options().dtype(at::kFloat);
  return {at::empty({x.size(0), x.size(1)}, x.options()), at::empty({x.size(0)}, f32), at::empty({x.size(0)}, f32)};
}
std::tuple<at::Tensor, at::Tensor> rms_norm_forward_meta(at::Tensor const& x, std::optional<at::Tensor> const&, double) {
  return {at::empty({x.size(0), x.size(1)}, x.options()), at::empty({x.size(0)}, x.options().dtype(at::kFloat))};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_backward_meta(at::Tensor const&, at::Tensor const& x, at::Tensor const&,
                                                                        at::Tensor const&,
                                                                        std::optional<at::Tensor> const& weight, bool bias_grad,
                                                                        std::optional<at::Tensor> const&, bool fp32_grads,
                                                                        bool weight_grad) {
  const bool w = weight.has_value() && weight->defined();
  const auto g = x.options().dtype(fp32_grads ? at::kFloat : w ? weight->scalar_type() : x.scalar_type());
  return {at::empty({x.size(0), x.size(1)}, x.options()), w && weight_grad ? at::empty({x.size(1)}, g) : at::Tensor(),
          bias_grad ? at::empty({x.size(1)}, g) : at::Tensor()};
}
std::tuple<at::Tensor, at::Tensor> rms_norm_backward_meta(at::Tensor const& dout, at::Tensor const& x, at::Tensor const& rstd,
                                                          std::optional<at::Tensor> const& weight,
                                                          std::optional<at::Tensor> const& residual, bool fp32_grads,
                                                          bool weight_grad) {
  auto g = layer_norm_backward_meta(dout, x, rstd, rstd, weight, false, residual, fp32_grads, weight_grad);
  return {std::get<0>(g), std::get<1>(g)};
}
void adamw_step_meta(at::TensorList, at::TensorList, at::TensorList, at::TensorList, int64_t, double, double, double, double,
                     double, at::TensorList, at::TensorList, at::TensorList, std::optional<at::Tensor> const&, int64_t,
                     std::optional<at::Tensor> const&, std::optional<at::Tensor> const&) {}
at::Tensor grad_norm_clip_meta(at::TensorList grads, double) {
  TORCH_CHECK(!grads.empty(), "grads must not be empty");
  return at::empty({2}, grads[0].options().dtype(at::kFloat));
}

namespace Fused_MLP {

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  m.def("fused_swiglu_bf16", &fused_swiglu_bf16, "fused SwiGLU for bf16");
  m.def("swiglu_fwd_bf16", &swiglu_fwd_bf16, "SwiGLU fwd bf16");
  m.def("rms_scale", &rms_scale, "rsqrt(mean(x^2) + eps) per row", py::arg("x"), py::arg("eps") = 1e-6);
  m.def("fused_swiglu_gateup_bf16", &fused_swiglu_gateup_bf16, "silu(s x Wg^T) * (s x Wu^T), split weights",
        py::arg("x"), py::arg("W_gate"), py::arg("W_up"), py::arg("row_scale") = py::none());
  m.def("swiglu_down_bf16", &swiglu_down_bf16, "(residual +) h Wd^T", py::arg("h"), py::arg("W_down"),
        py::arg("fp32_out") = false, py::arg("residual") = py::none());
  m.def("fused_swiglu_mlp_bf16", &fused_swiglu_mlp_bf16, "(residual +) (silu(s x Wg^T) * (s x Wu^T)) Wd^T",
        py::arg("x"), py::arg("W_gate"), py::arg("W_up"), py::arg("W_down"), py::arg("residual") = py::none(),
        py::arg("row_scale") = py::none(), py::arg("fp32_out") = false);
  m.def("layer_norm_forward", &layer_norm_forward, "(y, mean, rstd) of layer norm over the rows of x", py::arg("x"),
        py::arg("weight") = py::none(), py::arg("bias") = py::none(), py::arg("eps") = 1e-5);
  m.def("rms_norm_forward", &rms_norm_forward, "(y, rstd) of RMS norm over the rows of x", py::arg("x"),
        py::arg("weight") = py::none(), py::arg("eps") = 1e-6);
  m.def("layer_norm_backward", &layer_norm_backward, "(dx, dweight, dbias); residual is added to dx", py::arg("dout"),
        py::arg("x"), py::arg("mean"), py::arg("rstd"), py::arg("weight") = py::none(), py::arg("bias_grad") = false,
        py::arg("residual") = py::none(), py::arg("fp32_grads") = false, py::arg("weight_grad") = true);
  m.def("rms_norm_backward", &rms_norm_backward, "(dx, dweight); residual is added to dx", py::arg("dout"), py::arg("x"),
        py::arg("rstd"), py::arg("weight") = py::none(), py::arg("residual") = py::none(), py::arg("fp32_grads") = false,
        py::arg("weight_grad") = true);
  m.def("adamw_step",
        [](py::handle params, py::handle grads, py::handle exp_avgs, py::handle exp_avg_sqs, int64_t step, double lr,
           double beta1, double beta2, double eps, double weight_decay, py::handle masters, py::handle exp_avg_scales,
           py::handle exp_avg_sq_scales, const std::optional<at::Tensor>& grad_scale, int64_t seed,
           const std::optional<at::Tensor>& lr_tensor, const std::optional<at::Tensor>& step_tensor) {
          adamw_step_refs(refs_of(params, "params"), refs_of(grads, "grads"), refs_of(exp_avgs, "exp_avgs"),
                          refs_of(exp_avg_sqs, "exp_avg_sqs"), step, lr, beta1, beta2, eps, weight_decay,
                          refs_of(masters, "masters"), refs_of(exp_avg_scales, "exp_avg_scales"),
                          refs_of(exp_avg_sq_scales, "exp_avg_sq_scales"), grad_scale, seed, lr_tensor, step_tensor);
        },
        "one AdamW step over many tensors, in place", py::arg("params"), py::arg("grads"), py::arg("exp_avgs"),
        py::arg("exp_avg_sqs"), py::arg("step"), py::arg("lr"), py::arg("beta1") = 0.9, py::arg("beta2") = 0.999,
        py::arg("eps") = 1e-8, py::arg("weight_decay") = 0.01, py::arg("masters") = py::tuple(),
        py::arg("exp_avg_scales") = py::tuple(), py::arg("exp_avg_sq_scales") = py::tuple(), py::arg("grad_scale") = py::none(),
        py::arg("seed") = 0, py::arg("lr_tensor") = py::none(), py::arg("step_tensor") = py::none());
  m.def("grad_norm_clip",
        [](py::handle grads, double max_norm) { return grad_norm_clip_refs(refs_of(grads, "grads"), max_norm); },
        "[2-norm over all gradients, min(1, max_norm / (norm + 1e-6))]", py::arg("grads"), py::arg("max_norm"));
}

TORCH_LIBRARY(ASMLLM, m) {
  m.def("fused_swiglu_bf16(Tensor X, Tensor W1W3) -> Tensor");
  m.def("swiglu_fwd_bf16(int m, int n, int k, Tensor A, int ldA, Tensor B, int ldB, Tensor C, int ldC) -> ()");
  m.def("swiglu_fwd_bf16_out(int m, int n, int k, Tensor A, int ldA, Tensor B, int ldB, Tensor(a!) C, int ldC) -> ()");
  m.def("rms_scale(Tensor x, float eps=1e-6) -> Tensor");
  m.def("fused_swiglu_gateup_bf16(Tensor x, Tensor W_gate, Tensor W_up, Tensor? row_scale=None) -> Tensor");
  m.def("swiglu_down_bf16(Tensor h, Tensor W_down, bool fp32_out=False, Tensor? residual=None) -> Tensor");
  m.def("fused_swiglu_mlp_bf16(Tensor x, Tensor W_gate, Tensor W_up, Tensor W_down, Tensor? residual=None, "
        "Tensor? row_scale=None, bool fp32_out=False) -> Tensor");
  m.def("layer_norm_forward(Tensor x, Tensor? weight=None, Tensor? bias=None, float eps=1e-05) -> (Tensor, Tensor, Tensor)");
  m.def("rms_norm_forward(Tensor x, Tensor? weight=None, float eps=1e-06) -> (Tensor, Tensor)");
  m.def("layer_norm_backward(Tensor dout, Tensor x, Tensor mean, Tensor rstd, Tensor? weight=None, bool bias_grad=False, "
        "Tensor? residual=None, bool fp32_grads=False, bool weight_grad=True) -> (Tensor, Tensor, Tensor)");
  m.def("rms_norm_backward(Tensor dout, Tensor x, Tensor rstd, Tensor? weight=None, Tensor? residual=None, "
        "bool fp32_grads=False, bool weight_grad=True) -> (Tensor, Tensor)");
  m.def("adamw_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, Tensor(c!)[] exp_avg_sqs, int step, float lr, "
        "float beta1, float beta2, float eps, float weight_decay, Tensor(d!)[] masters, "
        "Tensor(e!)[] exp_avg_scales, Tensor(f!)[] exp_avg_sq_scales, Tensor? grad_scale=None, int seed=0, "
        "Tensor? lr_tensor=None, Tensor? step_tensor=None) -> ()");
  m.def("grad_norm_clip(Tensor[] grads, float max_norm) -> Tensor");
}

TORCH_LIBRARY_IMPL(ASMLLM, CUDA, m) {
  m.impl("fused_swiglu_bf16", &fused_swiglu_bf16);
  m.impl("swiglu_fwd_bf16", &swiglu_fwd_bf16);
  m.impl("swiglu_fwd_bf16_out", &swiglu_fwd_bf16_out);
  m.impl("rms_scale", &rms_scale);
  m.impl("fused_swiglu_gateup_bf16", &fused_swiglu_gateup_bf16);
  m.impl("swiglu_down_bf16", &swiglu_down_bf16);
  m.impl("fused_swiglu_mlp_bf16", &fused_swiglu_mlp_bf16);
  m.impl("layer_norm_forward", &layer_norm_forward);
  m.impl("rms_norm_forward", &rms_norm_forward);
  m.impl("layer_norm_backward", &layer_norm_backward);
  m.impl("rms_norm_backward", &rms_norm_backward);
  m.impl("adamw_step", &adamw_step);
  m.impl("grad_norm_clip", &grad_norm_clip);
}

TORCH_LIBRARY_IMPL(ASMLLM, Meta, m) {
  m.impl("fused_swiglu_bf16", &fused_swiglu_bf16_meta);
  m.impl("swiglu_fwd_bf16_out", &swiglu_fwd_bf16_out_meta);
  m.impl("rms_scale", &rms_scale_meta);
  m.impl("fused_swiglu_gateup_bf16", &fused_swiglu_gateup_bf16_meta);
  m.impl("swiglu_down_bf16", &swiglu_down_bf16_meta);
  m.impl("fused_swiglu_mlp_bf16", &fused_swiglu_mlp_bf16_meta);
  m.impl("layer_norm_forward", &layer_norm_forward_meta);
  m.impl("rms_norm_forward", &rms_norm_forward_meta);
  m.impl("layer_norm_backward", &layer_norm_backward_meta);
  m.impl("rms_norm_backward", &rms_norm_backward_meta);
  m.impl("adamw_step", &adamw_step_meta);
  m.impl("grad_norm_clip", &grad_norm_clip_meta);
}

}  // namespace Fused_MLP
