// The stateless operators (permute, fp8) as torch calls: argument checks, output
// tensors, the current stream and the gradients around the C entry points of
// b200moe.h. Written against torch's C++ interface because these calls are short:
// a decode step's operator runs 2-6 us on the GPU, where the same call through
// ctypes took 10-22 us of host time and a forward and backward through a Python
// autograd function 100 us.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <limits>
#include <string>
#include <tuple>

#include "../../include/b200moe.h"

namespace {

using at::ScalarType;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;
using OptDtype = std::optional<ScalarType>;

constexpr ScalarType kE4m3 = ScalarType::Float8_e4m3fn;
constexpr int64_t kBlock = 128, kMaxExperts = 1024, kMaxRoutes = int64_t(1) << 26, kMaxTopK = 1024;
constexpr int64_t kMaxAxis = INT32_MAX - 256;

// ------------------------------------------------------------------ errors
// A non-zero status of the library; becomes b200moe._lib.B200MoeError in Python.
struct StatusError : std::runtime_error {
  std::string where;
  int status;
  StatusError(const char* w, int s)
      : std::runtime_error(std::string(w) + ": " + b200moe_status_name(s)), where(w), status(s) {}
};
void check(const char* where, int status) {
  if (status) throw StatusError(where, status);
}

// ------------------------------------------------------------------ checks
enum Kind { kFloats, kFloatsOrE4m3, kOnlyE4m3, kF32, kI32 };

bool is_float(ScalarType t) {
  return t == ScalarType::BFloat16 || t == ScalarType::Half || t == ScalarType::Float;
}
bool fits(ScalarType t, Kind k) {
  switch (k) {
    case kFloats: return is_float(t);
    case kFloatsOrE4m3: return is_float(t) || t == kE4m3;
    case kOnlyE4m3: return t == kE4m3;
    case kF32: return t == ScalarType::Float;
    default: return t == ScalarType::Int;
  }
}
const char* kind_name(Kind k) {
  const char* names[] = {"bfloat16/float16/float32", "bfloat16/float16/float32/float8_e4m3fn", "float8_e4m3fn",
                         "float32", "int32"};
  return names[k];
}
int code(ScalarType t) {
  TORCH_CHECK_VALUE(is_float(t), "must be bfloat16, float16 or float32, got ", t);  // a wrong code is a wrong size
  return t == ScalarType::Half ? B200MOE_F16 : t == ScalarType::BFloat16 ? B200MOE_BF16 : B200MOE_F32;
}

// The operators have no forward-mode derivative: a tangent is refused instead of left out.
void no_tangent(const char* name, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), name,
                              " carries a forward-mode tangent, which this operator cannot differentiate");
}

// A CUDA tensor of the kind with `dim` axes, contiguous or (rows) with any distance between rows, on `like`'s device.
void want(const char* name, const Tensor& t, Kind kind, int64_t dim, const Tensor* like = nullptr, bool rows = false) {
  TORCH_CHECK_VALUE(t.defined() && t.is_cuda(), name, " must be a CUDA tensor, got ",
                    t.defined() ? t.device().str() : "none");
  TORCH_CHECK_VALUE(fits(t.scalar_type(), kind) && t.dim() == dim, name, " must be ", kind_name(kind), " with ", dim,
                    " axes, got ", t.scalar_type(), " ", t.sizes());
  TORCH_CHECK_VALUE(t.is_contiguous() || (rows && t.stride(-1) == 1 && t.stride(0) >= t.size(1)), name, " must ",
                    rows ? "have contiguous rows" : "be contiguous", ", got strides ", t.strides());
  // every axis: the kernels' sizes are 32 bits, and their round-ups to whole tiles stay below 2^31
  for (const int64_t n : t.sizes()) TORCH_CHECK_VALUE(n <= kMaxAxis, name, " is too large: ", t.sizes());
  TORCH_CHECK_VALUE(!like || t.device() == like->device(), name, " is on ", t.device(), ", the other arguments on ",
                    like ? like->device().str() : "");
  no_tangent(name, t);
}
void want_shape(const char* name, const Tensor& t, at::IntArrayRef shape) {
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
}

int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }

Tensor empty(at::IntArrayRef size, ScalarType dtype, const Tensor& like) {
  return at::detail::empty_cuda(size, dtype, like.device(), std::nullopt);
}
void* stream(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
const float* f32(const Tensor& t) { return t.defined() ? static_cast<const float*>(t.data_ptr()) : nullptr; }
float* f32_mut(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
const int32_t* i32(const Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }
int32_t* i32_mut(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }
void* mut(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool differentiable(const Tensor& t) { return t.defined() && t.requires_grad(); }

// ------------------------------------------------------------------ permute
void check_routes(const Tensor& ids, int64_t tokens, int64_t num_experts, const Tensor* like) {
  want("topk_ids", ids, kI32, 2, like);
  const int64_t k = ids.size(1);
  TORCH_CHECK_VALUE(ids.size(0) == tokens && k >= 1 && k <= kMaxTopK && tokens * k <= kMaxRoutes,
                    "bad routing shape ", ids.sizes(), " for ", tokens, " tokens");
  TORCH_CHECK_VALUE(num_experts >= 1 && num_experts <= kMaxExperts, "num_experts must be 1..", kMaxExperts, ", got ",
                    num_experts);
}

struct Tables {
  Tensor row_of_route, offsets, workspace;
  size_t bytes;
  Tables(const Tensor& ids, int64_t num_experts)
      : row_of_route(empty(ids.sizes(), ScalarType::Int, ids)),
        offsets(empty({num_experts + 1}, ScalarType::Int, ids)),
        bytes(ids.numel() ? b200moe_sort_workspace_bytes(int(ids.numel()), int(num_experts)) : 0) {
    if (bytes) workspace = empty({int64_t(bytes)}, ScalarType::Byte, ids);
  }
};

std::tuple<Tensor, Tensor> sort_routes(const Tensor& ids, int64_t num_experts) {
  want("topk_ids", ids, kI32, 2);
  check_routes(ids, ids.size(0), num_experts, nullptr);
  const c10::cuda::CUDAGuard guard(ids.device());
  Tables t(ids, num_experts);
  if (ids.numel() == 0)
    t.offsets.zero_();
  else
    check("b200moe_sort_routes",
          b200moe_sort_routes(stream(ids), i32(ids), int(ids.numel()), int(num_experts), i32_mut(t.row_of_route),
                              i32_mut(t.offsets), mut(t.workspace), t.bytes));
  return {t.row_of_route, t.offsets};
}

using Permuted = std::tuple<Tensor, Tensor, Tensor, Tensor>;  // rows, their scales (undefined: none), tables

Permuted run_permute(const Tensor& x, const Tensor& ids, int64_t num_experts, const Tensor& scale) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t t = x.size(0), h = x.size(1), k = ids.size(1), b = x.element_size();
  const int64_t n_scale = scale.defined() ? scale.size(1) : 0;
  Tables tab(ids, num_experts);
  Tensor rows = empty({t * k, h}, x.scalar_type(), x), row_scale;
  if (scale.defined()) row_scale = empty({t * k, n_scale}, ScalarType::Float, x);
  if (t == 0)
    tab.offsets.zero_();
  else
    check("b200moe_permute",
          b200moe_permute(stream(x), i32(ids), int(num_experts), x.data_ptr(), x.stride(0) * b, h * b, f32(scale),
                          n_scale ? scale.stride(0) : 0, int(n_scale), int(t), int(k), i32_mut(tab.row_of_route),
                          i32_mut(tab.offsets), rows.data_ptr(), f32_mut(row_scale), mut(tab.workspace), tab.bytes));
  return {rows, row_scale, tab.row_of_route, tab.offsets};
}

Tensor run_unpermute(const Tensor& rows, const Tensor& row_of_route, const Tensor& weights, ScalarType out_dtype) {
  const c10::cuda::CUDAGuard guard(rows.device());
  const int64_t t = row_of_route.size(0), k = row_of_route.size(1), h = rows.size(1);
  Tensor out = empty({t, h}, out_dtype, rows);
  if (t)
    check("b200moe_unpermute", b200moe_unpermute(stream(rows), rows.data_ptr(), code(rows.scalar_type()),
                                                 i32(row_of_route), f32(weights), int(t), int(k), int(h),
                                                 out.data_ptr(), code(out_dtype)));
  return out;
}

std::tuple<Tensor, Tensor> run_unpermute_grad(const Tensor& grad, const Tensor& rows, const Tensor& row_of_route,
                                              const Tensor& weights, bool need_rows, bool need_weights) {
  const c10::cuda::CUDAGuard guard(rows.device());
  const int64_t t = row_of_route.size(0), k = row_of_route.size(1), h = rows.size(1);
  need_weights = need_weights && weights.defined();
  Tensor grad_rows, grad_weights;
  if (need_rows) grad_rows = empty(rows.sizes(), rows.scalar_type(), rows);
  if (need_weights) grad_weights = empty(weights.sizes(), ScalarType::Float, rows);
  if (t && (need_rows || need_weights))
    check("b200moe_unpermute_grad",
          b200moe_unpermute_grad(stream(rows), grad.data_ptr(), code(grad.scalar_type()), grad.stride(0),
                                 rows.data_ptr(), code(rows.scalar_type()), i32(row_of_route), f32(weights), int(t),
                                 int(k), int(h), mut(grad_rows), f32_mut(grad_weights)));
  return {grad_rows, grad_weights};
}

// The gradients have no graph of their own: asked for one (create_graph), they refuse instead of leaving it out.
void once_differentiable(const Tensor& grad) {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), "this operator's gradient cannot be differentiated again");
  if (grad.defined()) no_tangent("the gradient", grad);
}

// A gradient as the kernels read it: contiguous columns, rows at any distance.
Tensor as_rows(const Tensor& grad) {
  return grad.stride(-1) == 1 && grad.stride(0) >= grad.size(1) ? grad : grad.contiguous();
}

struct PermuteFn : torch::autograd::Function<PermuteFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& ids, int64_t num_experts) {
    const auto [rows, scale, row_of_route, offsets] = run_permute(x, ids, num_experts, Tensor());
    ctx->save_for_backward({row_of_route});
    ctx->mark_non_differentiable({row_of_route, offsets});
    ctx->set_materialize_grads(false);
    return {rows, row_of_route, offsets};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_differentiable(grads[0]);
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    return {run_unpermute(grads[0].contiguous(), ctx->get_saved_variables()[0], Tensor(), grads[0].scalar_type()),
            Tensor(), Tensor()};
  }
};

struct UnpermuteFn : torch::autograd::Function<UnpermuteFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& row_of_route, const OptTensor& weights,
                        ScalarType out_dtype) {
    ctx->save_for_backward({rows, row_of_route, weights.value_or(Tensor())});
    return run_unpermute(rows, row_of_route, weights.value_or(Tensor()), out_dtype);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_differentiable(grads[0]);
    const auto saved = ctx->get_saved_variables();
    const bool need_weights = saved[2].defined() && ctx->needs_input_grad(2);
    const auto [grad_rows, grad_weights] = run_unpermute_grad(as_rows(grads[0]), saved[0], saved[1], saved[2],
                                                              ctx->needs_input_grad(0), need_weights);
    return {grad_rows, Tensor(), grad_weights, Tensor()};
  }
};

std::tuple<Tensor, OptTensor, Tensor, Tensor> permute(const Tensor& x, const Tensor& ids, int64_t num_experts,
                                                      const OptTensor& scale_arg) {
  const Tensor scale = scale_arg.value_or(Tensor());
  want("x", x, kFloatsOrE4m3, 2, nullptr, true);
  TORCH_CHECK_VALUE(x.size(1) >= 1, "x must have columns, got ", x.sizes());
  check_routes(ids, x.size(0), num_experts, &x);
  if (scale.defined()) {
    want("scale", scale, kF32, 2, &x, true);
    TORCH_CHECK_VALUE(scale.size(0) == x.size(0), "scale must have ", x.size(0), " rows, got ", scale.sizes());
  }
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    TORCH_CHECK_VALUE(!scale.defined() && is_float(x.scalar_type()),
                      "quantized rows (E4M3, or with scales) have no gradient: permute them without one");
    const variable_list out = PermuteFn::apply(x, ids, num_experts);
    return {out[0], std::nullopt, out[1], out[2]};
  }
  const auto [rows, row_scale, row_of_route, offsets] = run_permute(x, ids, num_experts, scale);
  return {rows, row_scale.defined() ? OptTensor(row_scale) : std::nullopt, row_of_route, offsets};
}

void check_row_of_route(const Tensor& rows, const Tensor& row_of_route, const Tensor& weights) {
  want("rows", rows, kFloats, 2);
  want("row_of_route", row_of_route, kI32, 2, &rows);
  const int64_t t = row_of_route.size(0), k = row_of_route.size(1);
  TORCH_CHECK_VALUE(k >= 1 && k <= kMaxTopK && t * k <= kMaxRoutes && rows.size(0) == t * k && rows.size(1) >= 1,
                    "rows ", rows.sizes(), " do not fit the routes ", row_of_route.sizes());
  if (weights.defined()) {
    want("weights", weights, kF32, 2, &rows);
    want_shape("weights", weights, {t, k});
  }
}

Tensor unpermute(const Tensor& rows, const Tensor& row_of_route, const OptTensor& weights_arg,
                 const OptDtype& out_dtype) {
  const Tensor weights = weights_arg.value_or(Tensor());
  check_row_of_route(rows, row_of_route, weights);
  const ScalarType dtype = out_dtype.value_or(rows.scalar_type());
  TORCH_CHECK_VALUE(dtype == rows.scalar_type() || dtype == ScalarType::Float, "out_dtype must be ",
                    rows.scalar_type(), " or Float, got ", dtype);
  if (at::GradMode::is_enabled() && (rows.requires_grad() || differentiable(weights)))
    return UnpermuteFn::apply(rows, row_of_route, weights_arg, dtype);
  return run_unpermute(rows, row_of_route, weights, dtype);
}

std::tuple<OptTensor, OptTensor> unpermute_grad(const Tensor& grad, const Tensor& rows, const Tensor& row_of_route,
                                                const OptTensor& weights_arg, bool need_rows, bool need_weights) {
  const Tensor weights = weights_arg.value_or(Tensor());
  check_row_of_route(rows, row_of_route, weights);
  want("grad", grad, kFloats, 2, &rows, true);
  TORCH_CHECK_VALUE(grad.scalar_type() == rows.scalar_type() || grad.scalar_type() == ScalarType::Float,
                    "grad must be ", rows.scalar_type(), " or Float, got ", grad.scalar_type());
  want_shape("grad", grad, {row_of_route.size(0), rows.size(1)});
  const auto [gr, gw] = run_unpermute_grad(grad, rows, row_of_route, weights, need_rows, need_weights);
  return {gr.defined() ? OptTensor(gr) : std::nullopt, gw.defined() ? OptTensor(gw) : std::nullopt};
}

// ---------------------------------------------------------------- quantizers
float check_limit(const std::optional<double>& limit) {
  const double v = limit.value_or(std::numeric_limits<double>::infinity());
  TORCH_CHECK_VALUE(v > 0, "limit must be above 0 or None, got ", v);
  return float(v);
}

std::tuple<Tensor, Tensor> run_quantize(const Tensor& x, int64_t width, bool swiglu, float limit) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0);
  Tensor q = empty({rows, width}, kE4m3, x), scale = empty({rows, blocks(width)}, ScalarType::Float, x);
  if (rows)
    check("b200moe_fp8_quantize",
          b200moe_fp8_quantize(stream(x), x.data_ptr(), code(x.scalar_type()), x.stride(0), int(rows), int(width),
                               swiglu, limit, q.data_ptr(), f32_mut(scale)));
  return {q, scale};
}

std::tuple<Tensor, Tensor> quantize(const Tensor& x) {
  want("x", x, kFloats, 2, nullptr, true);
  TORCH_CHECK_VALUE(x.size(1) >= 1, "x must have columns, got ", x.sizes());
  return run_quantize(x, x.size(1), false, 1.f);
}

void check_gate_up(const Tensor& h) {
  want("h", h, kFloats, 2, nullptr, true);
  TORCH_CHECK_VALUE(h.size(1) >= 2 && h.size(1) % 2 == 0, "h must have gate and up columns, got ", h.sizes());
}

std::tuple<Tensor, Tensor> swiglu_quantize(const Tensor& h, const std::optional<double>& limit) {
  check_gate_up(h);
  return run_quantize(h, h.size(1) / 2, true, check_limit(limit));
}

Tensor swiglu_grad(const Tensor& h, const Tensor& grad, const std::optional<double>& limit_arg) {
  check_gate_up(h);
  const int64_t rows = h.size(0), width = h.size(1) / 2;
  want("grad", grad, kFloats, 2, &h, true);
  TORCH_CHECK_VALUE(grad.scalar_type() == h.scalar_type(), "grad must be ", h.scalar_type(), ", got ",
                    grad.scalar_type());
  want_shape("grad", grad, {rows, width});
  const float limit = check_limit(limit_arg);
  const c10::cuda::CUDAGuard guard(h.device());
  Tensor out = empty({rows, 2 * width}, h.scalar_type(), h);
  if (rows)
    check("b200moe_swiglu_grad",
          b200moe_swiglu_grad(stream(h), h.data_ptr(), code(h.scalar_type()), h.stride(0), grad.data_ptr(),
                              grad.stride(0), int(rows), int(width), limit, out.data_ptr()));
  return out;
}

// The quantizer and the transpose of weights launch a CTA per block: grids of at most 65535 matrices and row blocks.
void check_launch(const char* name, const Tensor& w) {
  constexpr int64_t most = 65535;
  TORCH_CHECK_VALUE((w.dim() == 2 || w.size(0) <= most) && blocks(w.size(-2)) <= most, name, " is too large: ", w.sizes());
}

std::tuple<Tensor, Tensor> quantize_weight(const Tensor& w) {
  const bool many = w.defined() && w.dim() == 3;
  want("w", w, kFloats, many ? 3 : 2);
  TORCH_CHECK_VALUE(w.numel() > 0, "w must not be empty, got ", w.sizes());
  check_launch("w", w);
  const c10::cuda::CUDAGuard guard(w.device());
  const int64_t n = w.size(-2), k = w.size(-1), mats = many ? w.size(0) : 1;
  Tensor q = empty(w.sizes(), kE4m3, w);
  Tensor scale = many ? empty({mats, blocks(n), blocks(k)}, ScalarType::Float, w)
                      : empty({blocks(n), blocks(k)}, ScalarType::Float, w);
  check("b200moe_fp8_quantize_weight",
        b200moe_fp8_quantize_weight(stream(w), w.data_ptr(), code(w.scalar_type()), int(mats), int(n), int(k),
                                    q.data_ptr(), f32_mut(scale)));
  return {q, scale};
}

// Packed weights [(E,) N, K] with their blocks' scales.
void check_weight(const char* name, const char* scale_name, const Tensor& w, const Tensor& scale, int64_t dim,
                  const Tensor* like) {
  want(name, w, kOnlyE4m3, dim, like);
  want(scale_name, scale, kF32, dim, &w);
  TORCH_CHECK_VALUE(w.numel() > 0, name, " must not be empty, got ", w.sizes());
  const int64_t nb = blocks(w.size(-2)), kb = blocks(w.size(-1));
  if (dim == 3)
    want_shape(scale_name, scale, {w.size(0), nb, kb});
  else
    want_shape(scale_name, scale, {nb, kb});
}

std::tuple<Tensor, Tensor> run_transpose(const Tensor& w, const Tensor& scale) {
  check_launch("w", w);
  const c10::cuda::CUDAGuard guard(w.device());
  const bool many = w.dim() == 3;
  const int64_t n = w.size(-2), k = w.size(-1), mats = many ? w.size(0) : 1;
  Tensor out = many ? empty({mats, k, n}, kE4m3, w) : empty({k, n}, kE4m3, w);
  Tensor out_scale = many ? empty({mats, blocks(k), blocks(n)}, ScalarType::Float, w)
                          : empty({blocks(k), blocks(n)}, ScalarType::Float, w);
  check("b200moe_fp8_transpose_weight",
        b200moe_fp8_transpose_weight(stream(w), w.data_ptr(), f32(scale), int(mats), int(n), int(k), out.data_ptr(),
                                     f32_mut(out_scale)));
  return {out, out_scale};
}

std::tuple<Tensor, Tensor> transpose_weight(const Tensor& w, const Tensor& scale) {
  check_weight("w", "w_scale", w, scale, w.defined() && w.dim() == 3 ? 3 : 2, nullptr);
  return run_transpose(w, scale);
}

// ------------------------------------------------------------------ products
void check_k(const Tensor& w, int64_t k) {
  TORCH_CHECK_VALUE(w.size(-1) == k, "w has ", w.size(-1), " columns, the rows ", k);
  TORCH_CHECK_VALUE(k % 16 == 0, "the product's K must be a multiple of 16, got ", k);
}
void check_out(ScalarType t) {
  TORCH_CHECK_VALUE(is_float(t), "out_dtype must be bfloat16, float16 or float32, got ", t);
}
void check_rows(const Tensor& q, const Tensor& scale) {
  want("q", q, kOnlyE4m3, 2);
  want("scale", scale, kF32, 2, &q, true);
  want_shape("scale", scale, {q.size(0), blocks(q.size(1))});
}

Tensor run_product(const Tensor& q, const Tensor& scale, const Tensor& offsets, const Tensor& w, const Tensor& w_scale,
                   ScalarType out_dtype) {
  const c10::cuda::CUDAGuard guard(q.device());
  const int64_t s = q.size(0), k = q.size(1), n = w.size(-2);
  Tensor out = empty({s, n}, out_dtype, q);
  if (s)
    check("b200moe_fp8_matmul",
          b200moe_fp8_matmul(stream(q), q.data_ptr(), f32(scale), scale.stride(0), w.data_ptr(), f32(w_scale),
                             offsets.defined() ? i32(offsets) : nullptr, int(s), int(n), int(k),
                             offsets.defined() ? int(w.size(0)) : 1, out.data_ptr(), code(out_dtype)));
  return out;
}

Tensor matmul(const Tensor& q, const Tensor& scale, const Tensor& w, const Tensor& w_scale, ScalarType out_dtype) {
  check_rows(q, scale);
  check_weight("w", "w_scale", w, w_scale, 2, &q);
  check_k(w, q.size(1));
  check_out(out_dtype);
  return run_product(q, scale, Tensor(), w, w_scale, out_dtype);
}

Tensor grouped_matmul(const Tensor& q, const Tensor& scale, const Tensor& offsets, const Tensor& w,
                      const Tensor& w_scale, ScalarType out_dtype) {
  check_rows(q, scale);
  check_weight("w", "w_scale", w, w_scale, 3, &q);
  check_k(w, q.size(1));
  check_out(out_dtype);
  want("offsets", offsets, kI32, 1, &q);
  want_shape("offsets", offsets, {w.size(0) + 1});
  TORCH_CHECK_VALUE(w.size(0) <= kMaxExperts && w.size(0) * w.size(1) <= INT32_MAX - 256, "at most ", kMaxExperts,
                    " experts and 2^31 weight rows, got ", w.sizes());
  return run_product(q, scale, offsets, w, w_scale, out_dtype);
}

Tensor run_linear(const Tensor& x, const Tensor& w, const Tensor& w_scale, ScalarType out_dtype) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
  Tensor out = empty({m, n}, out_dtype, x), ws;
  if (m == 0) return out;
  // room for the quantized rows and their scales; few rows are quantized inside the product's kernel
  int64_t bytes = m * (k + 4 * blocks(k)) + 16;
  if (x.scalar_type() != ScalarType::Float && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 &&
      x.stride(0) % 8 == 0)
    bytes = int64_t(b200moe_fp8_linear_workspace_bytes(int(m), int(n), int(k)));
  if (bytes) ws = empty({bytes}, ScalarType::Byte, x);
  check("b200moe_fp8_linear",
        b200moe_fp8_linear(stream(x), x.data_ptr(), code(x.scalar_type()), x.stride(0), w.data_ptr(), f32(w_scale),
                           int(m), int(n), int(k), out.data_ptr(), code(out_dtype), mut(ws), size_t(bytes)));
  return out;
}

struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& w_scale,
                        const OptTensor& wt, const OptTensor& wt_scale, ScalarType out_dtype) {
    ctx->save_for_backward({wt.value_or(w), wt_scale.value_or(w_scale)});
    ctx->saved_data["transposed"] = wt.has_value();
    ctx->saved_data["dtype"] = int64_t(x.scalar_type());
    return run_linear(x, w, w_scale, out_dtype);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_differentiable(grads[0]);
    const auto saved = ctx->get_saved_variables();
    Tensor wt = saved[0], wt_scale = saved[1];
    if (!ctx->saved_data["transposed"].toBool()) std::tie(wt, wt_scale) = run_transpose(wt, wt_scale);
    const auto dtype = ScalarType(ctx->saved_data["dtype"].toInt());
    return {run_linear(as_rows(grads[0]), wt, wt_scale, dtype), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor linear(const Tensor& x, const Tensor& w, const Tensor& w_scale, const OptTensor& wt_arg,
              const OptTensor& wt_scale_arg, const OptDtype& out_dtype) {
  const Tensor wt = wt_arg.value_or(Tensor()), wt_scale = wt_scale_arg.value_or(Tensor());
  want("x", x, kFloats, 2, nullptr, true);
  check_weight("w", "w_scale", w, w_scale, 2, &x);
  check_k(w, x.size(1));
  const ScalarType dtype = out_dtype.value_or(x.scalar_type());
  check_out(dtype);
  TORCH_CHECK_VALUE(wt.defined() == wt_scale.defined(), "wt and wt_scale come together");
  if (wt.defined()) {
    check_weight("wt", "wt_scale", wt, wt_scale, 2, &x);
    want_shape("wt", wt, {w.size(1), w.size(0)});
  }
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    TORCH_CHECK_VALUE(w.size(0) % 16 == 0, "the gradient's product needs N a multiple of 16, got ", w.size(0));
    return LinearFn::apply(x, w, w_scale, wt_arg, wt_scale_arg, dtype);
  }
  return run_linear(x, w, w_scale, dtype);
}

PyObject* g_error_class = nullptr;  // b200moe._lib.B200MoeError

}  // namespace

PYBIND11_MODULE(b200moe_ops, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const StatusError& e) {
      if (!g_error_class) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return;
      }
      const py::object err = py::reinterpret_borrow<py::object>(g_error_class)(e.where, e.status);
      PyErr_SetObject(g_error_class, err.ptr());
    }
  });
  m.def("set_error_class", [](const py::object& c) { g_error_class = c.inc_ref().ptr(); });
  m.def("check_weight", [](const std::string& name, const Tensor& w, const Tensor& scale) {
    check_weight(name.c_str(), (name + "_scale").c_str(), w, scale, 3, nullptr);
  });
  m.def("sort_routes", &sort_routes);
  m.def("permute", &permute);
  m.def("unpermute", &unpermute);
  m.def("unpermute_grad", &unpermute_grad);
  m.def("quantize", &quantize);
  m.def("swiglu_quantize", &swiglu_quantize);
  m.def("swiglu_grad", &swiglu_grad);
  m.def("quantize_weight", &quantize_weight);
  m.def("transpose_weight", &transpose_weight);
  m.def("matmul", &matmul);
  m.def("grouped_matmul", &grouped_matmul);
  m.def("linear", &linear);
}
