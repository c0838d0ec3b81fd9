// The dense operators' autograd layer: argument checks, allocation, and the autograd nodes
// of layer norm and the linear layer, over the C ABI in ictc_o2_b200.h.
//
// In C++ because these operators are called on a few rows as often as on millions: an
// autograd.Function in Python over ctypes took 58 us a training call beside the engine's
// own 65 us, more than the arithmetic of every call below about 10^9 operations.  The
// kernel library is loaded by the Python package, which hands its entry points to bind().
//
// The functions work on the tensors' memory, past PyTorch's dispatcher.  Where something
// watches the dispatcher (a trace, fake tensors, a functional transform) they go through
// the registered custom operators instead, as under torch.compile.
#include <ATen/autocast_mode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <cstdint>
#include <optional>
#include <string>
#include <tuple>

#include "ictc_o2_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
  decltype(&ictc_o2_last_error) last_error;
  decltype(&ictc_o2_layer_norm_forward) norm_forward;
  decltype(&ictc_o2_layer_norm_workspace) norm_workspace;
  decltype(&ictc_o2_layer_norm_backward) norm_backward;
  decltype(&ictc_o2_linear_workspace) linear_workspace;
  decltype(&ictc_o2_linear_forward) linear_forward;
  decltype(&ictc_o2_linear_backward) linear_backward;
};

Api api{};

// The custom operators in Python, which run the raw directions at the end of this file.
struct Ops {
  PyObject *norm_forward, *norm_backward, *linear_forward, *linear_backward;
};

Ops ops{};

template <typename Result, typename... Args>
Result through_dispatcher(PyObject* op, const Args&... args) {
  const py::gil_scoped_acquire gil;
  return py::reinterpret_borrow<py::object>(op)(args...).template cast<Result>();
}

// Whether a call on these tensors has to be seen by the dispatcher.
bool watched(std::initializer_list<const Tensor*> tensors) {
  using K = c10::DispatchKey;
  constexpr c10::DispatchKeySet kWatchers(
      {K::Python, K::Tracer, K::Functionalize, K::FuncTorchDynamicLayerFrontMode,
       K::FuncTorchBatched, K::FuncTorchGradWrapper});
  const auto local = c10::impl::tls_local_dispatch_key_set();
  c10::DispatchKeySet keys = local.included_;
  for (const Tensor* t : tensors)
    if (t->defined()) keys = keys | t->key_set();
  return !((keys - local.excluded_) & kWatchers).empty();
}

void check(int32_t status, const char* what) {
  if (status == ICTC_OK) return;
  const std::string message = std::string(what) + ": " + api.last_error();
  TORCH_CHECK_VALUE(status != ICTC_ERR_INVALID, message);
  TORCH_CHECK_NOT_IMPLEMENTED(status != ICTC_ERR_UNSUPPORTED, message);
  TORCH_CHECK(false, message);
}

// ------------------------------------------------------------------------- arguments

int32_t code_of(at::ScalarType t) {
  return t == at::kFloat ? ICTC_DTYPE_F32 : t == at::kBFloat16 ? ICTC_DTYPE_BF16 : ICTC_DTYPE_F16;
}

void check_input(const char* what, const Tensor& x) {
  const auto t = x.scalar_type();
  TORCH_CHECK_TYPE(x.is_cuda() && (t == at::kFloat || t == at::kBFloat16 || t == at::kHalf), what,
                   " runs only on CUDA float32, bfloat16 or float16 tensors (there is no CPU or "
                   "other-dtype fallback); got ", t, " on ", x.device());
}

void check_like(const char* what, const char* name, const Tensor& t, const Tensor& x,
                bool float32_too = false) {
  TORCH_CHECK_VALUE(t.device() == x.device(), what, ": ", name, " is on ", t.device(),
                    ", the input on ", x.device());
  TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type() ||
                        (float32_too && t.scalar_type() == at::kFloat),
                    what, ": ", name, " is ", t.scalar_type(), ", the input ", x.scalar_type());
}

// A dual tensor's tangent would be left out without a word.
void check_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what,
                                " has no forward-mode derivative");
}

void check_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps) {
  check_input("layer_norm", x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1,
                    "layer_norm needs a last dimension of at least one element");
  TORCH_CHECK_VALUE(eps >= 0, "eps must be >= 0");
  const auto one = [&](const char* name, const Tensor& t) {
    if (!t.defined()) return;
    check_like("layer_norm", name, t, x, true);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == x.size(-1), "layer_norm: ", name,
                      " must have shape [", x.size(-1), "], got ", t.sizes());
  };
  one("weight", weight);
  one("bias", bias);
  TORCH_CHECK_VALUE(!weight.defined() || !bias.defined() ||
                        weight.scalar_type() == bias.scalar_type(),
                    "layer_norm: weight and bias must have the same type");
}

void check_linear(const Tensor& x, const Tensor& weight, const Tensor& bias,
                  const Tensor& residual, int64_t code) {
  check_input("linear", x);
  TORCH_CHECK_VALUE(code >= ICTC_ACT_NONE && code <= ICTC_ACT_GELU_TANH, "unknown activation");
  TORCH_CHECK_VALUE(weight.dim() == 2 && x.dim() >= 1 && x.size(-1) == weight.size(1),
                    "linear: x [..., in] and weight [out, in] do not match: ", x.sizes(), " and ",
                    weight.sizes());
  TORCH_CHECK_VALUE(weight.size(0) >= 1 && weight.size(1) >= 1,
                    "linear needs at least one input and one output feature");
  check_like("linear", "weight", weight, x);
  if (bias.defined()) {
    check_like("linear", "bias", bias, x);
    TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == weight.size(0),
                      "linear: bias must have shape [", weight.size(0), "], got ", bias.sizes());
  }
  if (residual.defined()) {
    check_like("linear", "residual", residual, x);
    bool same = residual.dim() == x.dim() && residual.size(-1) == weight.size(0);
    for (int64_t i = 0; same && i + 1 < x.dim(); ++i) same = residual.size(i) == x.size(i);
    TORCH_CHECK_VALUE(same, "linear: residual must have the output's shape, got ",
                      residual.sizes());
  }
}

// [rows, width] with unit stride inside a row; copies only when it must.  (A view whose
// sign is flipped by a bit on the tensor, such as the imaginary part of a conjugate, has
// other values than its memory.)
Tensor rows_of(const Tensor& t) {
  if (t.is_neg()) return rows_of(t.resolve_neg());
  const int64_t width = t.size(-1);
  if (t.dim() == 2 && (width == 1 || t.stride(1) == 1)) return t;
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
  const Tensor flat = t.dim() == 2 ? t : t.reshape({rows, width});
  return width == 1 || flat.stride(1) == 1 ? flat : flat.contiguous();
}

Tensor packed(const Tensor& t) { return t.defined() ? t.resolve_neg().contiguous() : t; }

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

float* floats(const Tensor& t) { return static_cast<float*>(data(t)); }

Tensor scratch(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte))
               : Tensor();
}

void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

// ------------------------------------------------------------------------ layer norm

std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& weight_in,
                                                const Tensor& bias_in, double eps, bool stats) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor rows = rows_of(x), weight = packed(weight_in), bias = packed(bias_in);
  const Tensor y = at::empty(x.sizes(), x.options());
  Tensor mean, rstd;
  if (stats) {
    mean = at::empty({rows.size(0)}, x.options().dtype(at::kFloat));
    rstd = at::empty({rows.size(0)}, x.options().dtype(at::kFloat));
  }
  const Tensor& p = weight.defined() ? weight : bias.defined() ? bias : x;
  check(api.norm_forward(rows.data_ptr(), rows.stride(0), data(weight), data(bias), y.data_ptr(),
                         floats(mean), floats(rstd), rows.size(0), rows.size(1),
                         static_cast<float>(eps), code_of(x.scalar_type()),
                         code_of(p.scalar_type()), stream_of(x)),
        "layer_norm_forward");
  return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> norm_backward(const Tensor& x, const Tensor& weight_in,
                                                 const Tensor& mean, const Tensor& rstd,
                                                 const Tensor& grad, at::ScalarType params,
                                                 bool need_x, bool need_w, bool need_b) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor rows = rows_of(x), g = rows_of(grad), weight = packed(weight_in);
  const int64_t width = x.size(-1);
  const int32_t dtype = code_of(x.scalar_type());
  Tensor dx, dw, db;
  if (need_x) dx = at::empty(x.sizes(), x.options());
  if (need_w) dw = at::empty({width}, x.options().dtype(params));
  if (need_b) db = at::empty({width}, x.options().dtype(params));
  size_t bytes = 0;
  if (need_w || need_b)
    check(api.norm_workspace(rows.size(0), width, dtype, x.device().index(), &bytes),
          "layer_norm_workspace");
  const Tensor space = scratch(bytes, x);
  check(api.norm_backward(rows.data_ptr(), rows.stride(0), data(weight), floats(mean),
                          floats(rstd), g.data_ptr(), g.stride(0), data(dx), data(dw), data(db),
                          data(space), bytes, rows.size(0), width, dtype, code_of(params),
                          stream_of(x)),
        "layer_norm_backward");
  return {dx, dw, db};
}

Tensor wanted(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

std::optional<Tensor> given(const Tensor& t) {
  return t.defined() ? std::optional<Tensor>(t) : std::nullopt;
}

class LayerNormFunction : public torch::autograd::Function<LayerNormFunction> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x,
                        const std::optional<Tensor>& weight_in,
                        const std::optional<Tensor>& bias_in, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor weight = wanted(weight_in), bias = wanted(bias_in);
    auto [y, mean, rstd] = norm_forward(x, weight, bias, eps, true);
    ctx->save_for_backward({x, weight, mean, rstd});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["has_bias"] = bias.defined();
    ctx->saved_data["params"] = static_cast<int64_t>(
        (weight.defined() ? weight : bias.defined() ? bias : x).scalar_type());
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor& grad = grads[0];
    if (!grad.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1];
    const auto params = static_cast<at::ScalarType>(ctx->saved_data["params"].toInt());
    // inputs are counted without those that were not given
    const bool nx = ctx->needs_input_grad(0);
    const bool nw = weight.defined() && ctx->needs_input_grad(1);
    const bool nb = ctx->saved_data["has_bias"].toBool() &&
                    ctx->needs_input_grad(weight.defined() ? 2 : 1);
    if (!at::GradMode::is_enabled()) {
      if (watched({&grad, &x, &weight})) {
        const auto [dx, dw, db] = through_dispatcher<std::tuple<Tensor, Tensor, Tensor>>(
            ops.norm_backward, x, weight, saved[2], saved[3], grad, params == at::kFloat);
        return {nx ? dx : Tensor(), nw ? dw : Tensor(), nb ? db : Tensor(), Tensor()};
      }
      auto [dx, dw, db] =
          norm_backward(x, weight, saved[2], saved[3], grad, params, nx, nw, nb);
      return {dx, dw, db, Tensor()};
    }
    // second derivatives: the formula in differentiable operations
    const double eps = ctx->saved_data["eps"].toDouble();
    const Tensor xf = x.to(at::kFloat), g = grad.to(at::kFloat);
    const Tensor centred = xf - xf.mean(-1, true);
    const Tensor rstd = (centred.square().mean(-1, true) + eps).rsqrt();
    const Tensor u = centred * rstd;
    const Tensor h = weight.defined() ? g * weight.to(at::kFloat) : g;
    const Tensor dx = rstd * (h - h.mean(-1, true) - u * (h * u).mean(-1, true));
    const auto columns = [&](const Tensor& t) {
      return t.reshape({-1, x.size(-1)}).sum(0).to(params);
    };
    return {nx ? dx.to(x.scalar_type()) : Tensor(), nw ? columns(g * u) : Tensor(),
            nb ? columns(g) : Tensor(), Tensor()};
  }
};

bool any_grad(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight_in,
                  const std::optional<Tensor>& bias_in, double eps) {
  const Tensor weight = wanted(weight_in), bias = wanted(bias_in);
  check_norm(x, weight, bias, eps);
  check_tangents("layer_norm", {&x, &weight, &bias});
  if (watched({&x, &weight, &bias}))
    return std::get<0>(through_dispatcher<std::tuple<Tensor, Tensor, Tensor>>(
        ops.norm_forward, x, weight, bias, eps));
  if (any_grad({&x, &weight, &bias})) return LayerNormFunction::apply(x, given(weight), given(bias), eps);
  return std::get<0>(norm_forward(x, weight, bias, eps, false));
}

// ---------------------------------------------------------------------------- linear

// What the operands' row starts allow (the C ABI's layout flags).
int32_t layout_of(const Tensor& x, const Tensor& w, const Tensor* g) {
  const int64_t block = 16 / x.element_size();
  const auto start = [](const Tensor& t) {
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  };
  bool aligned = start(w) && w.stride(0) % block == 0, packed_rows = true;
  for (const Tensor* t : {&x, g}) {
    if (!t) continue;
    aligned = aligned && start(*t) && t->stride(0) % block == 0;
    packed_rows = packed_rows && start(*t) && (t->stride(0) == t->size(1) || t->size(0) <= 1);
  }
  return (aligned ? ICTC_LINEAR_ALIGNED : 0) | (packed_rows ? ICTC_LINEAR_PACKED : 0);
}

std::tuple<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& weight,
                                          const Tensor& bias_in, const Tensor& residual,
                                          int64_t code, bool save) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor rows = rows_of(x), w = rows_of(weight), bias = packed(bias_in);
  const Tensor r = residual.defined() ? rows_of(residual) : Tensor();
  const int64_t m = rows.size(0), k = rows.size(1), n = w.size(0);
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  const Tensor y = at::empty(shape, x.options());
  Tensor preact;
  if (save) preact = at::empty({m, n}, x.options().dtype(at::kFloat));
  const int32_t dtype = code_of(x.scalar_type()), act = static_cast<int32_t>(code);
  size_t bytes = 0, other = 0;
  check(api.linear_workspace(m, k, n, dtype, act, layout_of(rows, w, nullptr),
                             x.device().index(), &bytes, &other),
        "linear_workspace");
  const Tensor space = scratch(bytes, x);
  check(api.linear_forward(rows.data_ptr(), rows.stride(0), w.data_ptr(), w.stride(0), data(bias),
                           data(r), r.defined() ? r.stride(0) : 0, y.data_ptr(), floats(preact),
                           data(space), bytes, m, k, n, dtype, act, stream_of(x)),
        "linear_forward");
  return {y, preact};
}

std::tuple<Tensor, Tensor, Tensor> linear_backward(const Tensor& x, const Tensor& weight,
                                                   const Tensor& preact, const Tensor& grad,
                                                   int64_t code, bool need_x, bool need_w,
                                                   bool need_b) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor rows = rows_of(x), w = rows_of(weight), g = rows_of(grad);
  const int64_t m = rows.size(0), k = rows.size(1), n = w.size(0);
  Tensor dx, dw, db;
  if (need_x) dx = at::empty(x.sizes(), x.options());
  if (need_w) dw = at::empty({n, k}, x.options());
  if (need_b) db = at::empty({n}, x.options());
  const int32_t dtype = code_of(x.scalar_type()), act = static_cast<int32_t>(code);
  size_t bytes = 0, other = 0;
  check(api.linear_workspace(m, k, n, dtype, act, layout_of(rows, w, &g), x.device().index(),
                             &other, &bytes),
        "linear_workspace");
  const Tensor space = scratch(bytes, x);
  check(api.linear_backward(rows.data_ptr(), rows.stride(0), w.data_ptr(), w.stride(0),
                            floats(preact), g.data_ptr(), g.stride(0), data(dx), data(dw),
                            data(db), data(space), bytes, m, k, n, dtype, act, stream_of(x)),
        "linear_backward");
  return {dx, dw, db};
}

// act'(p) in differentiable operations.
Tensor slope_formula(const Tensor& p, int64_t code) {
  if (code == ICTC_ACT_RELU) return (p > 0).to(p.scalar_type());
  if (code == ICTC_ACT_SILU) {
    const Tensor s = p.sigmoid();
    return s * (1 + p * (1 - s));
  }
  if (code == ICTC_ACT_GELU)
    return 0.5 * (1 + (p * M_SQRT1_2).erf()) + p * (-0.5 * p * p).exp() * (M_2_SQRTPI * M_SQRT1_2 / 2);
  const double c = M_2_SQRTPI * M_SQRT1_2;  // sqrt(2 / pi)
  const Tensor t = (c * (p + 0.044715 * p * p * p)).tanh();
  return 0.5 * (1 + t) + 0.5 * p * (1 - t * t) * c * (1 + 3 * 0.044715 * p * p);
}

Tensor linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_in,
              const std::optional<Tensor>& residual_in, int64_t code);

// `value` with the derivatives of p, which has the same value but for its rounding.
class ValueOf : public torch::autograd::Function<ValueOf> {
 public:
  static Tensor forward(AutogradContext*, const Tensor&, const Tensor& value) {
    at::AutoDispatchBelowADInplaceOrView below;
    return at::alias(value);
  }
  static variable_list backward(AutogradContext*, variable_list grads) {
    return {grads[0], Tensor()};
  }
};

class LinearFunction : public torch::autograd::Function<LinearFunction> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                        const std::optional<Tensor>& bias_in,
                        const std::optional<Tensor>& residual_in, int64_t code) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor bias = wanted(bias_in), residual = wanted(residual_in);
    auto [y, preact] = linear_forward(x, weight, bias, residual, code, code != ICTC_ACT_NONE);
    ctx->save_for_backward({x, weight, bias, preact});
    ctx->saved_data["code"] = code;
    ctx->saved_data["has_residual"] = residual.defined();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor& grad = grads[0];
    if (!grad.defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1];
    const int64_t code = ctx->saved_data["code"].toInt();
    const bool has_bias = saved[2].defined();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1);
    const bool nb = has_bias && ctx->needs_input_grad(2);
    const bool nr = ctx->saved_data["has_residual"].toBool() &&
                    ctx->needs_input_grad(has_bias ? 3 : 2);
    const Tensor dr = nr ? grad : Tensor();
    if (!nx && !nw && !nb) return {Tensor(), Tensor(), Tensor(), dr, Tensor()};
    if (!at::GradMode::is_enabled()) {
      if (watched({&grad, &x, &weight})) {
        const Tensor preact =
            saved[3].defined() ? saved[3] : at::empty({0}, x.options().dtype(at::kFloat));
        const auto [dx, dw, db] = through_dispatcher<std::tuple<Tensor, Tensor, Tensor>>(
            ops.linear_backward, x, weight, preact, grad, code);
        return {nx ? dx : Tensor(), nw ? dw : Tensor(), nb ? db : Tensor(), dr, Tensor()};
      }
      auto [dx, dw, db] = linear_backward(x, weight, saved[3], grad, code, nx, nw, nb);
      return {dx, dw, db, dr, Tensor()};
    }
    // second derivatives: a differentiable composition whose products are linear layers
    // again, on the same kernels
    const Tensor rows = rows_of(x);
    Tensor d = rows_of(grad), wide = d.to(at::kFloat);
    if (code != ICTC_ACT_NONE) {
      // p again, for its graph; in 16-bit types it is rounded, so the float32 p that the
      // forward kept is where the slope is taken, as in the kernels
      const Tensor p = linear(rows, weight, given(saved[2]), std::nullopt, ICTC_ACT_NONE);
      wide = wide * slope_formula(ValueOf::apply(p.to(at::kFloat), saved[3]), code);
      d = wide.to(x.scalar_type());
    }
    const auto product = [](const Tensor& a, const Tensor& b) {
      return linear(a, b, std::nullopt, std::nullopt, ICTC_ACT_NONE);
    };
    return {nx ? product(d, weight.t()).reshape(x.sizes()) : Tensor(),
            // a sum over no rows is no linear layer, but has its (zero) value and graph
            nw ? (rows.size(0) > 0 ? product(d.t(), rows.t()) : at::matmul(d.t(), rows)) : Tensor(),
            nb ? wide.sum(0).to(x.scalar_type()) : Tensor(), dr, Tensor()};
  }
};

// Under autocast, operands of different types take autocast's; equal ones are left alone.
bool cast_mixed(std::initializer_list<Tensor*> tensors) {
  const auto first = (*tensors.begin())->scalar_type();
  bool mixed = false;
  for (const Tensor* t : tensors) mixed |= t->defined() && t->scalar_type() != first;
  if (!mixed || !at::autocast::is_autocast_enabled(at::kCUDA)) return false;
  for (const Tensor* t : tensors) {
    if (!t->defined()) continue;
    const auto type = t->scalar_type();
    if (!t->is_cuda() || (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf))
      return false;
  }
  const auto type = at::autocast::get_autocast_dtype(at::kCUDA);
  for (Tensor* t : tensors)
    if (t->defined()) *t = t->to(type);
  return true;
}

Tensor linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_in,
              const std::optional<Tensor>& residual_in, int64_t code) {
  const Tensor bias = wanted(bias_in), residual = wanted(residual_in);
  Tensor cast[4] = {x, weight, bias, residual};
  if (cast_mixed({&cast[0], &cast[1], &cast[2], &cast[3]}))
    return linear(cast[0], cast[1], given(cast[2]), given(cast[3]), code);
  check_linear(x, weight, bias, residual, code);
  check_tangents("linear", {&x, &weight, &bias, &residual});
  const bool grad = any_grad({&x, &weight, &bias, &residual});
  if (watched({&x, &weight, &bias, &residual}))
    return std::get<0>(through_dispatcher<std::tuple<Tensor, Tensor>>(
        ops.linear_forward, x, weight, bias, residual, code, grad && code != ICTC_ACT_NONE));
  if (grad)
    return LinearFunction::apply(x, weight, given(bias), given(residual), code);
  return std::get<0>(linear_forward(x, weight, bias, residual, code, false));
}

// ---------------------------------------------- raw directions, for the custom operators

std::tuple<Tensor, Tensor, Tensor> norm_forward_op(const Tensor& x,
                                                   const std::optional<Tensor>& weight,
                                                   const std::optional<Tensor>& bias, double eps) {
  check_norm(x, wanted(weight), wanted(bias), eps);
  return norm_forward(x, wanted(weight), wanted(bias), eps, true);
}

std::tuple<Tensor, Tensor, Tensor> norm_backward_op(const Tensor& x,
                                                    const std::optional<Tensor>& weight,
                                                    const Tensor& mean, const Tensor& rstd,
                                                    const Tensor& grad, bool float_params) {
  return norm_backward(x, wanted(weight), mean, rstd, grad,
                       float_params ? at::kFloat : x.scalar_type(), true, true, true);
}

std::tuple<Tensor, Tensor> linear_forward_op(const Tensor& x, const Tensor& weight,
                                             const std::optional<Tensor>& bias,
                                             const std::optional<Tensor>& residual, int64_t code,
                                             bool save) {
  check_linear(x, weight, wanted(bias), wanted(residual), code);
  auto [y, preact] = linear_forward(x, weight, wanted(bias), wanted(residual), code, save);
  if (!save) preact = at::empty({0}, x.options().dtype(at::kFloat));
  return {y, preact};
}

std::tuple<Tensor, Tensor, Tensor> linear_backward_op(const Tensor& x, const Tensor& weight,
                                                      const Tensor& preact, const Tensor& grad,
                                                      int64_t code) {
  return linear_backward(x, weight, code == ICTC_ACT_NONE ? Tensor() : preact, grad, code, true,
                         true, true);
}

// The custom operators, held for the life of the process.
void bind_operators(py::object norm_fwd, py::object norm_bwd, py::object linear_fwd,
                    py::object linear_bwd) {
  ops = {norm_fwd.release().ptr(), norm_bwd.release().ptr(), linear_fwd.release().ptr(),
         linear_bwd.release().ptr()};
}

// Entry points of the loaded kernel library, by address.
void bind(uintptr_t last_error, uintptr_t norm_fwd, uintptr_t norm_ws, uintptr_t norm_bwd,
          uintptr_t linear_ws, uintptr_t linear_fwd, uintptr_t linear_bwd) {
  const auto set = [](auto& fn, uintptr_t at) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at); };
  set(api.last_error, last_error);
  set(api.norm_forward, norm_fwd);
  set(api.norm_workspace, norm_ws);
  set(api.norm_backward, norm_bwd);
  set(api.linear_workspace, linear_ws);
  set(api.linear_forward, linear_fwd);
  set(api.linear_backward, linear_bwd);
}

}  // namespace

PYBIND11_MODULE(_dense_autograd, m) {
  m.def("bind", &bind);
  m.def("bind_operators", &bind_operators);
  m.def("layer_norm", &layer_norm);
  m.def("linear", &linear);
  m.def("norm_forward", &norm_forward_op);
  m.def("norm_backward", &norm_backward_op);
  m.def("linear_forward", &linear_forward_op);
  m.def("linear_backward", &linear_backward_op);
}
