// torch.ops.st.* of a query tower's layers: layer norm, dropout, their sum with
// a residual, rows held in 8 bits and their products.  No reference
// counterparts.
//
// As in torch_head_ops.cpp, GPU tensors run on their device's current stream and
// CPU tensors are copied to the current GPU and the results back.  What a tower
// is trained through carries its gradients (Autograd key); the 8-bit operators
// refuse to be differentiated.  Below that key every kernel is called through the
// dispatcher, so that a dispatch mode sees it: a pass that keeps something for its
// gradients is an operator of its own (_with_state, _with_stats), and so is
// layer_norm_backward.
#include <torch/library.h>

#include "torch_autograd.hpp"

namespace {

using at::Tensor;
using st_torch::bytes_or_null;
using st_torch::check_st;
using st_torch::current_stream;
using st_torch::data_or_null;
using st_torch::find_op;
using st_torch::gpu_for_cpu_call;
using st_torch::if_defined;
using st_torch::moved;
using st_torch::OnceDifferentiable;
using st_torch::OptTensor;
using st_torch::refuse_tangents;
using st_torch::score_type;
using st_torch::with_adjacent_columns;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Pair = std::tuple<Tensor, Tensor>;
using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;

constexpr int64_t kMaxNormColumns = 32768;

Tensor given(const OptTensor& t) { return t.value_or(Tensor()); }

// The rows of a tensor of any shape, [rows, columns], columns adjacent.
Tensor as_rows(const Tensor& t) {
  if (t.dim() == 2) return with_adjacent_columns(t);
  const int64_t columns = t.size(-1);
  return t.contiguous().view({t.numel() / columns, columns});
}

// `t` on d; what is there already does not go through the dispatcher, which counts
// where a pass is a few launches.
Tensor placed(const Tensor& t, at::Device d) { return !t.defined() || t.device() == d ? t : t.to(d); }

// A gradient as the kernels take it.
Tensor grad_rows(const Tensor& g, at::ScalarType type, at::Device d) {
  const Tensor t = placed(g, d);
  return !t.defined() || (t.scalar_type() == type && t.is_contiguous()) ? t : t.to(type).contiguous();
}

Tensor back(const Tensor& t, bool on_gpu) { return t.defined() && !on_gpu ? t.cpu() : t; }

bool requires_grad(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

void refuse_tangents_of(std::initializer_list<const Tensor*> inputs, const char* op) {
  for (const Tensor* t : inputs)
    if (t->defined()) refuse_tangents({t}, op);
}

Tensor differentiable_once(const Tensor& grad, const Tensor& of, const Tensor& weight, const variable_list& outer,
                           const char* op) {
  if (!at::GradMode::is_enabled() || !grad.defined()) return grad;
  return OnceDifferentiable::apply(grad, of, if_defined(weight), if_defined(outer[0]),
                                   outer.size() > 1 ? if_defined(outer[1]) : OptTensor(), OptTensor(), std::string(op));
}

// ------------------------------------------ dropout

void check_dropout(const Tensor& x, double p, const Tensor& state, const char* op) {
  TORCH_CHECK(p >= 0.0 && p <= 1.0, "p must be in [0, 1], got ", p);
  TORCH_CHECK(!state.defined() || (state.dim() == 1 && state.size(0) == 2 && state.scalar_type() == at::kLong),
              "state must be an int64 tensor of 2: seed and offset");
  TORCH_CHECK(!state.defined() || state.device() == x.device(), op, " inputs must be on one device");
}

// (result, the state that was used if `with_used`)
Pair dropout_gpu(const Tensor& x_in, double p, const Tensor& state_in, bool with_used) {
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x_in.device());
  const Tensor x = x_in.contiguous(), state = state_in.contiguous();
  Tensor y = at::empty(x.sizes(), x.options()), used;
  if (with_used) used = at::empty({2}, state.options());
  check_st(st_dropout(bytes_or_null(x), score_type(x.scalar_type(), "x"), x.numel(), p, data_or_null<int64_t>(state),
                      bytes_or_null(y), data_or_null<int64_t>(used), current_stream(x)),
           "dropout");
  return {y, used};
}

Pair dropout_any(const Tensor& x, double p, const Tensor& state, bool with_used) {
  score_type(x.scalar_type(), "x");
  check_dropout(x, p, state, "dropout");
  if (x.is_cuda()) return dropout_gpu(x, p, state, with_used);
  const at::Device gpu = gpu_for_cpu_call();
  auto [y, used] = dropout_gpu(x.to(gpu), p, state.to(gpu), with_used);
  return {y.cpu(), back(used, false)};
}

Tensor dropout(const Tensor& x, double p, const Tensor& state) { return std::get<0>(dropout_any(x, p, state, false)); }

Pair dropout_with_state(const Tensor& x, double p, const Tensor& state) { return dropout_any(x, p, state, true); }

using DropoutOp = Tensor(const Tensor&, double, const Tensor&);
using DropoutKeepOp = Pair(const Tensor&, double, const Tensor&);

Tensor dropout_below(const Tensor& x, double p, const Tensor& state) {
  static const auto op = find_op<DropoutOp>("st::dropout");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, p, state);
}

Pair dropout_with_state_below(const Tensor& x, double p, const Tensor& state) {
  static const auto op = find_op<DropoutKeepOp>("st::dropout_with_state");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, p, state);
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, const Tensor& state) {
    auto [y, used] = dropout_with_state_below(x, p, state);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({used});
    ctx->saved_data["p"] = p;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor grad;
    if (grads[0].defined()) grad = dropout_below(grads[0], ctx->saved_data["p"].toDouble(), ctx->get_saved_variables()[0]);
    return {differentiable_once(grad, grads[0], Tensor(), grads, "dropout"), Tensor(), Tensor()};
  }
};

Tensor dropout_autograd(const Tensor& x, double p, const Tensor& state) {
  refuse_tangents({&x}, "dropout");
  return requires_grad({&x}) ? DropoutFunction::apply(x, p, state) : dropout_below(x, p, state);
}

// ------------------------------------------ layer norm

void check_weights(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, const char* op) {
  TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
  score_type(x.scalar_type(), "x");
  const int64_t dim = x.size(-1);
  TORCH_CHECK(dim >= 1 && dim <= kMaxNormColumns, "x must have between 1 and ", kMaxNormColumns, " columns, got ", dim);
  for (const Tensor* t : {&weight, &bias}) {
    if (!t->defined()) continue;
    score_type(t->scalar_type(), "weight and bias");
    TORCH_CHECK(t->dim() == 1 && t->size(0) == dim, "weight and bias must have one entry for each of ", dim,
                " columns, got ", t->sizes());
    TORCH_CHECK(t->device() == x.device(), op, " inputs must be on one device");
  }
  TORCH_CHECK(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(),
              "weight and bias must be of one type");
  TORCH_CHECK(eps >= 1e-30 && eps <= 1e30, "eps must be in [1e-30, 1e30], got ", eps);
}

int weights_type(const Tensor& weight, const Tensor& bias) {
  if (weight.defined()) return score_type(weight.scalar_type(), "weight");
  return bias.defined() ? score_type(bias.scalar_type(), "bias") : ST_SCORE_F32;
}

struct NormIn {
  Tensor x, residual, weight, bias, state;  // all but x may be undefined
  double p, eps;
};

struct NormOut {
  Tensor y, sum, stats, used;
};

void check_norm(const NormIn& in, const char* op) {
  check_weights(in.x, in.weight, in.bias, in.eps, op);
  if (!in.residual.defined()) return;
  score_type(in.residual.scalar_type(), "residual");
  TORCH_CHECK(in.residual.sizes() == in.x.sizes(), "residual must be of x's shape ", in.x.sizes(), ", got ",
              in.residual.sizes());
  TORCH_CHECK(in.residual.scalar_type() == in.x.scalar_type() || in.residual.scalar_type() == at::kFloat,
              "residual must be of x's type or float32, got ", in.residual.scalar_type());
  TORCH_CHECK(in.residual.device() == in.x.device(), op, " inputs must be on one device");
  check_dropout(in.x, in.p, in.state, op);
  TORCH_CHECK(in.p == 0.0 || in.state.defined(), "dropout needs a state");
}

NormOut norm_gpu(const NormIn& in, bool with_grad) {
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(in.x.device());
  const Tensor x = as_rows(in.x);
  Tensor residual, weight, bias, state;
  if (in.residual.defined()) residual = as_rows(in.residual);
  if (in.weight.defined()) weight = in.weight.contiguous();
  if (in.bias.defined()) bias = in.bias.contiguous();
  if (in.p > 0.0) state = in.state.contiguous();
  const int64_t rows = x.size(0), dim = x.size(1);
  NormOut o{at::empty(in.x.sizes(), x.options()), Tensor(), Tensor(), Tensor()};
  if (residual.defined()) o.sum = at::empty(in.x.sizes(), residual.options());
  if (with_grad) o.stats = at::empty({rows, ST_NORM_STATS}, x.options().dtype(at::kFloat));
  if (with_grad && state.defined()) o.used = at::empty({2}, state.options());
  check_st(st_layer_norm(bytes_or_null(x), score_type(x.scalar_type(), "x"), rows, dim, x.stride(0),
                         residual.defined() ? bytes_or_null(residual) : nullptr,
                         residual.defined() ? score_type(residual.scalar_type(), "residual") : ST_SCORE_F32,
                         residual.defined() ? residual.stride(0) : 0, bytes_or_null(weight), bytes_or_null(bias),
                         weights_type(weight, bias), in.eps, in.residual.defined() && rows > 0 ? in.p : 0.0,
                         data_or_null<int64_t>(state), bytes_or_null(o.y), bytes_or_null(o.sum),
                         data_or_null<float>(o.stats), data_or_null<int64_t>(o.used), current_stream(x)),
           "layer_norm");
  return o;
}

NormIn moved_in(const NormIn& in, at::Device d) {
  auto to = [&](const Tensor& t) { return t.defined() ? t.to(d) : t; };
  return {to(in.x), to(in.residual), to(in.weight), to(in.bias), to(in.state), in.p, in.eps};
}

NormOut norm_any(const NormIn& in, bool with_grad, const char* op) {
  check_norm(in, op);
  if (in.x.is_cuda()) return norm_gpu(in, with_grad);
  NormOut o = norm_gpu(moved_in(in, gpu_for_cpu_call()), with_grad);
  for (Tensor* t : {&o.y, &o.sum, &o.stats, &o.used}) *t = back(*t, false);
  return o;
}

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  return norm_any({x, Tensor(), given(weight), given(bias), Tensor(), 0.0, eps}, false, "layer_norm").y;
}

Pair layer_norm_with_stats(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  NormOut o = norm_any({x, Tensor(), given(weight), given(bias), Tensor(), 0.0, eps}, true, "layer_norm");
  return {o.y, o.stats};
}

Pair dropout_add_layer_norm(const Tensor& x, const Tensor& residual, const OptTensor& weight, const OptTensor& bias,
                            double p, const OptTensor& state, double eps) {
  NormOut o = norm_any({x, residual, given(weight), given(bias), given(state), p, eps}, false, "dropout_add_layer_norm");
  return {o.y, o.sum};
}

Four dropout_add_layer_norm_with_stats(const Tensor& x, const Tensor& residual, const OptTensor& weight,
                                       const OptTensor& bias, double p, const OptTensor& state, double eps) {
  NormOut o = norm_any({x, residual, given(weight), given(bias), given(state), p, eps}, true, "dropout_add_layer_norm");
  return {o.y, o.sum, o.stats, o.used};
}

void check_gradients(const Tensor& h, at::ScalarType y_type, const Tensor& weight, at::ScalarType weights,
                     const Tensor& stats, double p, const Tensor& used, const Tensor& grad_y, const Tensor& grad_sum) {
  check_weights(h, weight, Tensor(), 1.0, "layer_norm_backward");
  score_type(y_type, "x");
  score_type(weights, "weight and bias");
  TORCH_CHECK(!weight.defined() || weight.scalar_type() == weights, "weight must be of weight_type ", weights, ", got ",
              weight.scalar_type());
  TORCH_CHECK(h.scalar_type() == y_type || h.scalar_type() == at::kFloat, "the sum must be of x's type or float32, got ",
              h.scalar_type());
  TORCH_CHECK(stats.dim() == 2 && stats.size(0) == h.numel() / h.size(-1) && stats.size(1) == ST_NORM_STATS &&
                  stats.scalar_type() == at::kFloat && stats.device() == h.device(),
              "stats must be float32 [rows, ", ST_NORM_STATS, "] of the forward pass, got ", stats.sizes());
  for (const Tensor* t : {&grad_y, &grad_sum})
    TORCH_CHECK(!t->defined() || (t->sizes() == h.sizes() && t->device() == h.device()),
                "gradients must be of the results' shape ", h.sizes(), " and device");
  check_dropout(h, p, used, "layer_norm_backward");
  TORCH_CHECK(p == 0.0 || used.defined(), "dropout needs the state that was used");
}

// h: x, or the sum; used: the state that the forward pass used, if it dropped.  The
// gradients come on h's device, undefined where they are not wanted.
Four layer_norm_backward(const OptTensor& grad_y_in, const OptTensor& grad_sum_in, const Tensor& h_in,
                         const OptTensor& weight_opt, const Tensor& stats_in, const OptTensor& used_opt, double p,
                         at::ScalarType y_type, at::ScalarType weights, std::array<bool, 4> wanted) {
  const Tensor grad_y = given(grad_y_in), grad_sum = given(grad_sum_in), weight_in = given(weight_opt), used_in = given(used_opt);
  check_gradients(h_in, y_type, weight_in, weights, stats_in, p, used_in, grad_y, grad_sum);
  const bool on_gpu = h_in.is_cuda();
  const at::Device dev = on_gpu ? h_in.device() : gpu_for_cpu_call();
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(dev);
  const Tensor h = as_rows(placed(h_in, dev)), stats = placed(stats_in, dev).contiguous();
  Tensor used;
  if (used_in.defined()) used = placed(used_in, dev).contiguous();
  const int64_t rows = h.size(0), dim = h.size(1);
  const auto options = h.options();
  Tensor weight;
  if (weight_in.defined()) weight = placed(weight_in, dev).contiguous();
  // without a gradient of its own the norm's result has one of zeros
  const Tensor gy = grad_y.defined() ? grad_rows(grad_y, y_type, dev) : at::zeros(h_in.sizes(), options.dtype(y_type));
  const Tensor gsum = grad_rows(grad_sum, h.scalar_type(), dev);
  Tensor gx, gr, gw, gb, ws;
  if (wanted[0]) gx = at::empty(h_in.sizes(), options.dtype(y_type));
  if (wanted[1]) gr = at::empty(h_in.sizes(), options);
  if (wanted[2]) gw = at::empty({dim}, options.dtype(weights));
  if (wanted[3]) gb = at::empty({dim}, options.dtype(weights));
  if (wanted[2] || wanted[3])
    ws = at::empty({st_layer_norm_workspace_bytes(rows, dim)}, options.dtype(at::kByte));
  check_st(st_layer_norm_backward(bytes_or_null(gy), score_type(y_type, "x"), bytes_or_null(gsum), bytes_or_null(h),
                                  score_type(h.scalar_type(), "residual"), rows, dim, h.stride(0), bytes_or_null(weight),
                                  score_type(weights, "weight"), data_or_null<float>(stats), used.defined() ? p : 0.0,
                                  data_or_null<int64_t>(used), bytes_or_null(ws), bytes_or_null(gx),
                                  bytes_or_null(gr), bytes_or_null(gw), bytes_or_null(gb), current_stream(h)),
           "layer_norm_backward");
  return {back(gx, on_gpu), back(gr, on_gpu), back(gw, on_gpu), back(gb, on_gpu)};
}

using NormOp = Tensor(const Tensor&, const OptTensor&, const OptTensor&, double);
using NormKeepOp = Pair(const Tensor&, const OptTensor&, const OptTensor&, double);
using ResidualOp = Pair(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, double, const OptTensor&, double);
using ResidualKeepOp = Four(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, double, const OptTensor&, double);
using NormBackwardOp = Four(const OptTensor&, const OptTensor&, const Tensor&, const OptTensor&, const Tensor&,
                            const OptTensor&, double, at::ScalarType, at::ScalarType, std::array<bool, 4>);

Tensor norm_below(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  static const auto op = find_op<NormOp>("st::layer_norm");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, weight, bias, eps);
}

Pair norm_with_stats_below(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  static const auto op = find_op<NormKeepOp>("st::layer_norm_with_stats");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, weight, bias, eps);
}

Pair residual_below(const Tensor& x, const Tensor& residual, const OptTensor& weight, const OptTensor& bias, double p,
                    const OptTensor& state, double eps) {
  static const auto op = find_op<ResidualOp>("st::dropout_add_layer_norm");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, residual, weight, bias, p, state, eps);
}

Four residual_with_stats_below(const Tensor& x, const Tensor& residual, const OptTensor& weight, const OptTensor& bias,
                               double p, const OptTensor& state, double eps) {
  static const auto op = find_op<ResidualKeepOp>("st::dropout_add_layer_norm_with_stats");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, residual, weight, bias, p, state, eps);
}

Four norm_backward_below(AutogradContext* ctx, const Tensor& grad_y, const Tensor& grad_sum, const Tensor& h,
                         const Tensor& weight, const Tensor& stats, const Tensor& used, std::array<bool, 4> wanted) {
  static const auto op = find_op<NormBackwardOp>("st::layer_norm_backward");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(if_defined(grad_y), if_defined(grad_sum), h, if_defined(weight), stats, if_defined(used),
                 ctx->saved_data["p"].toDouble(), static_cast<at::ScalarType>(ctx->saved_data["y"].toInt()),
                 static_cast<at::ScalarType>(ctx->saved_data["weights"].toInt()), wanted);
}

at::ScalarType weights_scalar_type(const Tensor& weight, const Tensor& bias) {
  return weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : at::kFloat;
}

// Gradients wanted of weight and bias: the graph's edges count the tensors that
// were given, `first` of them ahead of the weight.
std::array<bool, 4> wanted(AutogradContext* ctx, size_t first) {
  const bool weight = ctx->saved_data["weight"].toBool(), bias = ctx->saved_data["bias"].toBool();
  return {ctx->needs_input_grad(0), first > 1 && ctx->needs_input_grad(1), weight && ctx->needs_input_grad(first),
          bias && ctx->needs_input_grad(first + (weight ? 1 : 0))};
}

void keep(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& bias, double p) {
  ctx->set_materialize_grads(false);
  ctx->saved_data["weight"] = weight.defined();
  ctx->saved_data["bias"] = bias.defined();
  ctx->saved_data["weights"] = static_cast<int64_t>(weights_scalar_type(weight, bias));
  ctx->saved_data["y"] = static_cast<int64_t>(x.scalar_type());
  ctx->saved_data["p"] = p;
}

struct LayerNormFunction : torch::autograd::Function<LayerNormFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    auto [y, stats] = norm_with_stats_below(x, weight, bias, eps);
    keep(ctx, x, given(weight), given(bias), 0.0);
    ctx->save_for_backward({x, given(weight), stats});
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    auto [gx, gr, gw, gb] =
        norm_backward_below(ctx, grads[0], Tensor(), saved[0], saved[1], saved[2], Tensor(), wanted(ctx, 1));
    auto once = [&](const Tensor& t) { return differentiable_once(t, saved[0], saved[1], grads, "layer_norm"); };
    return {once(gx), once(gw), once(gb), Tensor()};
  }
};

Tensor layer_norm_autograd(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  const Tensor w = given(weight), b = given(bias);
  refuse_tangents_of({&x, &w, &b}, "layer_norm");
  return requires_grad({&x, &w, &b}) ? LayerNormFunction::apply(x, weight, bias, eps) : norm_below(x, weight, bias, eps);
}

struct ResidualFunction : torch::autograd::Function<ResidualFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const OptTensor& weight,
                               const OptTensor& bias, double p, const OptTensor& state, double eps) {
    auto [y, sum, stats, used] = residual_with_stats_below(x, residual, weight, bias, p, state, eps);
    keep(ctx, x, given(weight), given(bias), used.defined() ? p : 0.0);
    ctx->save_for_backward({sum, given(weight), stats, used});
    return {y, sum};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(7);
    auto [gx, gr, gw, gb] =
        norm_backward_below(ctx, grads[0], grads[1], saved[0], saved[1], saved[2], saved[3], wanted(ctx, 2));
    auto once = [&](const Tensor& t) { return differentiable_once(t, saved[0], saved[1], grads, "dropout_add_layer_norm"); };
    return {once(gx), once(gr), once(gw), once(gb), Tensor(), Tensor(), Tensor()};
  }
};

Pair dropout_add_layer_norm_autograd(const Tensor& x, const Tensor& residual, const OptTensor& weight,
                                     const OptTensor& bias, double p, const OptTensor& state, double eps) {
  const Tensor w = given(weight), b = given(bias);
  refuse_tangents_of({&x, &residual, &w, &b}, "dropout_add_layer_norm");
  if (!requires_grad({&x, &residual, &w, &b})) return residual_below(x, residual, weight, bias, p, state, eps);
  const variable_list o = ResidualFunction::apply(x, residual, weight, bias, p, state, eps);
  return {o[0], o[1]};
}

// ------------------------------------------ rows in 8 bits

std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
  std::vector<int64_t> s(sizes.begin(), sizes.end());
  s.back() = last;
  return s;
}

// Codes and scales of x's rows, empty.
Pair empty_codes(const Tensor& x) {
  return {at::empty(with_last(x.sizes(), st_int8_columns(x.size(-1))), x.options().dtype(at::kChar)),
          at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat))};
}

void check_quantize(const Tensor& x) {
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "x must have at least one column");
  score_type(x.scalar_type(), "x");
}

Pair int8_quantize_gpu(const Tensor& x_in) {
  check_quantize(x_in);
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x_in.device());
  const Tensor x = as_rows(x_in);
  auto [codes, scales] = empty_codes(x_in);
  check_st(st_int8_quantize(bytes_or_null(x), score_type(x.scalar_type(), "x"), x.size(0), x.size(1), x.stride(0),
                            data_or_null<int8_t>(codes), data_or_null<float>(scales), current_stream(x)),
           "int8_quantize");
  return {codes, scales};
}

Pair int8_quantize_cpu(const Tensor& x) {
  check_quantize(x);
  auto [codes, scales] = int8_quantize_gpu(x.to(gpu_for_cpu_call()));
  return {codes.cpu(), scales.cpu()};
}

Pair layer_norm_int8_gpu(const Tensor& x_in, const OptTensor& weight_in, const OptTensor& bias_in, double eps) {
  Tensor weight = given(weight_in), bias = given(bias_in);
  check_weights(x_in, weight, bias, eps, "layer_norm_int8");
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x_in.device());
  const Tensor x = as_rows(x_in);
  if (weight.defined()) weight = weight.contiguous();
  if (bias.defined()) bias = bias.contiguous();
  auto [codes, scales] = empty_codes(x_in);
  check_st(st_layer_norm_int8(bytes_or_null(x), score_type(x.scalar_type(), "x"), x.size(0), x.size(1), x.stride(0),
                              bytes_or_null(weight), bytes_or_null(bias), weights_type(weight, bias), eps,
                              data_or_null<int8_t>(codes), data_or_null<float>(scales), current_stream(x)),
           "layer_norm_int8");
  return {codes, scales};
}

Pair layer_norm_int8_cpu(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  check_weights(x, given(weight), given(bias), eps, "layer_norm_int8");
  const at::Device gpu = gpu_for_cpu_call();
  auto [codes, scales] = layer_norm_int8_gpu(x.to(gpu), if_defined(moved(weight, gpu)), if_defined(moved(bias, gpu)), eps);
  return {codes.cpu(), scales.cpu()};
}

at::ScalarType result_type(const Tensor& x, std::optional<at::ScalarType> out_dtype) {
  return out_dtype.value_or(x.scalar_type() == at::kChar ? at::kFloat : x.scalar_type());
}

void check_matmul(const Tensor& codes, const Tensor& scales, const Tensor& x, const Tensor& x_scales, const Tensor& bias,
                  at::ScalarType out_type) {
  TORCH_CHECK(codes.dim() == 2 && codes.scalar_type() == at::kChar, "codes must be a 2-D int8 tensor");
  const int64_t n = codes.size(0), columns = codes.size(1);
  TORCH_CHECK(columns >= 16 && columns % 16 == 0, "rows of codes are whole blocks of 16 columns, got ", columns);
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "x must have at least one column");
  if (x.scalar_type() == at::kChar) {
    TORCH_CHECK(x.size(-1) == columns, "x has rows of ", x.size(-1), " codes, the table of ", columns);
    TORCH_CHECK(x_scales.defined(), "x of codes comes with x_scales");
    TORCH_CHECK(x_scales.scalar_type() == at::kFloat && x_scales.sizes() == x.sizes().slice(0, x.dim() - 1),
                "x_scales must be float32 with one entry for each row of x, ", x.sizes().slice(0, x.dim() - 1), ", got ",
                x_scales.sizes());
  } else {
    score_type(x.scalar_type(), "x that is not int8");
    TORCH_CHECK(!x_scales.defined(), "x_scales go with x of codes");
    TORCH_CHECK(st_int8_columns(x.size(-1)) == columns, "the table's rows have ", columns, " columns, vectors of ",
                x.size(-1), " take ", st_int8_columns(x.size(-1)));
  }
  score_type(out_type, "out_dtype");
  TORCH_CHECK(scales.dim() == 1 && scales.size(0) == n && scales.scalar_type() == at::kFloat,
              "scales must be float32 with one entry for each of ", n, " rows, got ", scales.sizes());
  TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == n && bias.scalar_type() == at::kFloat),
              "bias must be float32 with one entry for each of ", n, " rows");
  for (const Tensor* t : {&scales, &x, &x_scales, &bias})
    TORCH_CHECK(!t->defined() || t->device() == codes.device(), "int8_matmul inputs must be on one device");
}

Tensor aligned(const Tensor& t_in) {
  const Tensor t = t_in.contiguous();
  return t.numel() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0 ? t.clone() : t;
}

Tensor int8_matmul_gpu(const Tensor& codes_in, const Tensor& scales_in, const Tensor& x_in, const OptTensor& x_scales_in,
                       const OptTensor& bias_in, std::optional<at::ScalarType> out_dtype) {
  const at::ScalarType out_type = result_type(x_in, out_dtype);
  Tensor x_scales = given(x_scales_in), bias = given(bias_in);
  check_matmul(codes_in, scales_in, x_in, x_scales, bias, out_type);
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(codes_in.device());
  const bool coded = x_in.scalar_type() == at::kChar;
  const Tensor codes = aligned(codes_in), scales = scales_in.contiguous();
  Tensor x = as_rows(x_in);
  if (coded) x = aligned(x);
  if (x_scales.defined()) x_scales = x_scales.contiguous();
  if (bias.defined()) bias = bias.contiguous();
  const int x_type = coded ? ST_CODE_I8 : score_type(x.scalar_type(), "x");
  const int64_t tokens = x.size(0), columns = codes.size(1);
  Tensor y = at::empty(with_last(x_in.sizes(), codes.size(0)), x.options().dtype(out_type)), ws;
  const int64_t bytes = y.numel() ? st_int8_matmul_workspace_bytes(x_type, tokens, codes.size(0), columns) : 0;
  if (bytes > 0) ws = at::empty({bytes}, x.options().dtype(at::kByte));
  check_st(st_int8_matmul(data_or_null<int8_t>(codes), data_or_null<float>(scales), codes.size(0), columns,
                          bytes_or_null(x), x_type, data_or_null<float>(x_scales), tokens, x.size(1),
                          coded ? columns : x.stride(0), data_or_null<float>(bias), bytes_or_null(y),
                          score_type(out_type, "out_dtype"), bytes_or_null(ws), current_stream(x)),
           "int8_matmul");
  return y;
}

Tensor int8_matmul_cpu(const Tensor& codes, const Tensor& scales, const Tensor& x, const OptTensor& x_scales,
                       const OptTensor& bias, std::optional<at::ScalarType> out_dtype) {
  check_matmul(codes, scales, x, given(x_scales), given(bias), result_type(x, out_dtype));
  const at::Device gpu = gpu_for_cpu_call();
  return int8_matmul_gpu(codes.to(gpu), scales.to(gpu), x.to(gpu), if_defined(moved(x_scales, gpu)),
                         if_defined(moved(bias, gpu)), out_dtype)
      .cpu();
}

// The 8-bit operators have no gradients.  Their results say so when one is asked
// for, where they would otherwise count as constants.
using CodesOp = Pair(const Tensor&);
using NormCodesOp = Pair(const Tensor&, const OptTensor&, const OptTensor&, double);
using MatmulOp = Tensor(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                        std::optional<at::ScalarType>);

Pair quantize_below(const Tensor& x) {
  static const auto op = find_op<CodesOp>("st::int8_quantize");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x);
}

Pair norm_codes_below(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  static const auto op = find_op<NormCodesOp>("st::layer_norm_int8");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, weight, bias, eps);
}

Tensor matmul_below(const Tensor& codes, const Tensor& scales, const Tensor& x, const OptTensor& x_scales,
                    const OptTensor& bias, std::optional<at::ScalarType> out_dtype) {
  static const auto op = find_op<MatmulOp>("st::int8_matmul");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(codes, scales, x, x_scales, bias, out_dtype);
}

struct CodesFunction : torch::autograd::Function<CodesFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x) {
    auto [codes, scales] = quantize_below(x);
    ctx->mark_non_differentiable({codes});
    return {codes, scales};
  }
  static variable_list backward(AutogradContext* /*ctx*/, variable_list /*grads*/) {
    TORCH_CHECK(false, "int8_quantize has no gradient");
  }
};

struct NormCodesFunction : torch::autograd::Function<NormCodesFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                               double eps) {
    auto [codes, scales] = norm_codes_below(x, weight, bias, eps);
    ctx->mark_non_differentiable({codes});
    return {codes, scales};
  }
  static variable_list backward(AutogradContext* /*ctx*/, variable_list /*grads*/) {
    TORCH_CHECK(false, "layer_norm_int8 has no gradient");
  }
};

struct MatmulFunction : torch::autograd::Function<MatmulFunction> {
  static Tensor forward(AutogradContext* /*ctx*/, const Tensor& codes, const Tensor& scales, const Tensor& x,
                        const OptTensor& x_scales, const OptTensor& bias, std::optional<at::ScalarType> out_dtype) {
    return matmul_below(codes, scales, x, x_scales, bias, out_dtype);
  }
  static variable_list backward(AutogradContext* /*ctx*/, variable_list /*grads*/) {
    TORCH_CHECK(false, "int8_matmul has no gradient");
  }
};

Pair int8_quantize_autograd(const Tensor& x) {
  refuse_tangents({&x}, "int8_quantize");
  if (!requires_grad({&x})) return quantize_below(x);
  const variable_list o = CodesFunction::apply(x);
  return {o[0], o[1]};
}

Pair layer_norm_int8_autograd(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  const Tensor w = given(weight), b = given(bias);
  refuse_tangents_of({&x, &w, &b}, "layer_norm_int8");
  if (!requires_grad({&x, &w, &b})) return norm_codes_below(x, weight, bias, eps);
  const variable_list o = NormCodesFunction::apply(x, weight, bias, eps);
  return {o[0], o[1]};
}

Tensor int8_matmul_autograd(const Tensor& codes, const Tensor& scales, const Tensor& x, const OptTensor& x_scales,
                            const OptTensor& bias, std::optional<at::ScalarType> out_dtype) {
  const Tensor xs = given(x_scales), b = given(bias);
  refuse_tangents_of({&scales, &x, &xs, &b}, "int8_matmul");
  if (!requires_grad({&scales, &x, &xs, &b})) return matmul_below(codes, scales, x, x_scales, bias, out_dtype);
  return MatmulFunction::apply(codes, scales, x, x_scales, bias, out_dtype);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(st, m) {
  m.def("layer_norm(Tensor x, Tensor? weight=None, Tensor? bias=None, float eps=1e-05) -> Tensor");
  // state: int64 [2], seed and offset
  m.def("dropout(Tensor x, float p, Tensor state) -> Tensor");
  // (the sum's layer norm, residual + dropout(x))
  m.def("dropout_add_layer_norm(Tensor x, Tensor residual, Tensor? weight=None, Tensor? bias=None, float p=0.0, "
        "Tensor? state=None, float eps=1e-05) -> (Tensor, Tensor)");
  // What the gradients call: (result, state that was used), (result, stats), (norm, sum, stats, state that was used or
  // none), gradients of (x, residual, weight, bias) or none where not wanted.
  m.def("dropout_with_state(Tensor x, float p, Tensor state) -> (Tensor, Tensor)");
  m.def("layer_norm_with_stats(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor)");
  m.def("dropout_add_layer_norm_with_stats(Tensor x, Tensor residual, Tensor? weight, Tensor? bias, float p, "
        "Tensor? state, float eps) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("layer_norm_backward(Tensor? grad_y, Tensor? grad_sum, Tensor h, Tensor? weight, Tensor stats, Tensor? used, "
        "float p, ScalarType y_type, ScalarType weight_type, bool[4] wanted) -> (Tensor, Tensor, Tensor, Tensor)");
  // codes int8 [..., D up to a multiple of 16], scales [...]
  m.def("int8_quantize(Tensor x) -> (Tensor, Tensor)");
  m.def("layer_norm_int8(Tensor x, Tensor? weight=None, Tensor? bias=None, float eps=1e-05) -> (Tensor, Tensor)");
  // x [..., D], or its codes and scales, times the table transposed
  m.def("int8_matmul(Tensor codes, Tensor scales, Tensor x, Tensor? x_scales=None, Tensor? bias=None, "
        "ScalarType? out_dtype=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(st, CUDA, m) {
  m.impl("layer_norm", TORCH_FN(layer_norm));
  m.impl("dropout", TORCH_FN(dropout));
  m.impl("dropout_add_layer_norm", TORCH_FN(dropout_add_layer_norm));
  m.impl("dropout_with_state", TORCH_FN(dropout_with_state));
  m.impl("layer_norm_with_stats", TORCH_FN(layer_norm_with_stats));
  m.impl("dropout_add_layer_norm_with_stats", TORCH_FN(dropout_add_layer_norm_with_stats));
  m.impl("layer_norm_backward", TORCH_FN(layer_norm_backward));
  m.impl("int8_quantize", TORCH_FN(int8_quantize_gpu));
  m.impl("layer_norm_int8", TORCH_FN(layer_norm_int8_gpu));
  m.impl("int8_matmul", TORCH_FN(int8_matmul_gpu));
}

TORCH_LIBRARY_IMPL(st, CPU, m) {
  m.impl("layer_norm", TORCH_FN(layer_norm));
  m.impl("dropout", TORCH_FN(dropout));
  m.impl("dropout_add_layer_norm", TORCH_FN(dropout_add_layer_norm));
  m.impl("dropout_with_state", TORCH_FN(dropout_with_state));
  m.impl("layer_norm_with_stats", TORCH_FN(layer_norm_with_stats));
  m.impl("dropout_add_layer_norm_with_stats", TORCH_FN(dropout_add_layer_norm_with_stats));
  m.impl("layer_norm_backward", TORCH_FN(layer_norm_backward));
  m.impl("int8_quantize", TORCH_FN(int8_quantize_cpu));
  m.impl("layer_norm_int8", TORCH_FN(layer_norm_int8_cpu));
  m.impl("int8_matmul", TORCH_FN(int8_matmul_cpu));
}

TORCH_LIBRARY_IMPL(st, Autograd, m) {
  m.impl("layer_norm", TORCH_FN(layer_norm_autograd));
  m.impl("dropout", TORCH_FN(dropout_autograd));
  m.impl("dropout_add_layer_norm", TORCH_FN(dropout_add_layer_norm_autograd));
  m.impl("int8_quantize", TORCH_FN(int8_quantize_autograd));
  m.impl("layer_norm_int8", TORCH_FN(layer_norm_int8_autograd));
  m.impl("int8_matmul", TORCH_FN(int8_matmul_autograd));
}
