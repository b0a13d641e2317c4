// torch.ops.st.* of the retrieval head: 4-bit score tables, log-probabilities
// of given documents, cluster routing.  No reference counterparts.
//
// As in torch_ops.cpp, GPU tensors run on their device's current stream and
// CPU tensors are copied to the current GPU and the results back.  The two
// operators a model is trained through carry their gradients (Autograd key);
// the 4-bit ones refuse to be differentiated.
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "torch_common.hpp"

namespace {

using at::Tensor;
using st_torch::check_st;
using st_torch::current_stream;
using st_torch::gpu_for_cpu_call;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

int score_type(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat:
      return ST_SCORE_F32;
    case at::kHalf:
      return ST_SCORE_F16;
    case at::kBFloat16:
      return ST_SCORE_BF16;
    default:
      TORCH_CHECK(false, what, " must be float32, float16 or bfloat16, got ", t);
  }
}

template <typename T>
T* data_or_null(const Tensor& t) {
  return t.defined() && t.numel() ? t.data_ptr<T>() : nullptr;
}

void* bytes_or_null(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

// None of these operators has a forward-mode derivative: an input that carries
// a tangent is refused, where the result would otherwise come without one.
void refuse_tangents(std::initializer_list<const Tensor*> inputs, const char* op) {
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), op, " has no forward-mode derivative");
}

Tensor moved(const OptTensor& t, at::Device d) { return t.has_value() && t->defined() ? t->to(d) : Tensor(); }

// ------------------------------------------ 4-bit tables

constexpr int64_t kInt4Block = 32;  // columns of 16 bytes

void check_group(int64_t group_size) {
  TORCH_CHECK(group_size >= kInt4Block && group_size % kInt4Block == 0, "group_size must be a positive multiple of ",
              kInt4Block, ", got ", group_size);
}

void check_quantize(const Tensor& weight, int64_t group_size) {
  TORCH_CHECK(weight.dim() == 2 && weight.size(1) > 0, "weight must be a 2-D tensor with at least one column");
  score_type(weight.scalar_type(), "weight");
  check_group(group_size);
}

std::tuple<Tensor, Tensor, Tensor> int4_quantize_gpu(const Tensor& weight_in, int64_t group_size, bool symmetric) {
  check_quantize(weight_in, group_size);
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(weight_in.device());
  const Tensor weight = weight_in.contiguous();
  const int64_t n = weight.size(0), dim = weight.size(1), groups = (dim - 1) / group_size + 1;
  const auto bytes = weight.options().dtype(at::kByte);
  Tensor packed = at::empty({n, (dim + kInt4Block - 1) / kInt4Block * (kInt4Block / 2)}, bytes);
  Tensor scales = at::empty({n, groups}, weight.options());
  Tensor zeros = at::empty({n, groups}, bytes);
  check_st(st_int4_quantize(bytes_or_null(weight), score_type(weight.scalar_type(), "weight"), n, dim, group_size,
                            symmetric ? 1 : 0, data_or_null<uint8_t>(packed), bytes_or_null(scales),
                            data_or_null<uint8_t>(zeros), current_stream(weight)),
           "int4_quantize");
  return {packed, scales, zeros};
}

std::tuple<Tensor, Tensor, Tensor> int4_quantize_cpu(const Tensor& weight, int64_t group_size, bool symmetric) {
  check_quantize(weight, group_size);
  auto [p, s, z] = int4_quantize_gpu(weight.to(gpu_for_cpu_call()), group_size, symmetric);
  return {p.cpu(), s.cpu(), z.cpu()};
}

void check_matvec(const Tensor& packed, const Tensor& scales, const Tensor& x, int64_t group_size,
                  const OptTensor& zeros, at::ScalarType out_type) {
  check_group(group_size);
  TORCH_CHECK(packed.dim() == 2 && packed.scalar_type() == at::kByte, "packed must be a 2-D uint8 tensor");
  TORCH_CHECK(x.dim() == 1 || x.dim() == 2, "x must be a vector or a 2-D tensor of vectors");
  score_type(x.scalar_type(), "x");
  score_type(scales.scalar_type(), "scales");
  score_type(out_type, "out_dtype");
  const int64_t n = packed.size(0), dim = x.size(-1);
  TORCH_CHECK(dim >= 1, "x must have at least one column");
  const int64_t groups = (dim - 1) / group_size + 1;
  const int64_t row_bytes = (dim + kInt4Block - 1) / kInt4Block * (kInt4Block / 2);
  TORCH_CHECK(packed.size(1) == row_bytes, "packed has ", packed.size(1), " bytes a row, ", dim, " columns take ",
              row_bytes);
  TORCH_CHECK(scales.dim() == 2 && scales.size(0) == n && scales.size(1) == groups, "scales must be [", n, ", ",
              groups, "], got ", scales.sizes());
  const bool has_zeros = zeros.has_value() && zeros->defined();
  TORCH_CHECK(!has_zeros || (zeros->scalar_type() == at::kByte && zeros->sizes() == scales.sizes()),
              "zeros must be a uint8 tensor of the scales' shape");
  const auto dev = packed.device();
  TORCH_CHECK(scales.device() == dev && x.device() == dev && (!has_zeros || zeros->device() == dev),
              "int4_matvec inputs must be on one device");
}

Tensor int4_matvec_gpu(const Tensor& packed_in, const Tensor& scales_in, const Tensor& x_in, int64_t group_size,
                       const OptTensor& zeros_in, std::optional<at::ScalarType> out_dtype) {
  const at::ScalarType out_type = out_dtype.value_or(x_in.scalar_type());
  check_matvec(packed_in, scales_in, x_in, group_size, zeros_in, out_type);
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(packed_in.device());
  const int64_t n = packed_in.size(0), dim = x_in.size(-1), queries = x_in.dim() == 2 ? x_in.size(0) : 1;
  Tensor packed = packed_in.contiguous(), zeros;
  if (packed.numel() && reinterpret_cast<uintptr_t>(packed.data_ptr()) % 16 != 0) packed = packed.clone();
  if (zeros_in.has_value() && zeros_in->defined()) zeros = zeros_in->contiguous();
  const Tensor scales = scales_in.contiguous(), x = x_in.contiguous();
  Tensor y = x.dim() == 2 ? at::empty({queries, n}, x.options().dtype(out_type))
                          : at::empty({n}, x.options().dtype(out_type));
  check_st(st_int4_matvec(data_or_null<uint8_t>(packed), bytes_or_null(scales),
                          score_type(scales.scalar_type(), "scales"), data_or_null<uint8_t>(zeros), bytes_or_null(x),
                          score_type(x.scalar_type(), "x"), queries, n, dim, group_size, bytes_or_null(y),
                          score_type(out_type, "out_dtype"), current_stream(x)),
           "int4_matvec");
  return y;
}

Tensor int4_matvec_cpu(const Tensor& packed, const Tensor& scales, const Tensor& x, int64_t group_size,
                       const OptTensor& zeros, std::optional<at::ScalarType> out_dtype) {
  check_matvec(packed, scales, x, group_size, zeros, out_dtype.value_or(x.scalar_type()));
  const at::Device gpu = gpu_for_cpu_call();
  return int4_matvec_gpu(packed.to(gpu), scales.to(gpu), x.to(gpu), group_size, moved(zeros, gpu), out_dtype).cpu();
}

// The 4-bit operators have no gradients.  Their results say so when one is
// asked for, where they would otherwise count as constants.
template <typename Op>
auto find_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Op>();
}

using QuantizeOp = std::tuple<Tensor, Tensor, Tensor>(const Tensor&, int64_t, bool);
using MatvecOp = Tensor(const Tensor&, const Tensor&, const Tensor&, int64_t, const OptTensor&,
                        std::optional<at::ScalarType>);

std::tuple<Tensor, Tensor, Tensor> quantize_below(const Tensor& weight, int64_t group_size, bool symmetric) {
  static const auto op = find_op<QuantizeOp>("st::int4_quantize");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(weight, group_size, symmetric);
}

Tensor matvec_below(const Tensor& packed, const Tensor& scales, const Tensor& x, int64_t group_size,
                    const OptTensor& zeros, std::optional<at::ScalarType> out_dtype) {
  static const auto op = find_op<MatvecOp>("st::int4_matvec");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(packed, scales, x, group_size, zeros, out_dtype);
}

struct QuantizeFunction : torch::autograd::Function<QuantizeFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& weight, int64_t group_size, bool symmetric) {
    auto [packed, scales, zeros] = quantize_below(weight, group_size, symmetric);
    ctx->mark_non_differentiable({packed, zeros});
    return {packed, scales, zeros};
  }
  static variable_list backward(AutogradContext* /*ctx*/, variable_list /*grads*/) {
    TORCH_CHECK(false, "int4_quantize has no gradient");
  }
};

struct MatvecFunction : torch::autograd::Function<MatvecFunction> {
  static Tensor forward(AutogradContext* /*ctx*/, const Tensor& packed, const Tensor& scales, const Tensor& x,
                        int64_t group_size, const OptTensor& zeros, std::optional<at::ScalarType> out_dtype) {
    return matvec_below(packed, scales, x, group_size, zeros, out_dtype);
  }
  static variable_list backward(AutogradContext* /*ctx*/, variable_list /*grads*/) {
    TORCH_CHECK(false, "int4_matvec has no gradient");
  }
};

std::tuple<Tensor, Tensor, Tensor> int4_quantize_autograd(const Tensor& weight, int64_t group_size, bool symmetric) {
  refuse_tangents({&weight}, "int4_quantize");
  if (!at::GradMode::is_enabled() || !weight.requires_grad()) return quantize_below(weight, group_size, symmetric);
  const variable_list o = QuantizeFunction::apply(weight, group_size, symmetric);
  return {o[0], o[1], o[2]};
}

Tensor int4_matvec_autograd(const Tensor& packed, const Tensor& scales, const Tensor& x, int64_t group_size,
                            const OptTensor& zeros, std::optional<at::ScalarType> out_dtype) {
  refuse_tangents({&scales, &x}, "int4_matvec");
  if (!at::GradMode::is_enabled() || !(x.requires_grad() || scales.requires_grad()))
    return matvec_below(packed, scales, x, group_size, zeros, out_dtype);
  return MatvecFunction::apply(packed, scales, x, group_size, zeros, out_dtype);
}

// A score row is readable with any row stride; columns have to be adjacent.
Tensor with_adjacent_columns(const Tensor& t) { return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous(); }

// ------------------------------------------ log-probabilities of given documents

struct LogprobsIn {
  Tensor logits, targets, mask;  // on one GPU; mask may be undefined
  int64_t topk;
  double temperature;
  int type;
  int64_t mask_stride = 0, mask_words = 0;
};

void check_logprobs(const Tensor& logits, const Tensor& targets, int64_t topk, const Tensor& mask,
                    double temperature) {
  TORCH_CHECK(logits.dim() == 2, "logits must be a 2-D tensor");
  score_type(logits.scalar_type(), "logits");
  TORCH_CHECK(targets.dim() == 1 && targets.scalar_type() == at::kLong, "targets must be a 1-D int64 tensor");
  TORCH_CHECK(targets.size(0) == logits.size(0), "targets has ", targets.size(0), " entries, logits ", logits.size(0),
              " rows");
  TORCH_CHECK(logits.device() == targets.device() && (!mask.defined() || mask.device() == logits.device()),
              "target_logprobs inputs must be on one device");
  if (mask.defined()) {
    TORCH_CHECK(mask.dim() == 2 && mask.scalar_type() == at::kLong,
                "packed_mask must be the 2-D int64 packed search output");
    TORCH_CHECK(mask.size(0) == logits.size(0) || mask.size(0) == 1, "packed_mask has ", mask.size(0),
                " rows, logits ", logits.size(0));
    TORCH_CHECK(mask.size(1) * 64 >= logits.size(1), "packed_mask holds ", mask.size(1) * 64, " documents, logits ",
                logits.size(1));
  }
  TORCH_CHECK(topk >= 0 && topk <= 128, "topk must be in [0, 128], got ", topk);
  TORCH_CHECK(temperature >= 1e-6 && temperature <= 1e6, "temperature must be in [1e-6, 1e6], got ", temperature);
}

LogprobsIn logprobs_in(const Tensor& logits, const Tensor& targets, int64_t topk, const Tensor& mask,
                       double temperature) {
  LogprobsIn in{with_adjacent_columns(logits), targets.contiguous(), Tensor(), topk, temperature,
                score_type(logits.scalar_type(), "logits")};
  if (mask.defined() && mask.numel()) {
    in.mask = with_adjacent_columns(mask);
    in.mask_stride = in.mask.size(0) == 1 ? 0 : in.mask.stride(0);
    in.mask_words = in.mask.size(1);
  }
  return in;
}

struct LogprobsOut {
  Tensor logprobs, entropy, lse, top_ids, top_logprobs, stats;
};

LogprobsOut logprobs_gpu(const LogprobsIn& in, bool with_stats) {
  const Tensor& z = in.logits;
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(z.device());
  const int64_t n = z.size(0), v = z.size(1);
  const auto f = z.options().dtype(at::kFloat);
  LogprobsOut o{at::empty({n}, f), at::empty({n}, f), at::empty({n}, f),
                at::empty({n, in.topk}, z.options().dtype(at::kLong)), at::empty({n, in.topk}, f), Tensor()};
  if (with_stats) o.stats = at::empty({n, 2}, f);
  const int64_t bytes = st_target_logprobs_workspace_bytes(n, v, in.topk);
  Tensor ws;
  if (bytes > 0) ws = at::empty({bytes}, z.options().dtype(at::kByte));
  check_st(st_target_logprobs(bytes_or_null(z), in.type, n, v, z.stride(0), data_or_null<int64_t>(in.targets),
                              data_or_null<int64_t>(in.mask), in.mask_stride, in.mask_words, in.topk, in.temperature,
                              bytes_or_null(ws), data_or_null<float>(o.logprobs), data_or_null<float>(o.entropy),
                              data_or_null<float>(o.lse), data_or_null<int64_t>(o.top_ids),
                              data_or_null<float>(o.top_logprobs), data_or_null<float>(o.stats), current_stream(z)),
           "target_logprobs");
  return o;
}

LogprobsOut logprobs_any(const Tensor& logits, const Tensor& targets, int64_t topk, const Tensor& mask,
                         double temperature, bool with_stats) {
  check_logprobs(logits, targets, topk, mask, temperature);
  if (logits.is_cuda()) return logprobs_gpu(logprobs_in(logits, targets, topk, mask, temperature), with_stats);
  const at::Device gpu = gpu_for_cpu_call();
  LogprobsOut o = logprobs_gpu(
      logprobs_in(logits.to(gpu), targets.to(gpu), topk, mask.defined() ? mask.to(gpu) : mask, temperature),
      with_stats);
  for (Tensor* t : {&o.logprobs, &o.entropy, &o.lse, &o.top_ids, &o.top_logprobs, &o.stats})
    if (t->defined()) *t = t->cpu();
  return o;
}

// A gradient as the kernels take it: float32, contiguous, on the device.
Tensor gradient(const Tensor& g, at::Device d) {
  return g.defined() ? g.to(d, at::kFloat).contiguous() : g;
}

// A gradient with a graph over it (backward with create_graph): it depends on
// the scores and on the outputs' gradients, and refuses to be differentiated
// where it would otherwise count as a constant.
struct OnceDifferentiable : torch::autograd::Function<OnceDifferentiable> {
  static Tensor forward(AutogradContext* ctx, const Tensor& grad, const Tensor& /*logits*/, const OptTensor& /*g0*/,
                        const OptTensor& /*g1*/, const OptTensor& /*g2*/, const OptTensor& /*g3*/, std::string op) {
    ctx->saved_data["op"] = std::move(op);
    return grad;
  }
  static variable_list backward(AutogradContext* ctx, variable_list /*grads*/) {
    TORCH_CHECK(false, "the gradient of ", ctx->saved_data["op"].toStringRef(), " cannot be differentiated again");
  }
};

Tensor differentiable_once(const Tensor& grad, const Tensor& logits, const variable_list& outer, const char* op) {
  if (!at::GradMode::is_enabled()) return grad;
  auto given = [&](size_t i) { return outer[i].defined() ? OptTensor(outer[i]) : OptTensor(); };
  return OnceDifferentiable::apply(grad, logits, given(0), given(1), given(2), given(4), std::string(op));
}

struct LogprobsFunction : torch::autograd::Function<LogprobsFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, int64_t topk,
                               const OptTensor& packed_mask, double temperature) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor mask = packed_mask.value_or(Tensor());
    LogprobsOut o = logprobs_any(logits, targets, topk, mask, temperature, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, targets, mask, o.entropy, o.top_ids, o.stats});
    ctx->saved_data["topk"] = topk;
    ctx->saved_data["temperature"] = temperature;
    ctx->mark_non_differentiable({o.top_ids});
    return {o.logprobs, o.entropy, o.lse, o.top_ids, o.top_logprobs};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor grad = logits_gradient(ctx, saved, grads);
    return {differentiable_once(grad, saved[0], grads, "target_logprobs"), Tensor(), Tensor(), Tensor(), Tensor()};
  }

  static Tensor logits_gradient(AutogradContext* ctx, const variable_list& saved, const variable_list& grads) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor& logits = saved[0];
    const bool on_gpu = logits.is_cuda();
    const at::Device dev = on_gpu ? logits.device() : gpu_for_cpu_call();
    const LogprobsIn in = logprobs_in(logits.to(dev), saved[1].to(dev), ctx->saved_data["topk"].toInt(),
                                      saved[2].defined() ? saved[2].to(dev) : saved[2],
                                      ctx->saved_data["temperature"].toDouble());
    c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(dev);
    const Tensor entropy = saved[3].to(dev), top_ids = saved[4].to(dev), stats = saved[5].to(dev);
    const Tensor gl = gradient(grads[0], dev), ge = gradient(grads[1], dev), gs = gradient(grads[2], dev),
                 gt = gradient(grads[4], dev);
    const Tensor& z = in.logits;
    Tensor grad = at::empty(z.sizes(), z.options());
    check_st(st_target_logprobs_backward(
                 bytes_or_null(z), in.type, z.size(0), z.size(1), z.stride(0), data_or_null<int64_t>(in.targets),
                 data_or_null<int64_t>(in.mask), in.mask_stride, in.mask_words, in.topk, in.temperature,
                 data_or_null<float>(entropy), data_or_null<float>(stats), data_or_null<int64_t>(top_ids),
                 data_or_null<float>(gl), data_or_null<float>(ge), data_or_null<float>(gs), data_or_null<float>(gt),
                 bytes_or_null(grad), current_stream(z)),
             "target_logprobs");
    return on_gpu ? grad : grad.cpu();
  }
};

using Logprobs = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

Logprobs target_logprobs(const Tensor& logits, const Tensor& targets, int64_t topk, const OptTensor& mask,
                         double temperature) {
  LogprobsOut o = logprobs_any(logits, targets, topk, mask.value_or(Tensor()), temperature, false);
  return {o.logprobs, o.entropy, o.lse, o.top_ids, o.top_logprobs};
}

Logprobs target_logprobs_autograd(const Tensor& logits, const Tensor& targets, int64_t topk, const OptTensor& mask,
                                  double temperature) {
  refuse_tangents({&logits}, "target_logprobs");
  if (!at::GradMode::is_enabled() || !logits.requires_grad()) {
    at::AutoDispatchBelowADInplaceOrView below;
    return target_logprobs(logits, targets, topk, mask, temperature);
  }
  const variable_list o = LogprobsFunction::apply(logits, targets, topk, mask, temperature);
  return {o[0], o[1], o[2], o[3], o[4]};
}

// ------------------------------------------ cluster routing

void check_route(const Tensor& logits, int64_t probes, const Tensor& valid) {
  TORCH_CHECK(logits.dim() == 2, "logits must be a 2-D tensor");
  score_type(logits.scalar_type(), "logits");
  TORCH_CHECK(logits.size(1) >= 1 && logits.size(1) <= 32768, "clusters must be in [1, 32768], got ", logits.size(1));
  TORCH_CHECK(probes >= 1 && probes <= 64, "probes must be in [1, 64], got ", probes);
  if (valid.defined()) {
    TORCH_CHECK(valid.dim() == 1 && valid.scalar_type() == at::kBool && valid.size(0) == logits.size(0),
                "valid must be a bool tensor with one entry per row");
    TORCH_CHECK(valid.device() == logits.device(), "cluster_route inputs must be on one device");
  }
}

struct RouteOut {
  Tensor ids, weights, lse, counts, loss, stats, slopes;
};

RouteOut route_gpu(const Tensor& logits, int64_t probes, const Tensor& valid_in) {
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(logits.device());
  const Tensor z = with_adjacent_columns(logits);
  const Tensor valid = valid_in.defined() ? valid_in.contiguous() : valid_in;
  const int64_t n = z.size(0), e = z.size(1);
  const auto f = z.options().dtype(at::kFloat), l = z.options().dtype(at::kLong);
  RouteOut o{at::empty({n, probes}, l), at::empty({n, probes}, f), at::empty({n}, f), at::empty({e}, l),
             at::empty({}, f), at::empty({n, 2}, f), at::empty({e}, f)};
  const Tensor ws = at::empty({st_cluster_route_workspace_bytes(n, e)}, z.options().dtype(at::kByte));
  check_st(st_cluster_route(bytes_or_null(z), score_type(z.scalar_type(), "logits"), n, e, z.stride(0), probes,
                            static_cast<const uint8_t*>(bytes_or_null(valid)), ws.data_ptr(),
                            data_or_null<int64_t>(o.ids), data_or_null<float>(o.weights), data_or_null<float>(o.lse),
                            data_or_null<int64_t>(o.counts), o.loss.data_ptr<float>(), data_or_null<float>(o.stats),
                            data_or_null<float>(o.slopes), current_stream(z)),
           "cluster_route");
  return o;
}

RouteOut route_any(const Tensor& logits, int64_t probes, const Tensor& valid) {
  check_route(logits, probes, valid);
  if (logits.is_cuda()) return route_gpu(logits, probes, valid);
  const at::Device gpu = gpu_for_cpu_call();
  RouteOut o = route_gpu(logits.to(gpu), probes, valid.defined() ? valid.to(gpu) : valid);
  for (Tensor* t : {&o.ids, &o.weights, &o.lse, &o.counts, &o.loss, &o.stats, &o.slopes}) *t = t->cpu();
  return o;
}

struct RouteFunction : torch::autograd::Function<RouteFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t probes, const OptTensor& valid) {
    at::AutoDispatchBelowADInplaceOrView below;
    RouteOut o = route_any(logits, probes, valid.value_or(Tensor()));
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, o.ids, o.weights, o.stats, o.slopes});
    ctx->mark_non_differentiable({o.ids, o.counts});
    return {o.ids, o.weights, o.lse, o.counts, o.loss};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    return {differentiable_once(logits_gradient(saved, grads), saved[0], grads, "cluster_route"), Tensor(), Tensor()};
  }

  static Tensor logits_gradient(const variable_list& saved, const variable_list& grads) {
    at::AutoDispatchBelowADInplaceOrView below;
    const bool on_gpu = saved[0].is_cuda();
    const at::Device dev = on_gpu ? saved[0].device() : gpu_for_cpu_call();
    c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(dev);
    const Tensor z = with_adjacent_columns(saved[0].to(dev));
    const Tensor ids = saved[1].to(dev), weights = saved[2].to(dev), stats = saved[3].to(dev),
                 slopes = saved[4].to(dev);
    const Tensor gw = gradient(grads[1], dev), gs = gradient(grads[2], dev), gl = gradient(grads[4], dev);
    Tensor grad = at::empty(z.sizes(), z.options());
    check_st(st_cluster_route_backward(bytes_or_null(z), score_type(z.scalar_type(), "logits"), z.size(0), z.size(1),
                                       z.stride(0), ids.size(1), data_or_null<int64_t>(ids),
                                       data_or_null<float>(weights), data_or_null<float>(stats),
                                       data_or_null<float>(slopes), data_or_null<float>(gw), data_or_null<float>(gs),
                                       data_or_null<float>(gl), bytes_or_null(grad), current_stream(z)),
             "cluster_route");
    return on_gpu ? grad : grad.cpu();
  }
};

using Route = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

Route cluster_route(const Tensor& logits, int64_t probes, const OptTensor& valid) {
  RouteOut o = route_any(logits, probes, valid.value_or(Tensor()));
  return {o.ids, o.weights, o.lse, o.counts, o.loss};
}

Route cluster_route_autograd(const Tensor& logits, int64_t probes, const OptTensor& valid) {
  refuse_tangents({&logits}, "cluster_route");
  if (!at::GradMode::is_enabled() || !logits.requires_grad()) {
    at::AutoDispatchBelowADInplaceOrView below;
    return cluster_route(logits, probes, valid);
  }
  const variable_list o = RouteFunction::apply(logits, probes, valid);
  return {o[0], o[1], o[2], o[3], o[4]};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(st, m) {
  // packed uint8 [N, 16 ceil(D / 32)], scales [N, groups] of the weight's
  // type, zeros uint8 [N, groups]
  m.def("int4_quantize(Tensor weight, int group_size, bool symmetric=True) -> (Tensor, Tensor, Tensor)");
  // x [D] or [B, D] times the table transposed
  m.def("int4_matvec(Tensor packed, Tensor scales, Tensor x, int group_size, Tensor? zeros=None, "
        "ScalarType? out_dtype=None) -> Tensor");
  // (logprobs, entropy, lse, top_ids, top_logprobs)
  m.def("target_logprobs(Tensor logits, Tensor targets, int topk=0, Tensor? packed_mask=None, "
        "float temperature=1.0) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  // (cluster_ids, weights, lse, counts, balance_loss)
  m.def("cluster_route(Tensor logits, int probes, Tensor? valid=None) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(st, CUDA, m) {
  m.impl("int4_quantize", TORCH_FN(int4_quantize_gpu));
  m.impl("int4_matvec", TORCH_FN(int4_matvec_gpu));
  m.impl("target_logprobs", TORCH_FN(target_logprobs));
  m.impl("cluster_route", TORCH_FN(cluster_route));
}

TORCH_LIBRARY_IMPL(st, CPU, m) {
  m.impl("int4_quantize", TORCH_FN(int4_quantize_cpu));
  m.impl("int4_matvec", TORCH_FN(int4_matvec_cpu));
  m.impl("target_logprobs", TORCH_FN(target_logprobs));
  m.impl("cluster_route", TORCH_FN(cluster_route));
}

TORCH_LIBRARY_IMPL(st, Autograd, m) {
  m.impl("int4_quantize", TORCH_FN(int4_quantize_autograd));
  m.impl("int4_matvec", TORCH_FN(int4_matvec_autograd));
  m.impl("target_logprobs", TORCH_FN(target_logprobs_autograd));
  m.impl("cluster_route", TORCH_FN(cluster_route_autograd));
}
