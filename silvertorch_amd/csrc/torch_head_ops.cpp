// torch.ops.st.* of the retrieval head: 4-bit score tables, log-probabilities
// of given documents, cluster routing.  No reference counterparts.
//
// As in torch_ops.cpp, GPU tensors run on their device's current stream and
// CPU tensors are copied to the current GPU and the results back.  The two
// operators a model is trained through carry their gradients (Autograd key);
// the 4-bit ones refuse to be differentiated.  Below that key every kernel is
// called through the dispatcher, so that a dispatch mode sees it.
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
using st_torch::gradient;
using st_torch::if_defined;
using st_torch::moved;
using st_torch::OnceDifferentiable;
using st_torch::OptTensor;
using st_torch::refuse_tangents;
using st_torch::score_type;
using st_torch::with_adjacent_columns;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

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

Tensor differentiable_once(const Tensor& grad, const Tensor& logits, const variable_list& outer, const char* op) {
  if (!at::GradMode::is_enabled()) return grad;
  return OnceDifferentiable::apply(grad, logits, if_defined(outer[0]), if_defined(outer[1]), if_defined(outer[2]),
                                   if_defined(outer[4]), std::string(op));
}

using Logprobs = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;
using LogprobsStats = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

Logprobs target_logprobs(const Tensor& logits, const Tensor& targets, int64_t topk, const OptTensor& mask,
                         double temperature) {
  LogprobsOut o = logprobs_any(logits, targets, topk, mask.value_or(Tensor()), temperature, false);
  return {o.logprobs, o.entropy, o.lse, o.top_ids, o.top_logprobs};
}

LogprobsStats target_logprobs_with_stats(const Tensor& logits, const Tensor& targets, int64_t topk,
                                         const OptTensor& mask, double temperature) {
  LogprobsOut o = logprobs_any(logits, targets, topk, mask.value_or(Tensor()), temperature, true);
  return {o.logprobs, o.entropy, o.lse, o.top_ids, o.top_logprobs, o.stats};
}

// The gradients of logprobs, entropy, lse and top_logprobs, each absent where it is zero.
Tensor target_logprobs_backward(const Tensor& logits, const Tensor& targets, int64_t topk, const OptTensor& packed_mask,
                                double temperature, const Tensor& entropy_in, const Tensor& top_ids_in,
                                const Tensor& stats_in, const OptTensor& g_logprobs, const OptTensor& g_entropy,
                                const OptTensor& g_lse, const OptTensor& g_top) {
  const Tensor mask = packed_mask.value_or(Tensor());
  check_logprobs(logits, targets, topk, mask, temperature);
  const int64_t n = logits.size(0);
  auto check = [&](const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, const char* what) {
    TORCH_CHECK(t.sizes() == sizes && t.scalar_type() == type && t.device() == logits.device(), what, " must be ", type,
                " of ", sizes, " on the scores' device, got ", t.scalar_type(), " of ", t.sizes());
  };
  check(entropy_in, {n}, at::kFloat, "entropy");
  check(top_ids_in, {n, topk}, at::kLong, "top_ids");
  check(stats_in, {n, 2}, at::kFloat, "stats");
  for (const OptTensor* g : {&g_logprobs, &g_entropy, &g_lse, &g_top}) {
    if (!g->has_value() || !(*g)->defined()) continue;
    const bool of_rows = g != &g_top;
    TORCH_CHECK((of_rows ? (*g)->sizes() == at::IntArrayRef({n}) : (*g)->sizes() == at::IntArrayRef({n, topk})) &&
                    (*g)->device() == logits.device(),
                "gradients must be of the results' shapes and device, got ", (*g)->sizes());
  }
  const bool on_gpu = logits.is_cuda();
  const at::Device dev = on_gpu ? logits.device() : gpu_for_cpu_call();
  const LogprobsIn in =
      logprobs_in(logits.to(dev), targets.to(dev), topk, mask.defined() ? mask.to(dev) : mask, temperature);
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(dev);
  auto there = [&](const Tensor& t) { return t.to(dev).contiguous(); };
  const Tensor entropy = there(entropy_in), top_ids = there(top_ids_in), stats = there(stats_in);
  auto given = [&](const OptTensor& g) { return gradient(g.value_or(Tensor()), dev); };
  const Tensor gl = given(g_logprobs), ge = given(g_entropy), gs = given(g_lse), gt = given(g_top);
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

using LogprobsOp = Logprobs(const Tensor&, const Tensor&, int64_t, const OptTensor&, double);
using LogprobsKeepOp = LogprobsStats(const Tensor&, const Tensor&, int64_t, const OptTensor&, double);
using LogprobsBackwardOp = Tensor(const Tensor&, const Tensor&, int64_t, const OptTensor&, double, const Tensor&,
                                  const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                                  const OptTensor&);

Logprobs logprobs_below(const Tensor& logits, const Tensor& targets, int64_t topk, const OptTensor& mask,
                        double temperature) {
  static const auto op = find_op<LogprobsOp>("st::target_logprobs");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(logits, targets, topk, mask, temperature);
}

LogprobsStats logprobs_with_stats_below(const Tensor& logits, const Tensor& targets, int64_t topk, const OptTensor& mask,
                                        double temperature) {
  static const auto op = find_op<LogprobsKeepOp>("st::target_logprobs_with_stats");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(logits, targets, topk, mask, temperature);
}

struct LogprobsFunction : torch::autograd::Function<LogprobsFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, int64_t topk,
                               const OptTensor& packed_mask, double temperature) {
    auto [logprobs, entropy, lse, top_ids, top_logprobs, stats] =
        logprobs_with_stats_below(logits, targets, topk, packed_mask, temperature);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, targets, packed_mask.value_or(Tensor()), entropy, top_ids, stats});
    ctx->saved_data["topk"] = topk;
    ctx->saved_data["temperature"] = temperature;
    ctx->mark_non_differentiable({top_ids});
    return {logprobs, entropy, lse, top_ids, top_logprobs};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor grad = logits_gradient(ctx, saved, grads);
    return {differentiable_once(grad, saved[0], grads, "target_logprobs"), Tensor(), Tensor(), Tensor(), Tensor()};
  }

  static Tensor logits_gradient(AutogradContext* ctx, const variable_list& saved, const variable_list& grads) {
    static const auto op = find_op<LogprobsBackwardOp>("st::target_logprobs_backward");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(saved[0], saved[1], ctx->saved_data["topk"].toInt(), if_defined(saved[2]),
                   ctx->saved_data["temperature"].toDouble(), saved[3], saved[4], saved[5], if_defined(grads[0]),
                   if_defined(grads[1]), if_defined(grads[2]), if_defined(grads[4]));
  }
};

Logprobs target_logprobs_autograd(const Tensor& logits, const Tensor& targets, int64_t topk, const OptTensor& mask,
                                  double temperature) {
  refuse_tangents({&logits}, "target_logprobs");
  if (!at::GradMode::is_enabled() || !logits.requires_grad())
    return logprobs_below(logits, targets, topk, mask, temperature);
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

using Route = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;
using RouteStats = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

Route cluster_route(const Tensor& logits, int64_t probes, const OptTensor& valid) {
  RouteOut o = route_any(logits, probes, valid.value_or(Tensor()));
  return {o.ids, o.weights, o.lse, o.counts, o.loss};
}

RouteStats cluster_route_with_stats(const Tensor& logits, int64_t probes, const OptTensor& valid) {
  RouteOut o = route_any(logits, probes, valid.value_or(Tensor()));
  return {o.ids, o.weights, o.lse, o.counts, o.loss, o.stats, o.slopes};
}

// The gradients of weights, lse and the loss, each absent where it is zero.
Tensor cluster_route_backward(const Tensor& logits, const Tensor& ids_in, const Tensor& weights_in,
                              const Tensor& stats_in, const Tensor& slopes_in, const OptTensor& g_weights,
                              const OptTensor& g_lse, const OptTensor& g_loss) {
  TORCH_CHECK(ids_in.dim() == 2, "cluster_ids must be a 2-D tensor");
  const int64_t probes = ids_in.size(1);
  check_route(logits, probes, Tensor());
  const int64_t n = logits.size(0), e = logits.size(1);
  auto check = [&](const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, const char* what) {
    TORCH_CHECK(t.sizes() == sizes && t.scalar_type() == type && t.device() == logits.device(), what, " must be ", type,
                " of ", sizes, " on the scores' device, got ", t.scalar_type(), " of ", t.sizes());
  };
  check(ids_in, {n, probes}, at::kLong, "cluster_ids");
  check(weights_in, {n, probes}, at::kFloat, "weights");
  check(stats_in, {n, 2}, at::kFloat, "stats");
  check(slopes_in, {e}, at::kFloat, "slopes");
  auto check_gradient = [&](const OptTensor& g, at::IntArrayRef sizes) {
    TORCH_CHECK(!g.has_value() || !g->defined() || (g->sizes() == sizes && g->device() == logits.device()),
                "gradients must be of the results' shapes and device");
  };
  check_gradient(g_weights, {n, probes});
  check_gradient(g_lse, {n});
  check_gradient(g_loss, {});
  const bool on_gpu = logits.is_cuda();
  const at::Device dev = on_gpu ? logits.device() : gpu_for_cpu_call();
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(dev);
  const Tensor z = with_adjacent_columns(logits.to(dev));
  auto there = [&](const Tensor& t) { return t.to(dev).contiguous(); };
  const Tensor ids = there(ids_in), weights = there(weights_in), stats = there(stats_in), slopes = there(slopes_in);
  auto given = [&](const OptTensor& g) { return gradient(g.value_or(Tensor()), dev); };
  const Tensor gw = given(g_weights), gs = given(g_lse), gl = given(g_loss);
  Tensor grad = at::empty(z.sizes(), z.options());
  check_st(st_cluster_route_backward(bytes_or_null(z), score_type(z.scalar_type(), "logits"), z.size(0), z.size(1),
                                     z.stride(0), probes, data_or_null<int64_t>(ids), data_or_null<float>(weights),
                                     data_or_null<float>(stats), data_or_null<float>(slopes), data_or_null<float>(gw),
                                     data_or_null<float>(gs), data_or_null<float>(gl), bytes_or_null(grad),
                                     current_stream(z)),
           "cluster_route");
  return on_gpu ? grad : grad.cpu();
}

using RouteOp = Route(const Tensor&, int64_t, const OptTensor&);
using RouteKeepOp = RouteStats(const Tensor&, int64_t, const OptTensor&);
using RouteBackwardOp = Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                               const OptTensor&, const OptTensor&, const OptTensor&);

Route route_below(const Tensor& logits, int64_t probes, const OptTensor& valid) {
  static const auto op = find_op<RouteOp>("st::cluster_route");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(logits, probes, valid);
}

RouteStats route_with_stats_below(const Tensor& logits, int64_t probes, const OptTensor& valid) {
  static const auto op = find_op<RouteKeepOp>("st::cluster_route_with_stats");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(logits, probes, valid);
}

struct RouteFunction : torch::autograd::Function<RouteFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t probes, const OptTensor& valid) {
    auto [ids, weights, lse, counts, loss, stats, slopes] = route_with_stats_below(logits, probes, valid);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, ids, weights, stats, slopes});
    ctx->mark_non_differentiable({ids, counts});
    return {ids, weights, lse, counts, loss};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    return {differentiable_once(logits_gradient(saved, grads), saved[0], grads, "cluster_route"), Tensor(), Tensor()};
  }

  static Tensor logits_gradient(const variable_list& saved, const variable_list& grads) {
    static const auto op = find_op<RouteBackwardOp>("st::cluster_route_backward");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(saved[0], saved[1], saved[2], saved[3], saved[4], if_defined(grads[1]), if_defined(grads[2]),
                   if_defined(grads[4]));
  }
};

Route cluster_route_autograd(const Tensor& logits, int64_t probes, const OptTensor& valid) {
  refuse_tangents({&logits}, "cluster_route");
  if (!at::GradMode::is_enabled() || !logits.requires_grad()) return route_below(logits, probes, valid);
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
  // What its gradient calls: the same and the statistics; the gradient of the scores.
  m.def("target_logprobs_with_stats(Tensor logits, Tensor targets, int topk, Tensor? packed_mask, float temperature) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("target_logprobs_backward(Tensor logits, Tensor targets, int topk, Tensor? packed_mask, float temperature, "
        "Tensor entropy, Tensor top_ids, Tensor stats, Tensor? g_logprobs, Tensor? g_entropy, Tensor? g_lse, "
        "Tensor? g_top) -> Tensor");
  // (cluster_ids, weights, lse, counts, balance_loss)
  m.def("cluster_route(Tensor logits, int probes, Tensor? valid=None) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  // What its gradient calls: the same with statistics and slopes; the gradient of the scores.
  m.def("cluster_route_with_stats(Tensor logits, int probes, Tensor? valid) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("cluster_route_backward(Tensor logits, Tensor cluster_ids, Tensor weights, Tensor stats, Tensor slopes, "
        "Tensor? g_weights, Tensor? g_lse, Tensor? g_loss) -> Tensor");
}

TORCH_LIBRARY_IMPL(st, CUDA, m) {
  m.impl("int4_quantize", TORCH_FN(int4_quantize_gpu));
  m.impl("int4_matvec", TORCH_FN(int4_matvec_gpu));
  m.impl("target_logprobs", TORCH_FN(target_logprobs));
  m.impl("target_logprobs_with_stats", TORCH_FN(target_logprobs_with_stats));
  m.impl("target_logprobs_backward", TORCH_FN(target_logprobs_backward));
  m.impl("cluster_route", TORCH_FN(cluster_route));
  m.impl("cluster_route_with_stats", TORCH_FN(cluster_route_with_stats));
  m.impl("cluster_route_backward", TORCH_FN(cluster_route_backward));
}

TORCH_LIBRARY_IMPL(st, CPU, m) {
  m.impl("int4_quantize", TORCH_FN(int4_quantize_cpu));
  m.impl("int4_matvec", TORCH_FN(int4_matvec_cpu));
  m.impl("target_logprobs", TORCH_FN(target_logprobs));
  m.impl("target_logprobs_with_stats", TORCH_FN(target_logprobs_with_stats));
  m.impl("target_logprobs_backward", TORCH_FN(target_logprobs_backward));
  m.impl("cluster_route", TORCH_FN(cluster_route));
  m.impl("cluster_route_with_stats", TORCH_FN(cluster_route_with_stats));
  m.impl("cluster_route_backward", TORCH_FN(cluster_route_backward));
}

TORCH_LIBRARY_IMPL(st, Autograd, m) {
  m.impl("int4_quantize", TORCH_FN(int4_quantize_autograd));
  m.impl("int4_matvec", TORCH_FN(int4_matvec_autograd));
  m.impl("target_logprobs", TORCH_FN(target_logprobs_autograd));
  m.impl("cluster_route", TORCH_FN(cluster_route_autograd));
}
