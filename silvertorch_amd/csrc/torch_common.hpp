// Helpers shared by the files that register torch.ops.st.*.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/hip/HIPFunctions.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include "../../include/silvertorch_hip.h"

namespace st_torch {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

inline void check_st(int rc, const char* what) {
  TORCH_CHECK(rc == ST_OK, what, ": ", st_last_error());
}

inline void* current_stream(const at::Tensor& t) {
  return static_cast<void*>(
      c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream());
}

inline at::Device gpu_for_cpu_call() {
  TORCH_CHECK(c10::hip::device_count() > 0,
              "silvertorch_amd computes the bloom path with HIP kernels on an "
              "MI355X; no GPU is visible to this process");
  return at::Device(at::kCUDA, c10::hip::current_device());
}

inline int score_type(at::ScalarType t, const char* what) {
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

inline void* bytes_or_null(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

// None of these operators has a forward-mode derivative: an input that carries
// a tangent is refused, where the result would otherwise come without one.
inline void refuse_tangents(std::initializer_list<const Tensor*> inputs, const char* op) {
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), op, " has no forward-mode derivative");
}

inline Tensor moved(const OptTensor& t, at::Device d) { return t.has_value() && t->defined() ? t->to(d) : Tensor(); }

template <typename Op>
auto find_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Op>();
}

// A score row is readable with any row stride; columns have to be adjacent.
inline Tensor with_adjacent_columns(const Tensor& t) { return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous(); }

// A gradient as the kernels take it: float32, contiguous, on the device.
inline Tensor gradient(const Tensor& g, at::Device d) {
  return g.defined() ? g.to(d, at::kFloat).contiguous() : g;
}

}  // namespace st_torch
