// Gradients that cannot be differentiated again, for the files that register
// differentiable operators.
#pragma once

#include <torch/csrc/autograd/custom_function.h>

#include <string>

#include "torch_common.hpp"

namespace st_torch {

// A gradient with a graph over it (backward with create_graph): it depends on
// the input `of` and on the outputs' gradients, and refuses to be differentiated
// where it would otherwise count as a constant.
struct OnceDifferentiable : torch::autograd::Function<OnceDifferentiable> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& grad, const Tensor& /*of*/,
                        const OptTensor& /*g0*/, const OptTensor& /*g1*/, const OptTensor& /*g2*/, const OptTensor& /*g3*/,
                        std::string op) {
    ctx->saved_data["op"] = std::move(op);
    return grad;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list /*grads*/) {
    TORCH_CHECK(false, "the gradient of ", ctx->saved_data["op"].toStringRef(), " cannot be differentiated again");
  }
};

inline OptTensor if_defined(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

}  // namespace st_torch
