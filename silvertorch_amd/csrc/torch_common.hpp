// Helpers shared by the files that register torch.ops.st.*.
#pragma once

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include "../../include/silvertorch_hip.h"

namespace st_torch {

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

}  // namespace st_torch
