// Entry points of the layer norm (layer_norm_kernel.hpp holds the kernels), and
// the sum of its workgroups' parts of the weight's and bias's gradients.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "layer_norm_kernel.hpp"
#include "st_errors.hpp"

namespace st {
int cu_count();

template <>
NormShape norm_forward<ST_SCORE_F32>(int dim, bool wide_sum, bool codes);
template <>
NormShape norm_forward<ST_SCORE_F16>(int dim, bool wide_sum, bool codes);
template <>
NormShape norm_forward<ST_SCORE_BF16>(int dim, bool wide_sum, bool codes);
template <>
const void* norm_backward<ST_SCORE_F32>(int dim, bool wide_sum);
template <>
const void* norm_backward<ST_SCORE_F16>(int dim, bool wide_sum);
template <>
const void* norm_backward<ST_SCORE_BF16>(int dim, bool wide_sum);
template <>
const void* norm_columns<ST_SCORE_F32>(bool wide_sum);
template <>
const void* norm_columns<ST_SCORE_F16>(bool wide_sum);
template <>
const void* norm_columns<ST_SCORE_BF16>(bool wide_sum);

namespace {

void check_type(int type, const char* what) {
  ST_CHECK(type == ST_SCORE_F32 || type == ST_SCORE_F16 || type == ST_SCORE_BF16, what,
           " must be float32, float16 or bfloat16");
}

void check_rows(int64_t rows, int64_t dim) {
  ST_CHECK(rows >= 0, "negative number of rows");
  ST_CHECK(dim >= 1 && dim <= kMaxNormColumns, "columns must be in [1, ", kMaxNormColumns, "], got ", dim);
}

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw Error(ST_ERR_HIP, cat(what, " launch failed: ", hipGetErrorString(e)));
}

NormShape forward_shape_of(int type, int dim, bool wide_sum, bool codes) {
  if (type == ST_SCORE_F32) return norm_forward<ST_SCORE_F32>(dim, false, codes);
  if (type == ST_SCORE_F16) return norm_forward<ST_SCORE_F16>(dim, wide_sum, codes);
  return norm_forward<ST_SCORE_BF16>(dim, wide_sum, codes);
}

const void* backward_kernel_of(int type, int dim, bool wide_sum) {
  if (type == ST_SCORE_F32) return norm_backward<ST_SCORE_F32>(dim, false);
  if (type == ST_SCORE_F16) return norm_backward<ST_SCORE_F16>(dim, wide_sum);
  return norm_backward<ST_SCORE_BF16>(dim, wide_sum);
}

const void* columns_kernel_of(int type, bool wide_sum) {
  if (type == ST_SCORE_F32) return norm_columns<ST_SCORE_F32>(false);
  if (type == ST_SCORE_F16) return norm_columns<ST_SCORE_F16>(wide_sum);
  return norm_columns<ST_SCORE_BF16>(wide_sum);
}

void launch_kernel(const void* kernel, dim3 grid, int threads, void* args, const char* what, hipStream_t s) {
  void* list[] = {args};
  const hipError_t e = hipLaunchKernel(kernel, grid, dim3(threads), list, 0, s);
  if (e != hipSuccess) throw Error(ST_ERR_HIP, cat(what, " launch failed: ", hipGetErrorString(e)));
}

void launch_forward(NormArgs& a, int type, bool wide_sum, bool codes, hipStream_t s) {
  const NormShape shape = forward_shape_of(type, a.dim, wide_sum, codes);
  const int64_t grid = std::min<int64_t>((a.rows + shape.rows - 1) / shape.rows, static_cast<int64_t>(shape.per_cu) * cu_count());
  launch_kernel(shape.kernel, dim3(static_cast<unsigned>(grid)), shape.threads, &a, "norm_kernel", s);
}

// The backward kernel's workgroups, for the workspace and the launch: each adds two
// rows of sums in 32 bits to the traffic, so there are no more of them than the
// current device holds at once, and each takes four turns at least where that leaves
// one a CU.
int64_t backward_groups(int64_t rows, int64_t dim) {
  const NormLayout l = kNormLayouts[norm_layout(dim)];
  const int64_t turns = (rows + norm_rows(l.lanes) - 1) / norm_rows(l.lanes);
  const int64_t cus = cu_count(), most = cus * std::max(1, norm_backward_waves(l.lanes, l.steps) * 256 / norm_threads(l.lanes));
  return std::max<int64_t>(1, std::min(most, std::max(std::min(turns, cus), turns / 4)));
}

// out[c] = sum over the parts, for C columns of gw and gb side by side: 1,024 / C
// threads a column take turns with the parts.
template <int C>
__global__ __launch_bounds__(1024) void norm_finish_kernel(const float* partial, int parts, int dim, void* gw, void* gb,
                                                           int type) {
  __shared__ float sums[1024];
  const int column = blockIdx.x * C + threadIdx.x % C;
  float t = 0.0f;
  if (column < 2 * dim) {
    const float* from = partial + column;
    const int64_t step = 2 * static_cast<int64_t>(dim);
#pragma unroll 8
    for (int p = threadIdx.x / C; p < parts; p += 1024 / C) t += from[p * step];
  }
  sums[threadIdx.x] = t;
  __syncthreads();
  for (int half = 512; half >= C; half /= 2) {
    if (threadIdx.x < half) sums[threadIdx.x] += sums[threadIdx.x + half];
    __syncthreads();
  }
  if (threadIdx.x >= C || column >= 2 * dim) return;
  void* out = column < dim ? gw : gb;
  if (!out) return;
  const int c = column < dim ? column : column - dim;
  if (type == ST_SCORE_F32)
    store_score<ST_SCORE_F32>(out, c, sums[threadIdx.x]);
  else if (type == ST_SCORE_F16)
    store_score<ST_SCORE_F16>(out, c, sums[threadIdx.x]);
  else
    store_score<ST_SCORE_BF16>(out, c, sums[threadIdx.x]);
}

}  // namespace

// The codes and scales of rows as they are (int8_matmul.hip).
void launch_codes(const void* x, int x_type, int64_t rows, int64_t dim, int64_t x_stride, int8_t* codes, int64_t columns,
                  float* scales, hipStream_t s) {
  NormArgs a{};
  a.x = x;
  a.y = codes;
  a.scales = scales;
  a.rows = rows;
  a.x_stride = x_stride;
  a.dim = static_cast<int>(dim);
  a.code_columns = static_cast<int>(columns);
  launch_forward(a, x_type, false, true, s);
}

namespace {

float checked_eps(double eps) {
  ST_CHECK(eps >= 1e-30 && eps <= 1e30, "eps must be in [1e-30, 1e30], got ", eps);
  return static_cast<float>(eps);
}

}  // namespace
}  // namespace st

extern "C" int st_layer_norm(const void* x, int x_type, int64_t rows, int64_t dim, int64_t x_stride, const void* residual,
                             int residual_type, int64_t residual_stride, const void* weight, const void* bias,
                             int weight_type, double eps, double p, const int64_t* state, void* y, void* sum, float* stats,
                             int64_t* used, void* stream) {
  using namespace st;
  return guarded([&] {
    check_type(x_type, "x");
    check_type(weight_type, "weight and bias");
    check_rows(rows, dim);
    NormArgs a{};
    a.eps = checked_eps(eps);
    a.dropout = dropout_args(p, state, used);
    ST_CHECK(residual || a.dropout.dropped == 0, "dropout goes with a residual");
    ST_CHECK(a.dropout.dropped == 0 || state || rows == 0, "dropout needs a state");
    if (residual) {
      check_type(residual_type, "residual");
      ST_CHECK(residual_type == x_type || residual_type == ST_SCORE_F32, "residual must be of x's type or float32");
    }
    if (rows == 0) return;
    ST_CHECK(x && y && (!residual || sum), "null device pointer");
    if (a.dropout.dropped == 0 && !used) a.dropout.state = nullptr;
    ST_CHECK(!used || state, "null device pointer");
    a.x = x;
    a.residual = residual;
    a.weight = weight;
    a.bias = bias;
    a.y = y;
    a.sum = sum;
    a.stats = stats;
    a.rows = rows;
    a.x_stride = x_stride;
    a.residual_stride = residual_stride;
    a.dim = static_cast<int>(dim);
    a.weight_type = weight_type;
    a.normalise = 1;
    launch_forward(a, x_type, residual && residual_type != x_type, false, static_cast<hipStream_t>(stream));
  });
}

extern "C" int st_layer_norm_int8(const void* x, int x_type, int64_t rows, int64_t dim, int64_t x_stride,
                                  const void* weight, const void* bias, int weight_type, double eps, int8_t* codes,
                                  float* scales, void* stream) {
  using namespace st;
  return guarded([&] {
    check_type(x_type, "x");
    check_type(weight_type, "weight and bias");
    check_rows(rows, dim);
    NormArgs a{};
    a.eps = checked_eps(eps);
    if (rows == 0) return;
    ST_CHECK(x && codes && scales, "null device pointer");
    ST_CHECK(reinterpret_cast<uintptr_t>(codes) % 16 == 0, "codes must be 16-byte aligned");
    a.x = x;
    a.weight = weight;
    a.bias = bias;
    a.y = codes;
    a.scales = scales;
    a.rows = rows;
    a.x_stride = x_stride;
    a.dim = static_cast<int>(dim);
    a.code_columns = static_cast<int>((dim + 15) / 16 * 16);
    a.weight_type = weight_type;
    a.normalise = 1;
    a.dropout.times = 1.0f;
    launch_forward(a, x_type, false, true, static_cast<hipStream_t>(stream));
  });
}

extern "C" int64_t st_layer_norm_workspace_bytes(int64_t rows, int64_t dim) {
  using namespace st;
  if (rows <= 0 || dim < 1 || dim > kMaxNormColumns) return 0;
  return backward_groups(rows, dim) * 2 * dim * static_cast<int64_t>(sizeof(float));
}

extern "C" int st_layer_norm_backward(const void* grad_y, int y_type, const void* grad_sum, const void* h, int h_type,
                                      int64_t rows, int64_t dim, int64_t h_stride, const void* weight, int weight_type,
                                      const float* stats, double p, const int64_t* state, void* workspace, void* grad_x,
                                      void* grad_residual, void* grad_weight, void* grad_bias, void* stream) {
  using namespace st;
  return guarded([&] {
    check_type(y_type, "x");
    check_type(h_type, "residual");
    check_type(weight_type, "weight and bias");
    ST_CHECK(h_type == y_type || h_type == ST_SCORE_F32, "residual must be of x's type or float32");
    check_rows(rows, dim);
    NormBackwardArgs a{};
    a.dropout = dropout_args(p, state, nullptr);
    ST_CHECK(a.dropout.dropped == 0 || state || rows == 0, "dropout needs a state");
    const bool sums = grad_weight || grad_bias;
    if (!sums && !grad_x && !grad_residual) return;
    ST_CHECK(rows == 0 || (grad_y && h && stats), "null device pointer");
    ST_CHECK(rows == 0 || !sums || workspace, "null device pointer");
    hipStream_t s = static_cast<hipStream_t>(stream);
    int64_t groups = 0;
    if (rows > 0) {
      groups = backward_groups(rows, dim);
      if (a.dropout.dropped == 0) a.dropout.state = nullptr;
      a.gy = grad_y;
      a.gsum = grad_sum;
      a.h = h;
      a.weight = weight;
      a.gx = grad_x;
      a.gh = grad_residual;
      a.stats = stats;
      a.partial = sums ? static_cast<float*>(workspace) : nullptr;
      a.rows = rows;
      a.h_stride = h_stride;
      a.dim = static_cast<int>(dim);
      a.weight_type = weight_type;
      a.inverse_dim = 1.0f / static_cast<float>(dim);
      const bool apart = norm_columns_apart(dim), wide = h_type != y_type;
      if (!apart || grad_x || grad_residual)
        launch_kernel(backward_kernel_of(y_type, a.dim, wide), dim3(static_cast<unsigned>(groups)),
                      norm_threads(kNormLayouts[norm_layout(dim)].lanes), &a, "norm_backward_kernel", s);
      if (apart && sums) {
        groups = std::min<int64_t>(groups, 128);  // times 2,048 columns each
        launch_kernel(columns_kernel_of(y_type, wide), dim3(static_cast<unsigned>((dim + 2047) / 2048), static_cast<unsigned>(groups)),
                      256, &a, "norm_columns_kernel", s);
      }
    }
    if (sums) {  // without rows the sums are zeros
      const float* partial = static_cast<const float*>(workspace);
      const int columns = dim < 2048 ? 16 : 32, parts = static_cast<int>(groups), d = static_cast<int>(dim);
      hipLaunchKernelGGL(columns == 16 ? norm_finish_kernel<16> : norm_finish_kernel<32>,
                         dim3(static_cast<unsigned>((2 * dim + columns - 1) / columns)), dim3(1024), 0, s, partial, parts, d,
                         grad_weight, grad_bias, weight_type);
      check_launch("norm_finish_kernel");
    }
  });
}
