// Matrix-vector products with a table held in 4 bits, and the table's making.
//
// No reference operator.  A table row n has ceil(D / 32) * 16 bytes: column 2j
// in the low half of byte j, column 2j + 1 in the high half.  Each group of
// `group` columns (a multiple of 32; the last may be short) has a scale and,
// with `zeros`, a zero point (else 8):
//   y[b, n] = sum_g scale[n, g] sum_{d in g} (q[n, d] - zero[n, g]) x[b, d]
// What a row's last block of 32 holds past column D is not used.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "score_ops.hpp"
#include "st_errors.hpp"

namespace st {
int cu_count();

namespace {

constexpr int kBlock = 32;  // columns of 16 bytes

struct MatvecArgs {
  const uint8_t* packed;
  const void* scales;
  const uint8_t* zeros;  // null: 8
  const void* x;
  void* y;
  int64_t rows, dim, queries, group, groups, row_bytes;
  int scale_type, x_type, y_type;
};

__device__ __forceinline__ float load_any(const void* p, int64_t i, int type) {
  if (type == ST_SCORE_F32) return load_score<ST_SCORE_F32>(p, i);
  if (type == ST_SCORE_F16) return load_score<ST_SCORE_F16>(p, i);
  return load_score<ST_SCORE_BF16>(p, i);
}

__device__ __forceinline__ void store_any(void* p, int64_t i, float v, int type) {
  if (type == ST_SCORE_F32)
    store_score<ST_SCORE_F32>(p, i, v);
  else if (type == ST_SCORE_F16)
    store_score<ST_SCORE_F16>(p, i, v);
  else
    store_score<ST_SCORE_BF16>(p, i, v);
}

// A thread per table row and query.
__global__ __launch_bounds__(256) void matvec_kernel(MatvecArgs a) {
  const int64_t total = a.rows * a.queries;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t b = i / a.rows, n = i - b * a.rows;
    float y = 0.0f;
    for (int64_t g = 0; g < a.groups; ++g) {
      const float zero = a.zeros != nullptr ? static_cast<float>(a.zeros[n * a.groups + g]) : 8.0f;
      const int64_t end = min((g + 1) * a.group, a.dim);
      const float scale = load_any(a.scales, n * a.groups + g, a.scale_type);
      for (int64_t d = g * a.group; d < end; ++d) {
        const uint32_t byte = a.packed[n * a.row_bytes + d / 2];
        const float q = static_cast<float>((d & 1) ? byte >> 4 : byte & 15u);
        y = fmaf((q - zero) * scale, load_any(a.x, b * a.dim + d, a.x_type), y);
      }
    }
    store_any(a.y, i, y, a.y_type);
  }
}

struct QuantizeArgs {
  const void* weight;
  uint8_t* packed;
  void* scales;
  uint8_t* zeros;
  int64_t rows, dim, group, groups, row_bytes;
  int symmetric;
};

// A wave per row and group.  Symmetric: scale = max |w| / 7 rounded to the
// weights' type, code = w / scale to the nearest even, kept in [-8, 7], plus 8.
// Else lo = min(w, 0), hi = max(w, 0): scale = (hi - lo) / 15, zero = -lo /
// scale, code = w / scale + zero, each to the nearest even and kept in
// [0, 15].  A group of zeros has scale 0; one with a value that is not finite
// has scale NaN, so that its products say so.
template <int DT>
__global__ __launch_bounds__(256) void quantize_kernel(QuantizeArgs a) {
  const int lane = threadIdx.x % 64;
  const int64_t items = a.rows * a.groups;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 64; item < items;
       item += static_cast<int64_t>(gridDim.x) * 4) {
    const int64_t n = item / a.groups, g = item - n * a.groups;
    const int64_t first = g * a.group, end = min(first + a.group, a.dim);
    const char* row = static_cast<const char*>(a.weight) + n * a.dim * kScoreBytes<DT>;
    float lo = 0.0f, hi = 0.0f;
    bool finite = true;
    for (int64_t d = first + lane; d < end; d += 64) {
      const float w = load_score<DT>(row, d);
      finite &= __builtin_isfinite(w);
      lo = fminf(lo, w);
      hi = fmaxf(hi, w);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor(lo, o));
      hi = fmaxf(hi, __shfl_xor(hi, o));
    }
    finite = __all(finite);
    float scale = a.symmetric ? __fdiv_rn(fmaxf(-lo, hi), 7.0f) : __fdiv_rn(hi - lo, 15.0f);
    if (!finite) scale = __builtin_nanf("");
    scale = score_of_bits<DT>(score_bits<DT>(scale));
    const bool any = scale > 0.0f;
    float zero = 8.0f;
    if (!a.symmetric) zero = any ? fminf(fmaxf(rintf(__fdiv_rn(-lo, scale)), 0.0f), 15.0f) : 0.0f;
    if (lane == 0) {
      store_score<DT>(a.scales, item, scale);
      a.zeros[item] = static_cast<uint8_t>(zero);
    }
    // whole blocks of 32 columns, the codes past the last column 0
    const int64_t bytes_end = min((first + a.group) / 2, a.row_bytes);
    for (int64_t j = first / 2 + lane; j < bytes_end; j += 64) {
      uint32_t byte = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t d = 2 * j + h;
        if (d >= end) continue;
        const float q = any ? rintf(__fdiv_rn(load_score<DT>(row, d), scale)) + zero : zero;
        byte |= static_cast<uint32_t>(fminf(fmaxf(q, 0.0f), 15.0f)) << (4 * h);
      }
      a.packed[n * a.row_bytes + j] = static_cast<uint8_t>(byte);
    }
  }
}

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw Error(ST_ERR_HIP, cat(what, " launch failed: ", hipGetErrorString(e)));
}

void check_type(int type, const char* what) {
  ST_CHECK(type == ST_SCORE_F32 || type == ST_SCORE_F16 || type == ST_SCORE_BF16, what,
           " must be float32, float16 or bfloat16");
}

void check_table(int64_t rows, int64_t dim, int64_t group) {
  ST_CHECK(rows >= 0 && dim >= 1, "a table has at least one column, got ", rows, " x ", dim);
  ST_CHECK(dim < (1ll << 31), "columns must be below 2^31, got ", dim);
  ST_CHECK(group >= kBlock && group % kBlock == 0, "group_size must be a positive multiple of ", kBlock, ", got ", group);
}

}  // namespace
}  // namespace st

extern "C" int st_int4_quantize(const void* weight, int weight_type, int64_t rows, int64_t dim, int64_t group_size,
                                int symmetric, uint8_t* packed, void* scales, uint8_t* zeros, void* stream) {
  using namespace st;
  return guarded([&] {
    check_type(weight_type, "weight");
    check_table(rows, dim, group_size);
    if (rows == 0) return;
    ST_CHECK(weight && packed && scales && zeros, "null device pointer");
    QuantizeArgs a{weight, packed, scales, zeros, rows, dim, group_size, (dim + group_size - 1) / group_size,
                   (dim + kBlock - 1) / kBlock * (kBlock / 2), symmetric};
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((rows * a.groups + 3) / 4, 64ll * cu_count()));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (weight_type == ST_SCORE_F32)
      hipLaunchKernelGGL((quantize_kernel<ST_SCORE_F32>), dim3(grid), dim3(256), 0, s, a);
    else if (weight_type == ST_SCORE_F16)
      hipLaunchKernelGGL((quantize_kernel<ST_SCORE_F16>), dim3(grid), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((quantize_kernel<ST_SCORE_BF16>), dim3(grid), dim3(256), 0, s, a);
    check_launch("quantize_kernel");
  });
}

extern "C" int st_int4_matvec(const uint8_t* packed, const void* scales, int scale_type, const uint8_t* zeros,
                              const void* x, int x_type, int64_t queries, int64_t rows, int64_t dim,
                              int64_t group_size, void* y, int y_type, void* stream) {
  using namespace st;
  return guarded([&] {
    check_type(scale_type, "scales");
    check_type(x_type, "x");
    check_type(y_type, "the result");
    check_table(rows, dim, group_size);
    ST_CHECK(queries >= 0, "negative sizes");
    if (rows == 0 || queries == 0) return;
    ST_CHECK(packed && scales && x && y, "null device pointer");
    ST_CHECK(reinterpret_cast<uintptr_t>(packed) % 16 == 0, "the packed table must be 16-byte aligned");
    MatvecArgs a{packed, scales, zeros, x, y, rows, dim, queries, group_size, (dim + group_size - 1) / group_size,
                 (dim + kBlock - 1) / kBlock * (kBlock / 2), scale_type, x_type, y_type};
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((rows * queries + 255) / 256, 1 << 22));
    hipLaunchKernelGGL(matvec_kernel, dim3(grid), dim3(256), 0, static_cast<hipStream_t>(stream), a);
    check_launch("matvec_kernel");
  });
}
