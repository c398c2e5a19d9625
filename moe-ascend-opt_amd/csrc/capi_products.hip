// capi_products.hip -- C ABI of the products on rows sorted by expert and of
// the int8 row quantizer (include/mi_moe.h): checks of arguments, then one
// launch each.
#include <cstdarg>
#include <cstdio>

#include "expert_products.hpp"
#include "mi_moe.h"
#include "mi_moe_internal.hpp"

#define MI_API extern "C" __attribute__((visibility("default")))

using namespace mimoe;

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return api_fail(code, buf);
}

int launched(hipError_t e, const char* what) {
  if (e == hipSuccess) return MI_MOE_OK;
  return fail(MI_MOE_EHIP, "%s failed: %s", what, hipGetErrorString(e));
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// Offsets within a tile (256 rows, or 64 across) are 32 bits wide.
constexpr int64_t kMaxDim = (int64_t)1 << 20, kMaxRows = (int64_t)1 << 26, kMaxStride = (int64_t)1 << 22;
// Tiles and their places in the XCDs' runs are numbered in 32 bits; 2^22 tiles are
// 2^38 values of an operand or output.
constexpr int64_t kMaxTiles = (int64_t)1 << 22;

int check_sizes(int64_t M, int64_t N, int64_t K, int64_t E) {
  if (M < 0 || M > kMaxRows) return fail(MI_MOE_EINVAL, "rows=%lld must be in [0, 2^26]", (long long)M);
  if (N < 1 || N > kMaxDim || K < 1 || K > kMaxDim)
    return fail(MI_MOE_EINVAL, "N=%lld and K=%lld must be in [1, 2^20]", (long long)N, (long long)K);
  if (E < 1 || E > kGroupMaxE) return fail(MI_MOE_EINVAL, "experts=%lld must be in [1, %d]", (long long)E, kGroupMaxE);
  const int64_t rows = (M + 255) / 256 + E + 2, n = (N + 255) / 256, k = (K + 255) / 256;
  if (rows * n > kMaxTiles || rows * k > kMaxTiles || E * n * k > kMaxTiles)
    return fail(MI_MOE_EUNSUPPORTED, "more than 2^22 tiles of 256 x 256 outputs");
  return MI_MOE_OK;
}

// A matrix whose rows are read in 16-byte pieces.
int check_matrix(const char* name, const void* p, int64_t cols, int64_t stride, int64_t per16) {
  if (!p) return fail(MI_MOE_EINVAL, "null pointer: %s", name);
  if (!aligned16(p) || cols % per16 || stride % per16)
    return fail(MI_MOE_EINVAL, "%s, its rows and its row length must be whole 16-byte pieces (%lld elements)", name, (long long)per16);
  if (stride < cols || stride > kMaxStride)
    return fail(MI_MOE_EINVAL, "row stride %lld of %s must be in [%lld, 2^22]", (long long)stride, name, (long long)cols);
  return MI_MOE_OK;
}

int check_weights(const void* w, int64_t expert_stride, int64_t cols, int64_t stride, int64_t per16) {
  const int rc = check_matrix("w", w, cols, stride, per16);
  if (rc) return rc;
  if (expert_stride < 0 || expert_stride % per16)
    return fail(MI_MOE_EINVAL, "expert stride %lld of w must be whole 16-byte pieces", (long long)expert_stride);
  return MI_MOE_OK;
}

int check_16bit(int dtype) {
  if (dtype != MI_MOE_F16 && dtype != MI_MOE_BF16) return fail(MI_MOE_EINVAL, "dtype must be fp16 or bf16");
  return MI_MOE_OK;
}

int check_values(int dtype) {
  if (dtype != MI_MOE_F16 && dtype != MI_MOE_BF16 && dtype != MI_MOE_F32) return fail(MI_MOE_EINVAL, "values must be fp16, bf16 or fp32");
  return MI_MOE_OK;
}

#define CHECK(expr)      \
  do {                   \
    const int _rc = (expr); \
    if (_rc) return _rc; \
  } while (0)

// |code| <= 128: sums of 131071 products stay below 2^31; rows are whole pieces of 16.
constexpr int64_t kInt8MaxK = 131056;

int int8_product(const int8_t* x, int64_t x_stride, const float* xs, const int8_t* w, int64_t w_expert, int64_t w_stride,
                 const float* ws, const float* bias, const int32_t* starts, int64_t M, int64_t N, int64_t K, int64_t E, int out,
                 void* y, hipStream_t st) {
  CHECK(check_sizes(M, N, K, E));
  CHECK(check_values(out));
  if (K > kInt8MaxK) return fail(MI_MOE_EINVAL, "K=%lld: int32 sums hold at most %lld products", (long long)K, (long long)kInt8MaxK);
  if (M == 0) return MI_MOE_OK;
  if (!xs || !ws || !y) return fail(MI_MOE_EINVAL, "null pointer");
  CHECK(check_matrix("x", x, K, x_stride, 16));
  CHECK(check_weights(w, w_expert, K, w_stride, 16));
  const RowProductArgs a = {(const unsigned char*)x, (const unsigned char*)w, y, starts, xs, ws, bias, w_expert, N,
                            (uint32_t)x_stride, (uint32_t)w_stride, (int)M, (int)N, (int)K, (int)E};
  return launched(launch_row_product(a, 2, 0, out, st), "int8 product");
}

}  // namespace

MI_API int mi_moe_grouped_matmul(const void* x, int64_t x_stride, const void* w, int64_t w_expert_stride, int64_t w_stride,
                                 const int32_t* starts, int64_t M, int64_t N, int64_t K, int64_t E, int dtype, void* y,
                                 void* stream) {
  CHECK(check_sizes(M, N, K, E));
  CHECK(check_16bit(dtype));
  if (M == 0) return MI_MOE_OK;
  if (!starts || !y) return fail(MI_MOE_EINVAL, "null pointer");
  CHECK(check_matrix("x", x, K, x_stride, 8));
  CHECK(check_weights(w, w_expert_stride, K, w_stride, 8));
  const RowProductArgs a = {(const unsigned char*)x, (const unsigned char*)w, y, starts, nullptr, nullptr, nullptr,
                            2 * w_expert_stride, N, (uint32_t)(2 * x_stride), (uint32_t)(2 * w_stride), (int)M, (int)N, (int)K,
                            (int)E};
  return launched(launch_row_product(a, dtype, 0, dtype, (hipStream_t)stream), "grouped_matmul");
}

MI_API int mi_moe_grouped_matmul_dx(const void* dy, int64_t dy_stride, const void* w, int64_t w_expert_stride, int64_t w_stride,
                                    const int32_t* starts, int64_t M, int64_t N, int64_t K, int64_t E, int dtype, void* dx,
                                    void* stream) {
  CHECK(check_sizes(M, N, K, E));
  CHECK(check_16bit(dtype));
  if (M == 0) return MI_MOE_OK;
  if (!starts || !dx) return fail(MI_MOE_EINVAL, "null pointer");
  CHECK(check_matrix("dy", dy, N, dy_stride, 8));
  CHECK(check_weights(w, w_expert_stride, K, w_stride, 8));
  const RowProductArgs a = {(const unsigned char*)dy, (const unsigned char*)w, dx, starts, nullptr, nullptr, nullptr,
                            2 * w_expert_stride, K, (uint32_t)(2 * dy_stride), (uint32_t)(2 * w_stride), (int)M, (int)K, (int)N,
                            (int)E};
  return launched(launch_row_product(a, dtype, 1, dtype, (hipStream_t)stream), "grouped_matmul_dx");
}

MI_API int mi_moe_grouped_matmul_dw(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const int32_t* starts,
                                    int64_t M, int64_t N, int64_t K, int64_t E, int dtype, void* dw, void* stream) {
  CHECK(check_sizes(M, N, K, E));
  CHECK(check_16bit(dtype));
  if (!starts || !dw) return fail(MI_MOE_EINVAL, "null pointer");
  if (M > 0) {
    CHECK(check_matrix("dy", dy, N, dy_stride, 8));
    CHECK(check_matrix("x", x, K, x_stride, 8));
  }
  const WeightGradArgs a = {(const unsigned char*)dy, (const unsigned char*)x, dw, starts, (uint32_t)(2 * dy_stride),
                            (uint32_t)(2 * x_stride), (int)M, (int)N, (int)K, (int)E};
  return launched(launch_weight_grad(a, dtype, (hipStream_t)stream), "grouped_matmul_dw");
}

MI_API int mi_moe_grouped_matmul_int8(const int8_t* x, int64_t x_stride, const float* x_scales, const int8_t* w,
                                      int64_t w_expert_stride, int64_t w_stride, const float* w_scales, const int32_t* starts,
                                      int64_t M, int64_t N, int64_t K, int64_t E, int out_dtype, void* y, void* stream) {
  if (M > 0 && !starts) return fail(MI_MOE_EINVAL, "null pointer");
  return int8_product(x, x_stride, x_scales, w, w_expert_stride, w_stride, w_scales, nullptr, starts, M, N, K, E, out_dtype, y,
                      (hipStream_t)stream);
}

MI_API int mi_moe_int8_matmul(const int8_t* x, int64_t x_stride, const float* x_scales, const int8_t* w, int64_t w_stride,
                              const float* w_scales, const float* bias, int64_t M, int64_t N, int64_t K, int out_dtype, void* y,
                              void* stream) {
  return int8_product(x, x_stride, x_scales, w, 0, w_stride, w_scales, bias, nullptr, M, N, K, 1, out_dtype, y,
                      (hipStream_t)stream);
}

namespace {
int check_rows(int64_t rows, int64_t cols, int dtype) {
  CHECK(check_values(dtype));
  if (rows < 0 || cols < 1 || cols > ((int64_t)1 << 30) || rows > ((int64_t)1 << 40) / cols)
    return fail(MI_MOE_EINVAL, "rows=%lld of cols=%lld: cols must be in [1, 2^30], at most 2^40 values", (long long)rows, (long long)cols);
  return MI_MOE_OK;
}
}  // namespace

MI_API int mi_moe_int8_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, int8_t* codes,
                                float* scales, void* stream) {
  CHECK(check_rows(rows, cols, dtype));
  if (rows == 0) return MI_MOE_OK;
  if (!x || !codes || !scales) return fail(MI_MOE_EINVAL, "null pointer");
  if (row_stride < cols || row_stride > ((int64_t)1 << 40) / rows)
    return fail(MI_MOE_EINVAL, "row_stride=%lld must be at least cols", (long long)row_stride);
  return launched(launch_int8_quantize(x, dtype, rows, cols, row_stride, codes, scales, (hipStream_t)stream), "int8_quantize");
}

MI_API int mi_moe_int8_dequantize(const int8_t* codes, const float* scales, int64_t rows, int64_t cols, void* out, int dtype,
                                  void* stream) {
  CHECK(check_rows(rows, cols, dtype));
  if (rows == 0) return MI_MOE_OK;
  if (!out || !codes || !scales) return fail(MI_MOE_EINVAL, "null pointer");
  return launched(launch_int8_dequantize(codes, scales, rows, cols, out, dtype, (hipStream_t)stream), "int8_dequantize");
}
