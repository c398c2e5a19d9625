// expert_products.hpp -- arguments of the products on rows sorted by expert
// (expert_products.hip) and of the int8 row quantizer (int8_rows.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mimoe {

// Most experts of a product, as of the router.
constexpr int kGroupMaxE = 512;

// out[r][p] = sum_k w[e(r)](p, k) x[r][k], rows r of expert e: starts[e] <= r < starts[e+1].
struct RowProductArgs {
  const unsigned char* x;      // [M][K], ldx bytes a row
  const unsigned char* w;      // expert e at w + e * w_expert bytes, ldw bytes a row; [P][K], or [K][P] with w_cols
  void* y;                     // [M][P]
  const int32_t* starts;       // [E + 1], or null: one group of all rows
  const float* xs;             // int8: [M]
  const float* ws;             // int8: [E][P]
  const float* bias;           // int8: [P] or null
  int64_t w_expert;
  int64_t ldy;                 // elements
  uint32_t ldx, ldw;
  int M, P, K, E;
  int most;                    // rows of an item (set by the launcher)
};

// dw[e][n][k] = sum over rows r of e of dy[r][n] x[r][k]
struct WeightGradArgs {
  const unsigned char* dy;     // [M][N], lddy bytes a row
  const unsigned char* x;      // [M][K]
  void* dw;                    // [E][N][K], contiguous
  const int32_t* starts;
  uint32_t lddy, ldx;
  int M, N, K, E;
};

// dt: 0 fp16, 1 bf16, 2 int8 (then out: 0 fp16, 1 bf16, 2 fp32)
hipError_t launch_row_product(const RowProductArgs& a, int dt, int w_cols, int out, hipStream_t st);
hipError_t launch_weight_grad(const WeightGradArgs& a, int dt, hipStream_t st);
hipError_t launch_int8_quantize(const void* x, int dt, int64_t rows, int64_t cols, int64_t stride, int8_t* codes, float* scales,
                                hipStream_t st);
hipError_t launch_int8_dequantize(const int8_t* codes, const float* scales, int64_t rows, int64_t cols, void* out, int dt,
                                  hipStream_t st);

}  // namespace mimoe
