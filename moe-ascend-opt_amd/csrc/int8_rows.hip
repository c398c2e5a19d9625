// int8_rows.hip -- int8 codes with a scale for each row, and back.
//
//   s = max(amax / 127, 2^-126) rounded to fp32;  q = the integer nearest to x / s, ties to even
//
// A row with a NaN or an infinity gets s = NaN and codes 0, so that its
// products are NaN.
#pragma clang fp contract(off)
#include "expert_products.hpp"
#include "mi_moe_device.hpp"

namespace mimoe {

namespace {

// Eight elements of type DT (0 fp16, 1 bf16, 2 fp32) from element `at` on;
// elements past n are zeros.  ALIGNED: all eight there, 16-byte aligned.
template <int DT, bool ALIGNED>
__device__ __forceinline__ void load8(const void* x, int64_t at, int n, float (&v)[8]) {
  if constexpr (ALIGNED && DT == 2) {
    const f32x4_t* p = reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(x) + at);
    const f32x4_t a = p[0], b = p[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  } else if constexpr (ALIGNED) {
    const u32x4_t a = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint16_t*>(x) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = to_f32<DT>(a[i]);
      v[2 * i + 1] = to_f32<DT>(a[i] >> 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = 0.0f;
      if (i < n) {
        if constexpr (DT == 2) v[i] = reinterpret_cast<const float*>(x)[at + i];
        else v[i] = to_f32<DT>(reinterpret_cast<const uint16_t*>(x)[at + i]);
      }
    }
  }
}

__device__ __forceinline__ uint32_t amax8(const float (&v)[8], uint32_t m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
    m = a > m ? a : m;
  }
  return m;
}

// The codes of eight values: v * (1 / s) is off by less than 127 * 2^-22, so
// it names the nearest integer unless it lies within 2^-14 of a border; there
// the quotient in 64 bits does (x and s have 24 bits: a quotient that is no tie
// k + 1/2 is at least 2^-32 of itself away from one, since x - (k + 1/2) s is a
// multiple of half a unit of s, and k + 1/2 < 2^7; a tie is exact).
__device__ __forceinline__ u32x2_t codes8(const float (&v)[8], float s, float inv, bool bad) {
  float q[8];
  bool near = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = v[i] * inv;
    q[i] = __builtin_rintf(t);
    near |= __builtin_fabsf(t - q[i]) > 0.5f - 0x1p-14f;
  }
  if (near) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = (float)__builtin_rint((double)v[i] / (double)s);
  }
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i >> 2] |= ((uint32_t)(int)q[i] & 255u) << (8 * (i & 3));
  return bad ? u32x2_t{0, 0} : u32x2_t{w[0], w[1]};
}

template <bool ALIGNED>
__device__ __forceinline__ void store8(int8_t* codes, int64_t at, int n, const u32x2_t& c) {
  if constexpr (ALIGNED) {
    *reinterpret_cast<u32x2_t*>(codes + at) = c;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) codes[at + i] = (int8_t)(c[i >> 2] >> (8 * (i & 3)));
  }
}

// LANES threads a row (a wave, or the workgroup), NCH pieces of 8 elements
// each in registers (0: any number, read twice).  Bound by memory: 8191 x 4096
// fp16, 101 MB, in 20.5 us, 4.9 TB/s, the rate of a copy; 5 rows of 2048 2.7 us.
template <int DT, int LANES, int NCH, bool ALIGNED>
__global__ __launch_bounds__(256) void int8_quantize_kernel(const void* __restrict__ x, int64_t rows, int cols, int64_t stride,
                                                            int8_t* __restrict__ codes, float* __restrict__ scales) {
  const int t = threadIdx.x & (LANES - 1), nc = (cols + 7) >> 3;
  const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (LANES == kWave && row >= rows) return;   // a whole wave
  const int64_t src = row * stride, dst = row * cols;
  float v[NCH ? NCH : 1][8];
  uint32_t m = 0;
  if constexpr (NCH > 0) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int c = j * LANES + t;
      if (c < nc) {
        load8<DT, ALIGNED>(x, src + 8 * c, cols - 8 * c, v[j]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j) m = amax8(v[j], m);
  } else {
    for (int c = t; c < nc; c += LANES) {
      load8<DT, ALIGNED>(x, src + 8 * (int64_t)c, cols - 8 * c, v[0]);
      m = amax8(v[0], m);
    }
  }
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t o = __shfl_xor((int)m, d);
    m = o > m ? o : m;
  }
  if constexpr (LANES > kWave) {
    __shared__ uint32_t part[LANES / kWave];
    if ((t & 63) == 0) part[t >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LANES / kWave; ++i) m = part[i] > m ? part[i] : m;
  }
  const bool bad = m >= 0x7f800000u;
  float s = __uint_as_float(m) / 127.0f;
  s = bad || s < 0x1p-126f ? 0x1p-126f : s;
  const float inv = 1.0f / s;
  if (t == 0) scales[row] = bad ? __uint_as_float(0x7fc00000u) : s;
  if constexpr (NCH > 0) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int c = j * LANES + t;
      if (c < nc) store8<ALIGNED>(codes, dst + 8 * c, cols - 8 * c, codes8(v[j], s, inv, bad));
    }
  } else {
    for (int c = t; c < nc; c += LANES) {
      load8<DT, ALIGNED>(x, src + 8 * (int64_t)c, cols - 8 * c, v[0]);
      store8<ALIGNED>(codes, dst + 8 * (int64_t)c, cols - 8 * c, codes8(v[0], s, inv, bad));
    }
  }
}

// A code's value: the product in fp32, which the conversion that follows then
// rounds.  The empty asm keeps the two apart: for fp16 the compiler would make
// one instruction of them that rounds the exact product, other bits than those
// of the same codes and scales elsewhere.
__device__ __forceinline__ float value(int8_t code, float s) {
  float v = (float)code * s;
  asm("" : "+v"(v));
  return v;
}

// A thread per piece of 8 codes of a row: 8191 x 4096 to fp16 in 16.8 us, 6.0 TB/s.
template <int DT, bool ALIGNED>
__global__ __launch_bounds__(256) void int8_dequantize_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales,
                                                              int64_t rows, int cols, void* __restrict__ out) {
  const uint32_t nc = (uint32_t)((cols + 7) >> 3);
  const int64_t total = rows * nc;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = total < ((int64_t)1 << 32) ? (int64_t)((uint32_t)i / nc) : i / nc;
    const int c = 8 * (int)(i - row * nc), n = cols - c;
    const int64_t at = row * cols + c;
    const float s = scales[row];
    float v[8];
    if constexpr (ALIGNED) {
      const u32x2_t w = *reinterpret_cast<const u32x2_t*>(codes + at);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = value((int8_t)(w[k >> 2] >> (8 * (k & 3))), s);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = k < n ? value(codes[at + k], s) : 0.0f;
    }
    if constexpr (DT == 2) {
      float* o = reinterpret_cast<float*>(out) + at;
      if constexpr (ALIGNED) {
        reinterpret_cast<f32x4_t*>(o)[0] = f32x4_t{v[0], v[1], v[2], v[3]};
        reinterpret_cast<f32x4_t*>(o)[1] = f32x4_t{v[4], v[5], v[6], v[7]};
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < n) o[k] = v[k];
      }
    } else {
      uint16_t* o = reinterpret_cast<uint16_t*>(out) + at;
      if constexpr (ALIGNED) {
        u32x4_t w;
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = from_f32<DT>(v[2 * k]) | (uint32_t)from_f32<DT>(v[2 * k + 1]) << 16;
        *reinterpret_cast<u32x4_t*>(o) = w;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < n) o[k] = from_f32<DT>(v[k]);
      }
    }
  }
}

bool at16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

template <int DT>
void quantize(const void* x, int64_t rows, int cols, int64_t stride, int8_t* codes, float* scales, hipStream_t st) {
  const bool aligned = at16(x) && ((uintptr_t)codes & 7) == 0 && cols % 8 == 0 && stride % (DT == 2 ? 4 : 8) == 0;
  const unsigned per_row = (unsigned)rows, per_wave = (unsigned)((rows + 3) / 4);
  // A row a wave where there are rows enough for every SIMD, else a row a
  // workgroup, whose loads are all under way at once.
  if (!aligned) int8_quantize_kernel<DT, 256, 0, false><<<per_row, 256, 0, st>>>(x, rows, cols, stride, codes, scales);
  else if (rows >= 1024 && cols <= 512) int8_quantize_kernel<DT, 64, 1, true><<<per_wave, 256, 0, st>>>(x, rows, cols, stride, codes, scales);
  else if (rows >= 1024 && cols <= 2048) int8_quantize_kernel<DT, 64, 4, true><<<per_wave, 256, 0, st>>>(x, rows, cols, stride, codes, scales);
  else if (cols <= 2048) int8_quantize_kernel<DT, 256, 1, true><<<per_row, 256, 0, st>>>(x, rows, cols, stride, codes, scales);
  else if (cols <= 4096) int8_quantize_kernel<DT, 256, 2, true><<<per_row, 256, 0, st>>>(x, rows, cols, stride, codes, scales);
  else if (cols <= 16384) int8_quantize_kernel<DT, 256, 8, true><<<per_row, 256, 0, st>>>(x, rows, cols, stride, codes, scales);
  else int8_quantize_kernel<DT, 256, 0, true><<<per_row, 256, 0, st>>>(x, rows, cols, stride, codes, scales);
}

template <int DT>
void dequantize(const int8_t* codes, const float* scales, int64_t rows, int cols, void* out, hipStream_t st) {
  const int64_t total = rows * ((cols + 7) / 8), blocks = (total + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
  const bool aligned = ((uintptr_t)codes & 7) == 0 && at16(out) && cols % 8 == 0;
  if (aligned) int8_dequantize_kernel<DT, true><<<grid, 256, 0, st>>>(codes, scales, rows, cols, out);
  else int8_dequantize_kernel<DT, false><<<grid, 256, 0, st>>>(codes, scales, rows, cols, out);
}

}  // namespace

hipError_t launch_int8_quantize(const void* x, int dt, int64_t rows, int64_t cols, int64_t stride, int8_t* codes, float* scales,
                                hipStream_t st) {
  constexpr int64_t kRows = (int64_t)1 << 23;   // a launch has at most 2^32 threads
  for (int64_t r = 0; r < rows; r += kRows) {
    const void* p = (const char*)x + r * stride * (dt == 2 ? 4 : 2);
    const int64_t n = rows - r < kRows ? rows - r : kRows;
    if (dt == 0) quantize<0>(p, n, (int)cols, stride, codes + r * cols, scales + r, st);
    else if (dt == 1) quantize<1>(p, n, (int)cols, stride, codes + r * cols, scales + r, st);
    else quantize<2>(p, n, (int)cols, stride, codes + r * cols, scales + r, st);
  }
  return hipGetLastError();
}

hipError_t launch_int8_dequantize(const int8_t* codes, const float* scales, int64_t rows, int64_t cols, void* out, int dt,
                                  hipStream_t st) {
  if (dt == 0) dequantize<0>(codes, scales, rows, (int)cols, out, st);
  else if (dt == 1) dequantize<1>(codes, scales, rows, (int)cols, out, st);
  else dequantize<2>(codes, scales, rows, (int)cols, out, st);
  return hipGetLastError();
}

}  // namespace mimoe
