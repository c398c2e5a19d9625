// mx.hip -- MXFP4 expert layers on gfx950: weights in MXFP4 (E2M1, one E8M0
// scale per 32 along K), hidden states and the intermediate quantized to
// MXFP6 (E2M3), both products on the scaled matrix instructions, which take
// the codes as they are stored; and the MX quantizers.
//
//   x -> MXFP6;  g, u = W13[e] x;  h = silu(g) u -> MXFP6;  y = sum_k w_k W2[e_k] h_k
//
// Why E2M3: its products with E2M1 are exact in the instruction's group sums
// and run at the 4-bit rate, and its noise (2.8% of a Gaussian block, 2.6%
// for E4M3) stays far below that of the 4-bit weights (11%).
#pragma clang fp contract(off)
#include <algorithm>
#include <type_traits>

#include "mx_device.hpp"

namespace mimoe {

namespace {

constexpr int kMxWaves = 8;
constexpr int kMxThreads = kMxWaves * kWave;

__device__ __forceinline__ u32x4_t ld16(const void* p) { return *reinterpret_cast<const u32x4_t*>(p); }
__device__ __forceinline__ void st16(void* p, const u32x4_t& v) { *reinterpret_cast<u32x4_t*>(p) = v; }

// v[s] of lane row q <-> v[q] of lane row s (lane rows of 16): every lane
// ends with the four lane rows' values of one subtile.
__device__ __forceinline__ void transpose4(float& a0, float& a1, float& a2, float& a3) {
  auto swap16 = [](float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
  };
  auto swap32 = [](float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
  };
  swap16(a0, a1);
  swap16(a2, a3);
  swap32(a0, a2);
  swap32(a1, a3);
}

struct MxTile {
  int e, row0, rows, blk;
};
// Work item of this workgroup: row tile and block (of nblk) of output units.
// XCD x takes the x-th eighth of the tile list, which is in expert order, so
// that an expert's weights pass through one XCD's L2.
__device__ __forceinline__ bool mx_tile(const RouteGlobal& rg, int nblk, MxTile& t) {
  const int nt = *rg.ntiles, per = (nt + 7) >> 3;
  const int x = blockIdx.x & 7, j = blockIdx.x >> 3, i = j / nblk, tile = x * per + i;
  if (i >= per || tile >= nt) return false;
  const int4 v = *reinterpret_cast<const int4*>(rg.tiles + 4 * tile);
  t = MxTile{v.x, v.y, v.z, j - i * nblk};
  return true;
}

// The grouped products run one instance per number of 16-row subtiles of the
// work item (rounded up to 1, 2, 4 or 8): without branches in the K loop the
// loads of the next step stay in flight across it.
// A step is S k tiles (S * 128 B of a row): enough products between barriers
// to cover a load's latency, and a 16-byte piece for every thread.
constexpr int mx_step(int nsub) { return nsub == 1 ? 4 : 2; }
constexpr int mx_stage_bytes(int nsub) { return nsub * 16 * mx_step(nsub) * 128; }

// acc[t][s] = tile t of the wave's weight unit times the rows of subtile s,
// over all kt k tiles.  row(i): the packets of row i of the item; w, ws: the
// unit's codes and scales, at this lane.
// Rows are staged in LDS, double-buffered, through registers; a wave's weights
// go straight to its registers, each k tile's replaced as soon as it is used.
// LDS pieces of 16 B are permuted by the row, so that the 16 rows of an
// operand read lie in different banks.
template <int NSUB, class Row>
__device__ __forceinline__ void mx_gemm_core(unsigned char* smem, Row row, int kt, const unsigned char* w, const unsigned char* ws,
                                             f32x4_t (&acc)[4][NSUB]) {
  constexpr int S = mx_step(NSUB), STRIDE = S * 128, BYTES = mx_stage_bytes(NSUB);
  constexpr int NP = BYTES / (kMxThreads * 16), STEP = kMxThreads / (8 * S);   // pieces of a thread, STEP rows apart
  static_assert(NP >= 1 && NP * STEP == 16 * NSUB, "every thread stages whole pieces");
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, r = lane & 15;
  const int piece = tid % (8 * S), last = 8 * kt - 1, row0 = tid / (8 * S);
  const unsigned char* src[NP];
  int dst[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    src[p] = row(row0 + STEP * p);
    dst[p] = (row0 + STEP * p) * STRIDE + ((piece ^ ((row0 + STEP * p) & 15)) << 4);
  }
  u32x4_t sv[NP], wv[S][4];
  uint32_t sc[S];
  auto stage_load = [&](int c) {
    const int o = min(8 * S * c + piece, last) << 4;
#pragma unroll
    for (int p = 0; p < NP; ++p) sv[p] = ld16(src[p] + o);
  };
  auto stage_store = [&](unsigned char* buf) {
#pragma unroll
    for (int p = 0; p < NP; ++p) st16(buf + dst[p], sv[p]);
  };
  auto weights = [&](int k, u32x4_t (&v)[4], uint32_t& s) {
    const int kk = min(k, kt - 1);
#pragma unroll
    for (int t = 0; t < 4; ++t) v[t] = ld16(w + (size_t)kk * kMxTileBytes + t * 1024);
    s = *reinterpret_cast<const uint32_t*>(ws + (size_t)kk * kMxTileScaleBytes);
  };
  const int rd = r * STRIDE + (((2 * q) ^ r) << 4);
  auto products = [&](const unsigned char* buf, int k) {
    const int a0 = rd ^ (k << 7), a1 = a0 ^ 16;
#pragma unroll
    for (int s = 0; s < NSUB; ++s) {
      const u32x4_t lo = ld16(buf + a0 + s * 16 * STRIDE), hi = ld16(buf + a1 + s * 16 * STRIDE);
      acc[0][s] = mx_mfma<0>(wv[k][0], sc[k], lo, hi, acc[0][s]);
      acc[1][s] = mx_mfma<1>(wv[k][1], sc[k], lo, hi, acc[1][s]);
      acc[2][s] = mx_mfma<2>(wv[k][2], sc[k], lo, hi, acc[2][s]);
      acc[3][s] = mx_mfma<3>(wv[k][3], sc[k], lo, hi, acc[3][s]);
    }
  };
  stage_load(0);
#pragma unroll
  for (int k = 0; k < S; ++k) weights(k, wv[k], sc[k]);
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int s = 0; s < NSUB; ++s) acc[t][s] = f32x4_t{0, 0, 0, 0};
  stage_store(smem);
  __syncthreads();
  const int nc = kt / S, rest = kt - nc * S;
  for (int c = 0; c < nc; ++c) {
    const unsigned char* buf = smem + (c & 1) * BYTES;
    stage_load(c + 1);   // past the end: the last piece again
    __builtin_amdgcn_sched_barrier(0);   // loads stay where they are: sunk below the products they would be waited for at once
#pragma unroll
    for (int k = 0; k < S; ++k) {
      products(buf, k);
      __builtin_amdgcn_sched_barrier(0);
      weights(S * (c + 1) + k, wv[k], sc[k]);
      __builtin_amdgcn_sched_barrier(0);
    }
    stage_store(smem + ((c + 1) & 1) * BYTES);
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < S - 1; ++k)
    if (k < rest) products(smem + (nc & 1) * BYTES, k);   // uniform
}

// gate_up + SiLU*mul + MXFP6 of one work item: a unit is a slice of 32 rows of
// I (its gate and up tiles hold the same rows, so the product is in
// registers); a transpose between the wave's lane rows leaves every lane with
// the 32 values of one token's block.
template <int NSUB>
__device__ __forceinline__ void mx_gate_up(const MxArgs& a, unsigned char* smem, int e, int row0, int rows, int slice) {
  const int NS = a.I >> 5, kt = mx_ktiles(a.H), lane = threadIdx.x & 63;
  const size_t unit = ((size_t)e * NS + min(slice, NS - 1)) * kt;
  f32x4_t acc[4][NSUB];
  mx_gemm_core<NSUB>(
      smem, [&](int i) { return a.xq + (size_t)(a.rg.tok[row0 + min(i, rows - 1)] / a.K) * mx_row_bytes(a.H); }, kt,
      a.w13 + unit * kMxTileBytes + lane * 16, a.w13_s + unit * kMxTileScaleBytes + lane * 4, acc);
  if (slice >= 4 * mx_ktiles(a.I)) return;
#pragma unroll
  for (int g = 0; g < (NSUB + 3) / 4; ++g) {   // four subtiles at a time
    float v[32];   // [tile][q][4] after the transpose
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float h[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int ss = 4 * g + s < NSUB ? 4 * g + s : 0;
          h[s] = 4 * g + s < NSUB ? silu_mul_fast(acc[p][ss][i], acc[2 + p][ss][i]) : 0.0f;
        }
        transpose4(h[0], h[1], h[2], h[3]);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[16 * p + 4 * q + i] = h[q];
      }
    const int s = mx_scale_byte<kMxFp6>(mx_amax32(v));
    MxPacket pk = mx_packet(mx_fp6_codes32(v, s), s);
    if (slice >= NS) pk = MxPacket{u32x4_t{0, 0, 0, 0}, u32x4_t{0, 0, 0, 0}};   // past I
    const int i = 64 * g + lane;   // 16 subtile + row
    if (lane < 16 * NSUB && i < rows) {
      unsigned char* o = a.act + (size_t)(row0 + i) * mx_row_bytes(a.I) + slice * kMxPacketBytes;
      st16(o, pk.lo);
      st16(o + 16, pk.hi);
    }
  }
}

// down of one work item: a unit is 64 rows of H.  Expert outputs are fp32 up
// to the combine, as in decode calls: a column may be a thousand times its
// neighbours, so none shares a scale with them.  Lanes store where the
// products leave the values, four lanes 64 bytes of a token's row (T = 4096
// H=2048 top-8: 268 MB, the call 258 us; with a transpose, a lane per token's
// row, 271).
template <int NSUB>
__device__ __forceinline__ void mx_down(const MxArgs& a, unsigned char* smem, int e, int row0, int rows, int m) {
  const int NQ = a.H >> 6, kt = mx_ktiles(a.I), lane = threadIdx.x & 63;
  const size_t unit = ((size_t)e * NQ + min(m, NQ - 1)) * kt;
  f32x4_t acc[4][NSUB];
  mx_gemm_core<NSUB>(
      smem, [&](int i) { return a.act + (size_t)(row0 + min(i, rows - 1)) * mx_row_bytes(a.I); }, kt,
      a.w2 + unit * kMxTileBytes + lane * 16, a.w2_s + unit * kMxTileScaleBytes + lane * 4, acc);
  if (m >= NQ) return;
  int pair[NSUB];
#pragma unroll
  for (int s = 0; s < NSUB; ++s) pair[s] = a.rg.tok[row0 + min(16 * s + (lane & 15), rows - 1)];
#pragma unroll
  for (int s = 0; s < NSUB; ++s) {
    if (16 * s + (lane & 15) < rows) {
      float* o = a.eout + (size_t)pair[s] * a.H + 64 * m + 4 * (lane >> 4);
#pragma unroll
      for (int t = 0; t < 4; ++t) *reinterpret_cast<f32x4_t*>(o + 16 * t) = acc[t][s];
    }
  }
}

// Work item: 8 units, one a wave, and a row tile of an expert: up to 64 rows,
// or with BIG 128 (kRouteBigTiles).
template <bool BIG, bool DOWN>
__device__ __forceinline__ void mx_gemm_item(const MxArgs& a, unsigned char* smem) {
  const int units = DOWN ? a.H >> 6 : 4 * mx_ktiles(a.I);
  MxTile t;
  if (!mx_tile(a.rg, (units + kMxWaves - 1) / kMxWaves, t)) return;   // uniform
  const int nsub = (t.rows + 15) >> 4, unit = kMxWaves * t.blk + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto run = [&](auto n) {
    if constexpr (DOWN) mx_down<decltype(n)::value>(a, smem, t.e, t.row0, t.rows, unit);
    else mx_gate_up<decltype(n)::value>(a, smem, t.e, t.row0, t.rows, unit);
  };
  if (BIG && nsub > 4) run(std::integral_constant<int, BIG ? 8 : 4>{});
  else if (nsub > 2) run(std::integral_constant<int, 4>{});
  else if (nsub == 2) run(std::integral_constant<int, 2>{});
  else run(std::integral_constant<int, 1>{});
}

// 64-row items at four waves per SIMD, 128-row items at two (twice the accumulators).
//
// gate_up / down, H=2048 I=768 E=128 top-8: T = 333 skewed 49 / 40 us, 4.4 TB/s
// of weights and 3.2 of weights and outputs; T = 4096 94 / 116 us, 2.2 / 0.9
// PFLOP/s: the K loop alone runs at 5 (the instruction in registers at 5.9), the items'
// first loads and their epilogues, gate_up's quantization and down's 268 MB
// of expert outputs, take the rest.
template <bool DOWN>
__global__ __launch_bounds__(kMxThreads) __attribute__((amdgpu_waves_per_eu(4))) void mx_gemm_kernel(MxArgs a) {
  __shared__ __align__(16) unsigned char smem[2 * mx_stage_bytes(4)];
  mx_gemm_item<false, DOWN>(a, smem);
}
template <bool DOWN>
__global__ __launch_bounds__(kMxThreads) __attribute__((amdgpu_waves_per_eu(2))) void mx_gemm_big_kernel(MxArgs a) {
  __shared__ __align__(16) unsigned char smem[2 * mx_stage_bytes(8)];
  mx_gemm_item<true, DOWN>(a, smem);
}

// One block of 32 elements of type DT (0 fp16, 1 bf16, 2 fp32) as floats.
template <int DT>
__device__ __forceinline__ void ld_block(const void* x, size_t elem, float (&v)[32]) {
  if constexpr (DT == 2) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const f32x4_t f = *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(x) + elem + 4 * c);
      v[4 * c] = f.x; v[4 * c + 1] = f.y; v[4 * c + 2] = f.z; v[4 * c + 3] = f.w;
    }
  } else {
    uint32_t w[16];
    mx_load_words(reinterpret_cast<const uint16_t*>(x) + elem, w);
    mx_unpack16<DT>(w, v);
  }
}

// rows of cols elements (stride elements apart) -> codes [rows][cols/32][16
// or 24 B], scales [rows][cols/32].  One thread per block.  Bound by memory:
// 98304 x 2048 bf16 to MXFP4, 510 MB, in 111 us, 4.6 TB/s (a copy: 4.9).
template <int DT, int FMT>
__global__ void mx_quantize_kernel(const void* __restrict__ x, int64_t rows, int cols, int64_t stride, unsigned char* __restrict__ codes,
                                   unsigned char* __restrict__ scales) {
  const int nb = cols >> 5;
  const int64_t total = rows * nb;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / nb;
    float v[32];
    ld_block<DT>(x, (size_t)(row * stride + 32 * (i - row * nb)), v);
    const int s = mx_scale_byte<FMT>(mx_amax32(v));
    if constexpr (FMT == kMxFp4) {
      st16(codes + i * 16, mx_fp4_codes32(v, s));
    } else {
      const u32x6_t c = mx_fp6_codes32(v, s);
      u32x2_t* o = reinterpret_cast<u32x2_t*>(codes + i * 24);
      o[0] = u32x2_t{c[0], c[1]};
      o[1] = u32x2_t{c[2], c[3]};
      o[2] = u32x2_t{c[4], c[5]};
    }
    scales[i] = (unsigned char)s;
  }
}

// codes and scales -> values 2^(s-127) * element, rounded once to DT.  A
// thread writes one 16-byte piece (8 or 4 elements), so that a wave's stores
// are whole lines: 201M values MXFP4 to bf16 in 119 us, 4.3 TB/s (with a thread
// per block 152 us).
// An element's bits, as the top of a float's exponent and mantissa, are its
// value times 2^-126 (subnormal where the element is).
template <int DT, int FMT>
__global__ void mx_dequantize_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales, int64_t pieces,
                                     void* __restrict__ out) {
  constexpr int V = DT == 2 ? 4 : 8, BITS = FMT == kMxFp4 ? 4 : 6, BYTES = V * BITS / 8, M = FMT == kMxFp4 ? 1 : 3;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * blockDim.x) {
    const int s = scales[i / (32 / V)];
    const unsigned char* p = codes + i * BYTES;
    uint64_t c;
    if constexpr (BYTES == 4) c = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (BYTES == 2) c = *reinterpret_cast<const uint16_t*>(p);
    else if constexpr (BYTES == 3) c = p[0] | (uint32_t)p[1] << 8 | (uint32_t)p[2] << 16;
    else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
      c = h[0] | (uint32_t)h[1] << 16 | (uint64_t)h[2] << 32;
    }
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const uint32_t e = (uint32_t)(c >> (BITS * k));
      const uint32_t mag = (e & ((1u << (BITS - 1)) - 1)) << (23 - M), sign = (e >> (BITS - 1)) << 31;
      v[k] = s == 255 ? __uint_as_float(0x7fc00000u) : __builtin_ldexpf(__uint_as_float(mag | sign), s - 1);
    }
    if constexpr (DT == 2) {
      reinterpret_cast<f32x4_t*>(out)[i] = f32x4_t{v[0], v[1], v[2], v[3]};
    } else {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = from_f32<DT>(v[2 * k]) | ((uint32_t)from_f32<DT>(v[2 * k + 1]) << 16);
      st16(reinterpret_cast<uint16_t*>(out) + i * 8, u32x4_t{w[0], w[1], w[2], w[3]});
    }
  }
}

// Place of block b of row n in the device layout: projection rows as units of
// 64 rows (w13: of 32 rows of I, gate then up).
struct MxPlace {
  size_t code, scale;
};
__device__ __forceinline__ MxPlace mx_place(int64_t e, int n, int b, int which2, int H, int I) {
  int unit, tile, units, kt;
  if (!which2) {
    const int up = n >= I, i = n - (up ? I : 0);
    unit = i >> 5; tile = 2 * up + ((i >> 4) & 1); units = I >> 5; kt = mx_ktiles(H);
  } else {
    unit = n >> 6; tile = (n >> 4) & 3; units = H >> 6; kt = mx_ktiles(I);
  }
  const size_t k = ((size_t)e * units + unit) * kt + (b >> 2);
  const int lane = 16 * (b & 3) + (n & 15);
  return MxPlace{k * kMxTileBytes + tile * 1024 + lane * 16, k * kMxTileScaleBytes + lane * 4 + tile};
}

// Wire weights [E][N][K/2], scales [E][N][K/32] -> device layout; one thread per block.
__global__ void mx_repack_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales, int64_t E, int N,
                                 int nb, int which2, int H, int I, unsigned char* __restrict__ w, unsigned char* __restrict__ ws) {
  const int64_t total = E * N * nb;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / nb, e = row / N;
    const MxPlace p = mx_place(e, (int)(row - e * N), (int)(i - row * nb), which2, H, I);
    st16(w + p.code, ld16(codes + i * 16));
    ws[p.scale] = scales[i];
  }
}

// Rows [row0, row0 + N) of one expert's projection, quantized into the device layout.
template <int DT>
__global__ void mx_online_kernel(const void* __restrict__ x, int64_t e, int row0, int N, int nb, int which2, int H, int I,
                                 unsigned char* __restrict__ w, unsigned char* __restrict__ ws) {
  const int64_t total = (int64_t)N * nb;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int n = (int)(i / nb), b = (int)(i - (int64_t)n * nb);
    float v[32];
    ld_block<DT>(x, (size_t)i * 32, v);
    const int s = mx_scale_byte<kMxFp4>(mx_amax32(v));
    const MxPlace p = mx_place(e, row0 + n, b, which2, H, I);
    st16(w + p.code, mx_fp4_codes32(v, s));
    ws[p.scale] = (unsigned char)s;
  }
}

unsigned blocks_for(int64_t items) {
  const int64_t g = (items + 255) / 256;
  return (unsigned)(g > 65536 ? 65536 : g);
}

}  // namespace

// The grouped products of the sorted path, behind the routing (launch_route_mx).
hipError_t launch_mx_gemm(const MxArgs& a, int tiles_max, hipStream_t st, hipEvent_t mid) {
  const bool big = mx_big(a.n, a.E);
  const int tg = (tiles_max + 7) / 8 * 8;   // an eighth for each XCD
  const int b13 = (4 * mx_ktiles(a.I) + kMxWaves - 1) / kMxWaves, b2 = ((a.H >> 6) + kMxWaves - 1) / kMxWaves;
  if (big) hipLaunchKernelGGL(mx_gemm_big_kernel<false>, dim3(tg * b13), dim3(kMxThreads), 0, st, a);
  else hipLaunchKernelGGL(mx_gemm_kernel<false>, dim3(tg * b13), dim3(kMxThreads), 0, st, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  if (mid && (err = hipEventRecord(mid, st)) != hipSuccess) return err;
  if (big) hipLaunchKernelGGL(mx_gemm_big_kernel<true>, dim3(tg * b2), dim3(kMxThreads), 0, st, a);
  else hipLaunchKernelGGL(mx_gemm_kernel<true>, dim3(tg * b2), dim3(kMxThreads), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_mx_quantize(const void* x, int dt, int64_t rows, int cols, int64_t stride, int fmt, unsigned char* codes,
                              unsigned char* scales, hipStream_t st) {
  const unsigned g = blocks_for(rows * (cols >> 5));
#define MX_Q(D_, F_) \
  if (dt == D_ && fmt == F_) hipLaunchKernelGGL((mx_quantize_kernel<D_, F_>), dim3(g), dim3(256), 0, st, x, rows, cols, stride, codes, scales);
  MX_Q(0, 0) MX_Q(1, 0) MX_Q(2, 0) MX_Q(0, 1) MX_Q(1, 1) MX_Q(2, 1)
#undef MX_Q
  return hipGetLastError();
}

hipError_t launch_mx_dequantize(const unsigned char* codes, const unsigned char* scales, int64_t blocks, int fmt, void* out, int dt,
                                hipStream_t st) {
  const int64_t pieces = blocks * (dt == 2 ? 8 : 4);
  const unsigned g = blocks_for(pieces);
#define MX_D(D_, F_) \
  if (dt == D_ && fmt == F_) hipLaunchKernelGGL((mx_dequantize_kernel<D_, F_>), dim3(g), dim3(256), 0, st, codes, scales, pieces, out);
  MX_D(0, 0) MX_D(1, 0) MX_D(2, 0) MX_D(0, 1) MX_D(1, 1) MX_D(2, 1)
#undef MX_D
  return hipGetLastError();
}

// which2: 0 = w13 (N = 2I rows of H), 1 = w2 (N = H rows of I)
hipError_t launch_mx_repack(const void* codes, const void* scales, int64_t E, int which2, int H, int I, void* w, void* ws,
                            hipStream_t st) {
  const int N = which2 ? H : 2 * I, nb = (which2 ? I : H) >> 5;
  hipLaunchKernelGGL(mx_repack_kernel, dim3(blocks_for(E * N * nb)), dim3(256), 0, st, (const unsigned char*)codes,
                     (const unsigned char*)scales, E, N, nb, which2, H, I, (unsigned char*)w, (unsigned char*)ws);
  return hipGetLastError();
}

// proj: 0 gate, 1 up, 2 down
hipError_t launch_mx_online(const void* x, int dt, int64_t e, int proj, int H, int I, void* w, void* ws, hipStream_t st) {
  const int which2 = proj == 2, N = which2 ? H : I, nb = (which2 ? I : H) >> 5, row0 = proj == 1 ? I : 0;
  const unsigned g = blocks_for((int64_t)N * nb);
#define MX_O(D_) \
  if (dt == D_) hipLaunchKernelGGL(mx_online_kernel<D_>, dim3(g), dim3(256), 0, st, x, e, row0, N, nb, which2, H, I, (unsigned char*)w, (unsigned char*)ws);
  MX_O(0) MX_O(1) MX_O(2)
#undef MX_O
  return hipGetLastError();
}

}  // namespace mimoe
