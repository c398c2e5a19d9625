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
#include "mx_device.hpp"

namespace mimoe {

namespace {

constexpr int kMxWaves = 8;
constexpr int kMxThreads = kMxWaves * kWave;
constexpr int kMxChunkK = 2;                              // k tiles staged at a time
constexpr int kMxChunkRow = kMxChunkK * 4 * kMxPacketBytes;   // 256 B of a row
constexpr int kMxStage = kGemmRows * kMxChunkRow;         // 16 KB

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

// LDS position of 16-byte piece c of row r's chunk: pieces are permuted by
// the row, so that the 16 rows of an operand read lie in different banks.
__device__ __forceinline__ int mx_lds(int r, int c) { return r * kMxChunkRow + ((c ^ (r & 15)) << 4); }

// acc[t][s] = tile t of the wave's weight unit times the rows of subtile s,
// over all kt k tiles.  src: this thread's row of packets (row tid / 8) and
// part (tid % 8) of every chunk; w, ws: the unit's codes and scales, at this
// lane.  live: the wave has a unit (uniform); every wave stages.
__device__ __forceinline__ void mx_gemm_core(unsigned char* smem, const unsigned char* src, int kt, const unsigned char* w,
                                             const unsigned char* ws, int nsub, bool live, f32x4_t (&acc)[4][4]) {
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, r = lane & 15, srow = tid >> 3, part = tid & 7;
  const int nc = (kt + kMxChunkK - 1) / kMxChunkK, last = 4 * kt - 1;
  const bool stager = srow < 16 * nsub;
  auto stage_load = [&](int c, u32x4_t (&v)[2]) {
    const unsigned char* p = src + (size_t)min(8 * c + part, last) * kMxPacketBytes;
    v[0] = ld16(p);
    v[1] = ld16(p + 16);
  };
  u32x4_t sv[2], wv[kMxChunkK][4];
  uint32_t sc[kMxChunkK];
  auto weights = [&](int k, u32x4_t (&v)[4], uint32_t& s) {
    const int kk = min(k, kt - 1);
#pragma unroll
    for (int t = 0; t < 4; ++t) v[t] = ld16(w + (size_t)kk * kMxTileBytes + t * 1024);
    s = *reinterpret_cast<const uint32_t*>(ws + (size_t)kk * kMxTileScaleBytes);
  };
  stage_load(0, sv);
#pragma unroll
  for (int k = 0; k < kMxChunkK; ++k) weights(k, wv[k], sc[k]);
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int s = 0; s < 4; ++s) acc[t][s] = f32x4_t{0, 0, 0, 0};
  if (stager) {
    st16(smem + mx_lds(srow, 2 * part), sv[0]);
    st16(smem + mx_lds(srow, 2 * part + 1), sv[1]);
  }
  __syncthreads();
  for (int c = 0; c < nc; ++c) {
    const unsigned char* buf = smem + (c & 1) * kMxStage;
    if (c + 1 < nc) stage_load(c + 1, sv);
    if (live) {
#pragma unroll
      for (int k = 0; k < kMxChunkK; ++k) {
        if (kMxChunkK * c + k < kt) {   // uniform
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            if (s < nsub) {   // uniform
              const int row = 16 * s + r;
              const u32x4_t lo = ld16(buf + mx_lds(row, 2 * (4 * k + q))), hi = ld16(buf + mx_lds(row, 2 * (4 * k + q) + 1));
              acc[0][s] = mx_mfma<0>(wv[k][0], sc[k], lo, hi, acc[0][s]);
              acc[1][s] = mx_mfma<1>(wv[k][1], sc[k], lo, hi, acc[1][s]);
              acc[2][s] = mx_mfma<2>(wv[k][2], sc[k], lo, hi, acc[2][s]);
              acc[3][s] = mx_mfma<3>(wv[k][3], sc[k], lo, hi, acc[3][s]);
            }
          }
          // the weights of the same place in the next chunk, into the registers just used
          weights(kMxChunkK * (c + 1) + k, wv[k], sc[k]);
        }
      }
    }
    if (c + 1 < nc && stager) {
      unsigned char* nb = smem + ((c + 1) & 1) * kMxStage;
      st16(nb + mx_lds(srow, 2 * part), sv[0]);
      st16(nb + mx_lds(srow, 2 * part + 1), sv[1]);
    }
    __syncthreads();
  }
}

// gate_up + SiLU*mul + MXFP6: work item (row tile, 8 slices of 32 rows of I,
// one per wave).  A wave's gate and up tiles hold the same rows of I, so the
// product is in registers; a transpose between its lane rows leaves every
// lane with the 32 values of one token's block.
__global__ __launch_bounds__(kMxThreads) void mx_gemm13_kernel(MxArgs a) {
  __shared__ __align__(16) unsigned char smem[2 * kMxStage];
  const int NS = a.I >> 5, kt = mx_ktiles(a.H), NSP = 4 * mx_ktiles(a.I), nblk = (NSP + kMxWaves - 1) / kMxWaves;
  MxTile t;
  if (!mx_tile(a.rg, nblk, t)) return;   // uniform
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int slice = kMxWaves * t.blk + wave, nsub = (t.rows + 15) >> 4;
  const bool live = slice < NS;
  const int pair = a.rg.tok[t.row0 + min(tid >> 3, t.rows - 1)];
  const size_t unit = ((size_t)t.e * NS + (live ? slice : 0)) * kt;
  f32x4_t acc[4][4];
  mx_gemm_core(smem, a.xq + (size_t)(pair / a.K) * mx_row_bytes(a.H), kt, a.w13 + unit * kMxTileBytes + lane * 16,
               a.w13_s + unit * kMxTileScaleBytes + lane * 4, nsub, live, acc);
  if (slice >= NSP) return;
  float v[32];   // [q][tile][4] after the transpose
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float h[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) h[s] = silu_mul_fast(acc[p][s][i], acc[2 + p][s][i]);
      transpose4(h[0], h[1], h[2], h[3]);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[16 * p + 4 * q + i] = h[q];
    }
  MxPacket pk = {u32x4_t{0, 0, 0, 0}, u32x4_t{0, 0, 0, 0}};
  if (live) {
    const int s = mx_scale_byte<kMxFp6>(mx_amax32(v));
    pk = mx_packet(mx_fp6_codes32(v, s), s);
  }
  if (lane < t.rows) {   // lane = 16 subtile + row
    unsigned char* o = a.act + (size_t)(t.row0 + lane) * mx_row_bytes(a.I) + slice * kMxPacketBytes;
    st16(o, pk.lo);
    st16(o + 16, pk.hi);
  }
}

// Expert outputs between the down product and the combine: 16-bit integers
// with a power-of-two scale per 64 columns.  Half of fp32's bytes, and the
// rounding, at most 2^-15 of the 64 columns' largest, is far below that of
// the 16-bit result (16-bit floats would add as much as the result's own).
__device__ __forceinline__ float eout_scale(uint32_t amax_bits) {   // 2^(e - 14), NaN for NaN and infinity
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const int e = (int)(amax_bits >> 23);   // biased
  return __uint_as_float((uint32_t)(e > 15 ? e - 14 : 1) << 23);
}

// down: work item (row tile, 8 units of 64 rows of H, one per wave).
__global__ __launch_bounds__(kMxThreads) void mx_gemm2_kernel(MxArgs a) {
  __shared__ __align__(16) unsigned char smem[2 * kMxStage];
  const int NQ = a.H >> 6, kt = mx_ktiles(a.I), nblk = (NQ + kMxWaves - 1) / kMxWaves;
  MxTile t;
  if (!mx_tile(a.rg, nblk, t)) return;   // uniform
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int m = kMxWaves * t.blk + wave, nsub = (t.rows + 15) >> 4;
  const bool live = m < NQ;
  const size_t unit = ((size_t)t.e * NQ + (live ? m : 0)) * kt;
  f32x4_t acc[4][4];
  mx_gemm_core(smem, a.act + (size_t)(t.row0 + min(tid >> 3, t.rows - 1)) * mx_row_bytes(a.I), kt,
               a.w2 + unit * kMxTileBytes + lane * 16, a.w2_s + unit * kMxTileScaleBytes + lane * 4, nsub, live, acc);
  if (!live) return;
  float v[64];
#pragma unroll
  for (int p = 0; p < 4; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float h[4] = {acc[p][0][i], acc[p][1][i], acc[p][2][i], acc[p][3][i]};
      transpose4(h[0], h[1], h[2], h[3]);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[16 * p + 4 * q + i] = h[q];
    }
  if (lane >= t.rows) return;
  uint32_t am = 0;
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    am = b > am ? b : am;
  }
  const float d = eout_scale(am), id = 1.0f / d;   // powers of two
  const int pair = a.rg.tok[t.row0 + lane];
  int16_t* o = a.eout + (size_t)pair * a.H + 64 * m;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int z[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int n = (int)__builtin_rintf(v[8 * c + 2 * j + k] * id);
        z[k] = n > 32767 ? 32767 : n;   // the largest may round up to 2^15; -2^15 is there
      }
      w[j] = ((uint32_t)z[0] & 0xffffu) | ((uint32_t)z[1] << 16);
    }
    st16(o + 8 * c, u32x4_t{w[0], w[1], w[2], w[3]});
  }
  a.eout_d[(size_t)pair * NQ + m] = d;
}

// y[t,h] = cast(sum_k w[t,k] eout[t*K+k,h]) over the valid ids in k order, in
// fp32; a token without a valid id gets 0.  One thread per (t, 8 columns).
template <int ACT>
__global__ void mx_combine_kernel(const int16_t* __restrict__ eout, const float* __restrict__ eout_d, const float* __restrict__ tw,
                                  const int32_t* __restrict__ ids, uint16_t* __restrict__ y, int T, int K, int E, int H) {
  const int HV = H >> 3, NQ = H >> 6;
  const int64_t total = (int64_t)T * HV;
  for (int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; idx < total; idx += (int64_t)gridDim.x * blockDim.x) {
    const int t = (int)(idx / HV), h = (int)(idx - (int64_t)t * HV) * 8;
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    constexpr int kB = 8;   // pairs whose loads are issued together
    for (int k0 = 0; k0 < K; k0 += kB) {
      int ev[kB];
      float wv[kB], dv[kB];
      u32x4_t rv[kB];
#pragma unroll
      for (int j = 0; j < kB; ++j) {
        const int i = t * K + min(k0 + j, K - 1);
        ev[j] = k0 + j < K ? ids[i] : -1;
        wv[j] = tw[i];
        dv[j] = eout_d[(size_t)i * NQ + (h >> 6)];
        rv[j] = ld16(eout + (size_t)i * H + h);
      }
#pragma unroll
      for (int j = 0; j < kB; ++j) {
        if ((unsigned)ev[j] >= (unsigned)E) continue;
        const uint32_t u[4] = {rv[j].x, rv[j].y, rv[j].z, rv[j].w};
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const float lo = (float)(int16_t)(u[p] & 0xffffu) * dv[j], hi = (float)((int32_t)u[p] >> 16) * dv[j];   // exact
          acc[2 * p] = acc[2 * p] + wv[j] * lo;
          acc[2 * p + 1] = acc[2 * p + 1] + wv[j] * hi;
        }
      }
    }
    uint32_t o[4];
#pragma unroll
    for (int p = 0; p < 4; ++p)
      o[p] = from_f32<ACT>(acc[2 * p]) | ((uint32_t)from_f32<ACT>(acc[2 * p + 1]) << 16);
    st16(y + (size_t)t * H + h, u32x4_t{o[0], o[1], o[2], o[3]});
  }
}

__device__ __forceinline__ void ld_words(const void* p, uint32_t (&w)[16]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const u32x4_t v = ld16(reinterpret_cast<const unsigned char*>(p) + 16 * c);
    w[4 * c] = v.x; w[4 * c + 1] = v.y; w[4 * c + 2] = v.z; w[4 * c + 3] = v.w;
  }
}

// Hidden rows -> packets, one thread per block; blocks past H are zeros.
template <int ACT>
__global__ void mx_quant_rows_kernel(const uint16_t* __restrict__ x, int T, int H, unsigned char* __restrict__ xq) {
  const int nb = H >> 5, nbp = 4 * mx_ktiles(H);
  const int64_t total = (int64_t)T * nbp;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int t = (int)(i / nbp), b = (int)(i - (int64_t)t * nbp);
    MxPacket pk = {u32x4_t{0, 0, 0, 0}, u32x4_t{0, 0, 0, 0}};
    if (b < nb) {
      uint32_t w[16];
      ld_words(x + (size_t)t * H + 32 * b, w);
      const int s = mx_scale_byte<kMxFp6>(mx_amax16<ACT>(w));
      pk = mx_packet(mx_fp6_codes16<ACT>(w, s), s);
    }
    st16(xq + i * kMxPacketBytes, pk.lo);
    st16(xq + i * kMxPacketBytes + 16, pk.hi);
  }
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
    ld_words(reinterpret_cast<const uint16_t*>(x) + elem, w);
    mx_unpack16<DT>(w, v);
  }
}

// rows of cols elements (stride elements apart) -> codes [rows][cols/32][16
// or 24 B], scales [rows][cols/32].  One thread per block.
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

// codes and scales -> values 2^(s-127) * element, rounded once to DT.
template <int DT, int FMT>
__global__ void mx_dequantize_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales, int64_t total,
                                     void* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int s = scales[i];
    float v[32];
    if constexpr (FMT == kMxFp4) {
      const u32x4_t c = ld16(codes + i * 16);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const auto e0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[w], 1.0f, 0), e1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[w], 1.0f, 1),
                   e2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[w], 1.0f, 2), e3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[w], 1.0f, 3);
        v[8 * w] = e0[0]; v[8 * w + 1] = e0[1]; v[8 * w + 2] = e1[0]; v[8 * w + 3] = e1[1];
        v[8 * w + 4] = e2[0]; v[8 * w + 5] = e2[1]; v[8 * w + 6] = e3[0]; v[8 * w + 7] = e3[1];
      }
    } else {
      const u32x2_t* p = reinterpret_cast<const u32x2_t*>(codes + i * 24);
      const u32x2_t a = p[0], b = p[1], c = p[2];
      const auto f = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(u32x6_t{a.x, a.y, b.x, b.y, c.x, c.y}, 1.0f);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = f[j];
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = s == 255 ? __uint_as_float(0x7fc00000u) : __builtin_ldexpf(v[j], s - 127);
    if constexpr (DT == 2) {
      f32x4_t* o = reinterpret_cast<f32x4_t*>(out) + i * 8;
#pragma unroll
      for (int c = 0; c < 8; ++c) o[c] = f32x4_t{v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]};
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = from_f32<DT>(v[8 * c + 2 * j]) | ((uint32_t)from_f32<DT>(v[8 * c + 2 * j + 1]) << 16);
        st16(reinterpret_cast<uint16_t*>(out) + i * 32 + 8 * c, u32x4_t{w[0], w[1], w[2], w[3]});
      }
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

// The sorted path: the hidden rows quantized, both grouped products, the combine.
hipError_t launch_mx_sorted(const MxArgs& a, int act, int tiles_max, hipStream_t st, hipEvent_t mid) {
  const int64_t nbp = (int64_t)a.T * 4 * mx_ktiles(a.H);
  if (act == 1)
    hipLaunchKernelGGL(mx_quant_rows_kernel<1>, dim3(blocks_for(nbp)), dim3(256), 0, st, a.x, a.T, a.H, a.xq);
  else
    hipLaunchKernelGGL(mx_quant_rows_kernel<0>, dim3(blocks_for(nbp)), dim3(256), 0, st, a.x, a.T, a.H, a.xq);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const int tg = (tiles_max + 7) / 8 * 8;   // an eighth for each XCD
  const int b13 = (4 * mx_ktiles(a.I) + kMxWaves - 1) / kMxWaves, b2 = ((a.H >> 6) + kMxWaves - 1) / kMxWaves;
  hipLaunchKernelGGL(mx_gemm13_kernel, dim3(tg * b13), dim3(kMxThreads), 0, st, a);
  err = hipGetLastError();
  if (err != hipSuccess) return err;
  if (mid && (err = hipEventRecord(mid, st)) != hipSuccess) return err;
  hipLaunchKernelGGL(mx_gemm2_kernel, dim3(tg * b2), dim3(kMxThreads), 0, st, a);
  err = hipGetLastError();
  if (err != hipSuccess) return err;
  const unsigned g = blocks_for((int64_t)a.T * (a.H >> 3));
  if (act == 1)
    hipLaunchKernelGGL(mx_combine_kernel<1>, dim3(g), dim3(256), 0, st, a.eout, a.eout_d, a.tw, a.ids, a.y, a.T, a.K, a.E, a.H);
  else
    hipLaunchKernelGGL(mx_combine_kernel<0>, dim3(g), dim3(256), 0, st, a.eout, a.eout_d, a.tw, a.ids, a.y, a.T, a.K, a.E, a.H);
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
  const unsigned g = blocks_for(blocks);
#define MX_D(D_, F_) \
  if (dt == D_ && fmt == F_) hipLaunchKernelGGL((mx_dequantize_kernel<D_, F_>), dim3(g), dim3(256), 0, st, codes, scales, blocks, out);
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
