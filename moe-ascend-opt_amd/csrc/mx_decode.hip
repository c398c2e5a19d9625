// mx_decode.hip -- decode calls of MXFP4 expert layers (up to 64 routed
// pairs, top-k <= 16): no sort, no quantized copy of the hidden rows, the
// combine in the down product.
//
// gate_up item (pair, slice of 32 rows of I): serves its expert iff the pair
// is the expert's first (wave ballots over all ids).  The 8 waves split K.
// While the weights are on their way to registers, the tokens' rows are
// quantized into LDS, a lane per block.  The waves' sums meet in LDS, and one
// lane per token makes the slice's MXFP6 block.
//
// down item (token, 16 rows of H): wave k takes routed expert k over all of
// I; y = cast(sum_k w_k out_k) in k order.
//
// One launch (top-k <= 8): gate_up workgroups first, down workgroups behind
// them in the grid; a block travels as 8 tagged 8-byte units (handover.hpp):
// 6 words of codes, the scale byte, one word unused.  Two launches otherwise.
//
// One launch, H=2048 I=768 E=128 top-8, weights that no cache holds: T = 1
// 10.6 us for 20 MB, bound by its chain (ids, rows, weights, the sums' meeting,
// the hand-over, down); T = 8 28 us for the weights of some 50 experts, 4.6
// TB/s.  Two launches, H=2048 I=512 E=128 top-10: T = 1 6.1 + 5.1 us, T = 6
// 15.7 + 11.2 us for some 50 experts, 3.1 TB/s.
#pragma clang fp contract(off)
#include "handover.hpp"
#include "mi_moe_sched.hpp"
#include "mx_device.hpp"

namespace mimoe {

namespace {

constexpr int kDecWaves = 8;
constexpr int kMaxDecodeK = 16;
constexpr int kUnitsPerBlock = 8;
constexpr int kUnitBatch = 4;        // units per lane loaded together by a down wave
constexpr int kRedBytes = kDecWaves * 4 * 64 * 16;   // partial sums [wave][tile][lane][4]
constexpr int kHiddenStride = 33;    // floats of a token's slice in LDS

// Keeps loads in the order they are written in.
__device__ __forceinline__ void issue_order_fence() { asm volatile("" ::: "memory"); }
__device__ __forceinline__ u32x4_t ld16(const void* p) { return *reinterpret_cast<const u32x4_t*>(p); }
__device__ __forceinline__ void st16(void* p, const u32x4_t& v) { *reinterpret_cast<u32x4_t*>(p) = v; }

// ---------------------------------------------------------------- gate_up
// The columns (tokens of the expert) of a pass lie in LDS as packets, 16
// bytes apart from whole lines, so that 16 columns' packets of one block
// spread over the banks.  As many at a time as fit beside nothing (at least
// one, at most the matrix operand's 16).
__host__ __device__ inline int col_bytes(int H) { return (int)mx_row_bytes(H) + 16; }
__host__ __device__ inline int pass_cols(int H) {
  const int p = kRedBytes / col_bytes(H);
  return p < 1 ? 1 : p > 16 ? 16 : p;
}
// packets, then (the same memory) the partial sums; the slice's values
__host__ __device__ inline int gate_up_lds(int H) {
  const int p = pass_cols(H) * col_bytes(H);
  return (p > kRedBytes ? p : kRedBytes) + 16 * kHiddenStride * 4;
}

// NB: k tiles whose weights a wave has on their way together.
template <int ACT, int NB, bool FUSED>
__device__ __forceinline__ void gate_up_item(const MxArgs& a, int item, int js, unsigned char* smem) {
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int q = lane >> 4, r = lane & 15;
  const int NS = a.I >> 5, kt = mx_ktiles(a.H), nb = a.H >> 5, cb = col_bytes(a.H), P = pass_cols(a.H);
  SchedArgs c;
  c.ids = a.ids; c.n = a.n; c.E = a.E;
  const BallotCols cl = ballot_cols(c, item, lane);
  if (!cl.serve) return;   // uniform
  const int e = __builtin_amdgcn_readfirstlane(cl.e), cnt = __builtin_amdgcn_readfirstlane(cl.cnt);
  const float rk = 1.0f / (float)a.K;
  const size_t unit = ((size_t)e * NS + js) * kt;
  const unsigned char* w = a.w13 + unit * kMxTileBytes + lane * 16;
  const unsigned char* ws = a.w13_s + unit * kMxTileScaleBytes + lane * 4;
  const int k0 = kt * wave / kDecWaves, k1 = kt * (wave + 1) / kDecWaves;
  f32x4_t* red = reinterpret_cast<f32x4_t*>(smem);
  float* hid = reinterpret_cast<float*>(smem + gate_up_lds(a.H) - 16 * kHiddenStride * 4);
  for (int c0 = 0; c0 < cnt; c0 += P) {
    const int ncol = min(P, cnt - c0);
    u32x4_t wv[NB][4];
    uint32_t sc[NB];
    auto weights = [&](int kb) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int k = max(min(kb + i, k1 - 1), 0);
#pragma unroll
        for (int t = 0; t < 4; ++t) wv[i][t] = ld16(w + (size_t)k * kMxTileBytes + t * 1024);
        sc[i] = *reinterpret_cast<const uint32_t*>(ws + (size_t)k * kMxTileScaleBytes);
      }
    };
    // The hidden rows: a wave takes a column, a lane a block.  The first
    // blocks' loads go out before the weights' (loads return in order), which
    // are on their way during the quantization.
    uint32_t xv[16];
    auto row = [&](int col) { return a.x + (size_t)div_small(__shfl(cl.colpair, c0 + col), rk) * a.H; };
    if (wave < ncol) mx_load_words(row(wave) + 32 * min(lane, nb - 1), xv);   // uniform
    issue_order_fence();
    weights(k0);
    issue_order_fence();
    for (int col = wave; col < ncol; col += kDecWaves) {   // uniform
      const uint16_t* x = row(col);
      for (int b = lane; b < 4 * kt; b += 64) {
        if (col != wave || b != lane) mx_load_words(x + 32 * min(b, nb - 1), xv);
        MxPacket pk = {u32x4_t{0, 0, 0, 0}, u32x4_t{0, 0, 0, 0}};   // past H
        if (b < nb) {
          const int s = mx_scale_byte<kMxFp6>(mx_amax16<ACT>(xv));
          pk = mx_packet(mx_fp6_codes16<ACT>(xv, s), s);
        }
        st16(smem + col * cb + b * kMxPacketBytes, pk.lo);
        st16(smem + col * cb + b * kMxPacketBytes + 16, pk.hi);
      }
    }
    __syncthreads();
    f32x4_t acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = f32x4_t{0, 0, 0, 0};
    const unsigned char* cp = smem + min(r, ncol - 1) * cb + q * kMxPacketBytes;
    for (int kb = k0; kb < k1; kb += NB) {
      if (kb > k0) weights(kb);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        if (kb + i < k1) {   // uniform
          const unsigned char* p = cp + (kb + i) * 4 * kMxPacketBytes;
          const u32x4_t lo = ld16(p), hi = ld16(p + 16);
          acc[0] = mx_mfma<0>(wv[i][0], sc[i], lo, hi, acc[0]);
          acc[1] = mx_mfma<1>(wv[i][1], sc[i], lo, hi, acc[1]);
          acc[2] = mx_mfma<2>(wv[i][2], sc[i], lo, hi, acc[2]);
          acc[3] = mx_mfma<3>(wv[i][3], sc[i], lo, hi, acc[3]);
        }
      }
    }
    const int pair = __shfl(cl.colpair, c0 + min(lane, ncol - 1));   // of column lane
    __syncthreads();   // the packets are read: the sums take their place
#pragma unroll
    for (int t = 0; t < 4; ++t) red[(wave * 4 + t) * 64 + lane] = acc[t];
    __syncthreads();
    if (wave < 2 && r < ncol) {   // gate tile wave, up tile 2 + wave
      f32x4_t g = red[wave * 64 + lane], u = red[(2 + wave) * 64 + lane];
#pragma unroll
      for (int v = 1; v < kDecWaves; ++v) {
        g += red[(v * 4 + wave) * 64 + lane];
        u += red[(v * 4 + 2 + wave) * 64 + lane];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) hid[r * kHiddenStride + 16 * wave + 4 * q + i] = silu_mul_fast(g[i], u[i]);
    }
    __syncthreads();
    if (tid < ncol) {   // in wave 0: lane = column
      float h[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) h[i] = hid[tid * kHiddenStride + i];
      const int s = mx_scale_byte<kMxFp6>(mx_amax32(h));
      const MxPacket pk = mx_packet(mx_fp6_codes32(h, s), s);
      if constexpr (FUSED) {
        const unsigned long long tag = (unsigned long long)dispatch_tag32() << 32;
        unsigned long long* o = a.tact + ((size_t)pair * NS + js) * kUnitsPerBlock;
#pragma unroll
        for (int i = 0; i < 4; ++i) store_agent(o + i, tag | pk.lo[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) store_agent(o + 4 + i, tag | pk.hi[i]);
      } else {
        unsigned char* o = a.act + (size_t)pair * mx_row_bytes(a.I) + js * kMxPacketBytes;
        st16(o, pk.lo);
        st16(o + 16, pk.hi);
      }
    }
    // The next pass's packets take the place of the sums, which are read (the
    // barrier above); hid is written again behind two more barriers, which
    // wave 0 reaches with its reads of it done.
  }
}

// ---------------------------------------------------------------- down
// LDS: weighted outputs [K][16] f32 | state [K] (0 no expert, 1 valid, 2 a wait gave up) |
// fused: rows [K][NS packets].
__host__ __device__ inline size_t down_lds(int K, int I, bool fused) {
  return (size_t)K * 16 * 4 + (size_t)(K + 3) / 4 * 16 + (fused ? (size_t)K * (I >> 5) * kMxPacketBytes : 0);
}

template <int ACT, int NB, bool FUSED>
__device__ __forceinline__ void down_item(const MxArgs& a, int t, int tile0, unsigned char* smem) {
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, q = lane >> 4;
  const int NS = a.I >> 5, kt = mx_ktiles(a.I), NQ = a.H >> 6, K = a.K;
  float* outs = reinterpret_cast<float*>(smem);
  int* state = reinterpret_cast<int*>(outs + 16 * K);
  if (wave < K) {   // uniform
    const int i = t * K + wave;
    const int e = __builtin_amdgcn_readfirstlane(a.ids[i]);
    const float tw = a.tw[i];
    const bool ok = (unsigned)e < (unsigned)a.E;
    const size_t unit = ((size_t)(ok ? e : 0) * NQ + (tile0 >> 2)) * kt;
    const unsigned char* w = a.w2 + unit * kMxTileBytes + (tile0 & 3) * 1024 + lane * 16;
    const unsigned char* ws = a.w2_s + unit * kMxTileScaleBytes + lane * 4 + (tile0 & 3);
    u32x4_t wv[NB];
    uint32_t sc[NB];
    auto weights = [&](int kb) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int k = min(kb + j, kt - 1);
        wv[j] = ld16(w + (size_t)k * kMxTileBytes);
        sc[j] = ws[(size_t)k * kMxTileScaleBytes];
      }
    };
    int st = ok ? 1 : 0;
    f32x4_t acc = {0, 0, 0, 0};
    if (ok) {   // uniform
      weights(0);   // in flight during the wait
      const unsigned char* row;
      if constexpr (FUSED) {
        uint32_t* dst = reinterpret_cast<uint32_t*>(smem + down_lds(K, a.I, false)) + (size_t)wave * NS * kUnitsPerBlock;
        const unsigned tag = dispatch_tag32();
        const unsigned long long* src = a.tact + (size_t)i * NS * kUnitsPerBlock;
        const int nunits = NS * kUnitsPerBlock;
        auto read_row = [&]() {   // reads, checks and unpacks the whole row
          bool whole = true;
          for (int u0 = 0; u0 < nunits; u0 += 64 * kUnitBatch) {
            unsigned long long v[kUnitBatch];
#pragma unroll
            for (int b = 0; b < kUnitBatch; ++b) {
              const int u = u0 + 64 * b + lane;
              v[b] = u < nunits ? load_agent(src + u) : ((unsigned long long)tag << 32);
            }
#pragma unroll
            for (int b = 0; b < kUnitBatch; ++b) {
              const int u = u0 + 64 * b + lane;
              whole = whole && (unsigned)(v[b] >> 32) == tag;
              if (u < nunits) dst[u] = (uint32_t)v[b];
            }
          }
          return __all(whole);
        };
        for (int polls = 0; !read_row();) {
          if (++polls > kSpinMax) {
            st = 2;
            break;
          }
          __builtin_amdgcn_s_sleep(2);
        }
        row = reinterpret_cast<const unsigned char*>(dst);
      } else {
        row = a.act + (size_t)i * mx_row_bytes(a.I);
      }
      for (int kb = 0; kb < kt; kb += NB) {
        if (kb) weights(kb);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const int k = kb + j, b = 4 * k + q;
          if (k < kt) {   // uniform
            const unsigned char* p = row + min(b, NS - 1) * kMxPacketBytes;
            u32x4_t lo = ld16(p), hi = ld16(p + 16);
            if (b >= NS) { lo = u32x4_t{0, 0, 0, 0}; hi = lo; }   // past I
            acc = mx_mfma<0>(wv[j], sc[j], lo, hi, acc);
          }
        }
      }
    }
    if ((lane & 15) == 0) *reinterpret_cast<f32x4_t*>(outs + 16 * wave + 4 * q) = acc * tw;   // every column is the token
    if (lane == 0) state[wave] = st;
  }
  __syncthreads();
  if (tid < 16) {
    float yv = 0.0f;
    bool gave_up = false;
    for (int k = 0; k < K; ++k) {
      const int s = state[k];
      if (s) {
        gave_up |= s == 2;
        yv = yv + outs[16 * k + tid];
      }
    }
    a.y[(size_t)t * a.H + 16 * tile0 + tid] = gave_up ? (uint16_t)0x7fffu : from_f32<ACT>(yv);   // NaN in both types
  }
}

// The leading arguments repeat fields of a: they are preloaded into SGPRs at
// wave launch.
template <int ACT, int NB1, int NB2>
__global__ __launch_bounds__(kDecWaves * kWave) __attribute__((amdgpu_waves_per_eu(4)))
void mx_decode_kernel(const int32_t* ids, const uint16_t* x, const unsigned char* w13, const unsigned char* w13_s,
                      const unsigned char* w2, const unsigned char* w2_s, int n1, int ns, MxArgs a0) {
  extern __shared__ __align__(16) unsigned char smem[];
  MxArgs a = a0;
  a.ids = ids; a.x = x; a.w13 = w13; a.w13_s = w13_s; a.w2 = w2; a.w2_s = w2_s;
  const int b = blockIdx.x;
  if (b < n1) {   // uniform
    const int item = b / ns;
    gate_up_item<ACT, NB1, true>(a, item, b - item * ns, smem);
  } else {
    const int nt = a.H >> 4, d = b - n1, t = d / nt;
    down_item<ACT, NB2, true>(a, t, d - t * nt, smem);
  }
}

template <int ACT, int NB1>
__global__ __launch_bounds__(kDecWaves * kWave) __attribute__((amdgpu_waves_per_eu(4)))
void mx_gate_up_kernel(const int32_t* ids, const uint16_t* x, const unsigned char* w13, const unsigned char* w13_s, MxArgs a0) {
  extern __shared__ __align__(16) unsigned char smem[];
  MxArgs a = a0;
  a.ids = ids; a.x = x; a.w13 = w13; a.w13_s = w13_s;
  gate_up_item<ACT, NB1, false>(a, blockIdx.y, blockIdx.x, smem);
}

template <int ACT, int NB2>
__global__ __launch_bounds__(kMaxDecodeK * kWave) void mx_down_kernel(const int32_t* ids, const unsigned char* w2,
                                                                       const unsigned char* w2_s, MxArgs a0) {
  extern __shared__ __align__(16) unsigned char smem[];
  MxArgs a = a0;
  a.ids = ids; a.w2 = w2; a.w2_s = w2_s;
  down_item<ACT, NB2, false>(a, blockIdx.y, blockIdx.x, smem);
}

template <int ACT, int NB1, int NB2>
hipError_t launch_decode_t(const MxArgs& a, hipStream_t st, hipEvent_t mid) {
  const int NS = a.I >> 5, nt = a.H >> 4;
  if (mx_decode_fused(a.K, a.I)) {
    const size_t dl = down_lds(a.K, a.I, true), gl = gate_up_lds(a.H), lds = dl > gl ? dl : gl;
    if (lds > kMaxLds)   // H near its limit
      (void)hipFuncSetAttribute(reinterpret_cast<const void*>(mx_decode_kernel<ACT, NB1, NB2>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL((mx_decode_kernel<ACT, NB1, NB2>), dim3(a.n * NS + a.T * nt), dim3(kDecWaves * kWave), lds, st,
                       a.ids, a.x, a.w13, a.w13_s, a.w2, a.w2_s, a.n * NS, NS, a);
    return hipGetLastError();
  }
  if (gate_up_lds(a.H) > (int)kMaxLds)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(mx_gate_up_kernel<ACT, NB1>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, gate_up_lds(a.H));
  hipLaunchKernelGGL((mx_gate_up_kernel<ACT, NB1>), dim3(NS, a.n), dim3(kDecWaves * kWave), gate_up_lds(a.H), st, a.ids, a.x,
                     a.w13, a.w13_s, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  if (mid && (err = hipEventRecord(mid, st)) != hipSuccess) return err;
  hipLaunchKernelGGL((mx_down_kernel<ACT, NB2>), dim3(nt, a.T), dim3(a.K * kWave), down_lds(a.K, a.I, false), st, a.ids, a.w2,
                     a.w2_s, a);
  return hipGetLastError();
}

}  // namespace

// Decode calls: a.tact for the one-launch form (mx_decode_fused), a.act ([n]
// rows, row = pair) for the other.
hipError_t launch_mx_decode(const MxArgs& a, int act, hipStream_t st, hipEvent_t mid) {
  if (!mx_decode_ok(a.n, a.K, a.E, a.H, a.I)) return hipErrorInvalidValue;
  const int nb2 = mx_ktiles(a.I) <= 2 ? 2 : mx_ktiles(a.I) <= 4 ? 4 : 6;
  if (act == 1)
    return nb2 == 2 ? launch_decode_t<1, 2, 2>(a, st, mid) : nb2 == 4 ? launch_decode_t<1, 2, 4>(a, st, mid) : launch_decode_t<1, 2, 6>(a, st, mid);
  return nb2 == 2 ? launch_decode_t<0, 2, 2>(a, st, mid) : nb2 == 4 ? launch_decode_t<0, 2, 4>(a, st, mid) : launch_decode_t<0, 2, 6>(a, st, mid);
}

}  // namespace mimoe
