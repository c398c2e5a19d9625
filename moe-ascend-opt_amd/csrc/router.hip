// router.hip -- routing to experts by scores: softmax or sigmoid of the
// logits, a bias that only decides the choice, expert groups, top-k,
// renormalized and scaled weights.
//
//   s_e = sigmoid(l_e) or softmax(l)_e,  c_e = s_e + b_e
//   group score = the sum of the group's group_top largest c (1 or 2), of
//   the one that is left where the others are masked, -infinity of none
//   the topk_group groups of the largest scores, in them the K largest c
//   w_k = scale * s_k / sum of the picks' s  (renormalize), or scale * s_k
//
// Ties go to the lower group and the lower expert.  Scores are computed in 64
// bits: among some hundred experts two choices often lie within fp32's
// rounding of each other, and which expert is picked should follow from the
// logits, not from the order of a sum.
#include <algorithm>
#include <type_traits>

#include "mi_moe_device.hpp"
#include "mi_moe_internal.hpp"

namespace mimoe {

namespace {

constexpr int kScoreWaves = 4;
constexpr int kScoreMaxE = 512;
// Tokens from which a row of 16 lanes takes one (topk_scores_rows_kernel),
// not a wave.  us, row / wave: E=256 top-8 in groups T = 2048 7.1 / 6.2, 4096
// 7.2 / 8.5, 16384 15.4 / 22.6; E=128 top-8 2048 4.4 / 4.3, 4096 4.5 / 6.0;
// E=64 top-6 1024 3.4 / 3.2, 4096 3.5 / 4.6, 100000 24 / 55.
constexpr int kScoreRowsT = 3000;

// A lane's value from another lane of its row of 16 (DPP: no trip through
// LDS).  In this order the four controls leave every lane with the result
// over groups of 2, 4, 8 and 16 lanes.
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
  return __hiloint2double(__builtin_amdgcn_mov_dpp(__double2hiint(v), CTRL, 0xf, 0xf, false),
                          __builtin_amdgcn_mov_dpp(__double2loint(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float lane_value(float v, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); }
__device__ __forceinline__ double lane_value(double v, int l) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l), __builtin_amdgcn_readlane(__double2loint(v), l));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, false);
}
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ float larger(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }

// exp(x) for x <= 0, in 64 bits: x = n log 2 + r, |r| <= log(2) / 2, the
// Taylor series of exp(r) to r^13 (4e-18 left), scaled by 2^n.  NaN stays NaN.
__device__ __forceinline__ double exp_neg(double x) {
  x = x < -750.0 ? -750.0 : x;   // 0 after the scaling
  const double n = __builtin_rint(x * 1.4426950408889634);
  double r = __builtin_fma(n, -0x1.62e42fefa0000p-1, x);   // log 2 in two parts: n times the first, of 36 bits, is exact
  r = __builtin_fma(n, -0x1.cf79abc9e3b3ap-40, r);
  double p = 1.0 / 6227020800.0;
  p = __builtin_fma(p, r, 1.0 / 479001600.0);
  p = __builtin_fma(p, r, 1.0 / 39916800.0);
  p = __builtin_fma(p, r, 1.0 / 3628800.0);
  p = __builtin_fma(p, r, 1.0 / 362880.0);
  p = __builtin_fma(p, r, 1.0 / 40320.0);
  p = __builtin_fma(p, r, 1.0 / 5040.0);
  p = __builtin_fma(p, r, 1.0 / 720.0);
  p = __builtin_fma(p, r, 1.0 / 120.0);
  p = __builtin_fma(p, r, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}
// 1 / x for 1 <= x <= 2 or any other x of ordinary size: the hardware's
// estimate and two Newton steps.
__device__ __forceinline__ double reciprocal(double x) {
  double y = __builtin_amdgcn_rcp(x);
  y = __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
  return __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
}
// 1 / (1 + exp(-l)), from the exponential of -|l|, which cannot overflow
__device__ __forceinline__ double sigmoid(float l) {
  const double e = exp_neg(-__builtin_fabs((double)l)), y = reciprocal(1.0 + e);
  return l < 0.0f ? e * y : y;
}

// Over the 16 lanes of a row, and over the wave.
template <class T>
__device__ __forceinline__ T row_max(T v) {
  v = larger(v, dpp<kXor1>(v));
  v = larger(v, dpp<kXor2>(v));
  v = larger(v, dpp<kHalfMirror>(v));
  return larger(v, dpp<kMirror>(v));
}
template <class T>
__device__ __forceinline__ T wave_max(T v) {
  v = row_max(v);
  return larger(larger(lane_value(v, 0), lane_value(v, 16)), larger(lane_value(v, 32), lane_value(v, 48)));
}
__device__ __forceinline__ double row_sum(double v) {
  v += dpp<kXor1>(v);
  v += dpp<kXor2>(v);
  v += dpp<kHalfMirror>(v);
  return v + dpp<kMirror>(v);
}
__device__ __forceinline__ double wave_sum(double v) {
  v = row_sum(v);
  return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}

// The two largest of two sets, from each one's two largest.
struct Top2 {
  double a, b;
};
__device__ __forceinline__ void merge(Top2& x, double a, double b) {
  const double lo = __builtin_fmin(x.a, a);
  x.a = larger(x.a, a);
  x.b = larger(lo, larger(x.b, b));
}

// A lane's NJ consecutive elements from e0 on (any element for one past E).
// wide: in pieces of up to 16 bytes, which E and the alignment allow.
template <class T, int NJ>
__device__ __forceinline__ void load_run(const T* row, int e0, int E, bool wide, T (&v)[NJ]) {
  constexpr int P = NJ * sizeof(T) < 16 ? NJ : 16 / (int)sizeof(T);
  struct alignas(P * sizeof(T)) Piece {
    T v[P];
  };
  if (wide) {   // uniform
#pragma unroll
    for (int p = 0; p < NJ; p += P) {
      const Piece q = *reinterpret_cast<const Piece*>(row + min(e0 + p, E - P));
#pragma unroll
      for (int i = 0; i < P; ++i) v[p + i] = q.v[i];
    }
  } else {
#pragma unroll
    for (int j = 0; j < NJ; ++j) v[j] = row[min(e0 + j, E - 1)];
  }
}
// Logits (minus infinity past E) and bias of a lane's experts.
template <int LDT, int NJ>
__device__ __forceinline__ void load_lane(const void* logits, const float* bias, const ScoreArgs& a, bool wide, int t, int e0,
                                          float (&l)[NJ], float (&b)[NJ]) {
  using T = typename std::conditional<LDT == 2, float, uint16_t>::type;
  T v[NJ];
  load_run<T, NJ>(reinterpret_cast<const T*>(logits) + (size_t)t * a.E, e0, a.E, wide, v);
#pragma unroll
  for (int j = 0; j < NJ; ++j) b[j] = 0.0f;
  if (bias) load_run<float, NJ>(bias, e0, a.E, wide, b);   // uniform, around all loads: a branch for each would wait for each
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    float f;
    if constexpr (LDT == 2) f = v[j];
    else f = to_f32<LDT>(v[j]);
    l[j] = e0 + j < a.E ? f : -__builtin_inff();
  }
}

// One wave per token; lane l holds experts l NJ .. l NJ + NJ - 1, so that the
// lower of two experts is in the lower lane.
//
// A pick is the largest choice: found as a maximum of the choices rounded to
// fp32 (rounding keeps the order, so the largest is among those that reach
// it), and only where several experts reach it in 64 bits among them.
//
// Bound by a chain of dependent steps, the 64-bit scores and K maxima: T = 1
// E = 256 top-8 in 8 groups 4.2 us, E = 512 5.7, E = 384 (groups through LDS)
// 7.5.  More than 256 experts take it at any T: T = 16384 top-8 in 8 groups
// E = 512 36 us, E = 384 45 us.
template <int LDT, int NJ>   // logits: 0 fp16, 1 bf16, 2 fp32; NJ = ceil(E / 64), a power of two
__global__ __launch_bounds__(kScoreWaves * kWave) void topk_scores_kernel(const void* __restrict__ logits, const float* __restrict__ bias,
                                                                          ScoreArgs a, int32_t* __restrict__ ids_out,
                                                                          float* __restrict__ w_out) {
  __shared__ double cs[kScoreWaves][NJ * kWave];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int t = blockIdx.x * kScoreWaves + wave;
  if (t >= a.T) return;   // whole wave; no workgroup barrier follows
  const double ninf = -__builtin_inf();
  const int e0 = lane * NJ;
  float l[NJ], b[NJ];
  double s[NJ], c[NJ];
  load_lane<LDT, NJ>(logits, bias, a, a.wide, t, e0, l, b);
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) s[j] = sigmoid(l[j]);
  } else {
    float m = l[0];
#pragma unroll
    for (int j = 1; j < NJ; ++j) m = larger(m, l[j]);   // drops NaN, which shows in the scores
    m = wave_max(m);
    if (m == -__builtin_inff()) m = 0.0f;   // every expert masked
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      s[j] = exp_neg((double)l[j] - (double)m);
      sum += s[j];
    }
    sum = wave_sum(sum);
    const double inv = reciprocal(sum);   // 1 <= sum <= E; a sum of 0: every score is 0, and every expert masked
#pragma unroll
    for (int j = 0; j < NJ; ++j) s[j] = sum == 0.0 ? 0.0 : s[j] * inv;
  }
  bool nan = false;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    c[j] = s[j] + (double)b[j];
    nan |= c[j] != c[j];
    if (l[j] == -__builtin_inff()) c[j] = ninf;   // masked, or past E
  }
  int32_t* io = ids_out + (size_t)t * a.K;
  float* wo = w_out + (size_t)t * a.K;
  if (__ballot(nan)) {   // uniform: what the layer makes of this token is NaN
    if (lane < a.K) {
      io[lane] = lane;
      wo[lane] = __uint_as_float(0x7fc00000u);
    }
    return;
  }
  if (a.topk_group < a.n_group) {   // uniform
    const int gs = a.E / a.n_group;
    if (a.group_lanes) {
      // a group is 1, 2, 4, 8 or 16 whole lanes of a row
      Top2 x = {c[0], ninf};
#pragma unroll
      for (int j = 1; j < NJ; ++j) merge(x, c[j], ninf);
      if (a.group_lanes > 1) merge(x, dpp<kXor1>(x.a), dpp<kXor1>(x.b));
      if (a.group_lanes > 2) merge(x, dpp<kXor2>(x.a), dpp<kXor2>(x.b));
      if (a.group_lanes > 4) merge(x, dpp<kHalfMirror>(x.a), dpp<kHalfMirror>(x.b));
      if (a.group_lanes > 8) merge(x, dpp<kMirror>(x.a), dpp<kMirror>(x.b));
      const double g = a.group_top == 1 || x.b == ninf ? x.a : x.a + x.b;
      const int mine = lane / a.group_lanes;
      int ahead = 0;   // groups that come before this lane's
      for (int i = 0; i < a.n_group; ++i) {
        const double o = lane_value(g, i * a.group_lanes);
        ahead += o > g || (o == g && i < mine);
      }
      if (ahead >= a.topk_group)
#pragma unroll
        for (int j = 0; j < NJ; ++j) c[j] = ninf;
    } else {
      // any other size: a lane goes through its group in LDS
      double* cw = cs[wave];
#pragma unroll
      for (int j = 0; j < NJ; ++j) cw[e0 + j] = c[j];
      __builtin_amdgcn_wave_barrier();
      Top2 x = {ninf, ninf};
      if (lane < a.n_group)
        for (int i = 0; i < gs; ++i) merge(x, cw[lane * gs + i], ninf);
      const double g = a.group_top == 1 || x.b == ninf ? x.a : x.a + x.b;
      int ahead = 0;
      for (int i = 0; i < a.n_group; ++i) {
        const double o = lane_value(g, i);
        ahead += o > g || (o == g && i < lane);
      }
      const uint64_t open = __ballot(lane < a.n_group && ahead < a.topk_group);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        if (e0 + j < a.E && !((open >> ((e0 + j) / gs)) & 1)) c[j] = ninf;
    }
  }
  float f[NJ];   // the choices left, rounded to fp32
#pragma unroll
  for (int j = 0; j < NJ; ++j) f[j] = (float)c[j];
  int myid = -1;
  for (int k = 0; k < a.K; ++k) {
    float m = f[0];
#pragma unroll
    for (int j = 1; j < NJ; ++j) m = larger(m, f[j]);
    m = wave_max(m);
    if (m == -__builtin_inff()) break;   // uniform: only masked experts are left
    int reach = 0, id = 0;               // experts that reach it, and the (one) expert
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const uint64_t at = __ballot(f[j] == m);
      reach += __popcll(at);
      if (at) id = (__ffsll((long long)at) - 1) * NJ + j;   // uniform
    }
    if (reach > 1) {   // uniform: the 64-bit choices decide, then the lower expert
      double top = ninf;
#pragma unroll
      for (int j = 0; j < NJ; ++j) top = f[j] == m ? larger(top, c[j]) : top;
      top = wave_max(top);
      id = kScoreMaxE;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const uint64_t at = __ballot(f[j] == m && c[j] == top);
        const int lo = at ? (__ffsll((long long)at) - 1) * NJ + j : kScoreMaxE;
        id = lo < id ? lo : id;
      }
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if (e0 + j == id) f[j] = -__builtin_inff();
    if (lane == k) myid = id;
  }
  // lane k fetches the score of pick k
  double mys = 0.0;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int from = myid < 0 ? 0 : myid / NJ;
    const double v = __hiloint2double(__shfl(__double2hiint(s[j]), from), __shfl(__double2loint(s[j]), from));
    if (myid >= 0 && myid % NJ == j) mys = v;
  }
  const double sum = wave_sum(lane < a.K ? mys : 0.0);
  if (a.renorm) mys = sum > 0.0 ? mys / sum : 0.0;
  if (lane < a.K) {
    io[lane] = myid;
    wo[lane] = (float)(mys * a.scale);
  }
}

// Many tokens: a row of 16 lanes per token, so that a step of a reduction
// serves four.  Lane l holds experts l NJ .. l NJ + NJ - 1; K <= 16, lane k
// keeps pick k, groups are whole lanes, and rows load in pieces (element by
// element the E = 256 case below takes 22 us).  Scores are summed in the
// order of the other kernel: the same bits.
//
// Bound by vector issue, about half of it the scores, half the picks:
// T = 16384 E = 256 top-8 bf16 in 8 groups 15.4 us a call (17.1 traced by
// itself; reading its 8 MB: 2 us).
//
// Choices are compared as integers that order like their fp32 roundings; 0
// is one that is taken.
constexpr uint32_t kKeyMasked = 0x007fffffu;   // minus infinity
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

template <int LDT, int NJ>   // NJ = 4, 8 or 16: ceil(E / 16) rounded up
__global__ __launch_bounds__(kScoreWaves * kWave) void topk_scores_rows_kernel(const void* __restrict__ logits, const float* __restrict__ bias,
                                                                               ScoreArgs a, int32_t* __restrict__ ids_out,
                                                                               float* __restrict__ w_out) {
  __shared__ double ss[kScoreWaves * 4][NJ * 16];   // scores [token][j][lane]
  const int row = threadIdx.x >> 4, lane = threadIdx.x & 15, shift = threadIdx.x & 48;
  const int t = blockIdx.x * (kScoreWaves * 4) + row, tc = min(t, a.T - 1);
  const double ninf = -__builtin_inf();
  const int e0 = lane * NJ;
  auto of_row = [&](bool p) { return (uint32_t)(__ballot(p) >> shift) & 0xffffu; };   // p over the token's lanes
  float l[NJ], b[NJ];
  load_lane<LDT, NJ>(logits, bias, a, true, tc, e0, l, b);
  double s[NJ], c[NJ];
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) s[j] = sigmoid(l[j]);
  } else {
    float m = l[0];
#pragma unroll
    for (int j = 1; j < NJ; ++j) m = larger(m, l[j]);
    m = row_max(m);
    if (m == -__builtin_inff()) m = 0.0f;
    double part[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      part[p] = 0.0;
#pragma unroll
      for (int j = p * (NJ / 4); j < (p + 1) * (NJ / 4); ++j) {
        s[j] = exp_neg((double)l[j] - (double)m);
        part[p] += s[j];
      }
    }
    const double sum = row_sum((part[0] + part[1]) + (part[2] + part[3])), inv = reciprocal(sum);
#pragma unroll
    for (int j = 0; j < NJ; ++j) s[j] = sum == 0.0 ? 0.0 : s[j] * inv;
  }
  bool nan = false;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    ss[row][16 * j + lane] = s[j];
    c[j] = s[j] + (double)b[j];
    nan |= c[j] != c[j];
    if (l[j] == -__builtin_inff()) c[j] = ninf;
  }
  nan = of_row(nan) != 0;
  if (a.topk_group < a.n_group) {   // uniform; a.group_lanes lanes a group
    Top2 x = {c[0], ninf};
#pragma unroll
    for (int j = 1; j < NJ; ++j) merge(x, c[j], ninf);
    if (a.group_lanes > 1) merge(x, dpp<kXor1>(x.a), dpp<kXor1>(x.b));
    if (a.group_lanes > 2) merge(x, dpp<kXor2>(x.a), dpp<kXor2>(x.b));
    if (a.group_lanes > 4) merge(x, dpp<kHalfMirror>(x.a), dpp<kHalfMirror>(x.b));
    if (a.group_lanes > 8) merge(x, dpp<kMirror>(x.a), dpp<kMirror>(x.b));
    const double g = a.group_top == 1 || x.b == ninf ? x.a : x.a + x.b;
    const int mine = lane / a.group_lanes;
    int ahead = 0;
    for (int i = 0; i < a.n_group; ++i) {
      const int from = shift + i * a.group_lanes;
      const double o = __hiloint2double(__shfl(__double2hiint(g), from), __shfl(__double2loint(g), from));
      ahead += o > g || (o == g && i < mine);
    }
    if (ahead >= a.topk_group)
#pragma unroll
      for (int j = 0; j < NJ; ++j) c[j] = ninf;
  }
  uint32_t f[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) f[j] = order_key((float)c[j]);
  int myid = -1;
  for (int k = 0; k < a.K; ++k) {
    uint32_t m = f[0];
#pragma unroll
    for (int j = 1; j < NJ; ++j) m = larger(m, f[j]);
    m = row_max(m);
    const bool left = m > kKeyMasked;   // of the token: an expert to pick
    uint32_t at = 0;                    // bit j: expert j of the lane reaches the maximum
#pragma unroll
    for (int j = NJ - 1; j >= 0; --j) {
      at = at + at + (f[j] == m);
      f[j] = f[j] == m ? 0u : f[j];
    }
    const uint32_t where = of_row(at != 0);
    const bool several = ((at & (at - 1)) | (where & (where - 1))) != 0;
    if (__ballot(left & several)) {   // uniform: the 64-bit choices decide, then the lower expert
      double top = ninf;
#pragma unroll
      for (int j = 0; j < NJ; ++j) top = (at >> j) & 1 ? larger(top, c[j]) : top;
      top = row_max(top);
      uint32_t best = 0;
#pragma unroll
      for (int j = NJ - 1; j >= 0; --j) best = best + best + (((at >> j) & 1) && c[j] == top);
      const int first = __ffs((int)of_row(best != 0)) - 1;   // lane
      const uint32_t pick = lane == first ? best & (0u - best) : 0u;
#pragma unroll
      for (int j = 0; j < NJ; ++j) f[j] = ((at & ~pick) >> j) & 1 ? m : f[j];   // the others come back
      at = pick;
    }
    const uint32_t id1 = row_max(at ? (uint32_t)(e0 + __ffs((int)at)) : 0u);   // of the one lane that has it
    if (lane == k) myid = left ? (int)id1 - 1 : -1;
  }
  __builtin_amdgcn_wave_barrier();   // a token's scores are its own wave's
  double mys = myid < 0 ? 0.0 : ss[row][16 * (myid % NJ) + myid / NJ];
  const double sum = row_sum(mys);
  if (a.renorm) mys = sum > 0.0 ? mys / sum : 0.0;
  if (t < a.T && lane < a.K) {
    const size_t o = (size_t)t * a.K + lane;
    ids_out[o] = nan ? lane : myid;
    w_out[o] = nan ? __uint_as_float(0x7fc00000u) : (float)(mys * a.scale);
  }
}

template <int LDT>
void launch_rows_t(const void* logits, const float* bias, const ScoreArgs& a, int32_t* ids, float* w, hipStream_t st) {
  const dim3 grid((a.T + kScoreWaves * 4 - 1) / (kScoreWaves * 4)), block(kScoreWaves * kWave);
  if (a.E <= 64) hipLaunchKernelGGL((topk_scores_rows_kernel<LDT, 4>), grid, block, 0, st, logits, bias, a, ids, w);
  else if (a.E <= 128) hipLaunchKernelGGL((topk_scores_rows_kernel<LDT, 8>), grid, block, 0, st, logits, bias, a, ids, w);
  else hipLaunchKernelGGL((topk_scores_rows_kernel<LDT, 16>), grid, block, 0, st, logits, bias, a, ids, w);
}

template <int LDT>
void launch_t(const void* logits, const float* bias, const ScoreArgs& a, int32_t* ids, float* w, hipStream_t st) {
  const dim3 grid((a.T + kScoreWaves - 1) / kScoreWaves), block(kScoreWaves * kWave);
  if (a.E <= 64) hipLaunchKernelGGL((topk_scores_kernel<LDT, 1>), grid, block, 0, st, logits, bias, a, ids, w);
  else if (a.E <= 128) hipLaunchKernelGGL((topk_scores_kernel<LDT, 2>), grid, block, 0, st, logits, bias, a, ids, w);
  else if (a.E <= 256) hipLaunchKernelGGL((topk_scores_kernel<LDT, 4>), grid, block, 0, st, logits, bias, a, ids, w);
  else hipLaunchKernelGGL((topk_scores_kernel<LDT, 8>), grid, block, 0, st, logits, bias, a, ids, w);
}

}  // namespace

hipError_t launch_topk_scores(const void* logits, int ldt, const float* bias, ScoreArgs a, int32_t* ids, float* w,
                              hipStream_t st) {
  if (a.T == 0) return hipSuccess;
  if (a.E > kScoreMaxE) return hipErrorInvalidValue;
  const int nj = a.E <= 64 ? 1 : a.E <= 128 ? 2 : a.E <= 256 ? 4 : 8, gs = a.E / a.n_group;
  auto lanes = [&](int per) {   // lanes of a group at per experts a lane, 0: not whole lanes of a row
    const int gl = gs / per;
    return gs % per == 0 && gl <= 16 && (gl & (gl - 1)) == 0 ? gl : 0;
  };
  auto wide = [&](int per) {   // whole pieces of load_run in every row and in the bias
    const int size = ldt == 2 ? 4 : 2, p = std::min(per, 16 / size);
    return a.E % p == 0 && (uintptr_t)logits % (p * size) == 0 && (uintptr_t)bias % (4 * std::min(per, 4)) == 0;
  };
  a.group_lanes = lanes(4 * nj);
  if (a.T >= kScoreRowsT && a.E <= 256 && a.K <= 16 && wide(4 * nj) && (a.topk_group == a.n_group || a.group_lanes)) {
    if (ldt == 2) launch_rows_t<2>(logits, bias, a, ids, w, st);
    else if (ldt == 1) launch_rows_t<1>(logits, bias, a, ids, w, st);
    else launch_rows_t<0>(logits, bias, a, ids, w, st);
    return hipGetLastError();
  }
  a.group_lanes = lanes(nj);
  a.wide = wide(nj);
  if (ldt == 2) launch_t<2>(logits, bias, a, ids, w, st);
  else if (ldt == 1) launch_t<1>(logits, bias, a, ids, w, st);
  else launch_t<0>(logits, bias, a, ids, w, st);
  return hipGetLastError();
}

}  // namespace mimoe
