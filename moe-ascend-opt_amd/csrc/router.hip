// router.hip -- routing to experts by scores: softmax or sigmoid of the
// logits, a bias that only decides the choice, expert groups, top-k,
// renormalized and scaled weights.
//
//   s_e = sigmoid(l_e) or softmax(l)_e,  c_e = s_e + b_e
//   group score = the sum of the group's group_top largest c (1 or 2)
//   the topk_group groups of the largest scores, in them the K largest c
//   w_k = scale * s_k / sum of the picks' s  (renormalize), or scale * s_k
//
// Ties go to the lower group and the lower expert.  Scores are computed in 64
// bits: among some hundred experts two choices often lie within fp32's
// rounding of each other, and which expert is picked should follow from the
// logits, not from the order of a sum.
#include "mi_moe_device.hpp"
#include "mi_moe_internal.hpp"

namespace mimoe {

namespace {

constexpr int kScoreWaves = 4;
constexpr int kScoreMaxE = 512;
constexpr int kScoreMaxGroups = 64;

__device__ __forceinline__ double shfl_xor_f64(double v, int m) {
  const int lo = __shfl_xor(__double2loint(v), m), hi = __shfl_xor(__double2hiint(v), m);
  return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double shfl_f64(double v, int l) {
  return __hiloint2double(__shfl(__double2hiint(v), l), __shfl(__double2loint(v), l));
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += shfl_xor_f64(v, m);
  return v;
}

// One wave per token; lane l holds experts l, l + 64, ...
template <int LDT, int NJ>   // logits: 0 fp16, 1 bf16, 2 fp32; NJ = ceil(E / 64)
__global__ __launch_bounds__(kScoreWaves * kWave) void topk_scores_kernel(const void* __restrict__ logits, const float* __restrict__ bias,
                                                                          ScoreArgs a, int32_t* __restrict__ ids_out,
                                                                          float* __restrict__ w_out) {
  __shared__ double cs[kScoreWaves][NJ * kWave];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int t = blockIdx.x * kScoreWaves + wave;
  if (t >= a.T) return;   // whole wave; no workgroup barrier follows
  const double ninf = -__builtin_inf();
  float l[NJ];
  double s[NJ], c[NJ];
  bool nan = false;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = lane + kWave * j;
    const size_t off = (size_t)t * a.E + (e < a.E ? e : a.E - 1);
    float v;
    if constexpr (LDT == 2) v = reinterpret_cast<const float*>(logits)[off];
    else v = to_f32<LDT>(reinterpret_cast<const uint16_t*>(logits)[off]);
    l[j] = e < a.E ? v : -__builtin_inff();
  }
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) s[j] = 1.0 / (1.0 + exp(-(double)l[j]));
  } else {
    float m = l[0];
#pragma unroll
    for (int j = 1; j < NJ; ++j) m = fmaxf(m, l[j]);
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (m == -__builtin_inff()) m = 0.0f;   // every expert masked
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      s[j] = exp((double)l[j] - (double)m);
      sum += s[j];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < NJ; ++j) s[j] = sum == 0.0 ? 0.0 : s[j] / sum;
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = lane + kWave * j;
    c[j] = bias && e < a.E ? s[j] + (double)bias[e] : s[j];
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
  if (a.topk_group < a.n_group) {
    const int gs = a.E / a.n_group;
    double* cw = cs[wave];
#pragma unroll
    for (int j = 0; j < NJ; ++j) cw[lane + kWave * j] = c[j];
    __builtin_amdgcn_wave_barrier();
    double b1 = ninf, b2 = ninf;   // the group's two largest
    if (lane < a.n_group)
      for (int i = 0; i < gs; ++i) {
        const double v = cw[lane * gs + i];
        if (v > b1) { b2 = b1; b1 = v; }
        else if (v > b2) b2 = v;
      }
    const double g = a.group_top == 1 ? b1 : b2 == ninf ? ninf : b1 + b2;
    int ahead = 0;   // groups that come before this lane's
    for (int i = 0; i < a.n_group; ++i) {
      const double o = shfl_f64(g, i);
      ahead += o > g || (o == g && i < lane);
    }
    const uint64_t open = __ballot(lane < a.n_group && ahead < a.topk_group);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int e = lane + kWave * j;
      if (e < a.E && !((open >> (e / gs)) & 1)) c[j] = ninf;
    }
  }
  double mys = 0.0;
  int myid = -1;
  for (int k = 0; k < a.K; ++k) {
    double bv = ninf, bs = 0.0;
    int bi = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if (c[j] > bv) { bv = c[j]; bs = s[j]; bi = lane + kWave * j; }
#pragma unroll
    for (int m = 32; m; m >>= 1) {
      const double ov = shfl_xor_f64(bv, m), os = shfl_xor_f64(bs, m);
      const int oi = __shfl_xor(bi, m);
      if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bs = os; bi = oi; }
    }
    if (bi == 0x7fffffff) break;   // uniform: only masked experts are left
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if (bi == lane + kWave * j) c[j] = ninf;
    if (lane == k) { mys = bs; myid = bi; }
  }
  const double sum = wave_sum(lane < a.K ? mys : 0.0);
  if (a.renorm) mys = sum > 0.0 ? mys / sum : 0.0;
  if (lane < a.K) {
    io[lane] = myid;
    wo[lane] = (float)(mys * a.scale);
  }
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

hipError_t launch_topk_scores(const void* logits, int ldt, const float* bias, const ScoreArgs& a, int32_t* ids, float* w,
                              hipStream_t st) {
  if (a.T == 0) return hipSuccess;
  if (ldt == 2) launch_t<2>(logits, bias, a, ids, w, st);
  else if (ldt == 1) launch_t<1>(logits, bias, a, ids, w, st);
  else launch_t<0>(logits, bias, a, ids, w, st);
  return hipGetLastError();
}

}  // namespace mimoe
