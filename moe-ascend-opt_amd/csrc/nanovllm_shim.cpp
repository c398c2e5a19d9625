// nanovllm_shim.cpp -- PyTorch-ROCm binding of libmimoe.so with the schema of
// the reference extension (Int8-gemm/nanovllm_ops.cpp:349-412):
//   torch.classes.nanovllm.MoEInfer(E, H, I, quant_type)
//   torch.ops.nanovllm.moe_forward(hidden, topk_ids, topk_w, moe) -> Tensor
// plus the build-defined W4A16 loader store_awq_repack, the out variant
// moe_forward_out, and the router step the reference runs in its Python
// harness (make_topk_from_logits_cpu, Int8-gemm/test/fused_moe_cpu.py:20-37)
// as moe_topk_softmax / moe_forward_logits, the score router as moe_topk_scores /
// moe_forward_scores, and the MX formats: store_mxfp4_repack, mx_quantize,
// mx_dequantize.  Only this file sees torch types; it calls the C ABI of
// include/mi_moe.h: HIP tensors run the device kernels on the current HIP stream; CPU tensors run the
// host engine (the reference's CPU algorithm for Q8_0 / Q4_0; every expert on the host executor for
// W4A16), which needs weights stored from host tensors (kept by default when no HIP device is present,
// or with MIMOE_HOST_WEIGHTS=1; never with MIMOE_HOST_WEIGHTS=0).
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/custom_class.h>
#include <tuple>
#include <optional>
#include <vector>
#include <torch/library.h>
#include <ATen/ATen.h>

#include <cstdlib>
#include <string>
#include <chrono>
#include <algorithm>
#include <cmath>

#include "mi_moe.h"

namespace {

void check_status(int rc, const char* what) {
  TORCH_CHECK(rc == MI_MOE_OK, what, ": ", mi_moe_last_error(), " (status ", rc, ")");
}

int act_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return MI_MOE_BF16;
  TORCH_CHECK(t.scalar_type() == at::kHalf, "expected float16 or bfloat16, got ", t.scalar_type());
  return MI_MOE_F16;
}

void* stream_of(const at::Tensor& ref) {
  if (ref.is_cuda()) return (void*)c10::hip::getCurrentHIPStream(ref.get_device()).stream();
  return (void*)c10::hip::getCurrentHIPStream().stream();
}

// The reference's CPU layout variables (Int8-gemm/moe_infer.cpp:25,
// Int8-gemm/numa_threadpool.h:498-504, README.md:179): -1 when unset.
int64_t env_int(const char* name) {
  const char* s = getenv(name);
  if (!s || !*s) return -1;
  char* end = nullptr;
  const long long v = strtoll(s, &end, 10);
  TORCH_CHECK(end && *end == '\0', name, "=", s, " is not an integer");
  return v;
}

// Host threads of the CPU path: MIMOE_CPU_THREADS, else OMP_NUM_THREADS, else
// every CPU of the affinity mask (0).
int host_threads() {
  for (const char* v : {"MIMOE_CPU_THREADS", "OMP_NUM_THREADS"}) {
    const char* s = getenv(v);
    if (s && atoi(s) > 0) return atoi(s);
  }
  return 0;
}

bool hip_device_present() {
  int n = 0;
  return hipGetDeviceCount(&n) == hipSuccess && n > 0;
}

struct MoEInferHandle : torch::CustomClassHolder {
  int64_t E, H, I, quant_type;
  mi_moe_handle* h = nullptr;      // device weights (when a HIP device is present)
  mi_moe_cpu* cpu = nullptr;       // host engine, Q8_0 / Q4_0
  mi_moe_hybrid* hcpu = nullptr;   // W4A16 with every expert on the host executor
  bool keep_host = false;          // weights stored from host tensors also fill the host path
  bool last_cpu = false;           // the last forward ran on the host
  double last_cpu_ms = -1.0;

  // Int8-gemm/nanovllm_ops.cpp:28-30 (quant_type: 0 Q8_0, 1 Q4_0; 2 W4A16, 3 MXFP4)
  MoEInferHandle(int64_t E_, int64_t H_, int64_t I_, int64_t qt) : E(E_), H(H_), I(I_), quant_type(qt) {
    TORCH_CHECK(qt >= 0 && qt <= 3, "quant_type must be 0 (Q8_0), 1 (Q4_0), 2 (W4A16) or 3 (MXFP4)");
    const bool dev = hip_device_present();
    TORCH_CHECK(dev || qt != 3, "MoEInfer: MXFP4 layers need a HIP device");
    if (dev) check_status(mi_moe_create(E, H, I, (int)qt, &h), "MoEInfer");
    const char* kh = getenv("MIMOE_HOST_WEIGHTS");
    keep_host = kh ? atoi(kh) != 0 : !dev;
    if (qt == 3) keep_host = false;   // the host engines have no MXFP4
    else if (!dev) TORCH_CHECK(keep_host, "MoEInfer: no HIP device and MIMOE_HOST_WEIGHTS=0: nowhere to keep the weights");
  }
  ~MoEInferHandle() override {
    if (h) mi_moe_destroy(h);
    if (cpu) mi_moe_cpu_destroy(cpu);
    if (hcpu) mi_moe_hybrid_destroy(hcpu);
  }
  std::string get_quant_type() const {
    return quant_type == 1 ? "Q4_0" : quant_type == 2 ? "W4A16" : quant_type == 3 ? "MXFP4" : "Q8_0";
  }
  int64_t info(int which) const { return which == 0 ? E : (which == 1 ? H : I); }
  mi_moe_handle* dev() const {
    TORCH_CHECK(h != nullptr, "MoEInfer: no HIP device for this call");
    return h;
  }
  // NANOVLLM_TP_SIZE / NANOVLLM_TP_THREADS_PER_NODE, when set, give the
  // reference's layout: tp shards over NUMA nodes, that many threads per node
  // (the reference's default tp of 2 fails on one-node hosts, so unset means
  // one shard per NUMA node here); otherwise MIMOE_CPU_THREADS /
  // OMP_NUM_THREADS threads over whole nodes.
  mi_moe_cpu* host_engine() {
    if (!cpu) {
      const int64_t tp = env_int("NANOVLLM_TP_SIZE"), per = env_int("NANOVLLM_TP_THREADS_PER_NODE");
      if (tp >= 0 || per >= 0) {
        TORCH_CHECK(tp != 0 && tp < 0x10000, "tp_size must be >= 1 (NANOVLLM_TP_SIZE=", tp, ")");
        check_status(mi_moe_cpu_create_numa(E, H, I, (int)quant_type, tp > 0 ? (int)tp : 0,
                                            per > 0 ? (int)std::min<int64_t>(per, 1 << 20) : 0, &cpu),
                     "MoEInfer (host)");
      } else {
        check_status(mi_moe_cpu_create(E, H, I, (int)quant_type, host_threads(), 0, &cpu), "MoEInfer (host)");
      }
    }
    return cpu;
  }
  mi_moe_hybrid* host_w4() {
    if (!hcpu) {
      std::vector<uint8_t> all((size_t)E, 1);
      check_status(mi_moe_hybrid_create(E, H, I, MI_MOE_W4A16, all.data(), std::min(host_threads(), 16), &hcpu),
                   "MoEInfer (host)");
    }
    return hcpu;
  }
};

at::Tensor contig(const at::Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }

void check_forward_tensors(const at::Tensor& hidden, const at::Tensor& topk_ids, const at::Tensor& topk_w,
                           const c10::intrusive_ptr<MoEInferHandle>& moe, const at::Tensor& out) {
  TORCH_CHECK(hidden.dim() == 2 && topk_ids.dim() == 2 && topk_w.dim() == 2,
              "moe_forward: expected hidden [T,H], topk_ids [T,K], topk_w [T,K]");
  TORCH_CHECK(topk_ids.scalar_type() == at::kInt, "topk_ids must be int32");
  TORCH_CHECK(topk_w.scalar_type() == at::kFloat, "topk_w must be float32");
  TORCH_CHECK(topk_ids.size(0) == hidden.size(0) && topk_w.size(0) == hidden.size(0) &&
                  topk_w.size(1) == topk_ids.size(1),
              "moe_forward: token / top_k dimensions disagree");
  TORCH_CHECK(hidden.size(1) == moe->info(1), "hidden size ", hidden.size(1), " != handle H ",
              moe->info(1));
  TORCH_CHECK(topk_ids.device() == hidden.device() && topk_w.device() == hidden.device() &&
                  out.device() == hidden.device(),
              "all tensors must be on the same device");
  TORCH_CHECK(out.sizes() == hidden.sizes() && out.scalar_type() == hidden.scalar_type() &&
                  out.is_contiguous(),
              "out must be a contiguous tensor like hidden");
}

void forward_into(const at::Tensor& hidden, const at::Tensor& topk_ids, const at::Tensor& topk_w,
                  const c10::intrusive_ptr<MoEInferHandle>& moe, at::Tensor& out) {
  TORCH_CHECK(hidden.is_cuda(), "moe_forward: expected HIP tensors here");
  check_forward_tensors(hidden, topk_ids, topk_w, moe, out);
  at::Tensor x = contig(hidden), ids = contig(topk_ids), w = contig(topk_w);
  check_status(mi_moe_forward(moe->dev(), x.data_ptr(), out.data_ptr(), w.data_ptr<float>(),
                              ids.data_ptr<int32_t>(), x.size(0), ids.size(1), act_code(x),
                              stream_of(x)),
               "moe_forward");
  moe->last_cpu = false;
}

// The CPU key: the host engine (Q8_0 / Q4_0: the reference algorithm,
// Int8-gemm/nanovllm_ops.cpp:219-236 -> moe_infer.cpp:430-456) or, for W4A16,
// every expert on the host executor.
void forward_into_cpu(const at::Tensor& hidden, const at::Tensor& topk_ids, const at::Tensor& topk_w,
                      const c10::intrusive_ptr<MoEInferHandle>& moe, at::Tensor& out) {
  check_forward_tensors(hidden, topk_ids, topk_w, moe, out);
  TORCH_CHECK(moe->quant_type != 3, "moe_forward (CPU): MXFP4 layers run on HIP tensors only");
  at::Tensor x = contig(hidden), ids = contig(topk_ids), w = contig(topk_w);
  const int64_t T = x.size(0), K = ids.size(1);
  if (moe->quant_type == 2) {
    TORCH_CHECK(moe->hcpu != nullptr, "moe_forward (CPU): no host weights; store the weights from host tensors "
                "(with MIMOE_HOST_WEIGHTS=1 where a HIP device is present)");
    at::Tensor part = at::empty({T, moe->H}, x.options().dtype(at::kFloat));
    const auto t0 = std::chrono::steady_clock::now();
    check_status(mi_moe_hybrid_host_forward(moe->hcpu, x.data_ptr(), w.data_ptr<float>(), ids.data_ptr<int32_t>(),
                                            T, K, act_code(x), part.data_ptr<float>()),
                 "moe_forward (CPU)");
    out.copy_(part);   // fp32 -> the hidden dtype, round to nearest even
    moe->last_cpu_ms = std::chrono::duration<double, std::milli>(std::chrono::steady_clock::now() - t0).count();
  } else {
    TORCH_CHECK(moe->cpu != nullptr, "moe_forward (CPU): no host weights; store the weights from host tensors "
                "(with MIMOE_HOST_WEIGHTS=1 where a HIP device is present)");
    check_status(mi_moe_cpu_forward(moe->cpu, x.data_ptr(), out.data_ptr(), w.data_ptr<float>(),
                                    ids.data_ptr<int32_t>(), T, K, act_code(x)),
                 "moe_forward (CPU)");
    double ms = -1.0;
    check_status(mi_moe_cpu_get_info(moe->cpu, nullptr, nullptr, nullptr, nullptr, nullptr, &ms), "get_info");
    moe->last_cpu_ms = ms;
  }
  moe->last_cpu = true;
}

// Int8-gemm/nanovllm_ops.cpp:219-236
at::Tensor moe_forward_hip(const at::Tensor& hidden, const at::Tensor& topk_ids,
                           const at::Tensor& topk_w,
                           const c10::intrusive_ptr<MoEInferHandle>& moe) {
  at::Tensor out = at::empty_like(hidden, hidden.options().memory_format(at::MemoryFormat::Contiguous));
  forward_into(hidden, topk_ids, topk_w, moe, out);
  return out;
}

// Int8-gemm/nanovllm_ops.cpp:219-236 (CPU key, :410-412)
at::Tensor moe_forward_cpu(const at::Tensor& hidden, const at::Tensor& topk_ids, const at::Tensor& topk_w,
                           const c10::intrusive_ptr<MoEInferHandle>& moe) {
  at::Tensor out = at::empty_like(hidden, hidden.options().memory_format(at::MemoryFormat::Contiguous));
  forward_into_cpu(hidden, topk_ids, topk_w, moe, out);
  return out;
}

void moe_forward_out_cpu(const at::Tensor& hidden, const at::Tensor& topk_ids, const at::Tensor& topk_w,
                         const c10::intrusive_ptr<MoEInferHandle>& moe, at::Tensor out) {
  forward_into_cpu(hidden, topk_ids, topk_w, moe, out);
}

void moe_forward_out_hip(const at::Tensor& hidden, const at::Tensor& topk_ids,
                         const at::Tensor& topk_w, const c10::intrusive_ptr<MoEInferHandle>& moe,
                         at::Tensor out) {
  forward_into(hidden, topk_ids, topk_w, moe, out);
}

int logits_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kFloat) return MI_MOE_F32;
  if (t.scalar_type() == at::kBFloat16) return MI_MOE_BF16;
  TORCH_CHECK(t.scalar_type() == at::kHalf, "router logits must be float32, bfloat16 or float16");
  return MI_MOE_F16;
}

std::tuple<at::Tensor, at::Tensor> moe_topk_softmax_hip(const at::Tensor& logits, int64_t top_k,
                                                        bool renormalize) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "moe_topk_softmax: logits must be a [T,E] HIP tensor");
  at::Tensor x = contig(logits);
  const int64_t T = x.size(0), E = x.size(1);
  at::Tensor ids = at::empty({T, top_k}, x.options().dtype(at::kInt));
  at::Tensor w = at::empty({T, top_k}, x.options().dtype(at::kFloat));
  check_status(mi_moe_topk_softmax(x.data_ptr(), logits_code(x), T, E, top_k, renormalize ? 1 : 0,
                                   ids.data_ptr<int32_t>(), w.data_ptr<float>(), stream_of(x)),
               "moe_topk_softmax");
  return {ids, w};
}

// Router top-k + softmax on host tensors, the semantics of the device kernel
// (make_topk_from_logits_cpu, Int8-gemm/test/fused_moe_cpu.py:20-37): the K
// largest logits in descending order, equal logits lower expert id first,
// softmax over the K values (renormalize) or the full softmax gathered.
std::tuple<at::Tensor, at::Tensor> moe_topk_softmax_cpu(const at::Tensor& logits, int64_t top_k, bool renormalize) {
  TORCH_CHECK(logits.dim() == 2, "moe_topk_softmax: logits must be [T,E]");
  at::Tensor x = contig(logits).to(at::kFloat);
  const int64_t T = x.size(0), E = x.size(1);
  TORCH_CHECK(top_k >= 1 && top_k <= E && top_k <= 64, "top_k=", top_k, " must be in [1, min(E, 64)]");
  at::Tensor ids = at::empty({T, top_k}, x.options().dtype(at::kInt));
  at::Tensor w = at::empty({T, top_k}, x.options().dtype(at::kFloat));
  const float* g = x.data_ptr<float>();
  int32_t* oi = ids.data_ptr<int32_t>();
  float* ow = w.data_ptr<float>();
  check_status(mi_moe_cpu_topk_softmax(g, T, E, top_k, renormalize ? 1 : 0, oi, ow), "moe_topk_softmax");
  return {ids, w};
}

at::Tensor moe_forward_logits_hip(const at::Tensor& hidden, const at::Tensor& router_logits, int64_t top_k,
                                  bool renormalize, const c10::intrusive_ptr<MoEInferHandle>& moe) {
  TORCH_CHECK(hidden.is_cuda() && router_logits.is_cuda() && hidden.device() == router_logits.device(),
              "moe_forward_logits: hidden and router_logits must be HIP tensors on one device");
  TORCH_CHECK(hidden.dim() == 2 && router_logits.dim() == 2 && router_logits.size(0) == hidden.size(0),
              "moe_forward_logits: expected hidden [T,H], router_logits [T,E]");
  TORCH_CHECK(router_logits.size(1) == moe->info(0), "router_logits has ", router_logits.size(1),
              " experts, handle has ", moe->info(0));
  TORCH_CHECK(hidden.size(1) == moe->info(1), "hidden size ", hidden.size(1), " != handle H ", moe->info(1));
  at::Tensor x = contig(hidden), g = contig(router_logits);
  at::Tensor out = at::empty_like(x);
  check_status(mi_moe_forward_logits(moe->dev(), x.data_ptr(), out.data_ptr(), g.data_ptr(), logits_code(g),
                                     x.size(0), top_k, renormalize ? 1 : 0, act_code(x), nullptr, nullptr,
                                     stream_of(x)),
               "moe_forward_logits");
  moe->last_cpu = false;
  return out;
}

at::Tensor moe_forward_logits_cpu(const at::Tensor& hidden, const at::Tensor& router_logits, int64_t top_k,
                                  bool renormalize, const c10::intrusive_ptr<MoEInferHandle>& moe) {
  TORCH_CHECK(hidden.dim() == 2 && router_logits.dim() == 2 && router_logits.size(0) == hidden.size(0),
              "moe_forward_logits: expected hidden [T,H], router_logits [T,E]");
  TORCH_CHECK(router_logits.size(1) == moe->info(0), "router_logits has ", router_logits.size(1),
              " experts, handle has ", moe->info(0));
  auto picks = moe_topk_softmax_cpu(router_logits, top_k, renormalize);
  return moe_forward_cpu(hidden, std::get<0>(picks), std::get<1>(picks), moe);
}

// Score router: arguments as mi_moe_topk_scores, score "softmax" or "sigmoid".
int score_code(c10::string_view s) {
  TORCH_CHECK(s == "softmax" || s == "sigmoid", "score must be 'softmax' or 'sigmoid', got '", s, "'");
  return s == "sigmoid" ? MI_MOE_SCORE_SIGMOID : MI_MOE_SCORE_SOFTMAX;
}

// The selection bias as fp32 [E] beside the logits (an undefined tensor: none).
at::Tensor score_bias(const std::optional<at::Tensor>& bias, const at::Tensor& logits) {
  if (!bias.has_value() || !bias->defined()) return at::Tensor();
  TORCH_CHECK(bias->dim() == 1 && bias->size(0) == logits.size(1) && bias->scalar_type() == at::kFloat,
              "bias must be a float32 [E] tensor");
  TORCH_CHECK(bias->device() == logits.device(), "bias and logits must be on one device");
  return contig(*bias);
}

void check_scores(const at::Tensor& logits, int64_t top_k) {
  TORCH_CHECK(logits.dim() == 2, "router logits must be [T,E]");
  TORCH_CHECK(top_k >= 1 && top_k <= 64, "top_k=", top_k, " must be in [1, 64]");
}

std::tuple<at::Tensor, at::Tensor> moe_topk_scores_hip(const at::Tensor& logits, int64_t top_k,
                                                       const std::optional<at::Tensor>& bias, c10::string_view score,
                                                       int64_t n_group, int64_t topk_group, int64_t group_top,
                                                       bool renormalize, double scale) {
  check_scores(logits, top_k);
  TORCH_CHECK(logits.is_cuda(), "moe_topk_scores: bias and logits must be on one device");
  c10::hip::HIPGuard guard(logits.get_device());
  at::Tensor x = contig(logits), b = score_bias(bias, logits);
  const int64_t T = x.size(0), E = x.size(1);
  at::Tensor ids = at::empty({T, top_k}, x.options().dtype(at::kInt));
  at::Tensor w = at::empty({T, top_k}, x.options().dtype(at::kFloat));
  check_status(mi_moe_topk_scores(x.data_ptr(), logits_code(x), T, E, top_k, b.defined() ? b.data_ptr<float>() : nullptr,
                                  score_code(score), n_group, topk_group, group_top, renormalize ? 1 : 0, (float)scale,
                                  ids.data_ptr<int32_t>(), w.data_ptr<float>(), stream_of(x)),
               "moe_topk_scores");
  return {ids, w};
}

std::tuple<at::Tensor, at::Tensor> moe_topk_scores_cpu(const at::Tensor& logits, int64_t top_k,
                                                       const std::optional<at::Tensor>& bias, c10::string_view score,
                                                       int64_t n_group, int64_t topk_group, int64_t group_top,
                                                       bool renormalize, double scale) {
  check_scores(logits, top_k);
  logits_code(logits);
  at::Tensor x = contig(logits).to(at::kFloat), b = score_bias(bias, logits);
  const int64_t T = x.size(0), E = x.size(1);
  at::Tensor ids = at::empty({T, top_k}, x.options().dtype(at::kInt));
  at::Tensor w = at::empty({T, top_k}, x.options().dtype(at::kFloat));
  check_status(mi_moe_cpu_topk_scores(x.data_ptr<float>(), T, E, top_k, b.defined() ? b.data_ptr<float>() : nullptr,
                                      score_code(score), n_group, topk_group, group_top, renormalize ? 1 : 0, (float)scale,
                                      ids.data_ptr<int32_t>(), w.data_ptr<float>()),
               "moe_topk_scores");
  return {ids, w};
}

at::Tensor moe_forward_scores_hip(const at::Tensor& hidden, const at::Tensor& router_logits, int64_t top_k,
                                  const std::optional<at::Tensor>& bias, c10::string_view score, int64_t n_group,
                                  int64_t topk_group, int64_t group_top, bool renormalize, double scale,
                                  const c10::intrusive_ptr<MoEInferHandle>& moe) {
  check_scores(router_logits, top_k);
  TORCH_CHECK(hidden.is_cuda() && router_logits.is_cuda() && hidden.device() == router_logits.device(),
              "moe_forward_scores: hidden and router_logits must be HIP tensors on one device");
  TORCH_CHECK(hidden.dim() == 2 && router_logits.size(0) == hidden.size(0),
              "moe_forward_scores: expected hidden [T,H], router_logits [T,E]");
  TORCH_CHECK(router_logits.size(1) == moe->info(0), "router_logits has ", router_logits.size(1),
              " experts, handle has ", moe->info(0));
  TORCH_CHECK(hidden.size(1) == moe->info(1), "hidden size ", hidden.size(1), " != handle H ", moe->info(1));
  c10::hip::HIPGuard guard(hidden.get_device());
  at::Tensor x = contig(hidden), g = contig(router_logits), b = score_bias(bias, router_logits);
  at::Tensor out = at::empty_like(x);
  check_status(mi_moe_forward_scores(moe->dev(), x.data_ptr(), out.data_ptr(), g.data_ptr(), logits_code(g), x.size(0),
                                     top_k, b.defined() ? b.data_ptr<float>() : nullptr, score_code(score), n_group,
                                     topk_group, group_top, renormalize ? 1 : 0, (float)scale, act_code(x), nullptr, nullptr,
                                     stream_of(x)),
               "moe_forward_scores");
  moe->last_cpu = false;
  return out;
}

at::Tensor moe_forward_scores_cpu(const at::Tensor& hidden, const at::Tensor& router_logits, int64_t top_k,
                                  const std::optional<at::Tensor>& bias, c10::string_view score, int64_t n_group,
                                  int64_t topk_group, int64_t group_top, bool renormalize, double scale,
                                  const c10::intrusive_ptr<MoEInferHandle>& moe) {
  check_scores(router_logits, top_k);
  TORCH_CHECK(hidden.dim() == 2 && router_logits.size(0) == hidden.size(0),
              "moe_forward_scores: expected hidden [T,H], router_logits [T,E]");
  TORCH_CHECK(router_logits.size(1) == moe->info(0), "router_logits has ", router_logits.size(1),
              " experts, handle has ", moe->info(0));
  auto picks = moe_topk_scores_cpu(router_logits, top_k, bias, score, n_group, topk_group, group_top, renormalize, scale);
  return moe_forward_cpu(hidden, std::get<0>(picks), std::get<1>(picks), moe);
}

// MX block formats: "mxfp4" (E2M1) or "mxfp6" (E2M3), see mi_moe_mx_quantize.
int mx_format(c10::string_view f) {
  TORCH_CHECK(f == "mxfp4" || f == "mxfp6", "format must be 'mxfp4' or 'mxfp6', got '", f, "'");
  return f == "mxfp4" ? MI_MOE_MX_FP4 : MI_MOE_MX_FP6;
}
int64_t mx_block(int fmt) { return fmt == MI_MOE_MX_FP4 ? 16 : 24; }

int mx_value_code(at::ScalarType t) {
  if (t == at::kFloat) return MI_MOE_F32;
  if (t == at::kBFloat16) return MI_MOE_BF16;
  TORCH_CHECK(t == at::kHalf, "values must be float32, bfloat16 or float16, got ", t);
  return MI_MOE_F16;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// x [..., C] -> codes uint8 [..., C/2] (mxfp4) or [..., C/32*24] (mxfp6),
// scales uint8 [..., C/32].  A 2-D view whose rows are whole 16-byte pieces
// apart is read in place, any other layout is copied first.
std::tuple<at::Tensor, at::Tensor> mx_quantize_hip(const at::Tensor& x, c10::string_view format) {
  const int fmt = mx_format(format), dt = mx_value_code(x.scalar_type());
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) % 32 == 0,
              "mx_quantize: the last dimension must be a positive multiple of 32");
  c10::hip::HIPGuard guard(x.get_device());
  const int64_t C = x.size(-1), rows = x.numel() / C, per16 = dt == MI_MOE_F32 ? 4 : 8;
  const bool in_place = aligned16(x.data_ptr()) &&
                        (x.is_contiguous() || (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= C && x.stride(0) % per16 == 0));
  at::Tensor v = in_place ? x : x.contiguous();
  if (!aligned16(v.data_ptr())) v = v.clone(at::MemoryFormat::Contiguous);
  std::vector<int64_t> cs = x.sizes().vec(), ss = cs;
  cs.back() = C / 32 * mx_block(fmt);
  ss.back() = C / 32;
  at::Tensor codes = at::empty(cs, x.options().dtype(at::kByte)), scales = at::empty(ss, x.options().dtype(at::kByte));
  check_status(mi_moe_mx_quantize(v.data_ptr(), dt, rows, C, v.is_contiguous() ? C : v.stride(0), fmt,
                                  codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), stream_of(x)),
               "mx_quantize");
  return {codes, scales};
}

at::Tensor mx_dequantize_hip(const at::Tensor& codes, const at::Tensor& scales, c10::string_view format, at::ScalarType dtype) {
  const int fmt = mx_format(format), dt = mx_value_code(dtype);
  TORCH_CHECK(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, "codes and scales must be uint8");
  TORCH_CHECK(scales.is_cuda() && scales.device() == codes.device(), "codes and scales must be on one device");
  TORCH_CHECK(codes.dim() >= 1 && codes.dim() == scales.dim() && scales.size(-1) > 0 &&
                  codes.size(-1) == scales.size(-1) * mx_block(fmt) &&
                  codes.sizes().slice(0, codes.dim() - 1) == scales.sizes().slice(0, scales.dim() - 1),
              "mx_dequantize: codes and scales do not belong together in format ", format);
  c10::hip::HIPGuard guard(codes.get_device());
  at::Tensor c = contig(codes), s = contig(scales);
  if (!aligned16(c.data_ptr())) c = c.clone(at::MemoryFormat::Contiguous);
  std::vector<int64_t> os = s.sizes().vec();
  const int64_t C = 32 * os.back(), rows = s.numel() / os.back();
  os.back() = C;
  at::Tensor out = at::empty(os, c.options().dtype(dtype));
  check_status(mi_moe_mx_dequantize(c.data_ptr<uint8_t>(), s.data_ptr<uint8_t>(), rows, C, fmt, out.data_ptr(), dt,
                                    stream_of(c)),
               "mx_dequantize");
  return out;
}

// ------------------------------------------------------------------ products on rows sorted by expert
// An operand of the products: rows of whole 16-byte pieces (`per16` elements).
// A view that has them is read in place; others are copied, with zeros behind
// the values of a row where its length is no multiple.
at::Tensor rows16(const at::Tensor& t, int64_t per16) {
  const int64_t d = t.dim(), n = t.size(-1);
  bool ok = t.stride(-1) == 1 && n % per16 == 0 && aligned16(t.data_ptr());
  if (t.size(d - 2) > 1) ok = ok && t.stride(d - 2) >= n && t.stride(d - 2) % per16 == 0 && t.stride(d - 2) <= (1 << 22);
  if (d == 3 && t.size(0) > 1) ok = ok && t.stride(0) >= 0 && t.stride(0) % per16 == 0;
  if (ok) return t;
  if (n % per16) return at::constant_pad_nd(t, {0, per16 - n % per16}).contiguous();
  return t.is_contiguous() ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous();
}
int64_t row_stride(const at::Tensor& t) { return t.size(t.dim() - 2) > 1 ? t.stride(t.dim() - 2) : t.size(-1); }
int64_t expert_stride(const at::Tensor& w) { return w.size(0) > 1 ? w.stride(0) : 0; }

void check_starts(const at::Tensor& starts, int64_t E, const at::Tensor& x) {
  TORCH_CHECK(starts.dim() == 1 && starts.scalar_type() == at::kInt && starts.size(0) == E + 1,
              "starts must be int32 [E+1] with E=", E, " experts");
  TORCH_CHECK(starts.device() == x.device(), "all tensors must be on the same device");
}
void check_16bit(const at::Tensor& a, const at::Tensor& b) {
  TORCH_CHECK(a.is_cuda() && b.device() == a.device(), "all tensors must be on the same device");
  TORCH_CHECK(a.scalar_type() == b.scalar_type(), "operands must have one dtype, got ", a.scalar_type(), " and ", b.scalar_type());
}

// Weights stored as [E,K,N] (a view with its last two dimensions exchanged)
// are taken as they are.
bool stored_across(const at::Tensor& w) { return w.stride(2) != 1 && w.stride(1) == 1 && w.size(1) > 1; }

// out[r] = W[e] x[r] (across false: w [E,N,K]), or W[e]^T x[r] (w [E,K,N]).
at::Tensor grouped_rows(const at::Tensor& x, const at::Tensor& w, const at::Tensor& starts, bool across) {
  const int64_t M = x.size(0), E = w.size(0), P = w.size(across ? 2 : 1);
  at::Tensor a = rows16(x, 8), b = rows16(w, 8);
  const int64_t extra = a.size(1) - b.size(across ? 1 : 2);   // x was padded along the products' index
  if (across && extra > 0) b = at::constant_pad_nd(b, {0, 0, 0, extra});
  const int64_t K = a.size(1), P8 = across ? b.size(2) : P;
  at::Tensor s = contig(starts), out = at::empty({M, P8}, x.options().memory_format(at::MemoryFormat::Contiguous));
  if (across)
    check_status(mi_moe_grouped_matmul_dx(a.data_ptr(), row_stride(a), b.data_ptr(), expert_stride(b), row_stride(b),
                                          s.data_ptr<int32_t>(), M, K, P8, E, act_code(x), out.data_ptr(), stream_of(x)),
                 "moe_grouped_matmul");
  else
    check_status(mi_moe_grouped_matmul(a.data_ptr(), row_stride(a), b.data_ptr(), expert_stride(b), row_stride(b),
                                       s.data_ptr<int32_t>(), M, P8, K, E, act_code(x), out.data_ptr(), stream_of(x)),
                 "moe_grouped_matmul");
  return P8 == P ? out : out.narrow(1, 0, P).contiguous();
}

// x [M,K], w [E,N,K] -> y [M,N].
at::Tensor moe_grouped_matmul_hip(const at::Tensor& x, const at::Tensor& w, const at::Tensor& starts) {
  TORCH_CHECK(x.dim() == 2 && w.dim() == 3 && w.size(2) == x.size(1) && w.size(0) > 0 && w.size(1) > 0 && w.size(2) > 0,
              "moe_grouped_matmul: expected x [M,K], w [E,N,K]");
  check_16bit(x, w);
  check_starts(starts, w.size(0), x);
  c10::hip::HIPGuard guard(x.get_device());
  const bool across = stored_across(w);
  return grouped_rows(x, across ? w.transpose(1, 2) : w, starts, across);
}

// dy [M,N], w [E,N,K] -> dx [M,K].
at::Tensor moe_grouped_matmul_dx_hip(const at::Tensor& dy, const at::Tensor& w, const at::Tensor& starts) {
  TORCH_CHECK(dy.dim() == 2 && w.dim() == 3 && w.size(1) == dy.size(1) && w.size(0) > 0 && w.size(1) > 0 && w.size(2) > 0,
              "moe_grouped_matmul_dx: expected dy [M,N], w [E,N,K]");
  check_16bit(dy, w);
  check_starts(starts, w.size(0), dy);
  c10::hip::HIPGuard guard(dy.get_device());
  const bool across = stored_across(w);
  return grouped_rows(dy, across ? w.transpose(1, 2) : w, starts, !across);
}

// dy [M,N], x [M,K] -> dw [E,N,K].
at::Tensor moe_grouped_matmul_dw_hip(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& starts) {
  TORCH_CHECK(dy.dim() == 2 && x.dim() == 2 && dy.size(0) == x.size(0) && dy.size(1) > 0 && x.size(1) > 0,
              "moe_grouped_matmul_dw: expected dy [M,N], x [M,K]");
  check_16bit(dy, x);
  TORCH_CHECK(starts.dim() == 1 && starts.size(0) > 1, "starts must be int32 [E+1]");
  const int64_t E = starts.size(0) - 1, M = x.size(0), N = dy.size(1), K = x.size(1);
  check_starts(starts, E, x);
  c10::hip::HIPGuard guard(x.get_device());
  at::Tensor a = rows16(dy, 8), b = rows16(x, 8), s = contig(starts);
  const int64_t N8 = a.size(1), K8 = b.size(1);
  at::Tensor dw = at::empty({E, N8, K8}, x.options().memory_format(at::MemoryFormat::Contiguous));
  check_status(mi_moe_grouped_matmul_dw(a.data_ptr(), row_stride(a), b.data_ptr(), row_stride(b), s.data_ptr<int32_t>(), M, N8,
                                        K8, E, act_code(x), dw.data_ptr(), stream_of(x)),
               "moe_grouped_matmul_dw");
  return N8 == N && K8 == K ? dw : dw.narrow(1, 0, N).narrow(2, 0, K).contiguous();
}

// A product through the dispatcher, below autograd, so that dispatch modes
// (flop counters, selective checkpointing) and profilers see it.  The price of
// three such calls is within the noise of a small step's 37 to 62 us.
typedef at::Tensor ProductOp(const at::Tensor&, const at::Tensor&, const at::Tensor&);
c10::TypedOperatorHandle<ProductOp> product_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<ProductOp>();
}

// The differentiable form: each gradient is one of the products above.
struct GroupedMatmul : torch::autograd::Function<GroupedMatmul> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const at::Tensor& starts) {
    // what no gradient needs is not kept
    ctx->save_for_backward({w.requires_grad() ? x : at::Tensor(), x.requires_grad() ? w : at::Tensor(), starts});
    ctx->saved_data["across"] = w.dim() == 3 && stored_across(w);
    static const auto product = product_op("nanovllm::moe_grouped_matmul");
    at::AutoDispatchBelowADInplaceOrView guard;
    return product.call(x, w, starts);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "moe_grouped_matmul: no second derivatives (create_graph=True)");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &w = saved[1], &starts = saved[2], &dy = grads[0];
    at::Tensor dx, dw;
    if (!dy.defined()) return {dx, dw, at::Tensor()};
    static const auto product_dx = product_op("nanovllm::moe_grouped_matmul_dx"), product_dw = product_op("nanovllm::moe_grouped_matmul_dw");
    at::AutoDispatchBelowADInplaceOrView guard;
    if (ctx->needs_input_grad(0)) dx = product_dx.call(dy, w, starts);
    if (ctx->needs_input_grad(1))   // laid out as the weights are
      dw = ctx->saved_data["across"].toBool() ? product_dw.call(x, dy, starts).transpose(1, 2) : product_dw.call(dy, x, starts);
    return {dx, dw, at::Tensor()};
  }
};
at::Tensor moe_grouped_matmul_autograd(const at::Tensor& x, const at::Tensor& w, const at::Tensor& starts) {
  return GroupedMatmul::apply(x, w, starts);
}

int out_code(at::ScalarType t) {
  if (t == at::kFloat) return MI_MOE_F32;
  if (t == at::kBFloat16) return MI_MOE_BF16;
  TORCH_CHECK(t == at::kHalf, "dtype must be float32, bfloat16 or float16, got ", t);
  return MI_MOE_F16;
}
void check_int8(const at::Tensor& x, const at::Tensor& xs, const at::Tensor& w, const at::Tensor& ws) {
  TORCH_CHECK(x.scalar_type() == at::kChar && w.scalar_type() == at::kChar, "x and w must be int8");
  TORCH_CHECK(xs.scalar_type() == at::kFloat && ws.scalar_type() == at::kFloat, "scales must be float32");
  TORCH_CHECK(x.is_cuda() && w.device() == x.device() && xs.device() == x.device() && ws.device() == x.device(),
              "all tensors must be on the same device");
  TORCH_CHECK(x.dim() == 2 && w.size(-1) == x.size(1) && w.numel() > 0, "expected x [M,K] and w [...,N,K]");
  TORCH_CHECK(xs.sizes() == x.sizes().slice(0, 1), "x_scales must be [M], a scale for each row");
  TORCH_CHECK(ws.sizes() == w.sizes().slice(0, w.dim() - 1), "w_scales must be [...,N], a scale for each row of w");
}

// x [M,K] int8, w [N,K] int8, a scale for each row of both -> [M,N].
at::Tensor int8_matmul_hip(const at::Tensor& x, const at::Tensor& x_scales, const at::Tensor& w, const at::Tensor& w_scales,
                           const std::optional<at::Tensor>& bias, at::ScalarType dtype) {
  TORCH_CHECK(w.dim() == 2, "int8_matmul: expected w [N,K]");
  check_int8(x, x_scales, w, w_scales);
  const int out = out_code(dtype);
  const bool has = bias.has_value() && bias->defined();
  if (has)
    TORCH_CHECK(bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == w.size(0) && bias->device() == x.device(),
                "bias must be a float32 [N] tensor on the device of x");
  c10::hip::HIPGuard guard(x.get_device());
  at::Tensor a = rows16(x, 16), b = rows16(w, 16), xs = contig(x_scales), ws = contig(w_scales), bs = has ? contig(*bias) : at::Tensor();
  const int64_t M = a.size(0), K = a.size(1), N = b.size(0);
  at::Tensor y = at::empty({M, N}, x.options().dtype(dtype).memory_format(at::MemoryFormat::Contiguous));
  check_status(mi_moe_int8_matmul(a.data_ptr<int8_t>(), row_stride(a), xs.data_ptr<float>(), b.data_ptr<int8_t>(), row_stride(b),
                                  ws.data_ptr<float>(), has ? bs.data_ptr<float>() : nullptr, M, N, K, out, y.data_ptr(), stream_of(x)),
               "int8_matmul");
  return y;
}

// The same with a weight for each expert, w [E,N,K], and ragged rows.
at::Tensor moe_grouped_matmul_int8_hip(const at::Tensor& x, const at::Tensor& x_scales, const at::Tensor& w,
                                       const at::Tensor& w_scales, const at::Tensor& starts, at::ScalarType dtype) {
  TORCH_CHECK(w.dim() == 3, "moe_grouped_matmul_int8: expected w [E,N,K]");
  check_int8(x, x_scales, w, w_scales);
  check_starts(starts, w.size(0), x);
  const int out = out_code(dtype);
  c10::hip::HIPGuard guard(x.get_device());
  at::Tensor a = rows16(x, 16), b = rows16(w, 16), xs = contig(x_scales), ws = contig(w_scales), s = contig(starts);
  const int64_t M = a.size(0), K = a.size(1), N = b.size(1), E = b.size(0);
  at::Tensor y = at::empty({M, N}, x.options().dtype(dtype).memory_format(at::MemoryFormat::Contiguous));
  check_status(mi_moe_grouped_matmul_int8(a.data_ptr<int8_t>(), row_stride(a), xs.data_ptr<float>(), b.data_ptr<int8_t>(),
                                          expert_stride(b), row_stride(b), ws.data_ptr<float>(), s.data_ptr<int32_t>(), M, N, K, E,
                                          out, y.data_ptr(), stream_of(x)),
               "moe_grouped_matmul_int8");
  return y;
}

// x [...,C] -> int8 codes [...,C] and a scale for each row [...].
std::tuple<at::Tensor, at::Tensor> int8_quantize_hip(const at::Tensor& x) {
  const int dt = mx_value_code(x.scalar_type());
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "int8_quantize: expected [..., C] with C > 0");
  c10::hip::HIPGuard guard(x.get_device());
  const int64_t C = x.size(-1), rows = x.numel() / C;
  const bool in_place = x.is_contiguous() || (x.dim() == 2 && x.size(0) > 1 && x.stride(1) == 1 && x.stride(0) >= C);
  at::Tensor v = in_place ? x : x.contiguous();
  at::Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kChar).memory_format(at::MemoryFormat::Contiguous));
  at::Tensor scales = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  check_status(mi_moe_int8_quantize(v.data_ptr(), dt, rows, C, v.is_contiguous() ? C : v.stride(0), codes.data_ptr<int8_t>(),
                                    scales.data_ptr<float>(), stream_of(x)),
               "int8_quantize");
  return {codes, scales};
}

at::Tensor int8_dequantize_hip(const at::Tensor& codes, const at::Tensor& scales, at::ScalarType dtype) {
  const int dt = mx_value_code(dtype);
  TORCH_CHECK(codes.scalar_type() == at::kChar && scales.scalar_type() == at::kFloat, "codes must be int8, scales float32");
  TORCH_CHECK(codes.is_cuda() && scales.device() == codes.device(), "codes and scales must be on one device");
  TORCH_CHECK(codes.dim() >= 1 && codes.size(-1) > 0 && scales.sizes() == codes.sizes().slice(0, codes.dim() - 1),
              "int8_dequantize: expected codes [..., C] and scales [...]");
  c10::hip::HIPGuard guard(codes.get_device());
  at::Tensor c = contig(codes), s = contig(scales);
  at::Tensor out = at::empty(c.sizes(), c.options().dtype(dtype));
  check_status(mi_moe_int8_dequantize(c.data_ptr<int8_t>(), s.data_ptr<float>(), s.numel(), c.size(-1), out.data_ptr(), dt,
                                      stream_of(c)),
               "int8_dequantize");
  return out;
}

int scale_code(const at::Tensor& d) {
  if (d.scalar_type() == at::kBFloat16) return MI_MOE_BF16;
  TORCH_CHECK(d.scalar_type() == at::kHalf, "scales must be float16 or bfloat16");
  return MI_MOE_F16;
}

}  // namespace

// The graph-mode context of the reference's device op
// (MoEGraphContext, Int8-gemm/nanovllm_ops.cpp:160-201): built for a number
// of tokens, a top_k and an activation dtype (0 fp16, 1 bf16).  Here it
// grows the handle's device workspace to that size up front, so calls of at
// most num_tokens tokens at this top_k allocate nothing and can be captured
// into a HIP graph.  Any top_k >= 1 is accepted (the reference: 1, 8, 10).
struct MoEGraphContext : torch::CustomClassHolder {
  int64_t num_tokens, top_k, dtype;
  MoEGraphContext(const c10::intrusive_ptr<MoEInferHandle>& moe, int64_t T, int64_t K, int64_t dt)
      : num_tokens(T), top_k(K), dtype(dt) {
    TORCH_CHECK(T >= 0 && K >= 1, "MoEGraphContext: num_tokens >= 0 and top_k >= 1");
    TORCH_CHECK(dt == 0 || dt == 1, "MoEGraphContext: dtype must be 0 (float16) or 1 (bfloat16)");
    if (moe->h) check_status(mi_moe_reserve(moe->h, T, K, (void*)c10::hip::getCurrentHIPStream().stream()),
                             "MoEGraphContext");
  }
};

// The reference's callback report thread (NpuCallbackManager,
// Int8-gemm/nanovllm_ops.cpp:38-138) serves its host-callback op; the device
// op here needs none, so the class holds nothing (constructible, for callers
// that create one).
struct NpuCallbackManager : torch::CustomClassHolder {
  NpuCallbackManager(int64_t, int64_t) {}
};

// moe_forward_npu_graph_out (Int8-gemm/nanovllm_ops.cpp:308-342,406): the
// layer into `out` for the context's shape.
void moe_forward_graph_out_impl(const at::Tensor& hidden, const at::Tensor& topk_ids, const at::Tensor& topk_w,
                                const c10::intrusive_ptr<MoEInferHandle>& moe,
                                const c10::intrusive_ptr<MoEGraphContext>& ctx, at::Tensor out) {
  TORCH_CHECK(hidden.dim() == 2 && hidden.size(0) <= ctx->num_tokens,
              "moe_forward_npu_graph_out: more tokens than the MoEGraphContext was built for");
  TORCH_CHECK(topk_ids.dim() == 2 && topk_ids.size(1) == ctx->top_k,
              "moe_forward_npu_graph_out: top_k differs from the MoEGraphContext's");
  TORCH_CHECK((ctx->dtype == 1) == (hidden.scalar_type() == at::kBFloat16),
              "moe_forward_npu_graph_out: hidden dtype differs from the MoEGraphContext's");
  if (hidden.is_cuda()) {
    forward_into(hidden, topk_ids, topk_w, moe, out);
  } else {
    moe_forward_out_cpu(hidden, topk_ids, topk_w, moe, out);
  }
}

TORCH_LIBRARY_FRAGMENT(nanovllm, m) {
  m.class_<MoEInferHandle>("MoEInfer")
      .def(torch::init<int64_t, int64_t, int64_t, int64_t>())
      // Int8-gemm/nanovllm_ops.cpp:354-365
      .def("quantize_and_store_expert",
           [](const c10::intrusive_ptr<MoEInferHandle>& self, int64_t expert_idx,
              const std::string& proj_name, const at::Tensor& w) {
             TORCH_CHECK(self->quant_type == 0 || self->quant_type == 3,
                         "Q4_0 does not support online quantization. "
                         "Use store_quantized_repack() with pre-quantized weights.");
             int proj = proj_name == "gate_proj" ? 0 : proj_name == "up_proj" ? 1
                      : proj_name == "down_proj" ? 2 : -1;
             TORCH_CHECK(proj >= 0, "Unknown proj_name: ", proj_name);
             at::Tensor wc = contig(w);
             int wd = wc.scalar_type() == at::kFloat ? 2 : wc.scalar_type() == at::kBFloat16 ? 1
                    : wc.scalar_type() == at::kHalf ? 0 : -1;
             TORCH_CHECK(wd >= 0, "weight must be float32, float16 or bfloat16");
             const int64_t H = self->info(1), I = self->info(2);
             TORCH_CHECK(wc.dim() == 2, "weight must be 2D");
             if (proj < 2) {
               TORCH_CHECK(wc.size(0) == I && wc.size(1) == H, "gate/up weight must be [I,H]");
             } else {
               TORCH_CHECK(wc.size(0) == H && wc.size(1) == I, "down weight must be [H,I]");
             }
             if (wc.is_cuda() && !aligned16(wc.data_ptr())) wc = wc.clone(at::MemoryFormat::Contiguous);
             if (self->h)
               check_status(mi_moe_quantize_and_store_expert(self->h, expert_idx, proj, wc.data_ptr(),
                                                             wd, wc.is_cuda() ? 1 : 0, stream_of(wc)),
                            "quantize_and_store_expert");
             if (!wc.is_cuda() && self->keep_host)
               check_status(mi_moe_cpu_quantize_and_store_expert(self->host_engine(), expert_idx, proj,
                                                                 wc.data_ptr(), wd),
                            "quantize_and_store_expert (host)");
           })
      // Int8-gemm/nanovllm_ops.cpp:366-371
      .def("store_quantized_repack",
           [](const c10::intrusive_ptr<MoEInferHandle>& self, const at::Tensor& gate_up_qs,
              const at::Tensor& gate_up_d, const at::Tensor& down_qs, const at::Tensor& down_d) {
             TORCH_CHECK(self->quant_type == 0 || self->quant_type == 1,
                         "store_quantized_repack needs a Q8_0 or Q4_0 handle");
             TORCH_CHECK(gate_up_d.scalar_type() == down_d.scalar_type(),
                         "gate_up_d and down_proj_d must have the same dtype");
             const int64_t E = self->info(0), H = self->info(1), I = self->info(2);
             TORCH_CHECK(gate_up_qs.dim() == 3, "gate_up_qs must be [E,2I,H]");
             TORCH_CHECK(down_qs.dim() == 3, "down_proj_qs must be [E,H,I]");
             if (self->quant_type == 0) {
               TORCH_CHECK(gate_up_qs.scalar_type() == at::kChar && down_qs.scalar_type() == at::kChar,
                           "Q8_0 qs must be int8");
               TORCH_CHECK(gate_up_qs.size(0) == E && gate_up_qs.size(1) == 2 * I && gate_up_qs.size(2) == H &&
                               down_qs.size(0) == E && down_qs.size(1) == H && down_qs.size(2) == I,
                           "Q8_0 qs shapes must be [E,2I,H] and [E,H,I]");
             } else {
               TORCH_CHECK((gate_up_qs.scalar_type() == at::kInt || gate_up_qs.scalar_type() == at::kUInt32) &&
                               (down_qs.scalar_type() == at::kInt || down_qs.scalar_type() == at::kUInt32),
                           "Q4_0 qs must be int32 (uint32 storage)");
               TORCH_CHECK(gate_up_qs.size(0) == E && gate_up_qs.size(1) == 2 * I && gate_up_qs.size(2) == H / 8 &&
                               down_qs.size(0) == E && down_qs.size(1) == H && down_qs.size(2) == I / 8,
                           "Q4_0 qs shapes must be [E,2I,H/8] and [E,H,I/8]");
             }
             TORCH_CHECK(gate_up_d.numel() == E * 2 * I * (H / 32) && down_d.numel() == E * H * (I / 32),
                         "scale shapes must be [E,2I,H/32] and [E,H,I/32]");
             at::Tensor a = contig(gate_up_qs), b = contig(gate_up_d), c = contig(down_qs), d = contig(down_d);
             const bool dev = a.is_cuda();
             TORCH_CHECK(b.is_cuda() == dev && c.is_cuda() == dev && d.is_cuda() == dev,
                         "all weight tensors must be on one device");
             if (self->h)
               check_status(mi_moe_store_quantized(self->h, a.data_ptr(), b.data_ptr(), c.data_ptr(),
                                                   d.data_ptr(), scale_code(b), dev ? 1 : 0, stream_of(a)),
                            "store_quantized_repack");
             if (!dev && self->keep_host)
               check_status(mi_moe_cpu_store_quantized(self->host_engine(), a.data_ptr(), b.data_ptr(),
                                                       c.data_ptr(), d.data_ptr(), scale_code(b)),
                            "store_quantized_repack (host)");
           })
      // build-defined W4A16 (AWQ layout) loader; see include/mi_moe.h
      .def("store_awq_repack",
           [](const c10::intrusive_ptr<MoEInferHandle>& self, const at::Tensor& w13_qweight,
              const at::Tensor& w13_qzeros, const at::Tensor& w13_scales,
              const at::Tensor& w2_qweight, const at::Tensor& w2_qzeros,
              const at::Tensor& w2_scales, int64_t group_size) {
             TORCH_CHECK(self->quant_type == 2, "store_awq_repack needs a W4A16 handle (quant_type 2)");
             const int64_t E = self->info(0), H = self->info(1), I = self->info(2);
             TORCH_CHECK(group_size > 0 && H % group_size == 0 && I % group_size == 0, "bad group_size");
             const int64_t g = group_size;
             TORCH_CHECK(w13_qweight.sizes() == at::IntArrayRef({E, H, 2 * I / 8}) &&
                             w13_qzeros.sizes() == at::IntArrayRef({E, H / g, 2 * I / 8}) &&
                             w13_scales.sizes() == at::IntArrayRef({E, H / g, 2 * I}),
                         "w13 AWQ tensors must be [E,H,2I/8], [E,H/g,2I/8], [E,H/g,2I]");
             TORCH_CHECK(w2_qweight.sizes() == at::IntArrayRef({E, I, H / 8}) &&
                             w2_qzeros.sizes() == at::IntArrayRef({E, I / g, H / 8}) &&
                             w2_scales.sizes() == at::IntArrayRef({E, I / g, H}),
                         "w2 AWQ tensors must be [E,I,H/8], [E,I/g,H/8], [E,I/g,H]");
             TORCH_CHECK(w13_qweight.scalar_type() == at::kInt && w13_qzeros.scalar_type() == at::kInt &&
                             w2_qweight.scalar_type() == at::kInt && w2_qzeros.scalar_type() == at::kInt,
                         "qweight / qzeros must be int32");
             TORCH_CHECK(w13_scales.scalar_type() == w2_scales.scalar_type(), "scale dtypes differ");
             at::Tensor a = contig(w13_qweight), b = contig(w13_qzeros), c = contig(w13_scales),
                        d = contig(w2_qweight), e = contig(w2_qzeros), f = contig(w2_scales);
             const bool dev = a.is_cuda();
             TORCH_CHECK(b.is_cuda() == dev && c.is_cuda() == dev && d.is_cuda() == dev &&
                             e.is_cuda() == dev && f.is_cuda() == dev,
                         "all weight tensors must be on one device");
             if (self->h)
               check_status(mi_moe_store_awq(self->h, a.data_ptr<int32_t>(), b.data_ptr<int32_t>(),
                                             c.data_ptr(), d.data_ptr<int32_t>(), e.data_ptr<int32_t>(),
                                             f.data_ptr(), g, scale_code(c), dev ? 1 : 0, stream_of(a)),
                            "store_awq_repack");
             if (!dev && self->keep_host)
               check_status(mi_moe_hybrid_store_awq(self->host_w4(), a.data_ptr<int32_t>(), b.data_ptr<int32_t>(),
                                                    c.data_ptr(), d.data_ptr<int32_t>(), e.data_ptr<int32_t>(),
                                                    f.data_ptr(), g, scale_code(c), 0, nullptr),
                            "store_awq_repack (host)");
           })
      // MXFP4 weights as mx_quantize writes them; see mi_moe_store_mxfp4
      .def("store_mxfp4_repack",
           [](const c10::intrusive_ptr<MoEInferHandle>& self, const at::Tensor& gate_up_codes,
              const at::Tensor& gate_up_scales, const at::Tensor& down_codes, const at::Tensor& down_scales) {
             TORCH_CHECK(self->quant_type == 3, "store_mxfp4_repack needs an MXFP4 handle (quant_type 3)");
             const int64_t E = self->info(0), H = self->info(1), I = self->info(2);
             TORCH_CHECK(gate_up_codes.sizes() == at::IntArrayRef({E, 2 * I, H / 2}) &&
                             gate_up_scales.sizes() == at::IntArrayRef({E, 2 * I, H / 32}),
                         "gate_up tensors must be [E,2I,H/2] and [E,2I,H/32]");
             TORCH_CHECK(down_codes.sizes() == at::IntArrayRef({E, H, I / 2}) &&
                             down_scales.sizes() == at::IntArrayRef({E, H, I / 32}),
                         "down tensors must be [E,H,I/2] and [E,H,I/32]");
             at::Tensor t[4] = {contig(gate_up_codes), contig(gate_up_scales), contig(down_codes), contig(down_scales)};
             const bool dev = t[0].is_cuda();
             for (auto& v : t) {
               TORCH_CHECK(v.scalar_type() == at::kByte, "codes and scales must be uint8");
               TORCH_CHECK(v.device() == t[0].device(), "all weight tensors must be on one device");
               if (dev && !aligned16(v.data_ptr())) v = v.clone(at::MemoryFormat::Contiguous);
             }
             check_status(mi_moe_store_mxfp4(self->dev(), t[0].data_ptr<uint8_t>(), t[1].data_ptr<uint8_t>(),
                                             t[2].data_ptr<uint8_t>(), t[3].data_ptr<uint8_t>(), dev ? 1 : 0,
                                             stream_of(t[0])),
                          "store_mxfp4_repack");
           })
      .def("get_last_run_time_ms",
           [](const c10::intrusive_ptr<MoEInferHandle>& self) {
             if (self->last_cpu || !self->h) return self->last_cpu_ms;
             return mi_moe_get_last_run_time_ms(self->h);
           })
      .def("get_last_phase_times_ms",
           [](const c10::intrusive_ptr<MoEInferHandle>& self) {
             double ms[2] = {0.0, 0.0};
             const int n = mi_moe_get_last_phase_times_ms(self->dev(), ms, 2);
             TORCH_CHECK(n > 0, "get_last_phase_times_ms: ", mi_moe_last_error());
             return std::vector<double>(ms, ms + n);
           })
      .def("set_timing",
           [](const c10::intrusive_ptr<MoEInferHandle>& self, bool enable) {
             if (self->h) check_status(mi_moe_set_timing(self->h, enable ? 1 : 0), "set_timing");
           })
      .def("get_quant_type",
           [](const c10::intrusive_ptr<MoEInferHandle>& self) { return self->get_quant_type(); })
      .def("get_num_experts",
           [](const c10::intrusive_ptr<MoEInferHandle>& self) { return self->info(0); })
      .def("get_hidden_size",
           [](const c10::intrusive_ptr<MoEInferHandle>& self) { return self->info(1); })
      .def("get_intermediate_size",
           [](const c10::intrusive_ptr<MoEInferHandle>& self) { return self->info(2); });

  m.def("moe_forward(Tensor hidden, Tensor topk_ids, Tensor topk_w, "
        "__torch__.torch.classes.nanovllm.MoEInfer moe) -> Tensor");
  m.def("moe_forward_out(Tensor hidden, Tensor topk_ids, Tensor topk_w, "
        "__torch__.torch.classes.nanovllm.MoEInfer moe, Tensor(a!) out) -> ()");
  m.def("moe_topk_softmax(Tensor logits, int top_k, bool renormalize=True) -> (Tensor, Tensor)");
  // the reference's device-op names (Int8-gemm/nanovllm_ops.cpp:393-407): the
  // stream op is moe_forward, the graph op writes into out
  m.class_<NpuCallbackManager>("NpuCallbackManager").def(torch::init<int64_t, int64_t>());
  m.class_<MoEGraphContext>("MoEGraphContext")
      .def(torch::init<const c10::intrusive_ptr<MoEInferHandle>&, int64_t, int64_t, int64_t>());
  m.def("moe_forward_npu_stream(Tensor hidden, Tensor topk_ids, Tensor topk_w, "
        "__torch__.torch.classes.nanovllm.MoEInfer moe) -> Tensor");
  m.def("moe_forward_npu_graph_out(Tensor hidden, Tensor topk_ids, Tensor topk_w, "
        "__torch__.torch.classes.nanovllm.MoEInfer moe, __torch__.torch.classes.nanovllm.MoEGraphContext ctx, "
        "Tensor(a!) out) -> ()");
  m.def("moe_forward_logits(Tensor hidden, Tensor router_logits, int top_k, bool renormalize, "
        "__torch__.torch.classes.nanovllm.MoEInfer moe) -> Tensor");
  m.def("moe_topk_scores(Tensor logits, int top_k, Tensor? bias=None, str score='softmax', int n_group=1, "
        "int topk_group=1, int group_top=2, bool renormalize=True, float scale=1.0) -> (Tensor, Tensor)");
  m.def("moe_forward_scores(Tensor hidden, Tensor router_logits, int top_k, Tensor? bias, str score, int n_group, "
        "int topk_group, int group_top, bool renormalize, float scale, "
        "__torch__.torch.classes.nanovllm.MoEInfer moe) -> Tensor");
  m.def("mx_quantize(Tensor x, str format) -> (Tensor, Tensor)");
  m.def("mx_dequantize(Tensor codes, Tensor scales, str format, ScalarType dtype) -> Tensor");
  m.def("moe_grouped_matmul(Tensor x, Tensor w, Tensor starts) -> Tensor");
  m.def("moe_grouped_matmul_dx(Tensor dy, Tensor w, Tensor starts) -> Tensor");
  m.def("moe_grouped_matmul_dw(Tensor dy, Tensor x, Tensor starts) -> Tensor");
  m.def("moe_grouped_matmul_int8(Tensor x, Tensor x_scales, Tensor w, Tensor w_scales, Tensor starts, ScalarType dtype) -> Tensor");
  m.def("int8_matmul(Tensor x, Tensor x_scales, Tensor w, Tensor w_scales, Tensor? bias, ScalarType dtype) -> Tensor");
  m.def("int8_quantize(Tensor x) -> (Tensor, Tensor)");
  m.def("int8_dequantize(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
}

TORCH_LIBRARY_IMPL(nanovllm, AutogradCUDA, m) { m.impl("moe_grouped_matmul", &moe_grouped_matmul_autograd); }

TORCH_LIBRARY_IMPL(nanovllm, CUDA, m) {
  m.impl("moe_forward", &moe_forward_hip);
  m.impl("moe_forward_out", &moe_forward_out_hip);
  m.impl("moe_topk_softmax", &moe_topk_softmax_hip);
  m.impl("moe_forward_logits", &moe_forward_logits_hip);
  m.impl("moe_topk_scores", &moe_topk_scores_hip);
  m.impl("moe_forward_scores", &moe_forward_scores_hip);
  m.impl("mx_quantize", &mx_quantize_hip);
  m.impl("mx_dequantize", &mx_dequantize_hip);
  m.impl("moe_grouped_matmul", &moe_grouped_matmul_hip);
  m.impl("moe_grouped_matmul_dx", &moe_grouped_matmul_dx_hip);
  m.impl("moe_grouped_matmul_dw", &moe_grouped_matmul_dw_hip);
  m.impl("moe_grouped_matmul_int8", &moe_grouped_matmul_int8_hip);
  m.impl("int8_matmul", &int8_matmul_hip);
  m.impl("int8_quantize", &int8_quantize_hip);
  m.impl("int8_dequantize", &int8_dequantize_hip);
  m.impl("moe_forward_npu_stream", &moe_forward_hip);
  m.impl("moe_forward_npu_graph_out", &moe_forward_graph_out_impl);
}

TORCH_LIBRARY_IMPL(nanovllm, CPU, m) {
  m.impl("moe_forward", &moe_forward_cpu);
  m.impl("moe_forward_out", &moe_forward_out_cpu);
  m.impl("moe_topk_softmax", &moe_topk_softmax_cpu);
  m.impl("moe_forward_logits", &moe_forward_logits_cpu);
  m.impl("moe_topk_scores", &moe_topk_scores_cpu);
  m.impl("moe_forward_scores", &moe_forward_scores_cpu);
  m.impl("moe_forward_npu_stream", &moe_forward_cpu);
  m.impl("moe_forward_npu_graph_out", &moe_forward_graph_out_impl);
}
