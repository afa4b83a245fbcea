// Host launcher of the tensor-core kernel for calls whose scores are capped, biased or masked by prefix or document (score.cuh),
// for one (padded head dim, dtype).  Compiled once per pair like fwd_tc_inst.cu; the kernel is the same template (fwd_tc.cuh) with
// instantiations of its own.
#include <mutex>

#ifndef TFA_HDP
#error "compile with -DTFA_HDP=<64|128|192|256>"
#endif
#ifndef TFA_BF16
#error "compile with -DTFA_BF16=<0|1>"
#endif

#include "fwd_tc_host.cuh"

namespace tfa_b200 {

#define TFA_CAT3(a, b, c) a##b##c
#define TFA_NAME(hdp, bf) TFA_CAT3(launch_fwd_tc_score_hdp##hdp, _bf, bf)
#define TFA_NAME2(hdp, bf) TFA_NAME(hdp, bf)

namespace {

constexpr bool kBf = (TFA_BF16 != 0);
// Head dims 32 / 64: one-tile CTAs, two per SM, as without scores; key ranges: one-tile CTAs up to 128.
constexpr bool kSolo = TFA_HDP == 64;
constexpr bool kSoloParts = TFA_HDP <= 128;

template <int kMode, bool kSoloForm, int kScore, int kHD>
int launch_one(const FwdProblem& pr, int packShift, const TcSplit& split, int device) {
  using C = typename std::conditional<kSoloForm, typename std::conditional<TFA_HDP == 64, tc::CfgSolo64, tc::CfgSolo128>::type, tc::Cfg<TFA_HDP>>::type;
  auto kernel = tc::fwd_tc_kernel<TFA_HDP, kBf, kMode, kSoloForm, kHD, false, kScore>;
  static std::once_flag once[64];
  static cudaError_t attrErr[64];
  std::call_once(once[device], [&] {
    attrErr[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (kSoloForm && attrErr[device] == cudaSuccess) {  // two on an SM
      attrErr[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    }
  });
  if (attrErr[device] != cudaSuccess) {
    set_error_string("cudaFuncSetAttribute(%d bytes): %s", C::kSmemBytes, cudaGetErrorString(attrErr[device]));
    return kCudaError;
  }
  typename tc::ParamsOf<kMode, 1>::type p;
  long long numItems = 0;
  int rc = fill_tc_params(p, pr, packShift, split.parts, C::kNT, false, device, numItems);
  if (rc != kOk) return rc;
  static_cast<ScoreFields&>(p) = *pr.score;
  if constexpr (kMode == tc::kModeFixedSplit) {
    p.partBlocks = split.partBlocks;
    p.numItems = (int)numItems;
    p.rows = pr.totalQ * pr.headsQ;
    p.partO = split.partO;
    p.partLse = split.partLse;
  }
  // keys behind the last row's position are nobody's (a prefix may reach further): zeros, whatever they hold
  const long long reach = (long long)p.qStart + pr.seqLenQ, readable = pr.causal && p.prefix == nullptr && reach < pr.seqLenKV ? reach : pr.seqLenKV;
  CUtensorMap tmQ, tmK, tmV;
  if ((rc = make_map(&tmQ, pr.Q, pr.batch, pr.seqLenQ, pr.headsQ, pr.headDim, 1 << packShift, tc::kBlockM >> packShift)) != kOk) return rc;
  if ((rc = make_map(&tmK, pr.K, pr.batch, pr.seqLenKV, pr.headsKV, pr.headDim, 1, tc::kBlockN, readable)) != kOk) return rc;
  if ((rc = make_map(&tmV, pr.V, pr.batch, pr.seqLenKV, pr.headsKV, pr.headDim, 1, tc::kBlockN, readable)) != kOk) return rc;
  rc = kCudaError;
  p.workCounter = device_work_counter(device, pr.stream, &rc, nullptr);
  if (p.workCounter == nullptr) return rc;
  p.devMaps = nullptr;
  const long long slots = (long long)device_num_sms(device) * (kSoloForm ? 2 : 1);
  const int ctas = (int)(p.numWork < slots ? p.numWork : slots);
  const cudaError_t e = launch_kernel(kernel, dim3((unsigned)ctas), kSoloForm ? tc::kThreadsSolo : tc::kThreads, (size_t)C::kSmemBytes, pr.stream,
                                      pr.overlap, tmQ, tmK, tmV, p);
  if (e != cudaSuccess) {
    set_error_string("kernel launch failed: %s", cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

// kHD: head dims 32 and 96 have MMAs of their own shape in the 64- and 128-wide kernels.  (With key ranges they must: a partial result
// has rows of the head dim's width.)
template <int kScore, int kHD>
int launch_score(const FwdProblem& pr, int packShift, const TcSplit& split, int device) {
  if (split.parts > 1) return launch_one<tc::kModeFixedSplit, kSoloParts, kScore, kHD>(pr, packShift, split, device);
  return launch_one<tc::kModeFixed, kSolo, kScore, kHD>(pr, packShift, split, device);
}

template <int kHD>
int launch_head_dim(const FwdProblem& pr, int packShift, const TcSplit& split, int device) {
  const bool cap = pr.score->cap > 0.f, bias = pr.score->slopes != nullptr;
  if (cap && bias) return launch_score<tc::kScoreMask | tc::kScoreCap | tc::kScoreBias, kHD>(pr, packShift, split, device);
  if (cap) return launch_score<tc::kScoreMask | tc::kScoreCap, kHD>(pr, packShift, split, device);
  if (bias) return launch_score<tc::kScoreMask | tc::kScoreBias, kHD>(pr, packShift, split, device);
  return launch_score<tc::kScoreMask, kHD>(pr, packShift, split, device);
}

}  // namespace

int TFA_NAME2(TFA_HDP, TFA_BF16)(const FwdProblem& pr, int packShift, const TcSplit& split) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return kCudaError;
#if TFA_HDP == 64
  if (pr.headDim == 32) return launch_head_dim<32>(pr, packShift, split, device);
#endif
#if TFA_HDP == 128
  if (pr.headDim == 96) return launch_head_dim<96>(pr, packShift, split, device);
#endif
  return launch_head_dim<TFA_HDP>(pr, packShift, split, device);
}

}  // namespace tfa_b200
