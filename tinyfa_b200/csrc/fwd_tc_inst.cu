// Host launcher for one (padded head dim, dtype) instantiation of the tcgen05 attention kernel.
// Compiled once per pair with -DTFA_HDP=<64|128|192|256> -DTFA_BF16=<0|1> so that the instantiations
// build in parallel (the reference splits its instantiations the same way, one translation unit per
// dtype and architecture: reference csrc/flash_attn/kernels/tfa_fwd_*_sm8x.cu).
//
// Takes the place of the reference's host launcher (reference csrc/flash_attn/launcher.cuh:28-99):
// it derives the grid from the problem sizes, opts in to large dynamic shared memory and launches on
// the caller's stream; in addition it encodes the three TMA descriptors the kernel needs.
#include <cstdio>
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
#define TFA_NAME(hdp, bf) TFA_CAT3(launch_fwd_tc_hdp##hdp, _bf, bf)
#define TFA_NAME2(hdp, bf) TFA_NAME(hdp, bf)

int TFA_NAME2(TFA_HDP, TFA_BF16)(const FwdProblem& pr, int packShift, const TcSplit& split) {
  using C = tc::Cfg<TFA_HDP>;
  const bool varlen = (pr.cuQ != nullptr);
  constexpr bool kBf = (TFA_BF16 != 0);
  auto kernel = varlen ? tc::fwd_tc_kernel<TFA_HDP, kBf, tc::kModeVarlen> : tc::fwd_tc_kernel<TFA_HDP, kBf, tc::kModeFixed>;
  bool solo = false;  // one Q tile per CTA, two CTAs per SM (padded head dim 64; 128 with key ranges)
  int kNT = C::kNT, smemBytes = C::kSmemBytes, threads = tc::kThreads;
#if TFA_HDP == 128
  // head dim 96 has MMAs of its own shape in the 128-wide kernel (6 of 8 k-steps, 96 output columns)
  if (pr.headDim == 96 && option_narrow_mma() != 0) {
    kernel = varlen ? tc::fwd_tc_kernel<128, kBf, tc::kModeVarlen, false, 96> : tc::fwd_tc_kernel<128, kBf, tc::kModeFixed, false, 96>;
  }
#endif
#if TFA_HDP == 64
  // nothing to mask: not causal, and the key length fills its last 128-key block
  const bool noMask = !varlen && !pr.causal && pr.seqLenKV % tc::kBlockN == 0;
  if (noMask) kernel = tc::fwd_tc_kernel<64, kBf, tc::kModeFixedNoMask>;
  solo = option_solo64() != 0;
  if (solo) {
    const bool narrow = (pr.headDim == 32 && option_narrow_mma() != 0);  // head dim 32: 2 of 4 k-steps, 32 output columns
    if (narrow) {
      kernel = varlen ? tc::fwd_tc_kernel<64, kBf, tc::kModeVarlen, true, 32>
                      : (noMask ? tc::fwd_tc_kernel<64, kBf, tc::kModeFixedNoMask, true, 32>
                                : tc::fwd_tc_kernel<64, kBf, tc::kModeFixed, true, 32>);
    } else {
      kernel = varlen ? tc::fwd_tc_kernel<64, kBf, tc::kModeVarlen, true>
                      : (noMask ? tc::fwd_tc_kernel<64, kBf, tc::kModeFixedNoMask, true>
                                : tc::fwd_tc_kernel<64, kBf, tc::kModeFixed, true>);
    }
    kNT = 1;
    smemBytes = tc::CfgSolo64::kSmemBytes;
    threads = tc::kThreadsSolo;
  }
#endif

  const bool parts = split.parts > 1;  // key ranges: few query tiles, long keys (fixed length)
  if (parts) {
#if TFA_HDP <= 128
    solo = true;
    kNT = 1;
    smemBytes = TFA_HDP == 64 ? tc::CfgSolo64::kSmemBytes : tc::CfgSolo128::kSmemBytes;
    threads = tc::kThreadsSolo;
#endif
  }

  bool pair = false;  // clusters of two CTAs, one Q tile each, K/V shared (head dims 192 / 256, fixed length)
#if TFA_HDP >= 192
  // Measured (fp16, H16, batch x length = 16 K tokens, 600-800-launch loops, one-tile form -> pair form): head dim 256
  // non-causal S256 500 -> 497, S512 672 -> 789, S1024 791 -> 1010, S2048 872 -> 1168, S8192 957 -> 1244 TFLOP/s; causal
  // S512 444 -> 432, S1024 611 -> 673, S1536 702 -> 813, S2048 760 -> 896; head dim 192 non-causal S2048 1023 -> 1013,
  // S8192 1098 -> 1119, causal S2048 826 -> 764, S8192 1009 -> 1007 (three ring stages already keep its one-tile form
  // fed).  Causal pairs pay for the fully masked last block of their first tile and, with short sequences, for item
  // boundaries that are twice as heavy; "auto" is head dim 256 only, and its causal problems from 1024 query rows.
  const int pairOpt = option_pair_cta();
  const bool pairAuto = (TFA_HDP == 256) && (!pr.causal || pr.seqLenQ >= 1024);
  pair = !parts && !varlen && pr.seqLenQ > (tc::kBlockM >> packShift) && (pairOpt > 0 || (pairOpt < 0 && pairAuto));
  if (pair) {
    kernel = tc::fwd_tc_kernel<TFA_HDP, kBf, tc::kModeFixed, false, TFA_HDP, true>;
    kNT = 2;  // a work item is the two tiles of a pair
    smemBytes = tc::CfgPair<TFA_HDP>::kSmemBytes;
  }
#endif

  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return kCudaError;
  static std::once_flag once[64];
  static cudaError_t attrErr[64];
  if (device < 0 || device >= 64) return kBadArgument;
  std::call_once(once[device], [&] {
    auto bigAttr = [&](auto k) {
      if (attrErr[device] != cudaSuccess) return;
      attrErr[device] = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    };
    attrErr[device] = cudaSuccess;
    bigAttr(tc::fwd_tc_kernel<TFA_HDP, kBf, tc::kModeFixed>);
    bigAttr(tc::fwd_tc_kernel<TFA_HDP, kBf, tc::kModeVarlen>);
#if TFA_HDP >= 192
    bigAttr(tc::fwd_tc_kernel<TFA_HDP, kBf, tc::kModeFixedSplit>);
#endif
#if TFA_HDP <= 128
    // the two-CTAs-per-SM forms: 99 KB each, and the largest shared-memory carve-out so that two fit
    auto soloAttr = [&](auto k) {
      if (attrErr[device] != cudaSuccess) return;
      constexpr int bytes = TFA_HDP == 64 ? tc::CfgSolo64::kSmemBytes : tc::CfgSolo128::kSmemBytes;
      attrErr[device] = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      if (attrErr[device] == cudaSuccess) {
        attrErr[device] = cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
      }
    };
    soloAttr(tc::fwd_tc_kernel<TFA_HDP, kBf, tc::kModeFixedSplit, true>);
    soloAttr(tc::fwd_tc_kernel<TFA_HDP, kBf, tc::kModeFixedSplit, true, TFA_HDP == 64 ? 32 : 96>);
#endif
#if TFA_HDP >= 192
    if (attrErr[device] == cudaSuccess) {
      attrErr[device] = cudaFuncSetAttribute(tc::fwd_tc_kernel<TFA_HDP, kBf, tc::kModeFixed, false, TFA_HDP, true>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, tc::CfgPair<TFA_HDP>::kSmemBytes);
    }
#endif
#if TFA_HDP == 128
    bigAttr(tc::fwd_tc_kernel<128, kBf, tc::kModeFixed, false, 96>);
    bigAttr(tc::fwd_tc_kernel<128, kBf, tc::kModeVarlen, false, 96>);
#endif
#if TFA_HDP == 64
    bigAttr(tc::fwd_tc_kernel<64, kBf, tc::kModeFixedNoMask>);
    soloAttr(tc::fwd_tc_kernel<64, kBf, tc::kModeFixed, true>);
    soloAttr(tc::fwd_tc_kernel<64, kBf, tc::kModeVarlen, true>);
    soloAttr(tc::fwd_tc_kernel<64, kBf, tc::kModeFixedNoMask, true>);
    soloAttr(tc::fwd_tc_kernel<64, kBf, tc::kModeFixed, true, 32>);
    soloAttr(tc::fwd_tc_kernel<64, kBf, tc::kModeVarlen, true, 32>);
    soloAttr(tc::fwd_tc_kernel<64, kBf, tc::kModeFixedNoMask, true, 32>);
#endif
  });
  if (attrErr[device] != cudaSuccess) {
    set_error_string("cudaFuncSetAttribute(%d bytes): %s", C::kSmemBytes, cudaGetErrorString(attrErr[device]));
    return kCudaError;
  }

  const int gp = 1 << packShift;
  const int rowsPerTile = tc::kBlockM >> packShift;
  CUtensorMap tmQ, tmK, tmV;
  int rc;
  const long long nb = varlen ? 1 : pr.batch;
  // packed input with unknown totals: placeholder extent, completed on the device before the kernel runs
  const bool devMaps = varlen && (pr.totalQ < 0 || pr.totalKV < 0);
  const long long rowsQ = varlen ? (devMaps ? 1 : pr.totalQ) : pr.seqLenQ;
  const long long rowsKV = varlen ? (devMaps ? 1 : pr.totalKV) : pr.seqLenKV;
  if ((rc = make_map(&tmQ, pr.Q, nb, rowsQ, pr.headsQ, pr.headDim, gp, rowsPerTile)) != kOk) return rc;
  // pair form: each CTA loads 64 of a block's 128 keys
  if ((rc = make_map(&tmK, pr.K, nb, rowsKV, pr.headsKV, pr.headDim, 1, pair ? tc::kBlockN / 2 : tc::kBlockN)) != kOk) return rc;
  if ((rc = make_map(&tmV, pr.V, nb, rowsKV, pr.headsKV, pr.headDim, 1, tc::kBlockN)) != kOk) return rc;

  TcParams p;
  long long numItems = 0;
  if ((rc = fill_tc_params(p, pr, packShift, split.parts, kNT, pair, device, numItems)) != kOk) return rc;
  const long long numWork = p.numWork;
  int rcCounter = kCudaError;
  CUtensorMap* slotMaps = nullptr;
  p.workCounter = device_work_counter(device, pr.stream, &rcCounter, &slotMaps);
  if (p.workCounter == nullptr) return rcCounter;
  p.devMaps = nullptr;
  if (devMaps) {
    if ((rc = launch_patch_varlen_maps(tmQ, tmK, tmV, slotMaps, pr.cuQ, pr.cuKV, pr.batch, pr.stream)) != kOk) return rc;
    p.devMaps = slotMaps;
  }

  // persistent: one CTA per SM (512 tensor-memory columns and ~200 KB of shared memory each), or two of the small form
  const long long slots = (long long)device_num_sms(device) * (solo ? 2 : 1);
  const int ctas = (int)(numWork < slots ? numWork : slots);
  cudaError_t e;
  if (pair) {
    // one cluster of two CTAs per work item in flight; as many clusters as the device runs at once
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smemBytes;
    cfg.stream = pr.stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    static int maxClusters[64] = {0};
    if (maxClusters[device] == 0) {
      cfg.gridDim = dim3((unsigned)(2 * (device_num_sms(device) / 2)));
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
        (void)cudaGetLastError();
        n = device_num_sms(device) / 2;
      }
      maxClusters[device] = n;
    }
    const long long clusters = numWork < maxClusters[device] ? numWork : maxClusters[device];
    cfg.gridDim = dim3((unsigned)(2 * clusters));
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = pr.overlap ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kernel, tmQ, tmK, tmV, p);
  } else if (parts) {
    TcPartParams pp;
    static_cast<TcParams&>(pp) = p;
    pp.partBlocks = split.partBlocks;
    pp.numItems = (int)numItems;
    pp.rows = pr.totalQ * pr.headsQ;
    pp.partO = split.partO;
    pp.partLse = split.partLse;
    auto partKernel = tc::fwd_tc_kernel<TFA_HDP, kBf, tc::kModeFixedSplit, (TFA_HDP <= 128)>;
#if TFA_HDP <= 128
    if (pr.headDim != TFA_HDP) partKernel = tc::fwd_tc_kernel<TFA_HDP, kBf, tc::kModeFixedSplit, true, TFA_HDP == 64 ? 32 : 96>;
#endif
    e = launch_kernel(partKernel, dim3((unsigned)ctas), threads, (size_t)smemBytes, pr.stream, pr.overlap, tmQ, tmK, tmV, pp);
  } else {
    e = launch_kernel(kernel, dim3((unsigned)ctas), threads, (size_t)smemBytes, pr.stream, pr.overlap, tmQ, tmK, tmV, p);
  }
  if (e != cudaSuccess) {
    set_error_string("kernel launch failed: %s", cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}


}  // namespace tfa_b200
