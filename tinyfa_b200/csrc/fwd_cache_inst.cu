// Host launcher of the tensor-core kernel over the paged 8-bit cache (kModeCache of fwd_tc.cuh) for one (padded head dim, dtype).
// Compiled once per pair like fwd_tc_inst.cu.
#include <mutex>

#ifndef TFA_HDP
#error "compile with -DTFA_HDP=<64|128|192|256>"
#endif
#ifndef TFA_BF16
#error "compile with -DTFA_BF16=<0|1>"
#endif

#include "fwd_tc.cuh"

namespace tfa_b200 {

#define TFA_CAT3(a, b, c) a##b##c
#define TFA_NAME(hdp, bf) TFA_CAT3(launch_fwd_cache_hdp##hdp, _bf, bf)
#define TFA_NAME2(hdp, bf) TFA_NAME(hdp, bf)

namespace {

template <int kHD, int kScore>
int launch_one(const TcCacheParams& p, int ctas, bool overlap, int device, cudaStream_t stream) {
  constexpr int kSmem = tc::Cfg<TFA_HDP>::kSmemBytes + tc::kCacheSmem;
  static_assert(kSmem <= 227 * 1024, "shared memory");
  auto kernel = tc::fwd_tc_kernel<TFA_HDP, (TFA_BF16 != 0), tc::kModeCache, false, kHD, false, kScore>;
  static std::once_flag once[64];
  static cudaError_t attrErr[64];
  std::call_once(once[device], [&] { attrErr[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem); });
  if (attrErr[device] != cudaSuccess) {
    set_error_string("cudaFuncSetAttribute(%d bytes): %s", kSmem, cudaGetErrorString(attrErr[device]));
    return kCudaError;
  }
  const CUtensorMap none = {};  // nothing comes by TMA
  const cudaError_t e = launch_kernel(kernel, dim3((unsigned)ctas), tc::kThreads, (size_t)kSmem, stream, overlap, none, none, none, p);
  if (e != cudaSuccess) {
    set_error_string("cache attention kernel launch failed: %s", cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

template <int kHD, int kCodes>
int launch_codes(const TcCacheParams& p, int ctas, bool overlap, int device, cudaStream_t stream) {
  constexpr int kBase = tc::kScoreMask | kCodes;
  const bool cap = p.cap > 0.f, bias = p.slopes != nullptr;
  if (cap && bias) return launch_one<kHD, kBase | tc::kScoreCap | tc::kScoreBias>(p, ctas, overlap, device, stream);
  if (cap) return launch_one<kHD, kBase | tc::kScoreCap>(p, ctas, overlap, device, stream);
  if (bias) return launch_one<kHD, kBase | tc::kScoreBias>(p, ctas, overlap, device, stream);
  return launch_one<kHD, kBase>(p, ctas, overlap, device, stream);
}
template <int kHD>
int launch_head_dim(const TcCacheParams& p, int ctas, bool overlap, int device, cudaStream_t stream) {
  return p.int8 ? launch_codes<kHD, tc::kScoreInt8>(p, ctas, overlap, device, stream) : launch_codes<kHD, 0>(p, ctas, overlap, device, stream);
}

}  // namespace

int TFA_NAME2(TFA_HDP, TFA_BF16)(const TcCacheParams& p, int ctas, bool overlap, int device, cudaStream_t stream) {
#if TFA_HDP == 64
  if (p.headDim == 32) return launch_head_dim<32>(p, ctas, overlap, device, stream);
#endif
#if TFA_HDP == 128
  if (p.headDim == 96) return launch_head_dim<96>(p, ctas, overlap, device, stream);
#endif
  return launch_head_dim<TFA_HDP>(p, ctas, overlap, device, stream);
}

}  // namespace tfa_b200
