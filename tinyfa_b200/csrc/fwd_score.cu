// Attention with capped, biased or masked scores (score.cuh): argument checks, choice of the kernel, and the two small kernels that tell
// the attention kernels which key blocks a query tile can see when keys and queries belong to documents.
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>

#include "../../include/tinyfa_b200.h"
#include "build_config.cuh"
#include "ptx_sm100.cuh"
#include "score.cuh"
#include "tfa_common.cuh"

namespace tfa_b200 {

int device_num_sms(int device);  // c_abi.cu
int pack_shift_of(const FwdProblem& p);
int split_kv_option();
bool fp32_on_tensor_cores(const FwdProblem& p);
int dispatch_fp32(const FwdProblem& p, bool tensorCores);
TcSplit tc_split_of(const FwdProblem& p, int packShift, int qStart);
bool splitkv_applicable(const FwdProblem& p);  // fwd_decode.cu
SplitPlan splitkv_plan(const FwdProblem& p, int numSMs, int forced);
size_t splitkv_scratch_floats(const FwdProblem& p, const SplitPlan& plan);
int launch_fwd_splitkv(const FwdProblem& p, const SplitPlan& plan, float* scratch);
int launch_combine_parts(const FwdProblem& p, int packShift, const TcSplit& split);

#define TFA_DECLARE_SCORE(HDP)                                                             \
  int launch_fwd_tc_score_hdp##HDP##_bf0(const FwdProblem&, int, const TcSplit&);          \
  int launch_fwd_tc_score_hdp##HDP##_bf1(const FwdProblem&, int, const TcSplit&);          \
  static inline int score_call_hdp##HDP(const FwdProblem& p, int ps, const TcSplit& split) { \
    (void)p; (void)ps; (void)split;                                                        \
    if (p.dtype == kBf16) {                                                                \
      if constexpr (TFA_HAVE_BF16) return launch_fwd_tc_score_hdp##HDP##_bf1(p, ps, split); \
    } else {                                                                               \
      if constexpr (TFA_HAVE_FP16) return launch_fwd_tc_score_hdp##HDP##_bf0(p, ps, split); \
    }                                                                                      \
    return kBadDtype;                                                                      \
  }
#if TFA_HAVE_HDP64
TFA_DECLARE_SCORE(64)
#endif
#if TFA_HAVE_HDP128
TFA_DECLARE_SCORE(128)
#endif
#if TFA_HAVE_HDP192
TFA_DECLARE_SCORE(192)
#endif
#if TFA_HAVE_HDP256
TFA_DECLARE_SCORE(256)
#endif
#undef TFA_DECLARE_SCORE

namespace score {

constexpr int kWarps = 8;
constexpr int kScoreTileRows = 64, kScoreBlockKeys = 64;  // of the fp32 kernel; the tensor-core kernel has 128 >> packShift and 128

// Ascending order puts negative ids (no document) last, behind the largest id that a document can have.
__device__ __forceinline__ unsigned order_of(int id) { return id < 0 ? UINT_MAX : (unsigned)id; }

// Smallest and largest document of every key block, a warp each, and whether its keys and the one before it are in ascending order.
__global__ void __launch_bounds__(kWarps * 32) key_blocks_kernel(const int* docKV, int2* out, unsigned char* sorted, int seqLenKV, int blockKeys, int blocks,
                                                                 long long all) {
  ptx::grid_wait_previous();
  ptx::grid_allow_next();
  const long long i = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (i >= all) return;
  const long long b = i / blocks;
  const int k0 = (int)(i - b * blocks) * blockKeys, k1 = min(k0 + blockKeys, seqLenKV);
  const int* ids = docKV + b * seqLenKV;
  int lo = INT_MAX, hi = INT_MIN;
  bool ascends = true;
#pragma unroll 4
  for (int k = k0 + (threadIdx.x & 31); k < k1; k += 32) {
    const int d = ids[k], before = k > 0 ? ids[k - 1] : INT_MIN;
    lo = min(lo, d);
    hi = max(hi, d);
    ascends = ascends && (k == 0 || order_of(before) <= order_of(d));
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  ascends = __all_sync(0xffffffffu, ascends);
  if ((threadIdx.x & 31) == 0) {
    out[i] = make_int2(lo, hi);
    sorted[i] = ascends ? 1 : 0;
  }
}

// Key blocks [x, y) that some row of a query tile may see, a warp for each tile: from the first to the last block whose range of
// documents meets the tile's (documents in ascending order: exactly those with a visible key), as far as the causal mask reaches.
// Never empty: a tile that sees nothing gets one block, in which everything is masked, so that its rows are written.  Then the keys of every row's
// document, by bisection among those blocks, where all blocks as far as the mask reaches are in ascending order.
__global__ void __launch_bounds__(kWarps * 32) tile_range_kernel(const int* docQ, const int* docKV, const int2* keyBlocks, const unsigned char* sorted,
                                                                 const int* prefix, int2* out, int2* rowKeys, int seqLenQ, int seqLenKV, int tileRows,
                                                                 int tiles, int blockKeys, int blocks, int causal, int qStart, long long all) {
  ptx::grid_wait_previous();
  ptx::grid_allow_next();
  const long long i = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (i >= all) return;
  const int lane = threadIdx.x & 31;
  const long long b = i / tiles;
  const int r0 = (int)(i - b * tiles) * tileRows, r1 = min(r0 + tileRows, seqLenQ);
  int lo = INT_MAX, hi = INT_MIN;
#pragma unroll 4
  for (int r = r0 + lane; r < r1; r += 32) {
    const int d = docQ[b * seqLenQ + r];
    if (d >= 0) {
      lo = min(lo, d);
      hi = max(hi, d);
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  int end = blocks;
  if (causal) {
    long long see = (long long)qStart + r1;
    if (prefix != nullptr) see = max(see, (long long)prefix[b]);
    end = (int)min((long long)blocks, (see - 1) / blockKeys + 1);
  }
  int first = INT_MAX, last = -1;
  bool ascends = true;
#pragma unroll 4
  for (int k = lane; k < end; k += 32) {
    const int2 ids = keyBlocks[b * blocks + k];
    ascends = ascends && sorted[b * blocks + k] != 0;
    if (ids.y >= lo && ids.x <= hi) {
      first = min(first, k);
      last = k;
    }
  }
  first = __reduce_min_sync(0xffffffffu, first);
  last = __reduce_max_sync(0xffffffffu, last);
  ascends = __all_sync(0xffffffffu, ascends);
  if (last < 0) first = 0, last = 0;
  if (lane == 0) out[i] = make_int2(first, last + 1);
  const int* ids = docKV + b * seqLenKV;
  const int k0 = first * blockKeys, k1 = min((last + 1) * blockKeys, seqLenKV);
  for (int r = r0 + lane; r < r1; r += 32) {
    const int d = docQ[b * seqLenQ + r];
    int2 keys = make_int2(0, 0);
    if (!ascends) {
      keys = make_int2(-1, -1);
    } else if (d >= 0) {
      int from = k0, to = k1, from2 = k0, to2 = k1;  // first key not before the document, first behind it
      while (from < to || from2 < to2) {
        const int mid = (from + to) >> 1, mid2 = (from2 + to2) >> 1;
        const unsigned x = from < to ? order_of(ids[mid]) : 0u, y = from2 < to2 ? order_of(ids[mid2]) : 0u;
        if (from < to) {
          if (x < (unsigned)d) {
            from = mid + 1;
          } else {
            to = mid;
          }
        }
        if (from2 < to2) {
          if (y <= (unsigned)d) {
            from2 = mid2 + 1;
          } else {
            to2 = mid2;
          }
        }
      }
      keys = make_int2(from, from2);
    }
    rowKeys[b * seqLenQ + r] = keys;
  }
}

int run_tc(const FwdProblem& p, int ps, const TcSplit& split) {
  switch (p.headDim) {
#if TFA_HAVE_HDP64
    case 32:
    case 64: return score_call_hdp64(p, ps, split);
#endif
#if TFA_HAVE_HDP128
    case 96:
    case 128: return score_call_hdp128(p, ps, split);
#endif
#if TFA_HAVE_HDP192
    case 192: return score_call_hdp192(p, ps, split);
#endif
#if TFA_HAVE_HDP256
    case 256: return score_call_hdp256(p, ps, split);
#endif
    default: return kBadHeadDim;
  }
}

// The partial results of a call that is cut over its keys, and the tables of documents, live in one stream-ordered allocation that is
// released behind the last kernel.
int dispatch(FwdProblem p, ScoreFields& f, int device) {
  p.score = &f;
  p.overlap = may_overlap(p.stream);
  const bool docs = f.docKV != nullptr;
  const bool fp32 = p.dtype == kFp32;
  const int sms = device_num_sms(device);
  const int forced = split_kv_option();
  // few query rows: the split-KV kernel, which reads every key - with documents most keys may be none of the row's
  const bool rows = !fp32 && !docs && forced != 0 && splitkv_applicable(p);
  SplitPlan plan = {1, 0, 0};
  size_t floats = 0;
  int ps = 0;
  TcSplit split;
  if (rows) {
    plan = splitkv_plan(p, sms, forced);
    floats = splitkv_scratch_floats(p, plan);
  } else if (!fp32) {
    ps = pack_shift_of(p);
    if (!docs && f.prefix == nullptr) split = tc_split_of(p, ps, f.qStart);
    if (split.parts > 1) floats = (size_t)split.parts * p.totalQ * p.headsQ * (p.headDim + 1);
  }
  const bool cores = fp32 && !fp32_on_tensor_cores(p);
  if (fp32) ps = pack_shift_of(p);
  const int tileRows = cores ? kScoreTileRows : 128 >> ps, blockKeys = f.blockKeys = cores ? kScoreBlockKeys : 128;
  const int blocks = (p.seqLenKV + blockKeys - 1) / blockKeys;
  f.tiles = (p.seqLenQ + tileRows - 1) / tileRows;
  const size_t tableBytes = docs ? (size_t)p.batch * (sizeof(int2) * ((size_t)blocks + f.tiles + p.seqLenQ) + blocks) : 0;
  void* scratch = nullptr;
  int rc = kOk;
  if (floats > 0 || tableBytes > 0) {
    rc = scratch_alloc(&scratch, tableBytes > 0 ? tableBytes : floats * sizeof(float), device, p.stream);
    if (rc != kOk) return rc;
  }
  if (docs) {
    int2* keyBlocks = static_cast<int2*>(scratch);
    int2* tileRange = keyBlocks + (size_t)p.batch * blocks;
    int2* rowKeys = tileRange + (size_t)p.batch * f.tiles;
    unsigned char* sorted = reinterpret_cast<unsigned char*>(rowKeys + (size_t)p.batch * p.seqLenQ);
    const long long allBlocks = (long long)p.batch * blocks, allTiles = (long long)p.batch * f.tiles;
    cudaError_t e = launch_kernel(key_blocks_kernel, dim3((unsigned)((allBlocks + kWarps - 1) / kWarps)), kWarps * 32, 0, p.stream, p.overlap, f.docKV,
                                  keyBlocks, sorted, p.seqLenKV, blockKeys, blocks, allBlocks);
    if (e == cudaSuccess) {
      e = launch_kernel(tile_range_kernel, dim3((unsigned)((allTiles + kWarps - 1) / kWarps)), kWarps * 32, 0, p.stream, p.overlap, f.docQ, f.docKV, keyBlocks,
                        sorted, f.prefix, tileRange, rowKeys, p.seqLenQ, p.seqLenKV, tileRows, f.tiles, blockKeys, blocks, p.causal, f.qStart, allTiles);
    }
    if (e != cudaSuccess) {
      set_error_string("document table kernel launch failed: %s", cudaGetErrorString(e));
      rc = kCudaError;
    }
    f.keyBlocks = keyBlocks;
    f.tileRange = tileRange;
    f.rowKeys = rowKeys;
  }
  if (rc == kOk) {
    if (fp32) {
      rc = dispatch_fp32(p, !cores);
    } else if (rows) {
      rc = launch_fwd_splitkv(p, plan, static_cast<float*>(scratch));
    } else {
      if (split.parts > 1) {
        split.partO = static_cast<float*>(scratch);
        split.partLse = split.partO + (size_t)split.parts * p.totalQ * p.headsQ * p.headDim;
      }
      rc = run_tc(p, ps, split);
      if (rc == kOk && split.parts > 1) rc = launch_combine_parts(p, ps, split);
    }
  }
  if (scratch != nullptr) cudaFreeAsync(scratch, p.stream);
  return rc;
}

}  // namespace score
}  // namespace tfa_b200

using namespace tfa_b200;

extern "C" int tfa_b200_fwd_scored(const void* Q, const void* K, const void* V, void* O, int dtype, int batchSize, int seqLenQ, int seqLenKV,
                                   int numHeadsQ, int numHeadsKV, int headDim, int isCausal, int qStart, float softcap, const float* alibiSlopes,
                                   const int* prefixLens, const int* docIdsQ, const int* docIdsKV, void* stream) {
  int rc = validate_common(Q, K, V, O, dtype, batchSize, seqLenQ, seqLenKV, numHeadsQ, numHeadsKV, headDim);
  if (rc != kOk) return rc;
  if (qStart < 0 || !(softcap >= 0.f) || isinf(softcap)) {
    set_error_string("qStart and softcap must not be negative (qStart=%d softcap=%g)", qStart, softcap);
    return kBadArgument;
  }
  if (prefixLens != nullptr && !isCausal) {
    set_error_string("prefix lengths widen the causal mask: they need isCausal");
    return kBadArgument;
  }
  if ((docIdsQ == nullptr) != (docIdsKV == nullptr)) {
    set_error_string("document ids are given for queries and keys or for neither");
    return kBadArgument;
  }
  if (batchSize == 0 || seqLenQ == 0 || seqLenKV == 0) return kOk;  // nothing to write
  if ((long long)batchSize * seqLenQ > 0x7FFFFFFFll || (long long)batchSize * seqLenKV > 0x7FFFFFFFll || (long long)qStart + seqLenQ > 0x7FFFFF00ll) {
    set_error_string("batchSize * seqLen and qStart + seqLenQ must stay below 2^31 rows");
    return kTooLarge;
  }
  if ((rc = check_device()) != kOk) return rc;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return kCudaError;
  FwdProblem p;
  p.Q = Q;
  p.K = K;
  p.V = V;
  p.O = O;
  p.cuQ = nullptr;
  p.cuKV = nullptr;
  p.dtype = dtype;
  p.batch = batchSize;
  p.seqLenQ = seqLenQ;
  p.seqLenKV = seqLenKV;
  p.totalQ = (long long)batchSize * seqLenQ;
  p.totalKV = (long long)batchSize * seqLenKV;
  p.headsQ = numHeadsQ;
  p.headsKV = numHeadsKV;
  p.headDim = headDim;
  p.causal = isCausal ? 1 : 0;
  p.stream = static_cast<cudaStream_t>(stream);
  ScoreFields f = {qStart, score::usable_cap(softcap), alibiSlopes, prefixLens, docIdsQ, docIdsKV, nullptr, nullptr, nullptr, 0, 0,
                   {Q, K, V, seqLenQ, seqLenKV, numHeadsQ, numHeadsKV, p.causal}};
  return score::dispatch(p, f, device);
}
