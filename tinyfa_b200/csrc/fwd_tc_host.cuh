// What the launchers of the tensor-core kernels share: tensor maps and the parameters that follow from the problem.
// Included by translation units that define TFA_HDP and TFA_BF16.
#pragma once

#include "fwd_tc.cuh"

namespace tfa_b200 {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn get_encode_tiled();  // c_abi.cu
int* device_status_word(int device);  // c_abi.cu: per-device status word (device memory)
int next_epoch();                     // c_abi.cu
int* device_work_counter(int device, cudaStream_t stream, int* rc, CUtensorMap** maps);  // c_abi.cu
int launch_patch_varlen_maps(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, CUtensorMap* out,
                             const int* cuQ, const int* cuKV, int batch, cudaStream_t stream);  // c_abi.cu
int device_num_sms(int device);       // c_abi.cu
int option_narrow_mma();              // c_abi.cu: MMAs shaped for head dims 32 / 96 inside the 64- / 128-wide kernels
int option_solo64();                  // c_abi.cu: one-tile CTAs, two per SM, for head dims 32 / 64
int option_work_order();              // c_abi.cu: -1 auto, 0 pair index fastest, n > 0 chunk width
int option_pair_cta();                // c_abi.cu: head dims 192 / 256 in clusters of two CTAs that share K/V

// [batches, rows, heads, headDim] tensor, 16-bit elements (packed varlen: batches = 1, rows = total);
// box = 64 elements x boxHeads x boxRows x 1, 128-byte swizzle; out-of-range elements read as zero.
static int make_map(CUtensorMap* m, const void* base, long long batches, long long rows, int heads, int headDim,
                    int boxHeads, int boxRows, long long readable = -1 /* rows of an entry that are read; zeros behind them */) {
  EncodeTiledFn enc = get_encode_tiled();
  if (enc == nullptr) return kCudaError;
  cuuint64_t dims[4] = {(cuuint64_t)headDim, (cuuint64_t)heads, (cuuint64_t)(readable > 0 ? readable : rows), (cuuint64_t)batches};
  cuuint64_t strides[3] = {(cuuint64_t)headDim * 2, (cuuint64_t)heads * headDim * 2,
                           (cuuint64_t)rows * heads * headDim * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)boxHeads, (cuuint32_t)boxRows, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(m, TFA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                   const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error_string("cuTensorMapEncodeTiled failed with CUresult %d (batches=%lld rows=%lld heads=%d headDim=%d box=%d,%d)",
                     (int)r, batches, rows, heads, headDim, boxHeads, boxRows);
    return kCudaError;
  }
  return kOk;
}

// Everything of TcParams but the work counters and the maps on the device.
static int fill_tc_params(TcParams& p, const FwdProblem& pr, int packShift, int parts, int kNT, bool pair, int device, long long& numItems) {
  const int gp = 1 << packShift;
  const int rowsPerTile = tc::kBlockM >> packShift;
  p.O = pr.O;
  p.cuQ = pr.cuQ;
  p.cuKV = pr.cuKV;
  p.seqLenQ = pr.seqLenQ;
  p.seqLenKV = pr.seqLenKV;
  p.headsQ = pr.headsQ;
  p.headsKV = pr.headsKV;
  p.headDim = pr.headDim;
  p.group = pr.headsQ / pr.headsKV;
  p.packShift = packShift;
  const int seqPerCta = kNT * rowsPerTile;
  p.numPairs = (pr.seqLenQ + seqPerCta - 1) / seqPerCta;
  p.causal = pr.causal;
  p.scaleLog2 = (float)(1.4426950408889634 / sqrt((double)pr.headDim));
  p.status = device_status_word(device);
  p.epoch = next_epoch();
  if (p.status == nullptr) return kCudaError;
  p.numUnits = pr.headsQ / gp;
  numItems = (long long)p.numPairs * p.numUnits * pr.batch;
  const long long numWork = numItems * parts;
  if (numWork > 0x7FFFFFFFll) {
    set_error_string("too many work items (%lld)", numWork);
    return kTooLarge;
  }
  p.numWork = (int)numWork;
  // Causal problems: heaviest query tile pairs first inside chunks of (head unit, batch) entries.  A chunk is as wide
  // as the KV heads whose K and V fit a quarter of the L2 (32 MB) together, and at least wide enough to hold two
  // items per SM.  Option "work_order": -1 this rule, 0 pair index fastest, n > 0 chunks of n entries.
  const int order = option_work_order();
  p.chunk = 0;
  if (order > 0) {
    const long long per = (long long)p.numUnits * pr.batch;
    p.chunk = (int)(order < per ? order : per);
  } else if (order < 0 && pr.causal) {
    const long long kvPerHead = 4ll * pr.seqLenKV * pr.headDim;  // K and V of one KV head, 16-bit elements
    const int unitsPerKvHead = (p.group >> packShift) > 0 ? (p.group >> packShift) : 1;
    long long heads = (32ll << 20) / (kvPerHead > 0 ? kvPerHead : 1);
    if (heads < 1) heads = 1;
    long long width = heads * unitsPerKvHead;
    // two items per worker: a worker is a CTA, or in the pair form a cluster of two
    const long long workers = pair ? device_num_sms(device) / 2 : device_num_sms(device);
    const long long minWidth = (2ll * workers + p.numPairs - 1) / p.numPairs;
    if (width < minWidth) width = minWidth;
    const long long per = (long long)p.numUnits * pr.batch;
    if (width > per) width = per;
    // equal chunks: a narrow last chunk would start its heaviest items when everything else is about to finish
    const long long chunks = (per + width / 2) / width > 0 ? (per + width / 2) / width : 1;
    p.chunk = (int)((per + chunks - 1) / chunks);
  }
  return kOk;
}

}  // namespace tfa_b200
