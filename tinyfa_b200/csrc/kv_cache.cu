// The paged 8-bit K/V cache: block tables and slot maps (kv_cache_plan), and rows of K and V written into it (kv_cache_store).
//
// A cache is [numBlocks][Hkv][blockTokens][D] codes (int8 or e4m3) and one fp32 scale per (block, head); the value of a code is
// code * scale.  One (block, head) tile is contiguous and has one scale, which is what the attention kernel streams.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <float.h>

#include "../../include/tinyfa_b200.h"
#include "build_config.cuh"
#include "cta_scan.cuh"
#include "ptx_sm100.cuh"
#include "tfa_common.cuh"

namespace tfa_b200 {

bool aligned16(const void* p);  // c_abi.cu

namespace kvcache {

// ------------------------------------------------------------------------------------------------ tables and slots
struct PlanParams {
  int* table;  // [batch][width]
  const int* lens;
  const int* newLens;
  const unsigned char* finished;  // may be null
  int* freeBlocks;                // stack of free block ids, top at numFree - 1
  const int* numFree;
  long long* slots;  // [total]
  int* cu;           // [batch + 1]
  int* lensAfter;    // [batch]
  int* numFreeAfter;
  int batch, width, capacity, blockShift;
  long long total;
};

constexpr int kPlanThreads = 1024;

__device__ __forceinline__ int blocks_of(long long tokens, int shift) { return (int)((tokens + (1 << shift) - 1) >> shift); }
__device__ __forceinline__ long long length_before(const PlanParams& p, int b) {
  return min(max((long long)p.lens[b], 0ll), (long long)p.width << p.blockShift);
}

// Cell of the cache for packed row `row`, -1 for a row of no request or of one that was not served.
__device__ __forceinline__ long long slot_of_row(const PlanParams& p, long long row) {
  if (row >= p.cu[p.batch]) return -1;
  int lo = 0, hi = p.batch - 1;  // the request b with cu[b] <= row < cu[b + 1]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (row < p.cu[mid + 1]) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  const long long before = (p.finished != nullptr && p.finished[lo] != 0) ? 0 : length_before(p, lo);
  if (p.lensAfter[lo] == before) return -1;  // the row exists, so its request asked for tokens: it was not served
  const long long place = before + (row - p.cu[lo]);
  const int block = p.table[(long long)lo * p.width + (place >> p.blockShift)];
  return block < 0 ? -1 : ((long long)block << p.blockShift) + (place & ((1 << p.blockShift) - 1));
}

// One CTA: two prefix sums over the requests (blocks given back, blocks and rows asked for), the stack and the tables; the slots
// too where they are few.  Integers only; bound by latency of a handful of dependent reads.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p, bool withSlots) {
  __shared__ long long sWarp[32];
  const int lane = threadIdx.x & 31;
  ptx::grid_wait_previous();
  ptx::grid_allow_next();
  const long long free0 = min(max((long long)*p.numFree, 0ll), (long long)p.capacity);
  // blocks of finished requests go on top of the stack, in the order of the requests
  long long returned = 0;
  if (p.finished != nullptr) {
    for (int b0 = 0; b0 < p.batch; b0 += kPlanThreads) {
      const int b = b0 + threadIdx.x;
      const int n = (b < p.batch && p.finished[b] != 0) ? blocks_of(length_before(p, b), p.blockShift) : 0;
      long long sum;
      const long long at = free0 + returned + cta_scan(n, sWarp, sum) - n;
      for (unsigned todo = __ballot_sync(0xffffffffu, n > 0); todo != 0; todo &= todo - 1) {
        const int who = __ffs(todo) - 1;
        const int bw = __shfl_sync(0xffffffffu, b, who), nw = __shfl_sync(0xffffffffu, n, who);
        const long long aw = __shfl_sync(0xffffffffu, at, who);
        for (int i = lane; i < nw; i += 32) {
          if (aw + i < p.capacity) p.freeBlocks[aw + i] = p.table[(long long)bw * p.width + i];
        }
      }
      returned += sum;
    }
    __syncthreads();
  }
  const long long have = min(free0 + returned, (long long)p.capacity);
  // every request takes its new blocks from the top; one that finds too few, or whose row of the table is too short, keeps its length
  long long taken = 0, asked = 0, rows = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    long long before = 0, fresh = 0;
    int held = 0, need = 0;
    bool fits = true;
    if (b < p.batch) {
      before = (p.finished != nullptr && p.finished[b] != 0) ? 0 : length_before(p, b);
      fresh = max(p.newLens[b], 0);
      held = blocks_of(before, p.blockShift);
      fits = before + fresh <= ((long long)p.width << p.blockShift);
      need = fits ? blocks_of(before + fresh, p.blockShift) - held : 0;
    }
    long long sum, sumRows, sumTaken;
    const long long upto = asked + cta_scan(need, sWarp, sum);
    const long long row = rows + cta_scan(fresh, sWarp, sumRows);
    const bool served = fits && (need == 0 || upto <= have);
    cta_scan(served ? need : 0, sWarp, sumTaken);
    if (b < p.batch) {
      p.cu[b + 1] = (int)row;
      p.lensAfter[b] = (int)(served ? before + fresh : before);
    }
    const int n = served ? need : 0;
    const long long top = have - 1 - (upto - need);
    for (unsigned todo = __ballot_sync(0xffffffffu, n > 0); todo != 0; todo &= todo - 1) {
      const int who = __ffs(todo) - 1;
      const int bw = __shfl_sync(0xffffffffu, b, who), nw = __shfl_sync(0xffffffffu, n, who), hw = __shfl_sync(0xffffffffu, held, who);
      const long long tw = __shfl_sync(0xffffffffu, top, who);
      for (int i = lane; i < nw; i += 32) p.table[(long long)bw * p.width + hw + i] = p.freeBlocks[tw - i];
    }
    asked += sum;
    rows += sumRows;
    taken += sumTaken;
  }
  if (threadIdx.x == 0) {
    p.cu[0] = 0;
    *p.numFreeAfter = (int)(have - taken);
  }
  if (!withSlots) return;
  __syncthreads();
  for (long long row = threadIdx.x; row < p.total; row += kPlanThreads) p.slots[row] = slot_of_row(p, row);
}

__global__ void __launch_bounds__(256) slots_kernel(const PlanParams p) {
  ptx::grid_wait_previous();
  ptx::grid_allow_next();
  const long long row = (long long)blockIdx.x * 256 + threadIdx.x;
  if (row < p.total) p.slots[row] = slot_of_row(p, row);
}

// ------------------------------------------------------------------------------------------------------------ store
struct StoreParams {
  const void* x[2];      // K and V [rows][heads][D]
  uint8_t* codes[2];     // [numBlocks][heads][blockTokens][D]
  float* scales[2];      // [numBlocks][heads]
  const long long* slots;
  long long rows, cells;  // cells = numBlocks << blockShift
  int heads, headDim, blockShift, rowsPerCta;
};

constexpr int kStoreThreads = 128;
constexpr float kTinyScale = 1.17549435e-38f;  // 2^-126: the smallest scale of a block that holds anything but zeros

template <typename T>
__device__ __forceinline__ void load8(const T* src, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(src);
    const T* t = reinterpret_cast<const T*>(&a);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = static_cast<float>(t[i]);
  }
}

// x * num / den rounded to a code; beyond the largest code it is the largest code, a NaN is stored as zero.  The scale is den / num: given
// as two numbers, because a scale max |x| / 448 that is rounded before the division would move quotients off the border between two
// codes, where many lie.  (num x is exact for 16-bit x.)
template <bool kInt8>
__device__ __forceinline__ uint2 to_codes(const float (&x)[8], float num, float den) {
  uint2 out;
  uint8_t* c = reinterpret_cast<uint8_t*>(&out);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float q[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const float top = kInt8 ? 127.f : 448.f;
      q[j] = den > 0.f ? __fdiv_rn(x[i + j] * num, den) : 0.f;
      q[j] = (q[j] != q[j]) ? 0.f : fminf(fmaxf(q[j], -top), top);
    }
    if constexpr (kInt8) {
      c[i] = (uint8_t)(int8_t)__float2int_rn(q[0]);
      c[i + 1] = (uint8_t)(int8_t)__float2int_rn(q[1]);
    } else {
      *reinterpret_cast<__nv_fp8x2_storage_t*>(c + i) = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
    }
  }
  return out;
}

template <bool kInt8>
__device__ __forceinline__ void from_codes(uint2 in, float (&x)[8]) {
  const uint8_t* c = reinterpret_cast<const uint8_t*>(&in);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    if constexpr (kInt8) {
      x[i] = (float)(int8_t)c[i];
    } else {
      x[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw(c[i], __NV_E4M3)));
    }
  }
}

// One head of K or V (blockIdx.z) and rowsPerCta rows; the CTA that has the first row of a run of rows in one block does the run.
//   need = max |x| / largest code over the run's finite values;  scale' = max(scale before, need);  code = round(x / scale'),
// and codes that were in the block before are rounded anew where the scale grew: code' = round(code * scale / scale').  A run that begins
// at the block's first cell begins the block: what its scale was before says nothing.  Bound by memory (the rows once, the codes once;
// the second look at the rows comes from L2 or nearer).  All quotients are IEEE divisions, so that codes do not depend on how they are computed.
template <typename T, bool kInt8>
__global__ void __launch_bounds__(kStoreThreads) store_kernel(const StoreParams p) {
  __shared__ float sMax[kStoreThreads / 32];
  ptx::grid_wait_previous();
  ptx::grid_allow_next();
  const int h = blockIdx.y, which = blockIdx.z;
  const T* x = static_cast<const T*>(p.x[which]) + (long long)h * p.headDim;
  const long long rowStride = (long long)p.heads * p.headDim;
  const int chunks = p.headDim / 8, blockTokens = 1 << p.blockShift;
  auto block_of = [&](long long row) -> long long {  // -1: the row goes nowhere
    const long long s = p.slots[row];
    return (s < 0 || s >= p.cells) ? -1 : s >> p.blockShift;
  };
  const long long r0 = (long long)blockIdx.x * p.rowsPerCta, r1 = min(r0 + p.rowsPerCta, p.rows);
  long long before = r0 > 0 ? block_of(r0 - 1) : -1;
  for (long long r = r0; r < r1; r++) {
    const long long block = block_of(r);
    const bool begins = block >= 0 && block != before;
    before = block;
    if (!begins) continue;
    int n = 1;  // rows of the run; more than the block has cells only if a cell comes twice
    while (r + n < p.rows && n < blockTokens && block_of(r + n) == block) n++;
    const int first = (int)(p.slots[r] & (blockTokens - 1));
    float top = 0.f;
    for (int i = threadIdx.x; i < n * chunks; i += kStoreThreads) {
      float v[8];
      load8(x + (r + i / chunks) * rowStride + (i % chunks) * 8, v);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float a = fabsf(v[j]);
        if (a <= FLT_MAX) top = fmaxf(top, a);
      }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    __syncthreads();  // the run before may still read sMax
    if ((threadIdx.x & 31) == 0) sMax[threadIdx.x >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(sMax[0], sMax[1]), fmaxf(sMax[2], sMax[3]));
    float* scaleAt = p.scales[which] + block * p.heads + h;
    const float old = first == 0 ? 0.f : *scaleAt;
    const float need = top > 0.f ? fmaxf(__fdiv_rn(top, kInt8 ? 127.f : 448.f), kTinyScale) : 0.f;
    const float scale = fmaxf(old, need);
    // the scale is this run's (and not rounded up to a normal number, nor its numerator out of range)
    const bool fromRun = need >= old && need > kTinyScale && top <= 1e35f;
    const float num = fromRun ? (kInt8 ? 127.f : 448.f) : 1.f, den = fromRun ? top : scale;
    uint8_t* tile = p.codes[which] + ((block * p.heads + h) << p.blockShift) * p.headDim;
    for (int i = threadIdx.x; i < n * chunks; i += kStoreThreads) {
      const int cell = (int)(p.slots[r + i / chunks] & (blockTokens - 1));
      float v[8];
      load8(x + (r + i / chunks) * rowStride + (i % chunks) * 8, v);
      *reinterpret_cast<uint2*>(tile + (long long)cell * p.headDim + (i % chunks) * 8) = to_codes<kInt8>(v, num, den);
    }
    if (scale != old || first == 0) {
      for (int i = threadIdx.x; i < first * chunks; i += kStoreThreads) {
        uint2* at = reinterpret_cast<uint2*>(tile + i * 8);
        float v[8];
        from_codes<kInt8>(*at, v);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] *= old;
        *at = to_codes<kInt8>(v, num, den);
      }
      __syncthreads();  // every thread has read the scale
      if (threadIdx.x == 0) *scaleAt = scale;
    }
  }
}

template <typename T>
cudaError_t launch_store(const StoreParams& p, bool int8, dim3 grid, cudaStream_t stream) {
  auto kernel = int8 ? store_kernel<T, true> : store_kernel<T, false>;
  return launch_kernel(kernel, grid, kStoreThreads, 0, stream, may_overlap(stream), p);
}

int block_shift(int blockTokens) {
  switch (blockTokens) {
    case 16: return 4;
    case 32: return 5;
    case 64: return 6;
    case 128: return 7;
    default:
      set_error_string("blocks hold 16, 32, 64 or 128 tokens (got %d)", blockTokens);
      return -1;
  }
}

}  // namespace kvcache
}  // namespace tfa_b200

using namespace tfa_b200;

extern "C" int tfa_b200_kv_cache_plan(int* blockTable, const int* seqLens, const int* newLens, const unsigned char* finished, int* freeBlocks,
                                      const int* numFree, long long* slots, int* cuSeqLens, int* seqLensAfter, int* numFreeAfter, int batchSize,
                                      int maxBlocks, int freeCapacity, int blockTokens, long long totalNew, void* stream) {
  using namespace kvcache;
  const int shift = block_shift(blockTokens);
  if (shift < 0) return kBadArgument;
  if (batchSize < 0 || maxBlocks < 0 || freeCapacity < 0 || totalNew < 0) {
    set_error_string("negative size (batch=%d maxBlocks=%d freeCapacity=%d totalNew=%lld)", batchSize, maxBlocks, freeCapacity, totalNew);
    return kBadArgument;
  }
  if (totalNew > 0x7FFFFFFFll || ((long long)maxBlocks << shift) > 0x7FFFFFFFll) {
    set_error_string("more than 2^31 - 1 rows or tokens of a request");
    return kTooLarge;
  }
  if (numFree == nullptr || cuSeqLens == nullptr || numFreeAfter == nullptr || (totalNew > 0 && slots == nullptr) ||
      (batchSize > 0 && (seqLens == nullptr || newLens == nullptr || seqLensAfter == nullptr)) ||
      (batchSize > 0 && maxBlocks > 0 && blockTable == nullptr) || (freeCapacity > 0 && freeBlocks == nullptr)) {
    set_error_string("null pointer");
    return kBadArgument;
  }
  int rc = check_device();
  if (rc != kOk) return rc;
  PlanParams p = {blockTable, seqLens,      newLens,   finished,  freeBlocks,   numFree, slots,   cuSeqLens, seqLensAfter,
                  numFreeAfter, batchSize, maxBlocks, freeCapacity, shift, totalNew};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool overlap = may_overlap(s);
  const bool few = totalNew <= kPlanThreads;  // more rows than the CTA has threads: a kernel of as many CTAs as they need
  cudaError_t e = launch_kernel(plan_kernel, dim3(1), kPlanThreads, 0, s, overlap, p, few);
  if (e == cudaSuccess && !few) e = launch_kernel(slots_kernel, dim3((unsigned)((totalNew + 255) / 256)), 256, 0, s, overlap, p);
  if (e != cudaSuccess) {
    set_error_string("cache plan kernel launch failed: %s", cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

extern "C" int tfa_b200_kv_cache_store(const void* K, const void* V, void* kCache, void* vCache, float* kScales, float* vScales, const long long* slots,
                                       int dtype, int cacheType, long long totalNew, int numBlocks, int numHeadsKV, int headDim, int blockTokens,
                                       void* stream) {
  using namespace kvcache;
  int rc = validate_common(K, K, V, kCache, dtype, totalNew > 0 ? 1 : 0, 1, 1, numHeadsKV, numHeadsKV, headDim);
  if (rc != kOk) return rc;
  const int shift = block_shift(blockTokens);
  if (shift < 0) return kBadArgument;
  if (cacheType != TFA_B200_CACHE_INT8 && cacheType != TFA_B200_CACHE_E4M3) {
    set_error_string("unsupported cache type %d (1 = int8, 2 = e4m3)", cacheType);
    return kBadDtype;
  }
  if (totalNew < 0 || numBlocks < 0) {
    set_error_string("negative size (totalNew=%lld numBlocks=%d)", totalNew, numBlocks);
    return kBadArgument;
  }
  if (totalNew == 0 || numBlocks == 0) return kOk;
  if (vCache == nullptr || kScales == nullptr || vScales == nullptr || slots == nullptr) {
    set_error_string("null pointer");
    return kBadArgument;
  }
  if (!aligned16(vCache)) {
    set_error_string("K, V and the caches must be 16-byte aligned");
    return kBadArgument;
  }
  if (totalNew > 0x7FFFFFFFll) {
    set_error_string("more than 2^31 - 1 rows");
    return kTooLarge;
  }
  if ((rc = check_device()) != kOk) return rc;
  StoreParams p;
  p.x[0] = K, p.x[1] = V;
  p.codes[0] = static_cast<uint8_t*>(kCache), p.codes[1] = static_cast<uint8_t*>(vCache);
  p.scales[0] = kScales, p.scales[1] = vScales;
  p.slots = slots;
  p.rows = totalNew;
  p.cells = (long long)numBlocks << shift;
  p.heads = numHeadsKV;
  p.headDim = headDim;
  p.blockShift = shift;
  // Few rows are mostly runs of one row (a decode step), a CTA each; of many, sixteen rows hold the beginning of one run or two.
  p.rowsPerCta = totalNew <= 512 ? 1 : 16;
  const dim3 grid((unsigned)((totalNew + p.rowsPerCta - 1) / p.rowsPerCta), (unsigned)numHeadsKV, 2);
  const bool int8 = cacheType == TFA_B200_CACHE_INT8;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == kFp32   ? launch_store<float>(p, int8, grid, s)
                        : dtype == kBf16 ? launch_store<__nv_bfloat16>(p, int8, grid, s)
                                         : launch_store<__half>(p, int8, grid, s);
  if (e != cudaSuccess) {
    set_error_string("cache store kernel launch failed: %s", cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}
