// The paged 8-bit K/V cache: block tables and slot maps (kv_cache_plan), and rows of K and V written into it (kv_cache_store).
//
// A cache is [numBlocks][Hkv][blockTokens][D] codes (int8 or e4m3) and one fp32 scale per (block, head); the value of a code is
// code * scale.  One (block, head) tile is contiguous and has one scale, which is what the attention kernel streams.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/tinyfa_b200.h"
#include "build_config.cuh"
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

// Cell of the cache for packed row `row`, -1 for a row of no request or of one that was not served.  cu: p.cu or a copy of it.
__device__ __forceinline__ long long slot_of_row(const PlanParams& p, const int* cu, long long row) {
  if (row >= cu[p.batch]) return -1;
  int lo = 0, hi = p.batch - 1;  // the request b with cu[b] <= row < cu[b + 1]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (row < cu[mid + 1]) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  const int after = p.lensAfter[lo];
  const long long length = length_before(p, lo), before = (p.finished != nullptr && p.finished[lo] != 0) ? 0 : length;
  if (after == before) return -1;  // the row exists, so its request asked for tokens: it was not served
  const long long place = before + (row - cu[lo]);
  if (place < 0 || place >= (long long)p.width << p.blockShift) return -1;  // (rows of lengths whose sum does not fit 32 bits)
  const int block = p.table[(long long)lo * p.width + (place >> p.blockShift)];
  return block < 0 ? -1 : ((long long)block << p.blockShift) + (place & ((1 << p.blockShift) - 1));
}

// Inclusive sums of two values over the CTA, whose first threads have values other than zero.
__device__ __forceinline__ void cta_scan2(int& a, long long& b, int (&sA)[32], long long (&sB)[32], int& totalA, long long& totalB) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, a, d);
    const long long y = __shfl_up_sync(0xffffffffu, b, d);
    if (lane >= d) {
      a += x;
      b += y;
    }
  }
  if (lane == 31) {
    sA[warp] = a;
    sB[warp] = b;
  }
  __syncthreads();
  int wa = lane < warps ? sA[lane] : 0;  // every warp sums the warps' totals for itself
  long long wb = lane < warps ? sB[lane] : 0;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, wa, d);
    const long long y = __shfl_up_sync(0xffffffffu, wb, d);
    if (lane >= d) {
      wa += x;
      wb += y;
    }
  }
  totalA = __shfl_sync(0xffffffffu, wa, 31);
  totalB = __shfl_sync(0xffffffffu, wb, 31);
  const int beforeA = __shfl_sync(0xffffffffu, wa, (warp + 31) & 31);
  const long long beforeB = __shfl_sync(0xffffffffu, wb, (warp + 31) & 31);
  if (warp > 0) {
    a += beforeA;
    b += beforeB;
  }
}

// One CTA: two prefix sums over the requests (blocks given back, blocks and rows asked for), the stack and the tables; the slots
// too where they are few.  Integers only; bound by the latency of a handful of dependent reads: what does not depend on another read is asked for at
// once, a request's first new block is its thread's, further ones a warp's, and rows look for their request in shared memory.
// 256 requests of one token: 11 us on the device (15 with the requests handed to the warps one by one and a search in global memory); 64 of up to 2000
// tokens, 20 % of them finished: 16, and 4 for the slots.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p, bool withSlots) {
  __shared__ int sA[2][32];
  __shared__ long long sB[2][32];
  __shared__ int sCount[kPlanThreads], sHeld[kPlanThreads];
  __shared__ int sTop[kPlanThreads];
  __shared__ int sCu[kPlanThreads + 1];
  __shared__ int sTaken;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, threads = blockDim.x;
  ptx::grid_wait_previous();
  ptx::grid_allow_next();
  if (threadIdx.x == 0) sTaken = 0;
  const int free0 = min(max(*p.numFree, 0), p.capacity);
  // the thread's request of the first round
  const bool mine = (int)threadIdx.x < p.batch;
  const long long length0 = mine ? length_before(p, threadIdx.x) : 0;
  const int fresh0 = mine ? max(p.newLens[threadIdx.x], 0) : 0;
  const bool finished0 = mine && p.finished != nullptr && p.finished[threadIdx.x] != 0;
  // blocks of finished requests go on top of the stack, in the order of the requests
  long long returned = 0;
  int turn = 0;  // which half of sA, sB: a warp may still read the other one
  if (p.finished != nullptr && __syncthreads_or(finished0 || p.batch > threads)) {
    for (int b0 = 0; b0 < p.batch; b0 += threads, turn ^= 1) {
      const int b = b0 + threadIdx.x;
      const bool ended = b0 == 0 ? finished0 : b < p.batch && p.finished[b] != 0;
      int n = ended ? blocks_of(b0 == 0 ? length0 : length_before(p, b), p.blockShift) : 0, none = 0;
      sCount[threadIdx.x] = n;
      long long upto = n, sum;
      cta_scan2(none, upto, sA[turn], sB[turn], none, sum);
      sTop[threadIdx.x] = (int)min(free0 + returned + upto - sCount[threadIdx.x], (long long)p.capacity);
      __syncthreads();
      // requests warp, warp + warps, ... are this warp's
      for (unsigned some = __ballot_sync(0xffffffffu, sCount[warp + lane * warps] > 0); some != 0; some &= some - 1) {
        const int r = warp + (__ffs(some) - 1) * warps, count = sCount[r], at = sTop[r];
#pragma unroll 4
        for (int i = lane; i < min(count, p.capacity - at); i += 32) p.freeBlocks[at + i] = p.table[(long long)(b0 + r) * p.width + i];
      }
      returned += sum;
      __syncthreads();
    }
  }
  const int have = (int)min(free0 + returned, (long long)p.capacity);
  // every request takes its new blocks from the top; one that finds too few, or whose row of the table is too short, keeps its length
  long long asked = 0, rows = 0;
  for (int b0 = 0; b0 < p.batch; b0 += threads, turn ^= 1) {
    const int b = b0 + threadIdx.x;
    long long before = 0, fresh = 0;
    int held = 0, need = 0;
    bool fits = true;
    if (b < p.batch) {
      if (b0 == 0) {
        before = finished0 ? 0 : length0;
        fresh = fresh0;
      } else {
        before = (p.finished != nullptr && p.finished[b] != 0) ? 0 : length_before(p, b);
        fresh = max(p.newLens[b], 0);
      }
      held = blocks_of(before, p.blockShift);
      fits = before + fresh <= ((long long)p.width << p.blockShift);
      need = fits ? blocks_of(before + fresh, p.blockShift) - held : 0;
    }
    int sum, inclusive = need;
    long long row = fresh, sumRows;
    cta_scan2(inclusive, row, sA[turn], sB[turn], sum, sumRows);
    const long long upto = asked + inclusive;
    const bool served = fits && (need == 0 || upto <= have);
    const int top = (int)(served ? have - 1 - (upto - need) : 0);
    if (b < p.batch) {
      const int end = (int)(rows + row);
      p.cu[b + 1] = end;
      if (b0 == 0) sCu[b + 1] = end;
      p.lensAfter[b] = (int)(served ? before + fresh : before);
      if (served && need > 0) {
        p.table[(long long)b * p.width + held] = p.freeBlocks[top];
        atomicMax(&sTaken, (int)upto);  // the served ones are those that ask for no more than there is
      }
    }
    sCount[threadIdx.x] = served ? need : 0;
    sHeld[threadIdx.x] = held;
    sTop[threadIdx.x] = top;
    if (__syncthreads_or(served && need > 1)) {
      for (unsigned some = __ballot_sync(0xffffffffu, sCount[warp + lane * warps] > 1); some != 0; some &= some - 1) {
        const int r = warp + (__ffs(some) - 1) * warps, count = sCount[r], first = sTop[r];
        int* row0 = p.table + (long long)(b0 + r) * p.width + sHeld[r];
#pragma unroll 4
        for (int i = 1 + lane; i < count; i += 32) row0[i] = p.freeBlocks[first - i];
      }
    }
    asked += sum;
    rows += sumRows;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    p.cu[0] = sCu[0] = 0;
    *p.numFreeAfter = have - sTaken;
  }
  if (!withSlots) return;
  __syncthreads();
  const int* cu = p.batch <= threads ? sCu : p.cu;
  for (long long row = threadIdx.x; row < p.total; row += threads) p.slots[row] = slot_of_row(p, cu, row);
}

__global__ void __launch_bounds__(256) slots_kernel(const PlanParams p) {
  __shared__ int sCu[kPlanThreads + 1];
  ptx::grid_wait_previous();
  ptx::grid_allow_next();
  const bool few = p.batch <= kPlanThreads;
  if (few) {
    for (int i = threadIdx.x; i <= p.batch; i += 256) sCu[i] = p.cu[i];
    __syncthreads();
  }
  const long long row = (long long)blockIdx.x * 256 + threadIdx.x;
  if (row < p.total) p.slots[row] = slot_of_row(p, few ? sCu : p.cu, row);
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
struct Eight {  // eight elements as they come from memory
  uint4 raw[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* src) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) raw[i] = reinterpret_cast<const uint4*>(src)[i];
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    if constexpr (sizeof(T) == 4) {
      v[0] = __uint_as_float(raw[0].x), v[1] = __uint_as_float(raw[0].y), v[2] = __uint_as_float(raw[0].z), v[3] = __uint_as_float(raw[0].w);
      v[4] = __uint_as_float(raw[1].x), v[5] = __uint_as_float(raw[1].y), v[6] = __uint_as_float(raw[1].z), v[7] = __uint_as_float(raw[1].w);
    } else {
      const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float2 f;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
        } else {
          f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        }
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
};

// x * num / den rounded to a code; beyond the largest code it is the largest code, a NaN is stored as zero.  The scale is den / num: given
// as two numbers, because a scale max |x| / 448 that is rounded before the division would move quotients off the border between two
// codes, where many lie.  (num x is exact for 16-bit x.)
template <bool kInt8>
__device__ __forceinline__ uint2 to_codes(const float (&x)[8], float num, float den) {
  uint32_t word[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    float q[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float top = kInt8 ? 127.f : 448.f;
      q[j] = den > 0.f ? __fdiv_rn(x[h * 4 + j] * num, den) : 0.f;
      q[j] = (q[j] != q[j]) ? 0.f : fminf(fmaxf(q[j], -top), top);
    }
    if constexpr (kInt8) {
      uint32_t c[4];
#pragma unroll
      for (int j = 0; j < 4; j++) c[j] = (uint32_t)__float2int_rn(q[j]);
      word[h] = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    } else {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3);
      word[h] = lo | hi << 16;
    }
  }
  return make_uint2(word[0], word[1]);
}

// The same codes by multiplication: q = x * inv is within 5 x 2^-24 of the quotient, so a code that does not change within 2^-21 of q is the
// quotient's.  False where one of the eight is that near the border between two codes (about one in 10^4 eights of random values); x is finite.
template <bool kInt8>
__device__ __forceinline__ bool quick_codes(const float (&x)[8], float inv, uint2& out) {
  uint32_t word[2];
  bool certain = true;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    float q[4];
#pragma unroll
    for (int j = 0; j < 4; j++) q[j] = x[h * 4 + j] * inv;
    if constexpr (kInt8) {
      constexpr float kRound = 12582912.f;  // 1.5 x 2^23: added, it leaves the nearest integer in the low bits
      uint32_t c[4];
      float far = 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float r = __fadd_rn(q[j], kRound);
        c[j] = __float_as_uint(r);
        far = fmaxf(far, fabsf(q[j] - __fsub_rn(r, kRound)));
      }
      certain = certain && far < 0.4999f;  // 127 x 2^-21 from the border at least
      word[h] = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    } else {
      constexpr float kLess = 1.f - 0x1p-21f, kMore = 1.f + 0x1p-21f;
      uint32_t both[2];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const uint32_t less = __nv_cvt_float2_to_fp8x2(make_float2(q[2 * j] * kLess, q[2 * j + 1] * kLess), __NV_SATFINITE, __NV_E4M3);
        both[j] = __nv_cvt_float2_to_fp8x2(make_float2(q[2 * j] * kMore, q[2 * j + 1] * kMore), __NV_SATFINITE, __NV_E4M3);
        certain = certain && less == both[j];
      }
      word[h] = both[0] | both[1] << 16;
    }
  }
  out = make_uint2(word[0], word[1]);
  return certain;
}

template <bool kInt8>
__device__ __forceinline__ void from_codes(uint2 in, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t c = ((i < 4 ? in.x : in.y) >> (i % 4 * 8)) & 0xFFu;
    if constexpr (kInt8) {
      x[i] = (float)(int8_t)c;
    } else {
      x[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
    }
  }
}

// Largest |x| of elements as they come; +inf where one is not finite.
template <typename T>
struct Largest {
  float top = 0.f;
  __device__ __forceinline__ void add(const Eight<T>& e) {
    float v[8];
    e.values(v);
#pragma unroll
    for (int j = 0; j < 8; j++) top = fabsf(v[j]) <= FLT_MAX ? fmaxf(top, fabsf(v[j])) : INFINITY;
  }
  __device__ __forceinline__ float get() const { return top; }
};
template <typename T2, typename T>
struct LargestPair {  // 16-bit types: two at a time, NaN stays
  T2 top;
  __device__ __forceinline__ LargestPair() {
    const uint32_t zero = 0;
    top = *reinterpret_cast<const T2*>(&zero);
  }
  __device__ __forceinline__ void add(const Eight<T>& e) {
    const uint32_t w[4] = {e.raw[0].x, e.raw[0].y, e.raw[0].z, e.raw[0].w};
#pragma unroll
    for (int i = 0; i < 4; i++) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const T2*>(&w[i])));
  }
  __device__ __forceinline__ float get() const {
    const float a = to_float(top.x), b = to_float(top.y);
    return a <= FLT_MAX && b <= FLT_MAX ? fmaxf(a, b) : INFINITY;
  }
  static __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
  static __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
};
template <>
struct Largest<__half> : LargestPair<__half2, __half> {};
template <>
struct Largest<__nv_bfloat16> : LargestPair<__nv_bfloat162, __nv_bfloat16> {};

// One head of K or V (blockIdx.z) and rowsPerCta rows; the CTA that has the first row of a run of rows in one block does the run, whose cells may
// come in any order; what is below the lowest of them was in the block before.
//   need = max |x| / largest code over the run's finite values;  scale' = max(scale before, need);  code = round(x / scale'),
// and codes that were in the block before are rounded anew where the scale grew: code' = round(code * scale / scale').  A run that begins
// at the block's first cell begins the block: what its scale was before says nothing.  Bound by memory (the rows once, the codes once;
// the second look at the rows comes from registers, or from L2 behind 64 rows of 128).  Codes are those of IEEE divisions, whichever way they are computed.  8
// prompts, 8.4 k rows of 8 heads of 128, bf16 to e4m3: 24 us (a division for every element 34, the parameters in local memory as well 42).
template <typename T, bool kInt8, int D>
__global__ void __launch_bounds__(kStoreThreads) store_kernel(const StoreParams p) {
  constexpr int kChunks = D / 8, kWarps = kStoreThreads / 32;
  constexpr int kKept = 8;  // eights of a run that a thread keeps between the two looks: 64 rows of 128 elements; longer runs are read again
  __shared__ float sMax[kWarps];
  __shared__ int sEnd[kWarps], sLowest[kWarps];
  __shared__ int sCells[kStoreThreads];  // cells of the run's rows
  const int h = blockIdx.y, which = blockIdx.z, lane = threadIdx.x & 31;
  const int blockTokens = 1 << p.blockShift;
  ptx::grid_wait_previous();
  ptx::grid_allow_next();
  const bool second = which != 0;  // (indexing the parameters by it would copy them to local memory)
  const T* x = static_cast<const T*>(second ? p.x[1] : p.x[0]) + (long long)h * D;
  const long long rowStride = (long long)p.heads * D;
  auto block_of = [&](long long row) -> int {  // -1: the row goes nowhere
    if (row < 0 || row >= p.rows) return -1;
    const long long s = p.slots[row];
    return (s < 0 || s >= p.cells) ? -1 : (int)(s >> p.blockShift);
  };
  // which of the CTA's rows (32 at most) begin a run: every warp finds out for itself
  const long long r0 = (long long)blockIdx.x * p.rowsPerCta;
  const int mine = lane < p.rowsPerCta ? block_of(r0 + lane) : -1;
  int before = __shfl_up_sync(0xffffffffu, mine, 1);
  if (lane == 0) before = block_of(r0 - 1);
  unsigned begins = __ballot_sync(0xffffffffu, mine >= 0 && mine != before);
  for (; begins != 0; begins &= begins - 1) {
    const int from = __ffs(begins) - 1;
    const long long r = r0 + from;
    const int block = __shfl_sync(0xffffffffu, mine, from);
    // the run ends with the first row of another block; more rows than the block has cells only if a cell comes twice
    __syncthreads();  // the run before may still read sCells, sEnd and sMax
    bool other = (int)threadIdx.x >= blockTokens;
    int cell = blockTokens;
    if (!other) {
      other = block_of(r + threadIdx.x) != block;
      cell = other ? -1 : (int)(p.slots[r + threadIdx.x] & (blockTokens - 1));
      sCells[threadIdx.x] = cell;
    }
    // kStoreThreads rows are looked at, and a run has blockTokens <= kStoreThreads at most
    const unsigned others = __ballot_sync(0xffffffffu, other);
    const int mineEnd = others != 0 ? __ffs(others) - 1 : 32;  // lanes of the run, where it gets as far as this warp
    const int lowest = __reduce_min_sync(0xffffffffu, lane < mineEnd ? cell : blockTokens);
    if (lane == 0) {
      sEnd[threadIdx.x >> 5] = others != 0 ? (int)(threadIdx.x & ~31) + mineEnd : kStoreThreads;
      sLowest[threadIdx.x >> 5] = lowest;
    }
    __syncthreads();
    int n = kStoreThreads, first = blockTokens;  // rows of the run and its first cell: rows may come in any order of their cells
#pragma unroll
    for (int w = 0; w < kWarps; w++) n = min(n, sEnd[w]);
#pragma unroll
    for (int w = 0; w < kWarps; w++) first = w * 32 < n ? min(first, sLowest[w]) : first;
    const int items = n * kChunks;
    Eight<T> kept[kKept];
    auto at = [&](int i) { return x + (r + i / kChunks) * rowStride + i % kChunks * 8; };
    // maximum over the CTA's threads of a number that is not negative
    auto cta_max = [&](float v) {
      const unsigned m = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
      if (lane == 0) sMax[threadIdx.x >> 5] = __uint_as_float(m);
      __syncthreads();
      float all = sMax[0];
#pragma unroll
      for (int w = 1; w < kWarps; w++) all = fmaxf(all, sMax[w]);
      return all;
    };
    Largest<T> largest;
#pragma unroll
    for (int e = 0; e < kKept; e++) {
      const int i = threadIdx.x + e * kStoreThreads;
      if (i < items) kept[e].load(at(i));
    }
#pragma unroll
    for (int e = 0; e < kKept; e++) {
      if ((int)threadIdx.x + e * kStoreThreads < items) largest.add(kept[e]);
    }
#pragma unroll 4
    for (int i = threadIdx.x + kKept * kStoreThreads; i < items; i += kStoreThreads) {
      Eight<T> e;
      e.load(at(i));
      largest.add(e);
    }
    float top = cta_max(largest.get());
    const bool clean = top <= FLT_MAX;
    if (!clean) {  // the largest finite one
      top = 0.f;
#pragma unroll 1
      for (int i = threadIdx.x; i < items; i += kStoreThreads) {
        Eight<T> e;
        e.load(at(i));
        float v[8];
        e.values(v);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          if (fabsf(v[j]) <= FLT_MAX) top = fmaxf(top, fabsf(v[j]));
        }
      }
      __syncthreads();  // sMax is written again
      top = cta_max(top);
    }
    float* scaleAt = (second ? p.scales[1] : p.scales[0]) + (long long)block * p.heads + h;
    const float old = first == 0 ? 0.f : *scaleAt;
    const float need = top > 0.f ? fmaxf(__fdiv_rn(top, kInt8 ? 127.f : 448.f), kTinyScale) : 0.f;
    const float scale = fmaxf(old, need);
    // the scale is this run's (and not rounded up to a normal number, nor its numerator out of range)
    const bool fromRun = need >= old && need > kTinyScale && top <= 1e35f;
    const float num = fromRun ? (kInt8 ? 127.f : 448.f) : 1.f, den = fromRun ? top : scale;
    uint8_t* tile = (second ? p.codes[1] : p.codes[0]) + (((long long)block * p.heads + h) << p.blockShift) * D;
    auto put = [&](int i, uint2 codes) { *reinterpret_cast<uint2*>(tile + sCells[i / kChunks] * D + i % kChunks * 8) = codes; };
    auto divide = [&](int i) {
      Eight<T> e;
      float v[8];
      e.load(at(i));
      e.values(v);
      put(i, to_codes<kInt8>(v, num, den));
    };
    const float inv = __fdiv_rn(num, den);
    if (clean && inv > 1e-30f && inv < 1e30f) {
      unsigned again = 0;  // eights that are divided
#pragma unroll
      for (int e = 0; e < kKept; e++) {
        const int i = threadIdx.x + e * kStoreThreads;
        if (i < items) {
          float v[8];
          uint2 codes;
          kept[e].values(v);
          if (!quick_codes<kInt8>(v, inv, codes)) again |= 1u << e;
          put(i, codes);
        }
      }
#pragma unroll 1
      for (; again != 0; again &= again - 1) divide(threadIdx.x + (__ffs(again) - 1) * kStoreThreads);
#pragma unroll 4
      for (int i = threadIdx.x + kKept * kStoreThreads; i < items; i += kStoreThreads) {
        Eight<T> e;
        float v[8];
        uint2 codes;
        e.load(at(i));
        e.values(v);
        if (!quick_codes<kInt8>(v, inv, codes)) codes = to_codes<kInt8>(v, num, den);
        put(i, codes);
      }
    } else {
#pragma unroll 1
      for (int i = threadIdx.x; i < items; i += kStoreThreads) divide(i);
    }
    if (scale != old || first == 0) {
      for (int i = threadIdx.x; i < first * kChunks; i += kStoreThreads) {
        uint2* cell = reinterpret_cast<uint2*>(tile + i * 8);
        float v[8];
        from_codes<kInt8>(*cell, v);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] *= old;
        *cell = to_codes<kInt8>(v, num, den);
      }
      __syncthreads();  // every thread has read the scale
      if (threadIdx.x == 0) *scaleAt = scale;
    }
  }
}

template <typename T, int D>
cudaError_t launch_store(const StoreParams& p, bool int8, dim3 grid, cudaStream_t stream) {
  auto kernel = int8 ? store_kernel<T, true, D> : store_kernel<T, false, D>;
  return launch_kernel(kernel, grid, kStoreThreads, 0, stream, may_overlap(stream), p);
}
template <typename T>
cudaError_t launch_store(const StoreParams& p, bool int8, dim3 grid, cudaStream_t stream) {
  switch (p.headDim) {
    case 32: return launch_store<T, 32>(p, int8, grid, stream);
    case 64: return launch_store<T, 64>(p, int8, grid, stream);
    case 96: return launch_store<T, 96>(p, int8, grid, stream);
    case 128: return launch_store<T, 128>(p, int8, grid, stream);
    case 192: return launch_store<T, 192>(p, int8, grid, stream);
    default: return launch_store<T, 256>(p, int8, grid, stream);
  }
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
  // slots are worked out from the lengths before and after
  const uintptr_t before = reinterpret_cast<uintptr_t>(seqLens), after = reinterpret_cast<uintptr_t>(seqLensAfter), bytes = sizeof(int) * (uintptr_t)batchSize;
  if (batchSize > 0 && before < after + bytes && after < before + bytes) {
    set_error_string("seqLens and seqLensAfter overlap");
    return kBadArgument;
  }
  int rc = check_device();
  if (rc != kOk) return rc;
  PlanParams p = {blockTable, seqLens,      newLens,   finished,  freeBlocks,   numFree, slots,   cuSeqLens, seqLensAfter,
                  numFreeAfter, batchSize, maxBlocks, freeCapacity, shift, totalNew};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool overlap = may_overlap(s);
  const bool few = totalNew <= kPlanThreads;  // more rows than the CTA has threads: a kernel of as many CTAs as they need
  const int threads = batchSize <= 256 && totalNew <= 256 ? 256 : kPlanThreads;  // fewer warps to wait for
  cudaError_t e = launch_kernel(plan_kernel, dim3(1), threads, 0, s, overlap, p, few);
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
  // Few rows are mostly runs of one row (a decode step), a CTA each; of many, sixteen (blocks of 64 or more: 32) rows hold the beginning of one
  // run or two.
  p.rowsPerCta = totalNew <= 512 ? 1 : shift >= 6 ? 32 : 16;
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
