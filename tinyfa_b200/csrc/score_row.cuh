// One output row of scored attention from its definition, for rows that the matrix products cannot give.
//
// The products multiply what a mask hides by a weight of zero, and 0 x NaN is NaN: an infinity or a NaN in V at a key that shares a block
// with the row's own keys spoils the row.  The kernels notice a value of the row that is not finite, although its sum of weights is, while they store it
// (one multiply-add a value), and have the warp compute the row again, key by key, reading only what the row sees.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "score.cuh"

namespace tfa_b200 {
namespace score {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_float(float& y, float x) { y = x; }
__device__ __forceinline__ void from_float(__half& y, float x) { y = __float2half_rn(x); }
__device__ __forceinline__ void from_float(__nv_bfloat16& y, float x) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// Eight elements of 16 bits or four of 32
template <class T>
__device__ __forceinline__ float dot16(uint4 a, uint4 b, float x) {
  const uint32_t p[4] = {a.x, a.y, a.z, a.w}, q[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(T) == 4) {
      x = fmaf(__uint_as_float(p[i]), __uint_as_float(q[i]), x);
    } else {
      const T* u = reinterpret_cast<const T*>(&p[i]);
      const T* v = reinterpret_cast<const T*>(&q[i]);
      x = fmaf(to_float(u[0]), to_float(v[0]), fmaf(to_float(u[1]), to_float(v[1]), x));
    }
  }
  return x;
}

// kDocs: calls with documents come here too (they have neither few rows nor key ranges).
// All lanes of a warp call it for the same row (batch entry x seqLenQ + query, head), of which some columns are not finite in memory; the others
// stay as they are.  A lane scores every 32nd key and owns every 32nd column of O.  A value of V that the row does see stays what it is: nothing is
// done where no hidden key near the row has such a value (only the causal mask: a tile reads no more than 255 keys past its rows'), and
// keys are taken from the last to the first until none of the columns can become finite any more.  Capped causal prefill 2 x 4096, 32 heads of 128,
// 0.4 ms: 1.9 with all of V NaN,
// 3.0 with one value a head at key 2048.
template <class T, int D, bool kDocs = true>
__device__ __forceinline__ void exact_row(const ScoreFields& f, long long row, int head, void* O) {
  constexpr int kCols = D / 32, kPer = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 31;
  const ScoreSource& s = f.src;
  const bool docs = kDocs && f.docQ != nullptr;
  if (!s.causal && !docs) return;  // nothing is hidden
  const int b = (int)(row / s.seqLenQ), pos = bias_position(f.qStart + (int)(row - (long long)b * s.seqLenQ), s.seqLenKV);
  const long long kvStride = (long long)s.headsKV * D;
  const T* q = static_cast<const T*>(s.q) + (row * s.headsQ + head) * D;
  const long long kv0 = (long long)b * s.seqLenKV * kvStride + (long long)(head / (s.headsQ / s.headsKV)) * D;
  const T* k = static_cast<const T*>(s.k) + kv0;
  const T* v = static_cast<const T*>(s.v) + kv0 + lane;
  T* out = static_cast<T*>(O) + (row * s.headsQ + head) * D + lane;
  float acc[kCols], m = -INFINITY, l = 0.f;
  unsigned spoilt = 0;  // this lane's columns that are not finite, as bits
#pragma unroll
  for (int i = 0; i < kCols; i++) {
    acc[i] = 0.f;
    if (!finite(to_float(out[32 * i]))) spoilt |= 1u << i;
  }
  int end = s.seqLenKV;
  if (s.causal) end = min(end, max(pos, f.prefix != nullptr ? prefix_of(f, b, s.seqLenKV) - 1 : -1) + 1);
  if (!docs) {
    bool hidden = false;
    // (with a prefix, whose length only the device knows, the decode kernel reads all keys)
    const int stop = f.prefix != nullptr ? s.seqLenKV : min(min(s.seqLenKV, f.qStart + s.seqLenQ), end + 256);
#pragma unroll 1
    for (int k0 = end; k0 < stop; k0 += 8) {
      float x[8][kCols];
#pragma unroll
      for (int j = 0; j < 8; j++) {
#pragma unroll
        for (int i = 0; i < kCols; i++) x[j][i] = to_float(v[min(k0 + j, stop - 1) * kvStride + 32 * i]);
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
#pragma unroll
        for (int i = 0; i < kCols; i++) hidden |= (spoilt >> i & 1u) != 0 && !finite(x[j][i]);
      }
      if (__any_sync(0xffffffffu, hidden)) break;
    }
    if (!__any_sync(0xffffffffu, hidden)) return;
  }
  const int doc = docs ? f.docQ[row] : 0;
  int low = 0;
  if (docs && f.rowKeys[row].x >= 0) {  // documents in ascending order
    low = f.rowKeys[row].x;
    end = min(end, f.rowKeys[row].y);
  }
  const float scale = rsqrtf((float)D), slope = f.slopes != nullptr ? f.slopes[head] : 0.f;
#pragma unroll 1
  for (int k0 = (end - 1) / 32 * 32; k0 >= low / 32 * 32; k0 -= 32) {
    const int key = k0 + lane;
    const bool see = key < end && (!docs || (doc >= 0 && f.docKV[(long long)b * s.seqLenKV + key] == doc));
    const unsigned seen = __ballot_sync(0xffffffffu, see);
    if (seen == 0u) continue;
    float x = -INFINITY;
    if (see) {
      const uint4* k16 = reinterpret_cast<const uint4*>(k + key * kvStride);
      x = 0.f;
#pragma unroll 4
      for (int d = 0; d < D / kPer; d++) x = dot16<T>(reinterpret_cast<const uint4*>(q)[d], k16[d], x);
      x *= scale;
      if (f.cap > 0.f) x = f.cap * tanhf(x / f.cap);
      x = fmaf(-slope, fabsf((float)(pos - key)), x) * 1.44269504f;
    }
    float most = fmaxf(m, x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const float ref = most == -INFINITY ? 0.f : most, fade = exp2f(m - ref), weight = exp2f(x - ref);
    m = most;
    l = l * fade + weight;  // of this lane's keys
#pragma unroll
    for (int i = 0; i < kCols; i++) acc[i] *= fade;
#pragma unroll 1
    for (int j0 = 0; j0 < 32; j0 += 8) {
      float x[8][kCols];
#pragma unroll
      for (int j = 0; j < 8; j++) {  // in the place of a key that is not seen one that is, with weight zero
        const T* at = v + (k0 + ((seen >> (j0 + j) & 1u) != 0 ? j0 + j : __ffs(seen) - 1)) * kvStride;
#pragma unroll
        for (int i = 0; i < kCols; i++) x[j][i] = to_float(at[32 * i]);
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float w = __shfl_sync(0xffffffffu, weight, j0 + j);
#pragma unroll
        for (int i = 0; i < kCols; i++) acc[i] = fmaf(w, x[j][i], acc[i]);
      }
    }
    bool some = false;
#pragma unroll
    for (int i = 0; i < kCols; i++) some |= (spoilt >> i & 1u) != 0 && finite(acc[i]);
    if (!__any_sync(0xffffffffu, some)) return;  // as they are
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
  for (int i = 0; i < kCols; i++) {
    if (spoilt >> i & 1u) from_float(out[32 * i], acc[i] / l);
  }
}

// Rows of a warp's lanes, each bad or not: computes those that are.  Rows that several lanes name are computed once.
template <class T, int D, bool kDocs = true>
__device__ __forceinline__ void exact_rows(const ScoreFields& f, bool bad, long long row, int head, void* O) {
  unsigned left = __ballot_sync(0xffffffffu, bad);
  if (left == 0u) return;
  __syncwarp();  // what the lanes have stored
#pragma unroll 1
  while (left != 0u) {
    const int j = __ffs(left) - 1;
    const long long r = __shfl_sync(0xffffffffu, row, j);
    const int h = __shfl_sync(0xffffffffu, head, j);
    exact_row<T, D, kDocs>(f, r, h, O);
    left &= ~__ballot_sync(0xffffffffu, row == r && head == h);
  }
}

}  // namespace score
}  // namespace tfa_b200
