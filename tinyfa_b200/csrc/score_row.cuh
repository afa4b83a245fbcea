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

// All lanes of a warp call it for the same row (batch entry x seqLenQ + query, head).  A lane scores every 32nd key and owns every 32nd column
// of O.  Columns that are finite in memory stay as they are.  A value of V that the row does see stays what it is: the row ends
// where no column can become finite any more.
template <class T, int D>
__device__ __forceinline__ void exact_row(const ScoreFields& f, long long row, int head, void* O) {
  const int lane = threadIdx.x & 31;
  const ScoreSource& s = f.src;
  const int b = (int)(row / s.seqLenQ), pos = f.qStart + (int)(row - (long long)b * s.seqLenQ);
  const long long kvStride = (long long)s.headsKV * D;
  const T* q = static_cast<const T*>(s.q) + (row * s.headsQ + head) * D;
  const long long kv0 = (long long)b * s.seqLenKV * kvStride + (long long)(head / (s.headsQ / s.headsKV)) * D;
  const T* k = static_cast<const T*>(s.k) + kv0;
  const T* v = static_cast<const T*>(s.v) + kv0;
  int end = s.seqLenKV;
  if (s.causal) end = min(end, max(pos, f.prefix != nullptr ? f.prefix[b] - 1 : -1) + 1);
  const int doc = f.docQ != nullptr ? f.docQ[row] : 0;
  const float scale = rsqrtf((float)D), slope = f.slopes != nullptr ? f.slopes[head] : 0.f;
  float acc[D / 32], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; i++) acc[i] = 0.f;
#pragma unroll 1
  for (int k0 = 0; k0 < end; k0 += 32) {
    const int key = k0 + lane;
    const bool see = key < end && (f.docQ == nullptr || (doc >= 0 && f.docKV[(long long)b * s.seqLenKV + key] == doc));
    unsigned left = __ballot_sync(0xffffffffu, see);
    if (left == 0u) continue;
    float x = -INFINITY;
    if (see) {
      x = 0.f;
#pragma unroll 4
      for (int d = 0; d < D; d++) x = fmaf(to_float(q[d]), to_float(k[key * kvStride + d]), x);
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
    for (int i = 0; i < D / 32; i++) acc[i] *= fade;
#pragma unroll 1
    for (; left != 0u; left &= left - 1) {
      const int j = __ffs(left) - 1;
      const float w = __shfl_sync(0xffffffffu, weight, j);
#pragma unroll
      for (int i = 0; i < D / 32; i++) acc[i] = fmaf(w, to_float(v[(k0 + j) * kvStride + lane + 32 * i]), acc[i]);
    }
    bool some = false;
#pragma unroll
    for (int i = 0; i < D / 32; i++) some |= finite(acc[i]);
    if (!__any_sync(0xffffffffu, some)) break;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  T* out = static_cast<T*>(O) + (row * s.headsQ + head) * D;
#pragma unroll
  for (int i = 0; i < D / 32; i++) {
    if (!finite(to_float(out[lane + 32 * i]))) from_float(out[lane + 32 * i], acc[i] / l);
  }
}

// Rows of a warp's lanes, each bad or not: computes those that are.  Rows that several lanes name are computed once.
template <class T, int D>
__device__ __forceinline__ void exact_rows(const ScoreFields& f, bool bad, long long row, int head, void* O) {
  unsigned left = __ballot_sync(0xffffffffu, bad);
  if (left == 0u) return;
  __syncwarp();  // what the lanes have stored
#pragma unroll 1
  while (left != 0u) {
    const int j = __ffs(left) - 1;
    const long long r = __shfl_sync(0xffffffffu, row, j);
    const int h = __shfl_sync(0xffffffffu, head, j);
    exact_row<T, D>(f, r, h, O);
    left &= ~__ballot_sync(0xffffffffu, row == r && head == h);
  }
}

}  // namespace score
}  // namespace tfa_b200
