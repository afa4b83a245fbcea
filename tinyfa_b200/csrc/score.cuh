// Attention whose scores are capped, biased or masked: what the kernels need to know of it.
//
//   S_ij = q_i . k_j / sqrt(D);  cap > 0: S <- cap tanh(S / cap);  slopes: S <- S - slope_h |pos_i - j|, pos_i = qStart + i
//   visible: (not causal, or j <= pos_i, or j < prefix_b) and (no documents, or docQ_i == docKV_j >= 0)
// A row that sees nothing is zero.
#pragma once

#include <cuda_runtime.h>

namespace tfa_b200 {

struct ScoreSource {  // the call's tensors, for rows that are computed one by one (score_row.cuh)
  const void *q, *k, *v;
  int seqLenQ, seqLenKV, headsQ, headsKV, causal;
};

struct ScoreFields {
  int qStart;           // position of query row 0
  float cap;            // 0: none
  const float* slopes;  // [headsQ] or null
  const int* prefix;    // [batch] or null
  const int* docQ;      // [batch][seqLenQ] or null
  const int* docKV;     // [batch][seqLenKV]
  // documents: smallest and largest id of every key block, the key blocks [x, y) that some row of a query tile may see, and the keys [x, y) of
  // every row's document (x below zero where keys are not in ascending order of documents)
  const int2* keyBlocks;  // [batch][key blocks]
  const int2* tileRange;  // [batch][tiles]
  const int2* rowKeys;    // [batch][seqLenQ]
  int tiles;
  int blockKeys;  // keys of a block in those tables
  ScoreSource src;
};

namespace score {

// Prefix of batch entry b.  Any int may stand there: lengths below zero are none and those past the keys are all of them, which also keeps sums
// with it inside 32 bits.
__device__ __forceinline__ int prefix_of(const ScoreFields& f, long long b, int seqLenKV) { return min(max(f.prefix[b], 0), seqLenKV); }

// Position from which the bias of a row is measured (the masks are the same from there).  Behind the last key all distances share
// pos - (seqLenKV - 1), which is nothing to a softmax and, left in, would take the bits of the scores: at slope 1/2 and 2^24 keys past them they are
// rounded to whole numbers.
__device__ __forceinline__ int bias_position(int pos, int seqLenKV) { return min(pos, seqLenKV - 1); }

// tanh(t) / t = c0 + c1 t^2 + c2 t^4 + c3 t^6 for |t| <= 1/2, fitted to the smallest largest error of the tanh (1.3e-7)
constexpr float kTanh0 = 0.9999976754188538f, kTanh1 = -0.33320656418800354f, kTanh2 = 0.13145145773887634f, kTanh3 = -0.04337248206138611f;

// A cap stays where products with it neither overflow nor vanish; beyond, it changes no result (scores within 1e-30, or no cap at all).
inline float usable_cap(float cap) { return cap > 0.f ? (cap < 1e-30f ? 1e-30f : cap > 1e28f ? 1e28f : cap) : 0.f; }

// c tanh of a few scores, times log2(e); x: 2 log2(e) S / c.  Scores up to c / 2 (of the whole warp) by the polynomial; else c - 2 c / (e^2x + 1), which
// is off by 2^-22 c: no more than 2^-21 of the largest score then, but everything where c is far above all scores.
template <int N>
__device__ __forceinline__ void cap_few(float (&x)[N], float capLog2) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < N; i++) top = fmaxf(top, fabsf(x[i]));
  if (__all_sync(0xffffffffu, top <= 1.44269504f)) {  // (a NaN stays one on either way)
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float t = x[i] * 0.34657359f, u = t * t;
      x[i] = capLog2 * t * fmaf(fmaf(fmaf(kTanh3, u, kTanh2), u, kTanh1), u, kTanh0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) {
      float e, r;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x[i]));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.f));
      x[i] = fmaf(-2.f * capLog2, r, capLog2);
    }
  }
}

}  // namespace score
}  // namespace tfa_b200
