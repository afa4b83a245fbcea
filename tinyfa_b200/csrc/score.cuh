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

}  // namespace tfa_b200
