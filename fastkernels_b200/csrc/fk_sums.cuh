// Sums of softmax weights of a paged pool's tokens, from the logits that an attention has left.
#pragma once

#include "fk_common.cuh"

namespace fk {

struct SumsParams {
  const int32_t* lens;          // keys of each query token
  const int32_t* cu;            // query tokens of each sequence; null: one each
  const int32_t* tables; int64_t table_stride;
  int64_t capacity;
  int num_seqs, num_tokens, num_pages, page, hkv;
  int page_shift;               // set by launch_sums
  int block;                    // query tokens whose logits lie side by side
  int cols;                     // logits of a key: block * query heads
  const float2* ml; int64_t ml_pair, ml_col;   // of (token, head) and column
  const float* logits;
  const int64_t* first;         // steps of one head before a token's, null: logit_len keys each
  int64_t logit_len, logit_keys;
  float* weights;
  const int32_t* from;
};

cudaError_t launch_sums(SumsParams p, cudaStream_t s);

}  // namespace fk
