// The decode attention kernel as other entry points of the library launch it.
#pragma once

#include "fk_common.cuh"

namespace fk {

struct AttnParams {
  const uint16_t* q; int64_t q_stride;
  uint16_t* out; int64_t out_stride;
  const int32_t* context_lens;
  const int32_t* block_tables; int64_t bt_stride;
  int batch, hq, hkv, g;
  int block_size; int num_blocks;
  int sub_tokens;     // tokens per TMA copy = min(block_size, 64)
  int fused16;        // 16-token pages: one 5-D copy brings both 64-dim halves of a page
  int bs_shift;       // log2(block_size) when it is a power of two, else -1
  int hnd;            // 1: pool is [blocks, Hkv, block, D]; 0: [blocks, block, Hkv, D]
  float scale_log2;
  int max_splits;
  int direct;         // 1: no plan, no splits: CTA b handles (sequence, KV head) item b whole
  int beside;         // 1: runs beside the kernel before it, which has seen the plan's kernel end
  int* plan;          // header + chunk_start[batch+1]
  int sign;           // the plan's last header word if it is of these sizes (0: not compared)
  int4* chunk_info;   // per chunk: {seq, split | nsplits << 16, tok_begin, tok_end}
  float* part_o;      // [batch, hq, max_splits, D]
  float2* part_ml;    // [batch, hq, max_splits]
  int32_t* status;
  // selected blocks (launch_decode's `selected`): the keys of token i and KV head h are those of
  // selected[(i * hkv + h) * count ...]; `batch` counts tokens
  const int32_t* selected;
  const int32_t* rows;      // table of each token, null: its own number
  int count, sel_block;
  int num_tables;
  int64_t capacity;         // tokens that a table's row has pages for (0: block_size * bt_stride)
  int tiles;                // 128-token tiles of `count` blocks
  const int32_t* starts;    // groups of rows that a direct call only looks over
  int groups;
  int64_t unit;             // tiles of all tokens and heads, one after another, that a CTA takes
  // sums of weights: `rows` as above; logits of every key that a token and KV head sees
  float* logits;            // [batch, hkv, logit_len, g]
  int64_t logit_len;
};


// Tiles of the token and head `item` (token * hkv + head) lie in the runs of CTAs first .. last.
__host__ __device__ inline void selected_ctas(int64_t item, int tiles, int64_t unit, int* first,
                                              int* last) {
  *first = (int)(item * tiles / unit);
  *last = (int)(((item + 1) * tiles - 1) / unit);
}

constexpr int ATT_D = 128;                  // head_dim
constexpr int ATT_TILE = 128;               // tokens per pipeline stage
constexpr int ATT_BOX = 64;                 // tokens per TMA box

// g16: more than 8 query heads per KV head; split: softmax weights in two bf16 parts
cudaError_t launch_decode(bool g16, bool split, bool selected, int grid, const CUtensorMap& mk,
                          const CUtensorMap& mv, const AttnParams& p, cudaStream_t s);

// Tensor map of a pool for copies of `sub` tokens of one head inside one page; `fused`: one copy
// brings both 64-channel halves.
int get_kv_map(const void* cache, int64_t num_blocks, int block_size, int hkv,
               int64_t block_stride, int hnd, int sub, int fused, CUtensorMap* out);

}  // namespace fk
