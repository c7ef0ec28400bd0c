// Sums of softmax weights of a paged pool's tokens: to the entry of each cached token is added what
// all query tokens of its sequence and all query heads of its KV head give it, 2^(logit - M) / sum.
//
// The attention before has left the logits and, per query token and head, (M, 1 / sum).  Warps have
// equal runs of steps of 32 cached tokens, a lane each, four steps at a time so that four rows of
// logits and four entries are on their way; query tokens come in their order, so that the sum's
// roundings are always the same.  Bound by memory: the logits (4 bytes a query head) once, entries in
// and out; most of the logits are still in L2.
#include "fk_runs.cuh"
#include "fk_sums.cuh"

namespace fk {

constexpr int SUMS_THREADS = 256;

__device__ __forceinline__ int sums_len(const SumsParams& p, int token) {
  const int64_t n = p.lens[token];
  return n < 0 ? 0 : n > p.capacity ? (int)p.capacity : (int)n;
}
// Query tokens of a sequence, within the batch.
__device__ __forceinline__ int2 sums_tokens(const SumsParams& p, int seq) {
  if (!p.cu) return make_int2(seq, seq + 1);
  const int a = p.cu[seq], b = min(p.cu[seq + 1], p.num_tokens);
  return a < 0 || a >= b ? make_int2(0, 0) : make_int2(a, b);
}
__device__ __forceinline__ int sums_most(const SumsParams& p, int2 tokens) {
  int most = 0;
  for (int t = tokens.x; t < tokens.y; ++t) most = max(most, sums_len(p, t));
  return most;
}

constexpr int SUMS_CTAS = 3;                 // of an SM, all there are
// Place of a step behind the run's: beyond all lengths, those rounded up to whole steps among them, so
// that nothing is loaded for it.
constexpr int SUMS_NONE = 0x7fffffff;

// STEPS at a time: four where each sequence has one query token (64 sequences of 1024 to 5000: 72.5 us
// with the attention before, 85 by one), one where there are several, whose logits are loads enough (4
// windows of 32 tokens: 137 us, 161 by four; a bf16 pool and 8 x 4 tokens: 110 and 105).
template <int STEPS>
__global__ void __launch_bounds__(SUMS_THREADS, SUMS_CTAS)
    attn_sums_kernel(const SumsParams p) {
  __shared__ RunCount<SUMS_THREADS> counted;
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto steps = [&](int seq) { return (sums_most(p, sums_tokens(p, seq)) + 31) / 32; };
  count_runs<SUMS_THREADS>(counted, p.num_seqs, steps);
  const int64_t warps = (int64_t)gridDim.x * (SUMS_THREADS / 32);
  const int64_t total = counted.begins[SUMS_THREADS] * p.hkv;
  // (short runs would be all beginnings)
  const int64_t run = max(run_length(total, warps), (int64_t)STEPS);
  int64_t x = ((int64_t)blockIdx.x * (SUMS_THREADS / 32) + warp) * run;
  const int64_t x1 = min(total, x + run);
  while (x < x1) {
    const RunPlace at = find_run<SUMS_THREADS>(counted, p.num_seqs, p.hkv, x, steps);
    const int2 tokens = sums_tokens(p, at.entry);
    const int most = sums_most(p, tokens);
    const int end = (int)min((int64_t)(most + 31) / 32, at.step + (x1 - x));
    const int64_t from = p.from ? p.from[at.entry] : (int64_t)sums_len(p, tokens.x) - 1;
    const int32_t* table = p.tables + (int64_t)at.entry * p.table_stride;
    for (int s0 = at.step; s0 < end; s0 += STEPS) {
      int page[STEPS], place[STEPS], key[STEPS];
      float sum[STEPS], old[STEPS];
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        key[j] = s0 + j < end ? (s0 + j) * 32 + lane : SUMS_NONE;
        const int i = p.page_shift >= 0 ? key[j] >> p.page_shift : key[j] / p.page;
        place[j] = key[j] - i * p.page;
        page[j] = key[j] < most ? table[i] : -1;
        sum[j] = 0.f;
      }
      int t = tokens.x;
      if constexpr (STEPS == 1) {
        // blocks of 16 columns, two at a time (4 windows of 32 tokens: 137 us, 150 by the loop below,
        // which takes all others)
        if (p.first && p.cols == 16 && p.ml_col == 1) {
          for (; t + 2 * p.block <= tokens.y; t += 2 * p.block) {
            float4 v[2][4], m[2][8];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const int u = t + b * p.block;
              const int64_t before = p.first[u], n = p.first[u + 1] - before;
              const int64_t row = (before * p.hkv + at.head * n) * 32 + key[0];
              const bool live = key[0] < n * 32 && row < p.logit_keys;
              const float4* z = reinterpret_cast<const float4*>(p.logits + row * 16);
              const float4* ml = reinterpret_cast<const float4*>(
                  p.ml + ((int64_t)u * p.hkv + at.head) * p.ml_pair);
#pragma unroll
              for (int c = 0; c < 4; ++c)
                v[b][c] = live ? z[c] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
#pragma unroll
              for (int c = 0; c < 8; ++c) m[b][c] = ml[c];
            }
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                const float x = c & 1 ? v[b][c / 2].z : v[b][c / 2].x;
                const float y = c & 1 ? v[b][c / 2].w : v[b][c / 2].y;
                if (x != -INFINITY) sum[0] = fmaf(fast_exp2(x - m[b][c].x), m[b][c].y, sum[0]);
                if (y != -INFINITY) sum[0] = fmaf(fast_exp2(y - m[b][c].z), m[b][c].w, sum[0]);
              }
          }
        }
      }
      for (; t < tokens.y; t += p.block) {
        const int cols = p.cols / p.block * min(p.block, tokens.y - t);
        int64_t base;
        int len;
        if (p.first) {
          const int64_t before = p.first[t], n = p.first[t + 1] - before;
          base = (before * p.hkv + at.head * n) * 32;
          len = (int)n * 32;
        } else {
          base = ((int64_t)t * p.hkv + at.head) * p.logit_len;
          len = sums_len(p, t);
        }
        len = (int)min((int64_t)len, p.logit_keys - base);
        const float2* ml = p.ml + ((int64_t)t * p.hkv + at.head) * p.ml_pair;
        const float* z = p.logits + (base + s0 * 32 + lane) * p.cols;
        const int pitch = 32 * p.cols;
        // a logit that is none is -infinity
        auto add = [&](float2 m, int j, float l) {
          if (l != -INFINITY) sum[j] = fmaf(fast_exp2(l - m.x), m.y, sum[j]);
        };
        if (p.cols % 4 == 0) {
#pragma unroll 4 / STEPS
          for (int c = 0; c < cols; c += 4) {
            float4 v[STEPS];
            float2 m[4];
#pragma unroll
            for (int j = 0; j < STEPS; ++j)
              v[j] = key[j] < len
                         ? *reinterpret_cast<const float4*>(z + j * pitch + c)
                         : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              m[e] = c + e < cols ? ml[(c + e) * p.ml_col] : make_float2(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (c + e >= cols) break;
#pragma unroll
              for (int j = 0; j < STEPS; ++j)
                add(m[e], j, e == 0 ? v[j].x : e == 1 ? v[j].y : e == 2 ? v[j].z : v[j].w);
            }
          }
        } else {
          for (int c = 0; c < cols; ++c) {
            const float2 m = ml[c * p.ml_col];
            float v[STEPS];
#pragma unroll
            for (int j = 0; j < STEPS; ++j)
              v[j] = key[j] < len ? z[j * pitch + c] : -INFINITY;
#pragma unroll
            for (int j = 0; j < STEPS; ++j) add(m, j, v[j]);
          }
        }
      }
      float* entry[STEPS];
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        const bool there = page[j] >= 0 && page[j] < p.num_pages;     // else flagged by the attention
        entry[j] = there ? p.weights + ((int64_t)page[j] * p.hkv + at.head) * p.page + place[j]
                         : nullptr;
        old[j] = there && key[j] < from ? *entry[j] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < STEPS; ++j)
        if (entry[j]) *entry[j] = old[j] + sum[j];
    }
    x += max(1, end - at.step);
  }
}

template <int STEPS>
static cudaError_t launch_steps(const SumsParams& p, cudaStream_t s) {
  return launch_kernel(attn_sums_kernel<STEPS>, dim3(sm_count() * SUMS_CTAS),
                       dim3(SUMS_THREADS), (size_t)0, s, p);
}
cudaError_t launch_sums(SumsParams p, cudaStream_t s) {
  p.page_shift = (p.page & (p.page - 1)) == 0 ? __builtin_ctz(p.page) : -1;
  return p.num_tokens > p.num_seqs ? launch_steps<1>(p, s) : launch_steps<4>(p, s);
}

}  // namespace fk
