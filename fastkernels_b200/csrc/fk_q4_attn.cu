// Decode attention over a paged KV cache of 4 bits a value, which can also add up what every cached
// token is given.
//
//   logit  z_t = scale (s_t q.c_t + lo_t sum q)         per group of channels, summed
//   out    sum_t p_t (s_t c_t + lo_t) / sum_t p_t,      p_t = 2^(z_t - m)
//   sums   of query heads (and query tokens) of p_t / sum p, added to a pool of fp32
//
// The codes go to the tensor cores as they are.  Four bits at the lowest end of an fp16 are the
// number code 2^-24, four bits above them code 2^-20, exactly; so one AND makes two operands, and
// the scales, per token, are applied to logits and to softmax weights.  Products are those of the
// transposes, S^T = K Q^T and O^T = V^T P^T (m16n8k16), which have tokens or channels as rows and
// the up to 8 query heads of a KV head as the 8 columns: half the matrix instructions of the
// product with 16 rows of queries, of which most would be empty.  A warp takes 32 tokens a step;
// S^T becomes the operand P^T by one transposing move per 16 tokens.
//
// Rounding to fewer bits: q to fp16 with a power of two per head taken out (exact but for channels
// 2^-26 below the largest), the weights p s to fp16 (11 bits, where bf16 caches' decode has 8), taken by
// a power of two that the largest p s so far of the column and group decides: a scale counts by its
// weight, and what lies 2^-19 below the largest has fewer than 11 bits.  Sums, maxima, weights'
// lowest-value term (sum p lo) are fp32.
//
// Work: steps of 32 tokens of all (tokens, KV head) pairs, one after another, are cut into equal runs,
// one for each warp of the grid.  Warps share nothing: each has a ring of steps of its own,
// filled by bulk copies (a step is one contiguous copy of up to 4.6 KB), and no barrier between.
// What a warp does not have whole goes to one of its two places of partial results, joined by
// the kernel behind; where all warps of a CTA are at one pair their parts become one first.  The
// running maximum is raised only when a logit is 4 above it (weights up to 2^4 fit), so that in
// most steps nothing is reduced across lanes and nothing rescaled.
//
// What bounds it: long contexts of up to 8 columns run at 0.99 of the copy rate once they run (64 x 4096
// to 64 x 8192 tokens, 32 / 8 heads: 62.4 to 109.1 us for 302 MB more); the beginning of the runs
// takes some 9 us, the join 5.  A step is some 480 warp instructions at half of the issue slots.
// 16 columns are bound by waiting (256 sequences, 64 / 4 heads: 109.7 us, 2.9 TB/s): the registers leave
// 3 warps a scheduler, each a chain of copy, product, exponential, transpose and product; 0.45 of the
// issue slots are used, and a warp waits 1.9 times an instruction for the one before, 0.8 times each
// for a pipe and for instructions to be fetched.
#include "fk_q4.cuh"
#include "fk_runs.cuh"
#include "fk_sums.cuh"

namespace fk {

constexpr int QA_WARPS = 8;                  // of the joining kernel
constexpr int QA_THREADS = QA_WARPS * 32;
constexpr int QA_STEP = 32;                  // tokens of a warp's step
constexpr int QA_AHEAD = 16;                 // steps that are looked up at a time
constexpr float QA_NONE = -3e38f;            // reference before there is a key
constexpr int QA_RUN = 4;                    // steps of a warp, at least
// Logits may be this far above the reference (log2).
constexpr float QA_SLACK = 4.f;
// Weights times scales are taken by powers of two into fp16, each group of a column by its own.  Where a
// step's scale would be taken above 2^11, and so a product above 2^15, the step is looked at by its
// weights too, and its largest product taken to 2^6 at most.  So 2^5 is the least that the largest of
// all that has been summed is taken to, unless 2^118 makes less of it.
constexpr int QA_LARGE = 11, QA_PRODUCT = 5, QA_MOST = 118;
constexpr int64_t QA_LONGEST = 1ll << 30;    // tokens of a context

struct Q4AttnParams {
  const uint16_t* q; int64_t q_stride;
  uint16_t* out; int64_t out_stride;
  const uint8_t* pool;
  const int32_t* lens;
  const int32_t* cu;            // tokens of each sequence; null: one each
  const int32_t* tables; int64_t table_stride;
  int64_t capacity;             // tokens a table's row has pages for
  int num_tokens, num_seqs, num_pages, page, hkv, g;
  int block;                    // query tokens that go together
  int cols;                     // block * g <= 8 or 16
  int direct;                   // CTA b has pair b whole
  float scale_log2;
  int32_t* status;
  int64_t* run;                 // [0] steps of a warp's run
  int64_t* first;               // [tokens + 1] steps of one head before a token's
  float2* part_ml;              // [2 * warps, cols]
  float* part_o;                // [2 * warps, cols, 128]
  float2* whole_ml;             // [tokens * hkv, cols] (maximum, 1 / sum)
  float* logits;                // [steps, 32, cols]
  int64_t logit_steps;
};

__device__ __forceinline__ uint64_t qa_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// A wait of 2 s at most; all lanes get the same answer.
__device__ __forceinline__ bool qa_wait_warp(uint64_t* bar, uint32_t parity) {
  bool got = mbar_try_wait(bar, parity);
  if (__builtin_expect(!__all_sync(0xffffffffu, got), 0)) {
    const uint64_t t0 = qa_ns();
    bool late = false;
    do {
      for (int i = 0; i < 64 && !got; ++i) got = mbar_try_wait(bar, parity);
      late = qa_ns() - t0 > 2000000000ull;
    } while (!__all_sync(0xffffffffu, got) && !__any_sync(0xffffffffu, late));
  }
  return __all_sync(0xffffffffu, got);
}

// KEPT: at its place in the program, as instructions of whole warps whose results lanes choose among
// have to be; else where the compiler likes (3 % of the time with 16 columns).
#define FK_QA_MMA(ASM)                                                                          \
  ASM("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "                                      \
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"                                   \
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])                                          \
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
template <bool KEPT>
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (KEPT) FK_QA_MMA(asm volatile);
  else FK_QA_MMA(asm);
}
#undef FK_QA_MMA
#define FK_QA_MMA(ASM)                                                                          \
  ASM("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "                                      \
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"                               \
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])                                          \
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f))
// The same onto nothing.
template <bool KEPT>
__device__ __forceinline__ void mma_f16_16816_first(float (&c)[4], uint32_t a0, uint32_t a1,
                                                    uint32_t a2, uint32_t a3, uint32_t b0,
                                                    uint32_t b1) {
  if constexpr (KEPT) FK_QA_MMA(asm volatile);
  else FK_QA_MMA(asm);
}
#undef FK_QA_MMA
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t max_bf16(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// 2^(e - 127)
__device__ __forceinline__ float power_of_2(int e) { return __int_as_float(e << 23); }
// Two fp32 to fp16, lo = a.
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}

// A bulk load whose lines leave L2 first, so that logits and parts stay.  Also where several blocks of
// query tokens read a cache one after another (256 x 64 heads 109.7 us, 115.5 with lines that stay as
// long as others; drafts of 5 tokens 107 and 112; 4 windows of 32 tokens 136.5 and 137.4).
__device__ __forceinline__ uint64_t qa_policy() {
  uint64_t r;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(r));
  return r;
}
__device__ __forceinline__ void qa_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar,
                                        uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1], %2, [%3], %4;" ::"r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// Query tokens that go together, and what they see.
struct QaItem {
  int row;        // table
  int tokens;     // 0: the token is in another's block, or in no sequence
  int len;        // keys of the longest
  int steps;
};

__device__ __forceinline__ int qa_len(const Q4AttnParams& p, int token) {
  const int64_t n = p.lens[token];
  return n < 0 ? 0 : n > p.capacity ? (int)p.capacity : (int)n;
}

__device__ __forceinline__ QaItem qa_item(const Q4AttnParams& p, int token) {
  QaItem it{token, 1, 0, 0};
  if (p.cu) {
    int lo = 0, hi = p.num_seqs;              // the last sequence that begins at or before it
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.cu[mid] <= token) lo = mid; else hi = mid;
    }
    const int a = p.cu[lo], b = min(p.cu[lo + 1], p.num_tokens);
    it.row = lo;
    if (a < 0 || token < a || token >= b || (token - a) % p.block != 0) {
      it.tokens = 0;
      return it;
    }
    it.tokens = min(p.block, b - token);
  }
  for (int j = 0; j < it.tokens; ++j) it.len = max(it.len, qa_len(p, token + j));
  it.steps = (it.len + QA_STEP - 1) / QA_STEP;
  return it;
}

// A step in the row of all steps.
struct QaPlace {
  int token, head, step;
  QaItem it;
  // `n` steps on
  __device__ __forceinline__ void advance(const Q4AttnParams& p, int n) {
    step += n;
    while (step >= it.steps) {
      step -= it.steps;
      if (++head < p.hkv) continue;
      head = 0;
      do {
        if (++token >= p.num_tokens) {        // behind the last: no keys
          token = 0;
          it = QaItem{0, 0, 0, 1 << 30};
          return;
        }
        it = qa_item(p, token);
      } while (it.steps == 0);
    }
  }
};

// Columns of a warp's products.  Of up to 4 there are two sets side by side: one for the step's
// first 16 tokens, one for the others, so that what is done per logit is done once per 32 tokens
// and not on empty columns.
template <int NG, int COLS>
struct QaShape {
  static constexpr int kFold = COLS == 4 ? 2 : 1;          // units side by side
  static constexpr int kTiles = COLS == 16 ? 2 : 1;        // of 8 columns
  static constexpr int kUnit = q4_unit_bytes(NG);
  static constexpr int kStage = 2 * kUnit;
  static constexpr int kCtas = COLS == 16 ? 1 : 2;         // of an SM
  // 16 columns of two groups need the registers of 8 warps (4 windows of 32 tokens with sums: 137 us,
  // 163 with 12), of one group they do with those of 12 (256 x 64 heads: 109.7 us, 121.8 with 8)
  static constexpr int kWarps = COLS == 16 && NG == 1 ? 12 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kDepth = 2;                         // steps of a warp's ring
  // the operand Q^T in registers, or in shared memory: 4 KB a warp
  static constexpr bool kSharedQ = COLS == 16;
  // what weights are taken by in shared memory, where there are the fewest registers (256 x 64 heads:
  // 109.3 us, 111.1 in registers; 4 windows of 32 tokens, of two groups and 8 warps: 140.0 and 138.3)
  static constexpr bool kSharedTaken = COLS == 16 && NG == 1;
  static constexpr int kRing = kWarps * kDepth * kStage;
  static constexpr int kSmem = kRing + (kSharedQ ? kWarps * 4096 : 0);
};

// NG groups a row; SUMS: logits are kept for the sums of weights.
template <int NG, int COLS, bool SUMS>
__global__ void __launch_bounds__((QaShape<NG, COLS>::kThreads), (QaShape<NG, COLS>::kCtas))
    q4_attn_kernel(const Q4AttnParams p) {
  using S = QaShape<NG, COLS>;
  constexpr int DEPTH = S::kDepth, NT = S::kTiles, FOLD = S::kFold, SETS = 2 / FOLD;
  constexpr int WARPS = S::kWarps, THREADS = S::kThreads;
  constexpr bool KEPT = COLS != 16;
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ uint64_t bars[WARPS][DEPTH];
  __shared__ RunCount<THREADS> counted;
  __shared__ int2 where[WARPS][2 * QA_AHEAD];           // units of a step in the pool, -1: none
  __shared__ QaPlace places[WARPS], ahead[WARPS];       // of the pair a warp is at, of its copies
  __shared__ int ends[WARPS];
  __shared__ float2 taken_all[S::kSharedTaken ? WARPS : 1][NG][8];
  // (maximum, sum) of the warps' parts that become one, when runs have been counted
  static_assert(sizeof(RunCount<THREADS>) >= sizeof(float2) * WARPS * COLS, "they share a place");
  float2 (*part_ml)[COLS] = reinterpret_cast<float2 (*)[COLS]>(&counted);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = lane & 3, row = lane >> 2;
  if (lane == 0) {
    for (int i = 0; i < DEPTH; ++i) mbar_init(&bars[warp][i], 1);
    mbar_fence_init();
  }
  pdl_launch_dependents();
  pdl_wait();

  // ---- the run of this warp: from a place on, every step, or of its CTA's pair every WARPS-th ----
  QaPlace now;
  int64_t x0 = 0;
  int count, stride = 1;
  const int64_t me = (int64_t)blockIdx.x * WARPS + warp;
  if (p.direct) {
    now.token = blockIdx.x / p.hkv;
    now.head = blockIdx.x - now.token * p.hkv;
    now.step = warp;
    now.it = qa_item(p, now.token);
    if (now.it.tokens == 0) return;
    count = max(0, (now.it.steps - warp + WARPS - 1) / WARPS);
    stride = WARPS;
    if (p.status && now.head == 0 && threadIdx.x < now.it.tokens &&
        p.lens[now.token + threadIdx.x] > p.capacity)
      atomicOr(p.status, FK_DEV_BAD_PAGE);
  } else {
    auto steps = [&](int i) { return qa_item(p, i).steps; };
    int64_t before = count_runs<THREADS>(counted, p.num_tokens, steps);
    if (blockIdx.x == 0) {
      const int per = entries_of_thread(p.num_tokens, THREADS);
      const int a = min((int)threadIdx.x * per, p.num_tokens), b = min(a + per, p.num_tokens);
      for (int i = a; i < b; ++i) {
        p.first[i] = before;
        const QaItem it = qa_item(p, i);
        before += it.steps;
        if (p.status)
          for (int j = 0; j < it.tokens; ++j)
            if (p.lens[i + j] > p.capacity) atomicOr(p.status, FK_DEV_BAD_PAGE);
      }
      if (threadIdx.x == 0) p.first[p.num_tokens] = counted.begins[THREADS];
    }
    const int64_t total = counted.begins[THREADS] * p.hkv;
    // (short runs would be all beginnings, and many parts to join: but no longer than pairs are)
    const int64_t pairs = (int64_t)p.num_tokens * p.hkv;
    const int64_t least = total >= QA_RUN * pairs ? QA_RUN : 1;
    const int64_t run = max(run_length(total, (int64_t)gridDim.x * WARPS), least);
    if (blockIdx.x == 0 && threadIdx.x == 0) p.run[0] = run;
    x0 = me * run;
    count = (int)max((int64_t)0, min(total, x0 + run) - x0);
    if (count > 0) {
      const RunPlace r = find_run<THREADS>(counted, p.num_tokens, p.hkv, x0, steps);
      now = QaPlace{r.entry, r.head, r.step, qa_item(p, r.entry)};
    } else {
      now = QaPlace{-1, 0, 0, QaItem{0, 0, 0, 0}};
    }
  }
  if (lane == 0) places[warp] = ahead[warp] = now;
  // Whether all warps of the CTA are at one pair, to its run's end: their parts become one then.
  if (lane == 0) ends[warp] = now.step + count;
  __syncthreads();
  bool joint = p.direct;
  if (!p.direct) {
    const int w = min(lane, WARPS - 1);
    const QaPlace first = places[0], other = places[w];
    // (a pair that one run has whole is not joined: two warps have to be at it)
    joint = places[1].token >= 0 &&
            __all_sync(0xffffffffu, other.token < 0 || (other.token == first.token &&
                                                        other.head == first.head &&
                                                        ends[w] <= other.it.steps));
    __syncthreads();                                       // a warp's next pair takes its place there
    if (first.token < 0) return;
  }

  uint8_t* ring = ring_all + warp * DEPTH * S::kStage;
  uint64_t* full = bars[warp];
  const int units = p.page / Q4_UNIT;                      // of a page
  // Copies are looked up QA_AHEAD steps at a time, a lane for each unit, from the place before.
  auto look_up = [&](int k) {
    const int step = k + (lane >> 1), second = lane & 1;
    QaPlace r = ahead[warp];
    __syncwarp();
    int unit = -1;
    if (step < count) {
      r.advance(p, ((k > 0 ? QA_AHEAD : 0) + (lane >> 1)) * stride);
      const int t = r.step * QA_STEP + second * Q4_UNIT;
      if (t < r.it.len) {
        const int at = t / p.page;
        const int page = p.tables[(int64_t)r.it.row * p.table_stride + at];
        if (page >= 0 && page < p.num_pages)
          unit = (page * p.hkv + r.head) * units + (t - at * p.page) / Q4_UNIT;
        else if (p.status)
          atomicOr(p.status, FK_DEV_BAD_PAGE);
      }
    }
    if (lane == 0) ahead[warp] = r;
    reinterpret_cast<int*>(&where[warp][step & (2 * QA_AHEAD - 1)])[second] = unit;
    __syncwarp();
  };
  auto copy = [&](int k, int slot) {
    if (__builtin_expect((k & (QA_AHEAD - 1)) == 0, 0)) look_up(k);
    if (lane == 0) {
      const int2 w = where[warp][k & (2 * QA_AHEAD - 1)];
      uint8_t* dst = ring + slot * S::kStage;
      uint64_t* bar = &full[slot];
      const uint64_t policy = qa_policy();
      if (w.x >= 0 && w.y == w.x + 1) {                    // side by side in the pool
        mbar_arrive_expect_tx(bar, 2 * S::kUnit);
        qa_load(dst, p.pool + (int64_t)w.x * S::kUnit, 2 * S::kUnit, bar, policy);
      } else {
        mbar_arrive_expect_tx(bar, ((w.x >= 0) + (w.y >= 0)) * S::kUnit);
        if (w.x >= 0) qa_load(dst, p.pool + (int64_t)w.x * S::kUnit, S::kUnit, bar, policy);
        if (w.y >= 0)
          qa_load(dst + S::kUnit, p.pool + (int64_t)w.y * S::kUnit, S::kUnit, bar, policy);
      }
    }
  };
  for (int k = 0; k < DEPTH && k < count; ++k) copy(k, k);

  // ---- state of a pair: columns 8 nt + 2 quad + {0, 1} ----
  uint32_t qf[S::kSharedQ ? 1 : NT][8][2];
  uint4* qs = reinterpret_cast<uint4*>(ring_all + S::kRing) + warp * 256 + lane;
  float o[8][NT][4];
  // weights are 2^(logit - ref); their sums, and of weights times the value's lowest
  float ref[NT][2], l[NT][2], low[NG][NT][2];
  float factor[NT][2], qsum[NG][NT][2];       // of logits: of a product, of a token's lowest
  // what weights times scales of values are taken by
  float2 taken_own[NG][NT];
  auto taken = [&](int gr, int nt) -> float2& {
    if constexpr (S::kSharedTaken) return taken_all[warp][gr][nt * 4 + quad];
    else return taken_own[gr][nt];
  };
  float large[NG];                            // the scale that the largest of them takes to 2^QA_LARGE

  bool ok = true;
  int slot = 0, i = 0;
  uint32_t phase = 0;
  while (ok && i < count) {
    // ---------------------------------------------------------------- a new pair
    if (i > 0) {
      now = places[warp];
      now.advance(p, now.it.steps - now.step);
      __syncwarp();
      if (lane == 0) places[warp] = now;
      __syncwarp();
    }
    const int begin = i;
    const int last = p.direct ? count : i + max(1, min(now.it.steps - now.step, count - i));
    const int step0 = now.step - i * stride;               // of the pair, at i = 0
    int shortest = 0x7fffffff;
    {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int col = nt * 8 + (FOLD == 2 ? row & 3 : row);
        const int tok = col / p.g;
        const bool live = tok < now.it.tokens;
        uint4 w[4];
        float f = 0.f, sum[NG];
        int n = 0;
        if (live) {
          const uint4* src = reinterpret_cast<const uint4*>(
              p.q + (int64_t)(now.token + tok) * p.q_stride +
              (int64_t)(now.head * p.g + col - tok * p.g) * Q4_D);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = src[4 * i + quad];
          n = qa_len(p, now.token + tok);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        shortest = min(shortest, live ? n : 0x7fffffff);
        float big = 0.f;
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) sum[gr] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = bf16lo(u[e]), b = bf16hi(u[e]);
            big = fmaxf(big, fmaxf(fabsf(a), fabsf(b)));
            sum[i * NG / 4] += a + b;
          }
        }
#pragma unroll
        for (int sh = 1; sh < 4; sh <<= 1) {
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, sh));
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], sh);
        }
        // 2^(13 - E) for the largest channel in [2^E, 2^(E+1))
        const int e = max((int)(__float_as_uint(big) >> 23), 28);
        const float up = __uint_as_float((uint32_t)(127 + 13 + 127 - e) << 23);
        f = __uint_as_float((uint32_t)(e - 13) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // channels c, c + 4 | c + 1, c + 5, which meet codes 2^4 too large | c + 2, c + 6 | ...
          const float c0 = bf16lo(w[i].x) * up, c1 = bf16hi(w[i].x) * up;
          const float c2 = bf16lo(w[i].y) * up, c3 = bf16hi(w[i].y) * up;
          const float c4 = bf16lo(w[i].z) * up, c5 = bf16hi(w[i].z) * up;
          const float c6 = bf16lo(w[i].w) * up, c7 = bf16hi(w[i].w) * up;
          const uint4 q = make_uint4(pack_f16(c0, c4), pack_f16(c1 * 0.0625f, c5 * 0.0625f),
                                     pack_f16(c2, c6), pack_f16(c3 * 0.0625f, c7 * 0.0625f));
          if constexpr (S::kSharedQ) {
            qs[(i * NT + nt) * 32] = q;
          } else {
            qf[nt][2 * i][0] = q.x;
            qf[nt][2 * i][1] = q.y;
            qf[nt][2 * i + 1][0] = q.z;
            qf[nt][2 * i + 1][1] = q.w;
          }
        }
        f *= 16777216.f * p.scale_log2;                    // codes are 2^-24
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int from = (2 * quad + j) * 4;             // a lane of that column
          factor[nt][j] = __shfl_sync(0xffffffffu, f, from);
#pragma unroll
          for (int gr = 0; gr < NG; ++gr)
            qsum[gr][nt][j] = __shfl_sync(0xffffffffu, sum[gr], from) * p.scale_log2;
          ref[nt][j] = QA_NONE;
          l[nt][j] = 0.f;
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) low[gr][nt][j] = 0.f;
        }
#pragma unroll
        for (int mt = 0; mt < 8; ++mt)
          o[mt][nt][0] = o[mt][nt][1] = o[mt][nt][2] = o[mt][nt][3] = 0.f;
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
          taken(gr, nt) = make_float2(power_of_2(127 + QA_MOST), power_of_2(127 + QA_MOST));
      }
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) large[gr] = power_of_2(127 + QA_LARGE - QA_MOST);
      if constexpr (S::kSharedTaken) __syncwarp();
      shortest = __reduce_min_sync(0xffffffffu, shortest);
    }

    const int safe = shortest / QA_STEP;                   // whole steps for all columns
    for (; i < last; ++i) {
      if (!qa_wait_warp(&full[slot], phase)) {
        if (lane == 0 && p.status) atomicOr(p.status, FK_DEV_WAIT_TIMEOUT);
        ok = false;
        break;
      }
      const uint8_t* st = ring + slot * S::kStage;
      const int2 w = where[warp][i & (2 * QA_AHEAD - 1)];
      const int step = step0 + i * stride;
      const bool edge = step >= safe || (w.x | w.y) < 0;

      // ---- logits: rows are tokens row, row + 8 of unit `lu` ----
      float z[SETS][NT][4];                                 // [set][.][row: 2 columns, row + 8: 2]
      float vs[SETS][NG][2], vl[SETS][NG][2];               // the values' scale and lowest
#pragma unroll
      for (int u = 0; u < SETS; ++u) {
        const int lu = FOLD == 2 ? quad >> 1 : u;
        float acc[2 / SETS][NG][NT][4];
#pragma unroll
        for (int f = 0; f < FOLD; ++f) {
          const uint8_t* un = st + (u + f) * S::kUnit;
          const uint4 ka = *reinterpret_cast<const uint4*>(un + row * Q4_ROW + quad * 16);
          const uint4 kb = *reinterpret_cast<const uint4*>(un + (row + 8) * Q4_ROW + quad * 16);
          const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t ya = wa[w] >> 8, yb = wb[w] >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float (&c)[4] = acc[f][w * NG / 4][nt];
              uint4 q;
              if constexpr (S::kSharedQ) q = qs[(w * NT + nt) * 32];
              else q = make_uint4(qf[nt][2 * w][0], qf[nt][2 * w][1], qf[nt][2 * w + 1][0],
                                  qf[nt][2 * w + 1][1]);
              const uint32_t a0 = wa[w] & 0x000f000fu, a1 = wb[w] & 0x000f000fu;
              const uint32_t a2 = wa[w] & 0x00f000f0u, a3 = wb[w] & 0x00f000f0u;
              if (w % (4 / NG) == 0) mma_f16_16816_first<KEPT>(c, a0, a1, a2, a3, q.x, q.y);
              else mma_f16_16816<KEPT>(c, a0, a1, a2, a3, q.x, q.y);
              mma_f16_16816<KEPT>(c, ya & 0x000f000fu, yb & 0x000f000fu, ya & 0x00f000f0u,
                            yb & 0x00f000f0u, q.z, q.w);
            }
          }
        }
        if constexpr (FOLD == 2) {
#pragma unroll
          for (int gr = 0; gr < NG; ++gr)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[0][gr][0][e] = lu ? acc[1][gr][0][e] : acc[0][gr][0][e];
        }
        uint32_t kp[2][NG], vp[2][NG];
        const uint32_t* pairs = reinterpret_cast<const uint32_t*>(st + lu * S::kUnit + Q4_PAIRS);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if constexpr (NG == 2) {
            const uint2 a = *reinterpret_cast<const uint2*>(pairs + (row + 8 * r) * 2);
            const uint2 b = *reinterpret_cast<const uint2*>(pairs + (Q4_UNIT + row + 8 * r) * 2);
            kp[r][0] = a.x; kp[r][1] = a.y; vp[r][0] = b.x; vp[r][1] = b.y;
          } else {
            kp[r][0] = pairs[row + 8 * r];
            vp[r][0] = pairs[Q4_UNIT + row + 8 * r];
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            auto product = [&](int gr) {
              return pair_of(acc[0][gr][nt][2 * r], acc[0][gr][nt][2 * r + 1]);
            };
            auto q_sum = [&](int gr) { return pair_of(qsum[gr][nt][0], qsum[gr][nt][1]); };
            uint64_t t = mul2(pair_of(bf16lo(kp[r][0])), product(0));
            uint64_t b = mul2(pair_of(bf16hi(kp[r][0])), q_sum(0));
            if constexpr (NG == 2) {
              t = fma2(pair_of(bf16lo(kp[r][1])), product(1), t);
              b = fma2(pair_of(bf16hi(kp[r][1])), q_sum(1), b);
            }
            const float2 both = both_of(fma2(t, pair_of(factor[nt][0], factor[nt][1]), b));
            z[u][nt][2 * r] = both.x;
            z[u][nt][2 * r + 1] = both.y;
          }
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            vs[u][gr][r] = bf16lo(vp[r][gr]);
            vl[u][gr][r] = bf16hi(vp[r][gr]);
          }
        if (__builtin_expect(edge, 0)) {
          // what stands behind the context is any number, or none
          const QaPlace& at = places[warp];
          int len[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int tok = (FOLD == 2 ? 2 * (quad & 1) + j : nt * 8 + 2 * quad + j) / p.g;
              len[nt][j] = tok < at.it.tokens ? qa_len(p, at.token + tok) : 0;
            }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int t = step * QA_STEP + lu * Q4_UNIT + row + 8 * r;
            const bool there = (lu ? w.y : w.x) >= 0 && t < at.it.len;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              if (there && fabsf(vs[u][gr][r]) < INFINITY && fabsf(vl[u][gr][r]) < INFINITY) continue;
              // no weight makes nothing of a value that is no number: columns that see it have none
              // as their sum, the others are not told
              vs[u][gr][r] = vl[u][gr][r] = 0.f;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                  if (there && t < len[nt][j]) low[gr][nt][j] = NAN;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (!there || t >= len[nt][j]) z[u][nt][2 * r + j] = -INFINITY;
          }
        }
        if constexpr (SUMS) {
          if (x0 + i < p.logit_steps) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float* dst = p.logits + ((x0 + i) * QA_STEP + lu * Q4_UNIT + row + 8 * r) * p.cols;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const int c = FOLD == 2 ? 2 * (quad & 1) : nt * 8 + 2 * quad;
                if (c + 1 < p.cols && (p.cols & 1) == 0) {
                  *reinterpret_cast<float2*>(dst + c) =
                      make_float2(z[u][nt][2 * r], z[u][nt][2 * r + 1]);
                } else {
                  if (c < p.cols) dst[c] = z[u][nt][2 * r];
                  if (c + 1 < p.cols) dst[c + 1] = z[u][nt][2 * r + 1];
                }
              }
            }
          }
        }
      }

      // ---- new references, if a logit or a scale has left the old ones behind ----
      float top[NT][2];
      bool beyond = false;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        float most = fmaxf(vs[0][gr][0], vs[0][gr][1]);
        if constexpr (SETS == 2) most = fmaxf(most, fmaxf(vs[1][gr][0], vs[1][gr][1]));
        beyond |= most > large[gr];
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top[nt][j] = fmaxf(z[0][nt][j], z[0][nt][2 + j]);
          if constexpr (SETS == 2)
            top[nt][j] = fmaxf(top[nt][j], fmaxf(z[1][nt][j], z[1][nt][2 + j]));
          beyond |= top[nt][j] > ref[nt][j] + QA_SLACK;
        }
      if (__builtin_expect(__any_sync(0xffffffffu, beyond), 0)) {
        constexpr int kFrom = FOLD == 2 ? 2 : 4;            // lanes of the same column, and its twin
        int most[NG];
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) most[gr] = 0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float up[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float mx = top[nt][j];
#pragma unroll
            for (int sh = kFrom; sh < 32; sh <<= 1)
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, sh));
            const float next = fmaxf(ref[nt][j], ceilf(mx));
            up[j] = next - ref[nt][j];                       // whole, or all there is
            const float alpha = fast_exp2(-up[j]);
            ref[nt][j] = next;
            l[nt][j] *= alpha;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) low[gr][nt][j] *= alpha;
          }
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            float m[2] = {0.f, 0.f};                         // the largest product
#pragma unroll
            for (int u = 0; u < SETS; ++u)
#pragma unroll
              for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                  m[j] = fmaxf(m[j], fast_exp2(z[u][nt][2 * r + j] - ref[nt][j]) * vs[u][gr][r]);
            uint32_t both = pack_bf16(m[0], m[1]);
#pragma unroll
            for (int sh = kFrom; sh < 32; sh <<= 1)
              both = max_bf16(both, __shfl_xor_sync(0xffffffffu, both, sh));
            float2 by = taken(gr, nt);
            if constexpr (S::kSharedTaken) __syncwarp();
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // (what has been summed stays as it is where weights are taken by as much more as the
              // reference is higher)
              const float rise = (float)(__float_as_int(j ? by.y : by.x) >> 23) + up[j];
              const int at_most = min(127 + QA_MOST, 127 + QA_PRODUCT + 127 -
                                                         (int)(both >> (16 * j + 7) & 0xffu));
              const float e = fminf(rise, (float)at_most), back = fast_exp2(e - rise);
              (j ? by.y : by.x) = power_of_2((int)e);
              most[gr] = max(most[gr], (int)e);
#pragma unroll
              for (int mt = 0; mt < 8; ++mt)
                if (mt * NG / 8 == gr) {
                  o[mt][nt][j] *= back;
                  o[mt][nt][2 + j] *= back;
                }
            }
            taken(gr, nt) = by;
            if constexpr (S::kSharedTaken) __syncwarp();
          }
        }
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
          large[gr] = power_of_2(min(127 + QA_LARGE + 127 - most[gr], 254));
      }

      // ---- weights, and the operand P^T ----
      uint32_t pt[2][NG][NT][2];
#pragma unroll
      for (int u = 0; u < SETS; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint64_t w = pair_of(fast_exp2(z[u][nt][2 * r] - ref[nt][0]),
                                       fast_exp2(z[u][nt][2 * r + 1] - ref[nt][1]));
            auto add_to = [](float (&to)[2], uint64_t v) {
              const float2 both = both_of(v);
              to[0] = both.x;
              to[1] = both.y;
            };
            add_to(l[nt], add2(pair_of(l[nt][0], l[nt][1]), w));
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              float (&sum)[2] = low[gr][nt];
              add_to(sum, fma2(w, pair_of(vl[u][gr][r]), pair_of(sum[0], sum[1])));
            }
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              const float2 by = taken(gr, nt);
              const float2 ws = both_of(mul2(mul2(w, pair_of(by.x, by.y)), pair_of(vs[u][gr][r])));
              const uint32_t x = transpose_8x8(pack_f16(ws.x, ws.y));
              if constexpr (FOLD == 2) {
                pt[0][gr][nt][r] = row < 4 ? x : 0u;
                pt[1][gr][nt][r] = row < 4 ? 0u : x;
              } else {
                pt[u][gr][nt][r] = x;
              }
            }
          }

      // ---- O^T += V^T P^T: rows are channels, of lane `row` 8 row + {0 .. 7} (+ 64) ----
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint8_t* un = st + u * S::kUnit + Q4_VALUES + row * 8;
        const uint2 a0 = *reinterpret_cast<const uint2*>(un + (2 * quad) * Q4_ROW);
        const uint2 a1 = *reinterpret_cast<const uint2*>(un + (2 * quad + 1) * Q4_ROW);
        const uint2 b0 = *reinterpret_cast<const uint2*>(un + (2 * quad + 8) * Q4_ROW);
        const uint2 b1 = *reinterpret_cast<const uint2*>(un + (2 * quad + 9) * Q4_ROW);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t wa0 = h ? a0.y : a0.x, wa1 = h ? a1.y : a1.x;
          const uint32_t wb0 = h ? b0.y : b0.x, wb1 = h ? b1.y : b1.x;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // channels 4 half .. 4 half + 3 of the word, of two tokens side by side
            uint32_t xa = __byte_perm(wa0, wa1, half ? 0x7632 : 0x5410);
            uint32_t xb = __byte_perm(wb0, wb1, half ? 0x7632 : 0x5410);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int mt = 4 * h + 2 * half + k;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_f16_16816<KEPT>(o[mt][nt], xa & 0x000f000fu, xa & 0x00f000f0u, xb & 0x000f000fu,
                              xb & 0x00f000f0u, pt[u][h * NG / 2][nt][0],
                              pt[u][h * NG / 2][nt][1]);
              xa >>= 8;
              xb >>= 8;
            }
          }
        }
      }
      __syncwarp();
      if (i + DEPTH < count) copy(i + DEPTH, slot);
      if (++slot == DEPTH) { slot = 0; phase ^= 1; }
    }

    if (!ok) break;
    // ------------------------------------------------------------------- the pair's end
    const QaPlace done = places[warp];
    const bool whole = done.step == 0 && step0 + i == done.it.steps && !joint;
    const int64_t place = 2 * me + (begin > 0 ? 1 : 0);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = l[nt][j], lows[NG];
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) lows[gr] = low[gr][nt][j];
#pragma unroll
        for (int sh = FOLD == 2 ? 2 : 4; sh < 32; sh <<= 1) {
          sum += __shfl_xor_sync(0xffffffffu, sum, sh);
#pragma unroll
          for (int gr = 0; gr < NG; ++gr)
            lows[gr] += __shfl_xor_sync(0xffffffffu, lows[gr], sh);
        }
        if constexpr (FOLD == 2) {
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            o[mt][nt][j] += __shfl_xor_sync(0xffffffffu, o[mt][nt][j], 2);
            o[mt][nt][2 + j] += __shfl_xor_sync(0xffffffffu, o[mt][nt][2 + j], 2);
          }
          if (quad > 1) continue;
        }
        const int col = nt * 8 + 2 * quad + j;
        const int tok = col / p.g;
        if (tok >= done.it.tokens) continue;
        const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 by = taken(h * NG / 2, nt);
          const float back = __fdividef(1.f, j ? by.y : by.x);
          float v[8];
#pragma unroll
          for (int c = 0; c < 8; ++c)
            v[c] = fmaf(o[4 * h + (c >> 1)][nt][(c & 1) * 2 + j] *
                            ((c & 1) ? 1048576.f : 16777216.f),
                        back, lows[h * NG / 2]);
          if (whole) {
            uint4 w;
            w.x = pack_bf16(v[0] * inv, v[1] * inv);
            w.y = pack_bf16(v[2] * inv, v[3] * inv);
            w.z = pack_bf16(v[4] * inv, v[5] * inv);
            w.w = pack_bf16(v[6] * inv, v[7] * inv);
            *reinterpret_cast<uint4*>(p.out + (int64_t)(done.token + tok) * p.out_stride +
                                      (int64_t)(done.head * p.g + col - tok * p.g) * Q4_D + 64 * h +
                                      8 * row) = w;
          } else {
            float* part = joint ? reinterpret_cast<float*>(ring) + col * Q4_D
                                : p.part_o + (place * p.cols + col) * Q4_D;
            float4* dst = reinterpret_cast<float4*>(part + 64 * h + 8 * row);
            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
            dst[1] = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
        if (row == 0) {
          if (joint) part_ml[warp][col] = make_float2(ref[nt][j], sum);
          else if (!whole) p.part_ml[place * p.cols + col] = make_float2(ref[nt][j], sum);
          else if (SUMS)
            p.whole_ml[((int64_t)done.token * p.hkv + done.head) * p.cols + col] =
                make_float2(ref[nt][j], inv);
        }
      }
  }
  if (!ok) {
    // copies still on their way end before the shared memory goes
    for (int k = 0; k < DEPTH && k < count - i; ++k) {
      (void)qa_wait_warp(&full[slot], phase);
      if (++slot == DEPTH) { slot = 0; phase ^= 1; }
    }
  }
  if (!joint) return;

  // ---- parts of the CTA's warps, in their rings, become one ----
  if (count == 0 || !ok)
    for (int c = lane; c < COLS; c += 32) part_ml[warp][c] = make_float2(QA_NONE, 0.f);
  __syncthreads();
  const QaPlace done = places[0];
  const int64_t place = 2 * (int64_t)blockIdx.x * WARPS;
  for (int c = warp; c < done.it.tokens * p.g; c += WARPS) {
    float M = QA_NONE, L = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, part_ml[w][c].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float2 ml = part_ml[w][c];
      if (ml.y == 0.f) continue;
      const float f = fast_exp2(ml.x - M);
      const float4 v = reinterpret_cast<const float4*>(ring_all + w * DEPTH * S::kStage)[c * 32 + lane];
      L = fmaf(ml.y, f, L);
      acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y);
      acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
    }
    if (p.direct) {
      const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
      const int tok = c / p.g;
      reinterpret_cast<uint2*>(p.out + (int64_t)(done.token + tok) * p.out_stride +
                               (int64_t)(done.head * p.g + c - tok * p.g) * Q4_D)[lane] =
          make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
    } else {
      reinterpret_cast<float4*>(p.part_o + (place * p.cols + c) * Q4_D)[lane] = acc;
      // the first warp's part is all of them
      if (lane < WARPS)
        p.part_ml[(place + 2 * lane) * p.cols + c] =
            lane == 0 ? make_float2(M, L) : make_float2(QA_NONE, 0.f);
    }
  }
}

// ---------------------------------------------------------------------------
// join of partial results
// ---------------------------------------------------------------------------
// A CTA has `block_cols` columns of a pair, and as many warps for each as there are then: they take
// its parts in turn, QA_PARTS loads of a part on their way at a time.
constexpr int QA_PARTS = 4;

template <bool SUMS>
__global__ void __launch_bounds__(QA_THREADS) q4_attn_join_kernel(const Q4AttnParams p,
                                                                  int block_cols) {
  __shared__ float4 shares[QA_WARPS][32];
  __shared__ float2 totals[QA_WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int groups = (p.cols + block_cols - 1) / block_cols;
  const int pair = blockIdx.x / groups, group = blockIdx.x - pair * groups;
  const int token = pair / p.hkv, head = pair - token * p.hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slices = QA_WARPS / block_cols, slice = warp % slices;
  const int c = group * block_cols + warp / slices;
  const int64_t before = p.first[token], steps = p.first[token + 1] - before, run = p.run[0];
  const QaItem it = p.cu || steps == 0 ? qa_item(p, token) : QaItem{token, 1, 0, 0};
  const int tok = c / p.g;
  const bool mine = tok < it.tokens;
  uint2* out = reinterpret_cast<uint2*>(p.out + (int64_t)(token + tok) * p.out_stride +
                                        (int64_t)(head * p.g + c - tok * p.g) * Q4_D) + lane;
  if (steps == 0) {
    if (mine && slice == 0) *out = make_uint2(0u, 0u);
    return;
  }
  // the runs that the pair's steps lie in: a .. a + n - 1; the first has it in its second place
  // unless the pair begins with the run
  const int64_t px = before * p.hkv + head * steps, pe = px + steps - 1;
  const int64_t a = pe >> 31 ? px / run : (int64_t)((uint32_t)px / (uint32_t)run);
  const int n = (int)((pe >> 31 ? pe / run : (int64_t)((uint32_t)pe / (uint32_t)run)) - a) + 1;
  if (n == 1) return;
  const int second = px > a * run ? 1 : 0;
  auto place = [&](int w) { return (2 * (a + w) + (w == 0 ? second : 0)) * p.cols + c; };
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float2 all = make_float2(QA_NONE, 0.f);
  const int per = (n + slices - 1) / slices, end = min(n, (slice + 1) * per);
  for (int w0 = slice * per; mine && w0 < end; w0 += 32) {
    // (maximum, sum) of 32 parts, then those that are any
    const float2 ml = w0 + lane < end ? p.part_ml[place(w0 + lane)] : make_float2(QA_NONE, 0.f);
    float M = fmaxf(all.x, ml.x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float f = fast_exp2(ml.x - M), old = fast_exp2(all.x - M);
    float L = ml.y * f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    all = make_float2(M, fmaf(all.y, old, L));
    acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
    uint32_t any = __ballot_sync(0xffffffffu, ml.y != 0.f);
    while (any) {
      float4 v[QA_PARTS];
      float g[QA_PARTS];
#pragma unroll
      for (int i = 0; i < QA_PARTS; ++i) {
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        g[i] = 0.f;
        if (!any) continue;
        const int w = __ffs(any) - 1;
        any &= any - 1;
        v[i] = reinterpret_cast<const float4*>(p.part_o + place(w0 + w) * Q4_D)[lane];
        g[i] = __shfl_sync(0xffffffffu, f, w);
      }
#pragma unroll
      for (int i = 0; i < QA_PARTS; ++i) {
        acc.x = fmaf(v[i].x, g[i], acc.x); acc.y = fmaf(v[i].y, g[i], acc.y);
        acc.z = fmaf(v[i].z, g[i], acc.z); acc.w = fmaf(v[i].w, g[i], acc.w);
      }
    }
  }
  if (slices > 1) {
    shares[warp][lane] = acc;
    if (lane == 0) totals[warp] = all;
    __syncthreads();
    if (slice != 0) return;
    float M = all.x;
    for (int i = 1; i < slices; ++i) M = fmaxf(M, totals[warp + i].x);
    const float old = fast_exp2(all.x - M);
    acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
    all = make_float2(M, all.y * old);
    for (int i = 1; i < slices; ++i) {
      const float2 t = totals[warp + i];
      const float4 v = shares[warp + i][lane];
      const float f = fast_exp2(t.x - M);
      all.y = fmaf(t.y, f, all.y);
      acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y);
      acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
    }
  }
  if (!mine) return;
  const float inv = all.y > 0.f ? 1.f / all.y : all.y == 0.f ? 0.f : all.y;
  if (SUMS && lane == 0) p.whole_ml[(int64_t)pair * p.cols + c] = make_float2(all.x, inv);
  *out = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

struct QaLayout {
  size_t first, part_ml, part_o, whole_ml, logits, total;
  int64_t logit_steps;
};
static int qa_columns(int tokens, int seqs, int g, int* block) {
  // Query tokens of a sequence that go together: as many as 16 columns hold, and no more than there are
  // on average, since empty columns cost what full ones do.  Against as many as 16 columns hold, 4 query
  // heads, contexts of 4000: 64 x 1 token 66 us (101), 64 x 2 77 (108), 31 x 1 and one of 32 tokens
  // 56 (76); but 56 x 1 and 8 of 16 tokens 160 (143).
  int n = 16 / g;
  const int mean = seqs > 0 ? (tokens + seqs - 1) / seqs : 1;
  if (n > mean) n = mean;
  if (n < 1) n = 1;
  *block = n;
  return n * g;
}
// A small call -- each pair has a CTA of its own at once, and tables of at most 2048 tokens leave the
// CTA's warps little to do each -- is one launch, without runs, parts, join or workspace (1 x 500
// tokens: 7.4 us; 13 by runs).
static bool qa_direct(int tokens, int hkv, int cols, bool sums, int64_t max_len) {
  return !sums && max_len > 0 && max_len <= 2048 &&
         (int64_t)tokens * hkv <= (int64_t)(cols <= 8 ? 2 : 1) * sm_count();
}
static QaLayout qa_layout(int tokens, int seqs, int hkv, int g, bool sums, int64_t max_len) {
  auto up = [](size_t b) { return (b + 255) & ~size_t(255); };
  int block;
  const int cols = qa_columns(tokens, seqs, g, &block);
  const size_t places = (size_t)sm_count() * 16 * 2;       // two of each of at most 16 warps an SM
  QaLayout w{};
  if (qa_direct(tokens, hkv, cols, sums, max_len)) return w;
  w.first = 256;
  w.part_ml = w.first + up(((size_t)tokens + 1) * sizeof(int64_t));
  w.part_o = w.part_ml + up(places * cols * sizeof(float2));
  w.whole_ml = w.part_o + up(places * cols * Q4_D * sizeof(float));
  w.logits = w.total = w.whole_ml;
  if (sums) {
    w.logits = w.whole_ml + up((size_t)tokens * hkv * cols * sizeof(float2));
    const int64_t items = (int64_t)tokens / block + (block > 1 ? seqs : 0);
    w.logit_steps = items * hkv * ((max_len + QA_STEP - 1) / QA_STEP);
    w.total = w.logits + up((size_t)w.logit_steps * QA_STEP * cols * sizeof(float));
  }
  return w;
}

template <int NG, int COLS, bool SUMS>
static cudaError_t qa_launch(const Q4AttnParams& p, int sms, cudaStream_t s) {
  using Shape = QaShape<NG, COLS>;
  static PerDeviceOnce once;
  auto kernel = q4_attn_kernel<NG, COLS, SUMS>;
  const cudaError_t e = set_max_dynamic_smem(once, kernel, Shape::kSmem);
  if (e != cudaSuccess) return e;
  const int grid = p.direct ? p.num_tokens * p.hkv : sms * Shape::kCtas;
  return launch_kernel(kernel, dim3(grid), dim3(Shape::kThreads), (size_t)Shape::kSmem, s,
                       p);
}
template <int NG, bool SUMS>
static cudaError_t qa_launch(const Q4AttnParams& p, int sms, cudaStream_t s) {
  return p.cols <= 4 ? qa_launch<NG, 4, SUMS>(p, sms, s)
                     : p.cols <= 8 ? qa_launch<NG, 8, SUMS>(p, sms, s)
                                   : qa_launch<NG, 16, SUMS>(p, sms, s);
}

}  // namespace fk

using namespace fk;

extern "C" {

size_t fk_paged_decode_attn_q4_workspace_bytes(int num_tokens, int num_seqs, int num_q_heads,
                                               int num_kv_heads, int head_dim, int with_weights,
                                               int64_t max_context_len) {
  if (num_tokens <= 0 || num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads ||
      num_q_heads / num_kv_heads > 16 || head_dim != Q4_D || max_context_len < 0)
    return 0;
  return qa_layout(num_tokens, num_seqs, num_kv_heads, num_q_heads / num_kv_heads,
                   with_weights != 0, max_context_len).total;
}

int fk_paged_decode_attn_q4(const void* q, int64_t q_stride_token, void* out,
                            int64_t out_stride_token, const void* cache, int64_t num_pages,
                            int page_size, int group, const int32_t* context_lens,
                            const int32_t* block_tables, int64_t block_table_stride,
                            int64_t block_table_cols, const int32_t* cu_seqlens_q, int num_seqs,
                            int num_tokens, int num_q_heads, int num_kv_heads, int head_dim,
                            float softmax_scale, float* weights, const int32_t* weights_from,
                            int64_t max_context_len, void* workspace, size_t workspace_bytes,
                            int32_t* status, fk_stream_t stream) {
  static const char* what = "fk_paged_decode_attn_q4";
  FK_REQUIRE(num_tokens >= 0 && num_seqs >= 0, FK_ERR_INVALID_ARG, "%s: negative size", what);
  const int rc = q4_check_pool(what, cache, num_pages, page_size, num_kv_heads, head_dim, group);
  if (rc != FK_OK) return rc;
  if (num_tokens == 0 || num_seqs == 0) return FK_OK;
  FK_REQUIRE(q && out && context_lens && block_tables, FK_ERR_INVALID_ARG, "%s: null pointer",
             what);
  FK_REQUIRE(num_q_heads > 0 && num_q_heads % num_kv_heads == 0, FK_ERR_INVALID_ARG,
             "%s: num_q_heads must be a multiple of num_kv_heads", what);
  const int g = num_q_heads / num_kv_heads;
  FK_REQUIRE(g <= 16, FK_ERR_UNSUPPORTED, "%s: more than 16 query heads per KV head", what);
  FK_REQUIRE(cu_seqlens_q != nullptr || num_seqs == num_tokens, FK_ERR_INVALID_ARG,
             "%s: %d tokens of %d sequences need cu_seqlens_q", what, num_tokens, num_seqs);
  FK_REQUIRE(block_table_cols > 0 && block_table_stride >= 0, FK_ERR_INVALID_ARG, "%s: bad sizes",
             what);
  FK_REQUIRE(q_stride_token >= (int64_t)num_q_heads * head_dim &&
                 out_stride_token >= (int64_t)num_q_heads * head_dim,
             FK_ERR_INVALID_ARG, "%s: token stride too small", what);
  FK_REQUIRE(aligned16(q) && aligned16(out) && q_stride_token % 8 == 0 && out_stride_token % 8 == 0,
             FK_ERR_ALIGNMENT, "%s: 16-byte alignment required", what);
  FK_REQUIRE(max_context_len >= 0, FK_ERR_INVALID_ARG, "%s: negative size", what);
  FK_REQUIRE(num_pages * num_kv_heads < (1ll << 31) / (page_size / Q4_UNIT), FK_ERR_UNSUPPORTED,
             "%s: pool too large", what);
  Q4AttnParams p{};
  p.q = static_cast<const uint16_t*>(q); p.q_stride = q_stride_token;
  p.out = static_cast<uint16_t*>(out); p.out_stride = out_stride_token;
  p.pool = static_cast<const uint8_t*>(cache);
  p.lens = context_lens; p.cu = cu_seqlens_q;
  p.tables = block_tables; p.table_stride = block_table_stride;
  p.capacity = block_table_cols < QA_LONGEST / page_size ? block_table_cols * page_size
                                                         : QA_LONGEST;
  p.num_tokens = num_tokens; p.num_seqs = num_seqs; p.num_pages = (int)num_pages;
  p.page = page_size; p.hkv = num_kv_heads; p.g = g;
  p.cols = qa_columns(num_tokens, num_seqs, g, &p.block);
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.status = status;
  const bool sums = weights != nullptr;
  if (sums && max_context_len < p.capacity) p.capacity = max_context_len;
  const QaLayout w = qa_layout(num_tokens, num_seqs, num_kv_heads, g, sums, p.capacity);
  FK_REQUIRE(w.total == 0 || (workspace != nullptr && workspace_bytes >= w.total &&
                              (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0),
             FK_ERR_WORKSPACE, "%s: workspace needs %zu bytes, 256-byte aligned (got %zu)", what,
             w.total, workspace_bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.run = reinterpret_cast<int64_t*>(ws);
  p.first = reinterpret_cast<int64_t*>(ws + w.first);
  p.part_ml = reinterpret_cast<float2*>(ws + w.part_ml);
  p.part_o = reinterpret_cast<float*>(ws + w.part_o);
  p.whole_ml = reinterpret_cast<float2*>(ws + w.whole_ml);
  p.logits = reinterpret_cast<float*>(ws + w.logits);
  p.logit_steps = w.logit_steps;
  const int64_t pairs = (int64_t)num_tokens * num_kv_heads;
  const int sms = sm_count();
  p.direct = qa_direct(num_tokens, num_kv_heads, p.cols, sums, p.capacity);
  // Few pairs have many parts each: then all of a joining CTA's warps take one column.
  int block_cols = 1;
  while (block_cols < 8 && block_cols < p.cols &&
         pairs * ((p.cols + 2 * block_cols - 1) / (2 * block_cols)) >= 2 * sms)
    block_cols *= 2;
  const int64_t blocks = pairs * ((p.cols + block_cols - 1) / block_cols);
  FK_REQUIRE(blocks < (1ll << 31), FK_ERR_UNSUPPORTED, "%s: too many tokens", what);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      sums ? group == 64 ? qa_launch<2, true>(p, sms, s) : qa_launch<1, true>(p, sms, s)
           : group == 64 ? qa_launch<2, false>(p, sms, s) : qa_launch<1, false>(p, sms, s);
  FK_CUDA_OK(e);
  count_launch(1);
  if (p.direct) return FK_OK;
  auto join = sums ? q4_attn_join_kernel<true> : q4_attn_join_kernel<false>;
  FK_CUDA_OK(launch_kernel(join, dim3((unsigned)blocks), dim3(QA_THREADS), (size_t)0, s, p,
                           block_cols));
  count_launch(1);
  if (!sums) return FK_OK;
  SumsParams a{};
  a.lens = context_lens; a.cu = cu_seqlens_q;
  a.tables = block_tables; a.table_stride = block_table_stride;
  a.capacity = p.capacity;
  a.num_seqs = num_seqs; a.num_tokens = num_tokens; a.num_pages = p.num_pages;
  a.page = page_size; a.hkv = num_kv_heads;
  a.block = p.block; a.cols = p.cols;
  a.ml = p.whole_ml; a.ml_pair = p.cols; a.ml_col = 1;
  a.logits = p.logits; a.first = p.first; a.logit_keys = w.logit_steps * QA_STEP;
  a.weights = weights; a.from = weights_from;
  FK_CUDA_OK(launch_sums(a, s));
  count_launch(1);
  return FK_OK;
}

}  // extern "C"
