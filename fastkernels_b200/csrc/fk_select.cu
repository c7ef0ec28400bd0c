// Which blocks of a long cached context a query needs: bounds of the keys of every block, and for
// each query token and KV head the blocks with the largest bound of a logit.
//
//   fk_key_bounds      lo_d = min k_d, hi_d = max k_d over the cached keys of a block (any run of
//                      `block` positions that starts at a multiple of it)
//   fk_select_blocks   score(block) = max over the query heads h of a KV head of
//                      sum_d max(q_hd lo_d, q_hd hi_d), which no q_h . k of the block exceeds;
//                      the `count` best blocks in ascending order
#include "fk_common.cuh"

namespace fk {

constexpr int SEL_D = 128;                    // head_dim
constexpr int SEL_MAX_G = 16;                 // query heads per KV head
constexpr int SEL_MAX_BLOCKS = 16384;         // of one context
constexpr int SEL_WARP_BLOCKS = 1024;         // of one context, where a warp chooses

// ---------------------------------------------------------------------------
// bounds
// ---------------------------------------------------------------------------
struct BoundsParams {
  const uint16_t* k; int64_t page_stride;
  uint16_t* bounds;                   // [pages, hkv, blocks of a page, 2, D]
  const int32_t* context_lens;
  const int32_t* tables; int64_t table_stride;
  const int32_t* cu_new;              // null: one new token each
  int64_t capacity;                   // tokens that a table's row has pages for
  int num_pages, page, block, hkv, hnd;
  int max_new;                        // new tokens that the grid has CTAs for
  int32_t* status;
};

__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&a),
                                 *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a),
                                 *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}

// A CTA takes one block of one sequence and two KV heads: four warps a head, and a warp reads two
// keys at a time, 16 bytes a lane.  Bounds are made anew from all cached keys of the block, so they
// hang on the cache alone: tokens that were taken back and stored again leave nothing behind.
__global__ void __launch_bounds__(256) key_bounds_kernel(const BoundsParams p) {
  __shared__ uint4 part[2][2][4][16];        // [head][lo / hi][warp][16-byte piece]
  pdl_launch_dependents();
  pdl_wait();
  const int seq = blockIdx.y;
  int64_t len = p.context_lens[seq];
  if (len > p.capacity) {
    len = p.capacity;
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
  }
  int64_t fresh = p.cu_new ? (int64_t)p.cu_new[seq + 1] - p.cu_new[seq] : 1;
  if (fresh > p.max_new) {                   // the newest ones then
    fresh = p.max_new;
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, FK_DEV_BAD_POSITION);
  }
  if (len <= 0 || fresh <= 0) return;
  const int64_t first = (len > fresh ? len - fresh : 0) / p.block + blockIdx.x;
  if (first * p.block >= len) return;
  const int64_t pos = first * p.block;
  const int page = p.tables[(int64_t)seq * p.table_stride + pos / p.page];
  if (page < 0 || page >= p.num_pages) {
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
    return;
  }
  const int off = (int)(pos % p.page);
  const int keys = (int)(len - pos < p.block ? len - pos : p.block);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int side = warp >> 2, head = blockIdx.z * 2 + side;
  const int piece = lane & 15;
  uint4 lo = make_uint4(0x7f807f80u, 0x7f807f80u, 0x7f807f80u, 0x7f807f80u);   // +infinity
  uint4 hi = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
  if (head < p.hkv) {
    const int64_t row = p.hnd ? SEL_D : (int64_t)p.hkv * SEL_D;
    const uint16_t* base = p.k + (int64_t)page * p.page_stride +
                           (p.hnd ? ((int64_t)head * p.page + off) * SEL_D
                                  : (int64_t)off * p.hkv * SEL_D + (int64_t)head * SEL_D) +
                           piece * 8;
#pragma unroll 8
    for (int t = (warp & 3) * 2 + (lane >> 4); t < keys; t += 8) {
      const uint4 v = *reinterpret_cast<const uint4*>(base + t * row);
      lo.x = min2_nan(lo.x, v.x); lo.y = min2_nan(lo.y, v.y);
      lo.z = min2_nan(lo.z, v.z); lo.w = min2_nan(lo.w, v.w);
      hi.x = max2_nan(hi.x, v.x); hi.y = max2_nan(hi.y, v.y);
      hi.z = max2_nan(hi.z, v.z); hi.w = max2_nan(hi.w, v.w);
    }
  }
  lo.x = min2_nan(lo.x, __shfl_xor_sync(0xffffffffu, lo.x, 16));
  lo.y = min2_nan(lo.y, __shfl_xor_sync(0xffffffffu, lo.y, 16));
  lo.z = min2_nan(lo.z, __shfl_xor_sync(0xffffffffu, lo.z, 16));
  lo.w = min2_nan(lo.w, __shfl_xor_sync(0xffffffffu, lo.w, 16));
  hi.x = max2_nan(hi.x, __shfl_xor_sync(0xffffffffu, hi.x, 16));
  hi.y = max2_nan(hi.y, __shfl_xor_sync(0xffffffffu, hi.y, 16));
  hi.z = max2_nan(hi.z, __shfl_xor_sync(0xffffffffu, hi.z, 16));
  hi.w = max2_nan(hi.w, __shfl_xor_sync(0xffffffffu, hi.w, 16));
  if (lane < 16) {
    part[side][0][warp & 3][piece] = lo;
    part[side][1][warp & 3][piece] = hi;
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const int s = threadIdx.x >> 5, up = (threadIdx.x >> 4) & 1, at = threadIdx.x & 15;
  if ((int)blockIdx.z * 2 + s >= p.hkv) return;
  uint4 r = part[s][up][0][at];
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    const uint4 v = part[s][up][i][at];
    r.x = up ? max2_nan(r.x, v.x) : min2_nan(r.x, v.x);
    r.y = up ? max2_nan(r.y, v.y) : min2_nan(r.y, v.y);
    r.z = up ? max2_nan(r.z, v.z) : min2_nan(r.z, v.z);
    r.w = up ? max2_nan(r.w, v.w) : min2_nan(r.w, v.w);
  }
  const int64_t which = ((int64_t)page * p.hkv + blockIdx.z * 2 + s) * (p.page / p.block) +
                        off / p.block;
  reinterpret_cast<uint4*>(p.bounds + (which * 2 + up) * SEL_D)[at] = r;
}

// ---------------------------------------------------------------------------
// selection
// ---------------------------------------------------------------------------
struct SelectParams {
  const uint16_t* q; int64_t q_stride;
  const uint16_t* bounds;
  const int32_t* context_lens;
  const int32_t* rows;                // table row of each token, null: its own number
  const int32_t* tables; int64_t table_stride;
  int64_t capacity;
  int num_tokens, num_tables, num_pages, page, block, hkv, g;
  int count, keep_first, keep_last;
  int per_shift;                      // log2 of the blocks of a page, -1: no power of two
  int span;                           // tokens of a CTA of the scores
  int cols;                           // columns of a token in a product: g up to a power of two
  int most;                           // blocks that a table's row has pages for
  int pitch;                          // of the scores' rows: a multiple of four
  int chunk, chunks;                  // blocks of a CTA of the scores, of those CTAs per token
  uint32_t* scores;                   // [tokens, hkv, pitch], ordered
  float* largest;                     // [spans of tokens, hkv, chunks] largest |bound| of a chunk
  float* q_sum;                       // [tokens, hkv] largest sum of |q| of a query head
  int32_t* selected;                  // [tokens, hkv, count]
  int32_t* status;
};

// Numbers in an order of whole numbers: equal values (both zeros) alike, no-number above all.  Zero
// is below all of them.
__device__ __forceinline__ uint64_t order_of(double v) {
  if (v != v) return ~0ull;
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return ~0u;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b >> 31 ? ~b : b | (1u << 31);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

// The threads that choose for one token: a warp, or all eight.
template <int W>
struct Team {
  int hist[256];
  int count;
  int eq[W], gt[W];
  uint64_t lo[W], hi[W];
  uint64_t near[32];

  static __device__ __forceinline__ int rank() { return W == 1 ? threadIdx.x & 31 : threadIdx.x; }
  static __device__ __forceinline__ int warp() { return W == 1 ? 0 : threadIdx.x >> 5; }
  static __device__ __forceinline__ void sync() {
    if (W == 1) __syncwarp(); else __syncthreads();
  }
};

// The smallest and largest of all threads' values; ends behind a barrier.
template <int W, typename KEY>
__device__ __forceinline__ void range_of(KEY& lo, KEY& hi, Team<W>& s) {
  if (sizeof(KEY) == 4) {
    lo = (KEY)__reduce_min_sync(0xffffffffu, (uint32_t)lo);
    hi = (KEY)__reduce_max_sync(0xffffffffu, (uint32_t)hi);
  } else {
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) {
      lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
  }
  if (W > 1 && (threadIdx.x & 31) == 0) { s.lo[Team<W>::warp()] = lo; s.hi[Team<W>::warp()] = hi; }
  Team<W>::sync();
  if (W > 1) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      lo = min(lo, (KEY)s.lo[w]);
      hi = max(hi, (KEY)s.hi[w]);
    }
  }
}

// The want-th largest of n keys (1 <= want <= n) between lo and hi, and how many of the keys that
// equal it are among the want largest.  Counts of 256 parts of the range leave one part, which is
// the range of the next round, until 32 keys are left, which are ranked, or all that are left are
// equal.
template <int W, typename KEY>
__device__ __forceinline__ KEY border_of(const KEY* keys, int n, int want, KEY lo, KEY hi, int* left,
                                         Team<W>& s) {
  const int tid = Team<W>::rank(), lane = threadIdx.x & 31;
  constexpr int kBits = 8 * sizeof(KEY);
  while (lo != hi) {
    const int used = kBits - (kBits == 64 ? __clzll((long long)(hi - lo)) : __clz((int)(hi - lo)));
    const int shift = max(0, used - 8);
    for (int i = tid; i < 256; i += 32 * W) s.hist[i] = 0;
    if (tid == 0) s.count = 0;
    Team<W>::sync();
    for (int i = tid; i < n; i += 32 * W) {
      const KEY k = keys[i];
      if (k >= lo && k <= hi) atomicAdd(&s.hist[(int)((k - lo) >> shift)], 1);
    }
    Team<W>::sync();
    // parts from the largest down, eight a lane; every warp looks for itself
    const int4 p1 = reinterpret_cast<const int4*>(s.hist)[63 - lane * 2];
    const int4 p0 = reinterpret_cast<const int4*>(s.hist)[62 - lane * 2];
    const int own[8] = {p1.w, p1.z, p1.y, p1.x, p0.w, p0.z, p0.y, p0.x};
    int sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += own[j];
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    before -= sum;
    const bool mine = before < want && want <= before + sum;
    int part = 0, many = 0, ahead = 0;
    if (mine) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (before < want && want <= before + own[j]) {
          part = 255 - lane * 8 - j;
          many = own[j];
          ahead = before;
        }
        before += own[j];
      }
    }
    const int src = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
    part = __shfl_sync(0xffffffffu, part, src);
    many = __shfl_sync(0xffffffffu, many, src);
    want -= __shfl_sync(0xffffffffu, ahead, src);
    lo += (KEY)part << shift;
    hi = min(hi, (KEY)(lo + (((KEY)1 << shift) - 1)));
    if (shift == 0) break;                     // lo == hi
    if (many <= 32) {
      for (int i = tid; i < n; i += 32 * W) {
        const KEY k = keys[i];
        if (k >= lo && k <= hi) s.near[atomicAdd(&s.count, 1)] = k;
      }
      Team<W>::sync();
      const KEY k = lane < many ? (KEY)s.near[lane] : (KEY)0;
      int above = 0, equal = 0;
      for (int j = 0; j < many; ++j) {
        const KEY other = __shfl_sync(0xffffffffu, k, j);
        above += other > k ? 1 : 0;
        equal += other == k ? 1 : 0;
      }
      const bool is = lane < many && above < want && want <= above + equal;
      const int at = __ffs(__ballot_sync(0xffffffffu, is)) - 1;
      lo = __shfl_sync(0xffffffffu, k, at);
      want -= __shfl_sync(0xffffffffu, above, at);
      break;
    }
    Team<W>::sync();                           // the counts have been read
  }
  Team<W>::sync();
  *left = want;
  return lo;
}

// Score of a block in 64 bits, by a warp: the largest over the query heads.  Products of two bf16 are
// exact in fp32, and 128 of them all but always in a 64-bit sum.  (Code that runs once a launch
// costs what it takes to fetch it: four heads at a time and loops, not sixteen channels a lane
// unrolled, which took 8 us instead of 2.)
__device__ __forceinline__ uint64_t exact_score(const SelectParams& p, int token, int kvh,
                                                const uint16_t* at, int lane) {
  const uint2 lo = reinterpret_cast<const uint2*>(at)[lane];
  const uint2 hi = reinterpret_cast<const uint2*>(at + SEL_D)[lane];
  const float l[4] = {bf16lo(lo.x), bf16hi(lo.x), bf16lo(lo.y), bf16hi(lo.y)};
  const float u[4] = {bf16lo(hi.x), bf16hi(hi.x), bf16lo(hi.y), bf16hi(hi.y)};
  const uint16_t* qp = p.q + (int64_t)token * p.q_stride + (int64_t)kvh * p.g * SEL_D;
  double best = -INFINITY;
  bool nan = false;
#pragma unroll 1
  for (int h0 = 0; h0 < p.g; h0 += 4) {
    uint2 v[4];
#pragma unroll
    for (int h = 0; h < 4; ++h)                // the last head again behind the last
      v[h] = reinterpret_cast<const uint2*>(qp + min(h0 + h, p.g - 1) * SEL_D)[lane];
    double sum[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const float q[4] = {bf16lo(v[h].x), bf16hi(v[h].x), bf16lo(v[h].y), bf16hi(v[h].y)};
      sum[h] = 0.0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // one side of the maximum; no number, or zero times infinity, counts on either
        sum[h] += (double)q[k] * (double)(q[k] > 0.f ? u[k] : l[k]);
        const float other = q[k] > 0.f ? q[k] * l[k] : q[k] * u[k];
        nan |= other != other;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int h = 0; h < 4; ++h) sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], o);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      nan |= sum[h] != sum[h];
      best = fmax(best, sum[h]);
    }
  }
  return __any_sync(0xffffffffu, nan) ? ~0ull : order_of(best);
}

// The choice of one token, by a team: `keys` are the scores of its n - keep_first - keep_last blocks
// in the middle, `reach` bounds sum |q| max |bound|, key_lo and key_hi are
// the smallest and largest key.  exact and band: room for those blocks.
template <int W>
__device__ __forceinline__ void choose(const SelectParams& p, int token, int kvh, int n,
                                       const int32_t* table, uint32_t* keys, float reach,
                                       uint32_t key_lo, uint32_t key_hi, uint64_t* exact, uint16_t* band, Team<W>& s) {
  const int tid = Team<W>::rank(), warp = Team<W>::warp(), lane = threadIdx.x & 31;
  const uint32_t below = (1u << lane) - 1u;
  const int per = p.page / p.block;
  int32_t* out = p.selected + ((int64_t)token * p.hkv + kvh) * p.count;
  if (n <= p.count) {
    for (int i = tid; i < p.count; i += 32 * W) out[i] = i < n ? i : -1;
    return;
  }
  const int middle = n - p.keep_first - p.keep_last;
  const int want = p.count - p.keep_first - p.keep_last;     // of the middle ones
  for (int i = tid; i < p.keep_first; i += 32 * W) out[i] = i;
  for (int i = tid; i < p.keep_last; i += 32 * W)
    out[p.count - p.keep_last + i] = n - p.keep_last + i;
  if (want == 0) return;
  // scores past fp32's range, products below it, and what is no number: all in 64 bits
  const bool all = !(reach < INFINITY) || (reach > 0.f && reach < 7.9e-31f) || key_hi == ~0u;
  uint32_t above = ~0u, least = 0u;            // keys above are taken, keys below `least` are not
  bool same = false;                           // keys between are equal in truth
  if (!all) {
    int left;
    const uint32_t border = border_of<W, uint32_t>(keys, middle, want, key_lo, key_hi, &left, s);
    const float v = value_of(border), e2 = reach * (2.f / 262144.f);
    same = border == 0u || reach == 0.f;
    above = same ? border : order_of(v + e2);
    least = same ? border : order_of(v - e2);
  }
  // how many are above, and between; each warp has a run of blocks
  const int run = ((middle + W - 1) / W + 31) / 32 * 32;
  const int from = min(warp * run, middle), to = min(from + run, middle);
  auto count = [&](int* eqs, int* gts, int* eq_before, int* gt_before) {
    int eq = 0, gt = 0;
    for (int i = from + lane; i < to; i += 32) {
      gt += keys[i] > above ? 1 : 0;
      eq += keys[i] >= least && keys[i] <= above ? 1 : 0;
    }
    *eqs = __reduce_add_sync(0xffffffffu, eq);
    *gts = __reduce_add_sync(0xffffffffu, gt);
    *eq_before = *gt_before = 0;
    if (W == 1) return;
    Team<W>::sync();
    if (lane == 0) { s.eq[warp] = *eqs; s.gt[warp] = *gts; }
    Team<W>::sync();
    *eqs = *gts = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w == warp) { *eq_before = *eqs; *gt_before = *gts; }
      *eqs += s.eq[w];
      *gts += s.gt[w];
    }
  };
  int eqs, gts, eq_before, gt_before;
  count(&eqs, &gts, &eq_before, &gt_before);
  int ties = want - gts;                       // of those between, the first ones if they are equal
  if (!same && eqs > ties) {
    // score those between again; their keys become "taken" or "not"
    int at = eq_before;
    for (int i0 = from; i0 < to; i0 += 32) {
      const int i = i0 + lane;
      const bool is = i < to && keys[i] >= least && keys[i] <= above;
      const uint32_t votes = __ballot_sync(0xffffffffu, is);
      if (is) band[at + __popc(votes & below)] = (uint16_t)i;
      at += __popc(votes);
    }
    Team<W>::sync();
    for (int c = warp; c < eqs; c += W) {
      const int b = p.keep_first + band[c];
      uint64_t key = 0ull;                     // without a page
      if (keys[band[c]] != 0u) {
        const int at_page = p.per_shift >= 0 ? b >> p.per_shift : b / per;
        key = exact_score(p, token, kvh,
                          p.bounds + (((int64_t)table[at_page] * p.hkv + kvh) * per + b -
                                      at_page * per) * 2 * SEL_D, lane);
      }
      if (lane == 0) exact[c] = key;
    }
    Team<W>::sync();
    if (eqs <= 32) {
      // a lane per block: its rank, the lower index first among equals
      const uint64_t key = lane < eqs ? exact[lane] : 0ull;
      int rank = 0;
      for (int j = 0; j < eqs; ++j) {
        const uint64_t other = __shfl_sync(0xffffffffu, key, j);
        rank += other > key || (other == key && j < lane) ? 1 : 0;
      }
      if (warp == 0 && lane < eqs) keys[band[lane]] = rank < ties ? ~0u : 0u;
    } else {
      uint64_t lo = ~0ull, hi = 0ull;
      for (int c = tid; c < eqs; c += 32 * W) {
        lo = min(lo, exact[c]);
        hi = max(hi, exact[c]);
      }
      range_of<W, uint64_t>(lo, hi, s);
      int left;
      const uint64_t edge = border_of<W, uint64_t>(exact, eqs, ties, lo, hi, &left, s);
      // equal ones in order: a warp has a run of them, as above
      const int run_c = ((eqs + W - 1) / W + 31) / 32 * 32;
      const int fc = min(warp * run_c, eqs), tc = min(fc + run_c, eqs);
      int seen = 0;
      if (W > 1) {
        int n_eq = 0;
        for (int c = fc + lane; c < tc; c += 32) n_eq += exact[c] == edge ? 1 : 0;
        n_eq = __reduce_add_sync(0xffffffffu, n_eq);
        if (lane == 0) s.eq[warp] = n_eq;
        Team<W>::sync();
        for (int w = 0; w < warp; ++w) seen += s.eq[w];
      }
      for (int c0 = fc; c0 < tc; c0 += 32) {
        const int c = c0 + lane;
        const bool is = c < tc && exact[c] == edge;
        const uint32_t votes = __ballot_sync(0xffffffffu, is);
        if (c < tc)
          keys[band[c]] =
              exact[c] > edge || (is && seen + __popc(votes & below) < left) ? ~0u : 0u;
        seen += __popc(votes);
      }
    }
    Team<W>::sync();
    // taken ones are above now, and nothing is between
    above = min(above, ~0u - 1u);
    least = ~0u;
    count(&eqs, &gts, &eq_before, &gt_before);
    ties = 0;
    eq_before = 0;
  }
  // taken ones in order
  int seen = eq_before, at = gt_before + min(eq_before, ties);
  for (int i0 = from; i0 < to; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t key = i < to ? keys[i] : 0u;
    const bool is_eq = ties > 0 && i < to && key >= least && key <= above;
    const uint32_t votes = __ballot_sync(0xffffffffu, is_eq);
    const bool take = i < to && (key > above || (is_eq && seen + __popc(votes & below) < ties));
    const uint32_t takes = __ballot_sync(0xffffffffu, take);
    if (take) out[p.keep_first + at + __popc(takes & below)] = p.keep_first + i;
    seen += __popc(votes);
    at += __popc(takes);
  }
}

// a b with sums that begin at zero
__device__ __forceinline__ void mma_from_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// the larger one, or no number where either is none
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// two fp32 sums in one instruction
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}

constexpr int SEL_STAGES = 2;                  // 16 blocks each of a warp's bounds under way
constexpr int SEL_WARPS = 4;                   // of a CTA of the scores
constexpr int SEL_RING_BYTES = SEL_WARPS * SEL_STAGES * 16 * 32 * 16;

// 16 bytes into shared memory, or zeros.
__device__ __forceinline__ void copy16(uint4* dst, const uint16_t* src, bool have) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(have ? 16 : 0)
               : "memory");
}

// ---- scores: sum_d max(q_d lo_d, q_d hi_d) = q+ . hi + q- . lo with the positive and negative parts of
// q, a product of 16 blocks by 8 query heads by 256 on the tensor cores.  A lane takes 16 bytes of a
// row at a time, which are operands of two instructions when q's channels are taken in the same
// order.  Sums in fp32 are off by at most e = 2^-18 sum |q| max |bound|: an instruction adds 17 terms
// (its sum begins at zero), each off by at most 2^-23 of the sum of absolute values, and a term
// goes through at most six further additions of 2^-24: 20 x 2^-23 = 2^-18.7.

// 16 blocks (two of them with this lane's pieces: lower and upper bounds) by 8 columns; v: columns
// 2 (lane % 4) + 0, 1 of blocks lane / 4 and lane / 4 + 8.
__device__ __forceinline__ void score_tile(const uint4 (&l0)[4], const uint4 (&u0)[4],
                                           const uint4 (&l1)[4], const uint4 (&u1)[4],
                                           const uint32_t (&qp)[4][4], const uint32_t (&qm)[4][4],
                                           float (&v)[4]) {
  uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float c[4][4];
    mma_from_zero(c[0], u0[j].x, u1[j].x, u0[j].y, u1[j].y, qp[j][0], qp[j][1]);
    mma_from_zero(c[1], l0[j].x, l1[j].x, l0[j].y, l1[j].y, qm[j][0], qm[j][1]);
    mma_from_zero(c[2], u0[j].z, u1[j].z, u0[j].w, u1[j].w, qp[j][2], qp[j][3]);
    mma_from_zero(c[3], l0[j].z, l1[j].z, l0[j].w, l1[j].w, qm[j][2], qm[j][3]);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      sum[i] = add_pair(sum[i], add_pair(add_pair(pair_of(c[0][2 * i], c[0][2 * i + 1]),
                                                  pair_of(c[1][2 * i], c[1][2 * i + 1])),
                                         add_pair(pair_of(c[2][2 * i], c[2][2 * i + 1]),
                                                  pair_of(c[3][2 * i], c[3][2 * i + 1]))));
  }
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v[0]), "=f"(v[1]) : "l"(sum[0]));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v[2]), "=f"(v[3]) : "l"(sum[1]));
}

// The largest upper bound and the smallest lower one, two channels at once, from below and above zero:
// bits of bf16 as signed numbers order those above zero, and as unsigned ones those below it, the
// most negative last.  (A bound that is no number makes a score that is none.)
struct Extent {
  uint32_t top = 0u, low = 0x80008000u;
  __device__ __forceinline__ void add(const uint4& l, const uint4& u) {
    top = __vimax3_s16x2(top, u.x, u.y); top = __vimax3_s16x2(top, u.z, u.w);
    low = __vimax3_u16x2(low, l.x, l.y); low = __vimax3_u16x2(low, l.z, l.w);
  }
  // largest |bound| of a CTA's warps, as a number's bits; `scratch`: a word per warp
  __device__ __forceinline__ uint32_t of_cta(uint32_t* scratch) const {
    uint32_t most = max(max((top & 0xffffu) << 16, top & 0x7fff0000u),
                        max((low & 0x7fffu) << 16, low & 0x7fff0000u));
    most = __reduce_max_sync(0xffffffffu, most);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SEL_WARPS; ++w) most = max(most, scratch[w]);
    return most;
  }
};

__device__ __forceinline__ int select_length(const SelectParams& p, int token, int row) {
  const int64_t len = p.context_lens[token];
  if (len <= 0 || row < 0 || row >= p.num_tables) return 0;
  return (int)(len > p.capacity ? p.capacity : len);
}
// blocks keep_first .. of a context that are scored
__device__ __forceinline__ int select_scored(const SelectParams& p, int len) {
  const int blocks = (int)(((int64_t)len + p.block - 1) / p.block);
  return blocks > p.count ? blocks - p.keep_first - p.keep_last : 0;
}
// positive and negative parts of a column's channels 32 j + 8 (lane % 4) + 0 .. 7
__device__ __forceinline__ void split_q(const uint4 (&v)[4], uint32_t (&qp)[4][4],
                                        uint32_t (&qm)[4][4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      qp[j][i] = max2_nan(w[i], 0u);
      qm[j][i] = min2_nan(w[i], 0u);
    }
  }
}
// sum of |q| of a column, over its four lanes; no number counts as infinite
__device__ __forceinline__ float abs_q(const uint4 (&v)[4]) {
  float a = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) a += fabsf(bf16lo(w[i])) + fabsf(bf16hi(w[i]));
  }
  a += __shfl_xor_sync(0xffffffffu, a, 1);
  a += __shfl_xor_sync(0xffffffffu, a, 2);
  return a < INFINITY ? a : INFINITY;
}

// ---- a token for itself: a CTA per token, KV head and chunk of blocks.  A warp has 16 blocks at a time
// and as many on their way in shared memory.  Bounds: the bytes of the bounds (64 tokens of 8192 to
// 65536 keys, 148 MB: 31 us), and the instructions around the products.
template <int NT>                              // 8 query heads each
__global__ void __launch_bounds__(32 * SEL_WARPS, 3)
select_scores_kernel(const SelectParams p) {
  extern __shared__ __align__(16) uint8_t sel_smem[];
  uint4* ring = reinterpret_cast<uint4*>(sel_smem);
  pdl_launch_dependents();
  pdl_wait();
  const int kvh = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int token = blockIdx.x / p.chunks, chunk = blockIdx.x - token * p.chunks;
  const int per = p.page / p.block;
  const int r0 = lane >> 2, quad = lane & 3;
  const int row = token;
  const int scored = select_scored(p, select_length(p, token, row));
  const int begin = chunk * p.chunk, end = min(scored, begin + p.chunk);
  Extent extent;
  if (begin < end) {
    const int32_t* table = p.tables + (int64_t)row * p.table_stride;
    // pages of the two blocks that this lane copies pieces of
    auto page_of = [&](int at) -> int {
      const int b = p.keep_first + at;
      return at < end ? table[p.per_shift >= 0 ? b >> p.per_shift : b / per] : -1;
    };
    uint32_t have = 0;                         // two bits per stage
    auto copy = [&](int b0, int stage, int page0, int page1) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int page = half ? page1 : page0, at = b0 + half * 8 + r0;
        const bool ok = page >= 0 && page < p.num_pages;
        if (!ok && at < end && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
        const uint32_t bit = 1u << (stage * 2 + half);
        have = ok ? have | bit : have & ~bit;
        const int b = p.keep_first + at;
        const int in = p.per_shift >= 0 ? b & (per - 1) : b % per;
        const uint16_t* src =
            p.bounds + (ok ? (((int64_t)page * p.hkv + kvh) * per + in) * 2 * SEL_D : 0) + quad * 8;
        uint4* dst = ring + ((warp * SEL_STAGES + stage) * 16 + half * 8) * 32 + lane;
#pragma unroll
        for (int j = 0; j < 8; ++j) copy16(dst + j * 32, src + j * 32, ok);
      }
    };
    constexpr int kStep = 16 * SEL_WARPS;
    int ahead = begin + warp * 16;
#pragma unroll
    for (int i = 0; i < SEL_STAGES; ++i, ahead += kStep) {
      if (ahead < end) copy(ahead, i, page_of(ahead + r0), page_of(ahead + 8 + r0));
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    int page0 = page_of(ahead + r0), page1 = page_of(ahead + 8 + r0);
    // column lane / 4 of 8: a query head
    uint32_t qp[NT][4][4], qm[NT][4][4];
    float abs_sum = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = nt * 8 + r0;
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = head < p.g ? *reinterpret_cast<const uint4*>(
                                p.q + (int64_t)token * p.q_stride +
                                ((int64_t)kvh * p.g + head) * SEL_D + j * 32 + quad * 8)
                          : make_uint4(0u, 0u, 0u, 0u);
      split_q(v, qp[nt], qm[nt]);
      if (chunk == 0 && warp == 0) abs_sum = fmaxf(abs_sum, abs_q(v));
    }
    if (chunk == 0 && warp == 0) {
      abs_sum = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(abs_sum)));
      if (lane == 0) p.q_sum[(int64_t)token * p.hkv + kvh] = abs_sum;
    }
    int stage = 0;
    for (int b0 = begin + warp * 16; b0 < end; b0 += kStep) {
      asm volatile("cp.async.wait_group %0;" ::"n"(SEL_STAGES - 1) : "memory");
      const uint4* src = ring + (warp * SEL_STAGES + stage) * 512 + lane;
      uint4 l0[4], u0[4], l1[4], u1[4];        // blocks r0 and r0 + 8
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        l0[j] = src[j * 32]; u0[j] = src[(4 + j) * 32];
        l1[j] = src[(8 + j) * 32]; u1[j] = src[(12 + j) * 32];
        extent.add(l0[j], u0[j]);
        extent.add(l1[j], u1[j]);
      }
      float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float v[4];
        score_tile(l0, u0, l1, u1, qp[nt], qm[nt], v);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool live = nt * 8 + quad * 2 + i < p.g;
          m0 = max_nan(m0, live ? v[i] : -INFINITY);
          m1 = max_nan(m1, live ? v[2 + i] : -INFINITY);
        }
      }
      const bool ok0 = have >> (stage * 2) & 1u, ok1 = have >> (stage * 2 + 1) & 1u;
      // the stage has been read: its next blocks
      const int now0 = page0, now1 = page1;
      page0 = page_of(ahead + kStep + r0);
      page1 = page_of(ahead + kStep + 8 + r0);
      if (ahead < end) copy(ahead, stage, now0, now1);
      asm volatile("cp.async.commit_group;" ::: "memory");
      ahead += kStep;
      if (++stage == SEL_STAGES) stage = 0;
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        m0 = max_nan(m0, __shfl_xor_sync(0xffffffffu, m0, o));
        m1 = max_nan(m1, __shfl_xor_sync(0xffffffffu, m1, o));
      }
      uint32_t* scores = p.scores + ((int64_t)token * p.hkv + kvh) * p.pitch + b0 + r0;
      if (quad == 0 && b0 + r0 < end) scores[0] = ok0 ? order_of(m0) : 0u;
      if (quad == 0 && b0 + 8 + r0 < end) scores[8] = ok1 ? order_of(m1) : 0u;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  const uint32_t most = extent.of_cta(reinterpret_cast<uint32_t*>(ring));     // which has been read
  if (threadIdx.x == 0)
    p.largest[((int64_t)token * p.hkv + kvh) * p.chunks + chunk] = __uint_as_float(most);
}

// ---- tokens that may have one table: a CTA per span of tokens, KV head and 64 blocks.  A warp keeps the
// bounds of 16 blocks in registers and goes over the query heads of all tokens of the table.
// Bounds: instructions (some 350 for 16 blocks by 8 columns) at three warps a scheduler.
__global__ void __launch_bounds__(32 * SEL_WARPS, 3)
select_scores_many_kernel(const SelectParams p) {
  __shared__ uint32_t scratch[SEL_WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int kvh = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = blockIdx.x / p.chunks, chunk = blockIdx.x - group * p.chunks;
  const int per = p.page / p.block;
  const int r0 = lane >> 2, quad = lane & 3;
  const int shift = 31 - __clz(p.cols);
  const int end_token = min(p.num_tokens, (group + 1) * p.span);
  Extent extent;
  for (int t0 = group * p.span; t0 < end_token;) {
    // a run of tokens with one table, 32 looked at together
    const int row = p.rows[t0];
    int t1 = t0, longest = 0;
    for (;;) {
      const int t = t1 + lane;
      const bool same = t < end_token && p.rows[t] == row;
      const uint32_t others = ~__ballot_sync(0xffffffffu, same);
      const int many = others ? __ffs(others) - 1 : 32;
      longest = max(longest, __reduce_max_sync(0xffffffffu,
                                               lane < many ? select_length(p, t, row) : 0));
      t1 += many;
      if (many < 32) break;
    }
    const int scored = select_scored(p, longest);
    const int b0 = chunk * p.chunk + warp * 16;
    const int first = t0;
    t0 = t1;
    if (b0 >= scored) continue;
    const int32_t* table = p.tables + (int64_t)row * p.table_stride;
    uint4 l0[4], u0[4], l1[4], u1[4];          // blocks b0 + r0 and b0 + 8 + r0
    bool ok[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int at = b0 + half * 8 + r0, b = p.keep_first + at;
      const int page = at < scored ? table[p.per_shift >= 0 ? b >> p.per_shift : b / per] : -1;
      ok[half] = page >= 0 && page < p.num_pages;
      if (!ok[half] && at < scored && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
      const int in = p.per_shift >= 0 ? b & (per - 1) : b % per;
      const uint4* src = reinterpret_cast<const uint4*>(
          p.bounds + (ok[half] ? (((int64_t)page * p.hkv + kvh) * per + in) * 2 * SEL_D : 0) +
          quad * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 none = make_uint4(0u, 0u, 0u, 0u);
        const uint4 l = ok[half] ? src[j * 4] : none, u = ok[half] ? src[16 + j * 4] : none;
        if (half) { l1[j] = l; u1[j] = u; } else { l0[j] = l; u0[j] = u; }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      extent.add(l0[j], u0[j]);
      extent.add(l1[j], u1[j]);
    }
    // columns: p.cols a token, the last ones of them without a head
    const int tiles = ((t1 - first) * p.cols + 7) / 8;
    auto column = [&](int nt, uint4 (&v)[4]) {
      const int col = nt * 8 + r0, t = first + (col >> shift), head = col & (p.cols - 1);
      const bool live = t < t1 && head < p.g;
      const uint4* src = reinterpret_cast<const uint4*>(
          p.q + (int64_t)(live ? t : first) * p.q_stride +
          ((int64_t)kvh * p.g + (live ? head : 0)) * SEL_D + quad * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = live ? src[j * 4] : make_uint4(0u, 0u, 0u, 0u);
    };
    uint4 next[4];
    column(0, next);
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, a_max = 0.f;
    for (int nt = 0; nt < tiles; ++nt) {
      uint32_t qp[4][4], qm[4][4];
      split_q(next, qp, qm);
      float a = chunk == 0 && warp == 0 ? abs_q(next) : 0.f;
      if (nt + 1 < tiles) column(nt + 1, next);
      float v[4];
      score_tile(l0, u0, l1, u1, qp, qm, v);
      // a token's heads: columns 2 quad + 0, 1, then next lanes, then the next tile (of one head a
      // token, every column is another token)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int head = (nt * 8 + quad * 2 + (i & 1)) & (p.cols - 1);
        v[i] = head < p.g ? v[i] : -INFINITY;
      }
      if (p.cols > 1) {
        v[0] = v[1] = max_nan(v[0], v[1]);
        v[2] = v[3] = max_nan(v[2], v[3]);
      }
      for (int o = 1; o < min(p.cols, 8) / 2; o <<= 1) {
        v[0] = max_nan(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
        v[2] = max_nan(v[2], __shfl_xor_sync(0xffffffffu, v[2], o));
      }
      if (p.cols == 16) {
        const bool more = nt & 1;              // the token's second half
        v[0] = m[0] = more ? max_nan(m[0], v[0]) : v[0];
        v[2] = m[2] = more ? max_nan(m[2], v[2]) : v[2];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = nt * 8 + quad * 2 + i, t = first + (col >> shift);
        const int at = col & (p.cols - 1);
        if (at != (p.cols == 16 ? 8 : 0) || t >= t1) continue;
        uint32_t* scores = p.scores + ((int64_t)t * p.hkv + kvh) * p.pitch + b0 + r0;
        if (b0 + r0 < scored) scores[0] = ok[0] ? order_of(v[i]) : 0u;
        if (b0 + 8 + r0 < scored) scores[8] = ok[1] ? order_of(v[2 + i]) : 0u;
      }
      if (chunk == 0 && warp == 0) {
        // the largest sum of |q| of each token's heads
        for (int o = 1; o < min(p.cols, 8); o <<= 1)
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o * 4));
        if (p.cols == 16) a = a_max = nt & 1 ? fmaxf(a_max, a) : a;
        const int col = nt * 8 + r0, t = first + (col >> shift);
        if (quad == 0 && (col & (p.cols - 1)) == (p.cols == 16 ? 8 : 0) && t < t1)
          p.q_sum[(int64_t)t * p.hkv + kvh] = a;
      }
    }
  }
  const uint32_t most = extent.of_cta(scratch);
  if (threadIdx.x == 0)
    p.largest[((int64_t)group * p.hkv + kvh) * p.chunks + chunk] = __uint_as_float(most);
}

// ---- the choice: a team of W warps per token and KV head, a CTA of its own or, of one warp, eight in one
//
// Blocks above the want-th largest score by more than 2 e are taken, those below it by more are not,
// and those between are scored again in 64 bits if they do not all fit.  So the choice is that of
// 64 bits, ties to the lower index.
//
// Bounds: the latency of its steps.  Eight warps take the shortest time over one, a single warp the
// fewest instructions: the more there are to choose, the fewer warps for each.
template <int W>
__global__ void __launch_bounds__(W == 1 ? 256 : 32 * W) select_choose_kernel(const SelectParams p) {
  extern __shared__ __align__(16) uint8_t sel_smem[];
  constexpr int kTeams = W == 1 ? 8 : 1;
  __shared__ Team<W> teams[kTeams];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, team = W == 1 ? threadIdx.x >> 5 : 0;
  const int64_t item = (int64_t)blockIdx.x * kTeams + team;
  if (item >= (int64_t)p.num_tokens * p.hkv) return;
  const int token = (int)(item / p.hkv), kvh = (int)(item - (int64_t)token * p.hkv);
  const int row = p.rows ? p.rows[token] : token;
  int64_t len = p.context_lens[token];
  if (row < 0 || row >= p.num_tables || len > p.capacity) {
    if (Team<W>::rank() == 0 && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
    len = row < 0 || row >= p.num_tables ? 0 : p.capacity;
  }
  const int n = (int)((max(len, (int64_t)0) + p.block - 1) / p.block);
  // [teams][most] each
  uint64_t* exact = reinterpret_cast<uint64_t*>(sel_smem) + team * p.most;
  uint32_t* keys = reinterpret_cast<uint32_t*>(sel_smem + (size_t)kTeams * p.most * 8) +
                   team * p.most;
  uint16_t* band = reinterpret_cast<uint16_t*>(sel_smem + (size_t)kTeams * p.most * 12) +
                   team * p.most;
  float reach = 0.f;
  uint32_t key_lo = ~0u, key_hi = 0u;
  if (n > p.count) {
    const int middle = n - p.keep_first - p.keep_last;
    const uint4* src = reinterpret_cast<const uint4*>(p.scores + item * p.pitch);
    for (int i = Team<W>::rank() * 4; i < middle; i += 128 * W) {
      const uint4 v = src[i >> 2];
      const uint32_t k[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (i + h >= middle) break;
        keys[i + h] = k[h];
        key_lo = min(key_lo, k[h]);
        key_hi = max(key_hi, k[h]);
      }
    }
    // largest |bound|; no number counts as infinite
    const float* from = p.largest + ((int64_t)(token / p.span) * p.hkv + kvh) * p.chunks;
    float largest = 0.f;
    for (int i = lane; i < p.chunks; i += 32)
      largest = fmaxf(largest, from[i] < INFINITY ? from[i] : INFINITY);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    reach = p.q_sum[item] * largest;
    range_of<W, uint32_t>(key_lo, key_hi, teams[team]);
  }
  choose<W>(p, token, kvh, n, p.tables + (int64_t)row * p.table_stride, keys, reach, key_lo,
            key_hi, exact, band, teams[team]);
}

// Tokens of a CTA, its blocks, and what is in a workspace.
struct SelectLayout {
  int span, chunk, chunks, pitch;
  int64_t groups;
  size_t largest, q_sum, total;       // bytes
};
static SelectLayout select_layout(int64_t tokens, int hkv, bool rows, int64_t most) {
  SelectLayout s;
  const int sms = sm_count();
  s.span = 1;
  s.chunk = 256;
  if (rows) {
    // spans as long as leaves two rounds of work for every SM's three CTAs (1000 tokens of two
    // prompts 66 us; one round 79, eight 73)
    s.chunk = 64;
    s.chunks = (int)((most + s.chunk - 1) / s.chunk);
    s.span = 64;
    while (s.span > 1 && (tokens + s.span - 1) / s.span * hkv * s.chunks < 6ll * sms) s.span /= 2;
  } else {
    // long chunks for the pipeline's sake, unless that leaves SMs without work
    while (s.chunk > 64 && tokens * hkv * ((most + s.chunk - 1) / s.chunk) < 4ll * sms)
      s.chunk /= 2;
    s.chunks = (int)((most + s.chunk - 1) / s.chunk);
  }
  s.groups = (tokens + s.span - 1) / s.span;
  s.pitch = (int)((most + 3) & ~3ll);
  s.largest = ((size_t)tokens * hkv * s.pitch * 4 + 255) & ~size_t(255);
  s.q_sum = s.largest + (size_t)s.groups * hkv * s.chunks * 4;
  s.total = s.q_sum + (size_t)tokens * hkv * 4;
  return s;
}

// what the entry points of this file have in common
static int check_cache(const char* what, int page, int block, int hkv, int head_dim,
                       int64_t num_pages, int64_t table_cols) {
  FK_REQUIRE(head_dim == SEL_D, FK_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (128 only)", what,
             head_dim);
  FK_REQUIRE(block == 16 || block == 32 || (block >= 64 && block % 64 == 0), FK_ERR_UNSUPPORTED,
             "%s: block %d must be 16, 32 or a multiple of 64", what, block);
  FK_REQUIRE(page > 0 && page % block == 0, FK_ERR_INVALID_ARG,
             "%s: a page of %d tokens is not a whole number of blocks of %d", what, page, block);
  FK_REQUIRE(hkv > 0 && num_pages > 0 && num_pages < (1ll << 31) && table_cols > 0,
             FK_ERR_INVALID_ARG, "%s: bad sizes", what);
  return FK_OK;
}

}  // namespace fk

using namespace fk;

extern "C" {

int fk_key_bounds(const void* k_cache, int64_t num_pages, int page_size, int64_t kv_page_stride,
                  int kv_layout, int num_kv_heads, int head_dim, void* bounds, int block,
                  const int32_t* context_lens, const int32_t* block_tables,
                  int64_t block_table_stride, int64_t block_table_cols, const int32_t* cu_new,
                  int num_seqs, int max_new, int32_t* status, fk_stream_t stream) {
  FK_REQUIRE(num_seqs >= 0 && max_new >= 0, FK_ERR_INVALID_ARG, "fk_key_bounds: negative size");
  if (num_seqs == 0 || max_new == 0) return FK_OK;
  FK_REQUIRE(k_cache && bounds && context_lens && block_tables, FK_ERR_INVALID_ARG,
             "fk_key_bounds: null pointer");
  const int rc = check_cache("fk_key_bounds", page_size, block, num_kv_heads, head_dim, num_pages,
                             block_table_cols);
  if (rc != FK_OK) return rc;
  FK_REQUIRE(kv_layout == 0 || kv_layout == 1, FK_ERR_INVALID_ARG,
             "fk_key_bounds: kv_layout must be 0 (NHD) or 1 (HND)");
  FK_REQUIRE(kv_page_stride >= (int64_t)page_size * num_kv_heads * head_dim &&
                 block_table_stride >= 0,
             FK_ERR_INVALID_ARG, "fk_key_bounds: stride too small");
  FK_REQUIRE(cu_new != nullptr || max_new == 1, FK_ERR_INVALID_ARG,
             "fk_key_bounds: %d new tokens need cu_new", max_new);
  FK_REQUIRE(aligned16(k_cache) && aligned16(bounds) && kv_page_stride % 8 == 0, FK_ERR_ALIGNMENT,
             "fk_key_bounds: 16-byte alignment required");
  FK_REQUIRE(num_seqs <= 65535 && num_kv_heads <= 131070, FK_ERR_UNSUPPORTED,
             "fk_key_bounds: more than 65535 sequences");
  BoundsParams p{};
  p.k = static_cast<const uint16_t*>(k_cache); p.page_stride = kv_page_stride;
  p.bounds = static_cast<uint16_t*>(bounds);
  p.context_lens = context_lens;
  p.tables = block_tables; p.table_stride = block_table_stride;
  p.cu_new = cu_new;
  p.capacity = block_table_cols * page_size;
  p.num_pages = (int)num_pages; p.page = page_size; p.block = block; p.hkv = num_kv_heads;
  p.hnd = kv_layout;
  p.max_new = max_new;
  p.status = status;
  // a run of max_new tokens touches at most this many blocks
  const int64_t blocks = ((int64_t)max_new - 1 + block - 1) / block + 1;
  FK_CUDA_OK(launch_kernel(key_bounds_kernel,
                           dim3((unsigned)blocks, (unsigned)num_seqs,
                                (unsigned)((num_kv_heads + 1) / 2)),
                           dim3(256), (size_t)0, static_cast<cudaStream_t>(stream), p));
  count_launch(1);
  return FK_OK;
}

size_t fk_select_blocks_workspace_bytes(int num_tokens, int num_q_heads, int num_kv_heads,
                                        int page_size, int block, int64_t block_table_cols) {
  if (num_tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads ||
      block <= 0 || page_size < block || block_table_cols <= 0)
    return 0;
  // the larger of both ways to group tokens
  const int64_t most = block_table_cols * (page_size / block);
  const size_t a = select_layout(num_tokens, num_kv_heads, false, most).total;
  const size_t b = select_layout(num_tokens, num_kv_heads, true, most).total;
  return a > b ? a : b;
}

int fk_select_blocks(const void* q, int64_t q_stride_token, const void* bounds, int64_t num_pages,
                     int page_size, int block, const int32_t* context_lens,
                     const int32_t* table_rows, const int32_t* block_tables,
                     int64_t block_table_stride, int64_t block_table_cols, int num_tables,
                     int num_tokens, int num_q_heads, int num_kv_heads, int head_dim, int count,
                     int keep_first, int keep_last, int32_t* selected, void* workspace,
                     size_t workspace_bytes, int32_t* status, fk_stream_t stream) {
  FK_REQUIRE(num_tokens >= 0, FK_ERR_INVALID_ARG, "fk_select_blocks: negative size");
  if (num_tokens == 0) return FK_OK;
  FK_REQUIRE(q && bounds && context_lens && block_tables && selected, FK_ERR_INVALID_ARG,
             "fk_select_blocks: null pointer");
  const int rc = check_cache("fk_select_blocks", page_size, block, num_kv_heads, head_dim,
                             num_pages, block_table_cols);
  if (rc != FK_OK) return rc;
  FK_REQUIRE(num_q_heads > 0 && num_q_heads % num_kv_heads == 0, FK_ERR_INVALID_ARG,
             "fk_select_blocks: num_q_heads must be a multiple of num_kv_heads");
  FK_REQUIRE(num_q_heads / num_kv_heads <= SEL_MAX_G, FK_ERR_UNSUPPORTED,
             "fk_select_blocks: more than %d query heads per KV head", SEL_MAX_G);
  FK_REQUIRE(keep_first >= 0 && keep_last >= 1 && count >= 1 && keep_first <= count &&
                 keep_last <= count - keep_first,
             FK_ERR_INVALID_ARG,
             "fk_select_blocks: of %d blocks the first %d and the last %d are kept "
             "(at least the last one is)", count, keep_first, keep_last);
  FK_REQUIRE(q_stride_token >= (int64_t)num_q_heads * head_dim && block_table_stride >= 0,
             FK_ERR_INVALID_ARG, "fk_select_blocks: stride too small");
  FK_REQUIRE(table_rows != nullptr || num_tables >= num_tokens, FK_ERR_INVALID_ARG,
             "fk_select_blocks: %d tables for %d tokens", num_tables, num_tokens);
  FK_REQUIRE(aligned16(q) && aligned16(bounds) && q_stride_token % 8 == 0, FK_ERR_ALIGNMENT,
             "fk_select_blocks: 16-byte alignment required");
  const int64_t most = block_table_cols * (page_size / block);
  FK_REQUIRE(most <= SEL_MAX_BLOCKS, FK_ERR_UNSUPPORTED,
             "fk_select_blocks: tables of %lld blocks (at most %d)", (long long)most,
             SEL_MAX_BLOCKS);
  FK_REQUIRE(num_kv_heads <= 65535, FK_ERR_UNSUPPORTED, "fk_select_blocks: too many heads");
  SelectParams p{};
  p.q = static_cast<const uint16_t*>(q); p.q_stride = q_stride_token;
  p.bounds = static_cast<const uint16_t*>(bounds);
  p.context_lens = context_lens; p.rows = table_rows;
  p.tables = block_tables; p.table_stride = block_table_stride;
  p.capacity = block_table_cols * page_size;
  p.num_tokens = num_tokens; p.num_tables = num_tables; p.num_pages = (int)num_pages;
  p.page = page_size; p.block = block;
  p.hkv = num_kv_heads; p.g = num_q_heads / num_kv_heads;
  p.count = count; p.keep_first = keep_first; p.keep_last = keep_last;
  p.most = (int)most;
  const int per = page_size / block;
  p.per_shift = (per & (per - 1)) == 0 ? __builtin_ctz(per) : -1;
  p.selected = selected;
  p.status = status;
  const SelectLayout w =
      select_layout(num_tokens, num_kv_heads, table_rows != nullptr, most);
  FK_REQUIRE(workspace != nullptr && workspace_bytes >= w.total &&
                 (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0,
             FK_ERR_WORKSPACE,
             "fk_select_blocks: workspace needs %zu bytes, 256-byte aligned (got %zu)", w.total,
             workspace_bytes);
  FK_REQUIRE(w.groups * w.chunks < (1ll << 31), FK_ERR_UNSUPPORTED,
             "fk_select_blocks: too many tokens");
  p.span = w.span; p.pitch = w.pitch;
  p.cols = 1;
  while (p.cols < p.g) p.cols *= 2;
  p.chunk = w.chunk; p.chunks = w.chunks;
  p.scores = static_cast<uint32_t*>(workspace);
  p.largest = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + w.largest);
  p.q_sum = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + w.q_sum);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = p.g > 8;
  auto scores = table_rows ? select_scores_many_kernel
                           : wide ? select_scores_kernel<2> : select_scores_kernel<1>;
  const size_t ring = table_rows ? 0 : SEL_RING_BYTES;
  static PerDeviceOnce scores_once[2];
  if (ring) FK_CUDA_OK(set_max_dynamic_smem(scores_once[wide], scores, SEL_RING_BYTES));
  FK_CUDA_OK(launch_kernel(scores,
                           dim3((unsigned)(w.groups * w.chunks), (unsigned)num_kv_heads),
                           dim3(32 * SEL_WARPS), ring, s, p));
  count_launch(1);
  const int64_t items = (int64_t)num_tokens * num_kv_heads;
  const int sms = sm_count();
  const int warps = items <= 2ll * sms ? 8 : items < 16ll * sms || most > SEL_WARP_BLOCKS ? 4 : 1;
  const int teams = warps == 1 ? 8 : 1;
  static PerDeviceOnce once[3];
  auto kernel = warps == 8 ? select_choose_kernel<8>
                           : warps == 4 ? select_choose_kernel<4> : select_choose_kernel<1>;
  FK_CUDA_OK(set_max_dynamic_smem(once[warps == 8 ? 0 : warps == 4 ? 1 : 2], kernel,
                                  (warps == 1 ? 8 * SEL_WARP_BLOCKS : SEL_MAX_BLOCKS) * 14));
  FK_CUDA_OK(launch_kernel(kernel, dim3((unsigned)((items + teams - 1) / teams)),
                           dim3(warps == 1 ? 256 : 32 * warps), (size_t)most * 14 * teams, s, p));
  count_launch(1);
  return FK_OK;
}

}  // extern "C"
