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
constexpr int SEL_THREADS = 256;
constexpr int SEL_MAX_G = 16;                 // query heads per KV head
constexpr int SEL_MAX_BLOCKS = 16384;         // of one context

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
  const int64_t fresh = p.cu_new ? (int64_t)p.cu_new[seq + 1] - p.cu_new[seq] : 1;
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
  int together;                       // tokens of a CTA: 1, or up to 16 / g (a power of two)
  int most;                           // blocks that a table's row has pages for
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
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b >> 31 ? ~b : b | (1u << 31);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

struct SelectShared {
  int hist[256];
  int digit, left;
  int eq[8], gt[8];
  float q_sum[16];                    // of each token: largest sum of |q| of its query heads
  uint32_t most[8];                   // largest |bound|, as bf16 bits
  uint32_t lo[8], hi[8];
};

// The want-th largest of n keys (want >= 1), and in s.left how many of the keys equal to it are
// among the want largest.  All threads; ends behind a barrier.
template <typename KEY>
__device__ __forceinline__ KEY border_of(const KEY* keys, int n, int want, int top_shift,
                                         KEY fixed, SelectShared& s) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kBits = 8 * sizeof(KEY);
  if (tid == 0) s.left = want;
  KEY border = fixed;                        // the digits above that all keys share
  for (int shift = top_shift; shift >= 0; shift -= 8) {
    s.hist[tid] = 0;
    __syncthreads();
    const KEY mask = shift + 8 >= kBits ? (KEY)0 : (KEY)(~(KEY)0 << (shift + 8));
    for (int i = tid; i < n; i += SEL_THREADS)
      if ((keys[i] & mask) == border) atomicAdd(&s.hist[(int)(keys[i] >> shift) & 255], 1);
    __syncthreads();
    if (warp == 0) {
      // digits from the largest down, eight a lane
      int own[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += own[j] = s.hist[255 - lane * 8 - j];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const int left = s.left;
      int before = upto - sum;
      __syncwarp();
      if (before < left && left <= upto) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (before < left && left <= before + own[j]) {
            s.digit = 255 - lane * 8 - j;
            s.left = left - before;
          }
          before += own[j];
        }
      }
    }
    __syncthreads();
    border |= (KEY)s.digit << shift;
  }
  return border;
}

// Score of a block in 64 bits, by a warp: the largest over the query heads.  Products of two bf16 are
// exact in fp32, and 128 of them all but always in a 64-bit sum.
__device__ __forceinline__ uint64_t exact_score(const SelectParams& p, int token, int kvh,
                                                const uint16_t* at, int lane) {
  const uint2 lo = *reinterpret_cast<const uint2*>(at + lane * 4);
  const uint2 hi = *reinterpret_cast<const uint2*>(at + SEL_D + lane * 4);
  const double l[4] = {bf16lo(lo.x), bf16hi(lo.x), bf16lo(lo.y), bf16hi(lo.y)};
  const double u[4] = {bf16lo(hi.x), bf16hi(hi.x), bf16lo(hi.y), bf16hi(hi.y)};
  const uint16_t* qp = p.q + (int64_t)token * p.q_stride + (int64_t)kvh * p.g * SEL_D + lane * 4;
  double best = -INFINITY;
  bool nan = false;
  for (int h = 0; h < p.g; ++h) {
    const uint2 qv = *reinterpret_cast<const uint2*>(qp + h * SEL_D);
    const double q[4] = {bf16lo(qv.x), bf16hi(qv.x), bf16lo(qv.y), bf16hi(qv.y)};
    double sum = 0.0;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const double a = q[d] * l[d], c = q[d] * u[d];
      sum += a != a || c != c ? a + c : fmax(a, c);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    nan |= sum != sum;
    best = fmax(best, sum);
  }
  return nan ? ~0ull : order_of(best);
}

// One CTA per KV head and token, or several tokens of one table.
//
// Scores: sum_d max(q_d lo_d, q_d hi_d) = q+ . hi + q- . lo with the positive and negative parts of
// q, a product of 16 rows (query heads, of several tokens where they fit) by 8 blocks by 256 on the
// tensor cores, the blocks' bounds straight from memory: a lane loads 16 bytes, which are operands of
// two instructions when q's channels are taken in the same order.  Sums in fp32 are off by at most
// e = 2^-15 sum |q| max |bound| (16 instructions of 17 terms, each off by at most 2^-23 of the sums
// of absolute values: 2^-15.9).  Of the blocks between the kept ends those above the want-th largest
// score by more than 2 e are taken, those below it by more are not, and those between are scored
// again in 64 bits if they do not all fit.  So the choice is that of 64 bits, ties to the lower
// index.
//
// Bounds: the bytes of the bounds when there are many tokens (8 loads of 16 bytes are under way per
// lane, two CTAs on an SM), else the latency of the steps behind the scores.
__global__ void __launch_bounds__(SEL_THREADS, 2) select_blocks_kernel(const SelectParams p) {
  extern __shared__ uint64_t sel_smem[];
  __shared__ SelectShared s;
  uint64_t* exact = sel_smem;                                       // [most]
  uint32_t* scores = reinterpret_cast<uint32_t*>(exact + p.most);   // [together][most], ordered
  uint16_t* band = reinterpret_cast<uint16_t*>(scores + p.together * p.most);   // [most]
  pdl_launch_dependents();
  pdl_wait();
  const int kvh = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = p.page / p.block;
  auto length = [&](int token, int row) -> int {
    const int64_t len = p.context_lens[token];
    if (len <= 0 || row < 0 || row >= p.num_tables) return 0;
    return (int)(len > p.capacity ? p.capacity : len);
  };
  auto bounds_at = [&](int page, int b) -> const uint16_t* {
    return p.bounds + (((int64_t)page * p.hkv + kvh) * per + b % per) * 2 * SEL_D;
  };

  // runs of tokens with one table
  const int last_token = min(p.num_tokens, ((int)blockIdx.x + 1) * p.together);
  for (int t0 = blockIdx.x * p.together; t0 < last_token;) {
    const int row = p.rows ? p.rows[t0] : t0;
    int t1 = t0 + 1;
    while (t1 < last_token && p.rows[t1] == row) ++t1;
    int longest = 0;
    bool bad = row < 0 || row >= p.num_tables;
    for (int t = t0; t < t1; ++t) {
      bad |= p.context_lens[t] > p.capacity;
      longest = max(longest, length(t, row));
    }
    if (bad && tid == 0 && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
    const int32_t* table = p.tables + (int64_t)row * p.table_stride;
    // scores of blocks keep_first .. of the longest context; a shorter one uses fewer of them
    const int blocks = (longest + p.block - 1) / p.block;
    const int scored = blocks > p.count ? blocks - p.keep_first - p.keep_last : 0;
    if (scored > 0) {
      // rows lane / 4 and lane / 4 + 8 of q, channels 32 j + 8 (lane % 4) + 0 .. 7
      uint32_t qp[4][8], qm[4][8];
      const int r0 = lane >> 2, quad = lane & 3;
      float abs0 = 0.f, abs1 = 0.f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = r0 + half * 8, t = t0 + r / p.g;
        const bool live = t < t1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (live)
            v = *reinterpret_cast<const uint4*>(
                p.q + (int64_t)t * p.q_stride + ((int64_t)kvh * p.g + r % p.g) * SEL_D + j * 32 +
                quad * 8);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            qp[j][half * 4 + i] = max2_nan(w[i], 0u);
            qm[j][half * 4 + i] = min2_nan(w[i], 0u);
            const float a = fabsf(bf16lo(w[i])) + fabsf(bf16hi(w[i]));
            if (half) abs1 += a; else abs0 += a;
          }
        }
      }
      abs0 += __shfl_xor_sync(0xffffffffu, abs0, 1); abs1 += __shfl_xor_sync(0xffffffffu, abs1, 1);
      abs0 += __shfl_xor_sync(0xffffffffu, abs0, 2); abs1 += __shfl_xor_sync(0xffffffffu, abs1, 2);
      if (tid < 16) s.q_sum[tid] = 0.f;
      __syncthreads();
      if (warp == 0 && quad == 0) {
        // not a number counts as infinite; whole numbers order floats above zero
        auto put = [&](int r, float a) {
          if (r / p.g < p.together)
            atomicMax(reinterpret_cast<int*>(&s.q_sum[r / p.g]),
                      __float_as_int(a < INFINITY ? a : INFINITY));
        };
        put(r0, abs0);
        put(r0 + 8, abs1);
      }
      uint32_t most = 0u;                      // largest |bound|, two channels at once
      for (int b0 = warp * 8; b0 < scored; b0 += 8 * (SEL_THREADS / 32)) {
        const int mine = b0 + r0, b = p.keep_first + mine;
        int page = mine < scored ? table[b / per] : -1;
        if (mine < scored && (page < 0 || page >= p.num_pages)) {
          if (p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
          page = -1;
        }
        const bool have = page >= 0;
        uint4 lo[4], hi[4];
        const uint16_t* at = bounds_at(have ? page : 0, have ? b : 0) + quad * 8;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          hi[j] = lo[j] = make_uint4(0u, 0u, 0u, 0u);
          if (have) {
            hi[j] = *reinterpret_cast<const uint4*>(at + SEL_D + j * 32);
            lo[j] = *reinterpret_cast<const uint4*>(at + j * 32);
          }
        }
        float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t pa[4] = {qp[j][0], qp[j][4], qp[j][1], qp[j][5]};
          const uint32_t pb[4] = {qp[j][2], qp[j][6], qp[j][3], qp[j][7]};
          const uint32_t ma[4] = {qm[j][0], qm[j][4], qm[j][1], qm[j][5]};
          const uint32_t mb[4] = {qm[j][2], qm[j][6], qm[j][3], qm[j][7]};
          mma_bf16_16816(c0, pa, hi[j].x, hi[j].y);
          mma_bf16_16816(c1, ma, lo[j].x, lo[j].y);
          mma_bf16_16816(c0, pb, hi[j].z, hi[j].w);
          mma_bf16_16816(c1, mb, lo[j].z, lo[j].w);
          most = max2_nan(most, max2_nan(max2_nan(hi[j].x & 0x7fff7fffu, hi[j].y & 0x7fff7fffu),
                                         max2_nan(hi[j].z & 0x7fff7fffu, hi[j].w & 0x7fff7fffu)));
          most = max2_nan(most, max2_nan(max2_nan(lo[j].x & 0x7fff7fffu, lo[j].y & 0x7fff7fffu),
                                         max2_nan(lo[j].z & 0x7fff7fffu, lo[j].w & 0x7fff7fffu)));
        }
        // rows r0 and r0 + 8 of blocks b0 + 2 quad + 0, 1: the largest of each token's rows
        float v[4] = {c0[0] + c1[0], c0[1] + c1[1], c0[2] + c1[2], c0[3] + c1[3]};
        const uint32_t bads = __ballot_sync(0xffffffffu, mine < scored && !have);
        if (p.together == 1) {
          if (r0 >= p.g) v[0] = v[1] = -INFINITY;
          if (r0 + 8 >= p.g) v[2] = v[3] = -INFINITY;
          v[0] = v[2] = fmaxf(v[0], v[2]);
          v[1] = v[3] = fmaxf(v[1], v[3]);
        }
        const int across = p.together == 1 ? 8 : p.g;
        for (int o = 1; o < across; o <<= 1) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[i] = fmaxf(v[i], __shfl_xor_sync(0xffffffffu, v[i], o * 4));
        }
        if (r0 % across == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int col = quad * 2 + (i & 1);
            const int tq = p.together == 1 ? 0 : (r0 + (i >> 1) * 8) / p.g;
            if ((p.together == 1 && i > 1) || b0 + col >= scored || tq >= p.together) continue;
            scores[tq * p.most + b0 + col] = bads >> (col * 4) & 1u ? 0u : order_of(v[i]);
          }
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = max2_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (lane == 0) s.most[warp] = most;
      __syncthreads();
    }

    for (int token = t0; token < t1; ++token) {
      int32_t* out = p.selected + ((int64_t)token * p.hkv + kvh) * p.count;
      const int n = (length(token, row) + p.block - 1) / p.block;
      if (n <= p.count) {
        for (int i = tid; i < p.count; i += SEL_THREADS) out[i] = i < n ? i : -1;
        continue;
      }
      const int middle = n - p.keep_first - p.keep_last;
      const int want = p.count - p.keep_first - p.keep_last;     // of the middle ones
      for (int i = tid; i < p.keep_first; i += SEL_THREADS) out[i] = i;
      for (int i = tid; i < p.keep_last; i += SEL_THREADS)
        out[p.count - p.keep_last + i] = n - p.keep_last + i;
      if (want == 0) continue;
      uint32_t* keys = scores + (token - t0) * p.most;
      uint32_t most = s.most[0];
#pragma unroll
      for (int w = 1; w < 8; ++w) most = max2_nan(most, s.most[w]);
      const float reach = s.q_sum[token - t0] * __uint_as_float(max(most << 16, most & 0xffff0000u));
      // scores past fp32's range, products below it, and what is not a number: all in 64 bits
      const bool all = !(reach < INFINITY) || (reach > 0.f && reach < 7.9e-31f);
      uint32_t above, least;                 // keys above are taken, keys below `least` are not
      bool same = false;                     // keys between are equal in truth
      if (all) {
        above = ~0u; least = 0u;
      } else {
        // digits that all keys share need no pass
        uint32_t lo = ~0u, hi = 0u;
        for (int i = tid; i < middle; i += SEL_THREADS) {
          lo = min(lo, keys[i]);
          hi = max(hi, keys[i]);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        __syncthreads();
        if (lane == 0) { s.lo[warp] = lo; s.hi[warp] = hi; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) { lo = min(lo, s.lo[w]); hi = max(hi, s.hi[w]); }
        const int shift = lo == hi ? 0 : (31 - __clz(lo ^ hi)) / 8 * 8;
        const uint32_t border = border_of<uint32_t>(
            keys, middle, want, shift, shift == 24 ? 0u : hi & ~0u << (shift + 8), s);
        const float v = value_of(border), e2 = reach * (2.f / 32768.f);
        same = border == 0u || reach == 0.f;
        above = same ? border : order_of(v + e2);
        least = same ? border : order_of(v - e2);
      }
      // how many are above, and between
      int eq = 0, gt = 0;
      const int run = ((middle + 7) / 8 + 31) / 32 * 32;       // blocks of a warp
      const int from = min(warp * run, middle), to = min(from + run, middle);
      for (int i = from + lane; i < to; i += 32) {
        gt += keys[i] > above ? 1 : 0;
        eq += keys[i] >= least && keys[i] <= above ? 1 : 0;
      }
      eq = __reduce_add_sync(0xffffffffu, eq);
      gt = __reduce_add_sync(0xffffffffu, gt);
      __syncthreads();
      if (lane == 0) { s.eq[warp] = eq; s.gt[warp] = gt; }
      __syncthreads();
      int eqs = 0, gts = 0, eq_before = 0, gt_before = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        if (w == warp) { eq_before = eqs; gt_before = gts; }
        eqs += s.eq[w];
        gts += s.gt[w];
      }
      int ties = want - gts;                 // of those between, the first ones if they are equal
      if (!same && eqs > ties) {
        // score those between again; their keys become "taken" or "not"
        int at = eq_before;
        for (int i0 = from; i0 < to; i0 += 32) {
          const int i = i0 + lane;
          const bool is = i < to && keys[i] >= least && keys[i] <= above;
          const uint32_t votes = __ballot_sync(0xffffffffu, is);
          if (is) band[at + __popc(votes & ((1u << lane) - 1u))] = (uint16_t)i;
          at += __popc(votes);
        }
        __syncthreads();
        for (int c = warp; c < eqs; c += 8) {
          const int b = p.keep_first + band[c];
          uint64_t key = 0ull;               // without a page
          if (keys[band[c]] != 0u)
            key = exact_score(p, token, kvh, bounds_at(table[b / per], b), lane);
          if (lane == 0) exact[c] = key;
        }
        __syncthreads();
        if (eqs <= 32) {
          // a lane per block: its rank, the lower index first among equals
          if (warp == 0) {
            const uint64_t key = lane < eqs ? exact[lane] : 0ull;
            int rank = 0;
            for (int j = 0; j < eqs; ++j) {
              const uint64_t other = __shfl_sync(0xffffffffu, key, j);
              rank += other > key || (other == key && j < lane) ? 1 : 0;
            }
            if (lane < eqs) keys[band[lane]] = rank < ties ? ~0u : 0u;
          }
          __syncthreads();
        } else {
          const uint64_t edge = border_of<uint64_t>(exact, eqs, ties, 56, 0ull, s);
          const int left = s.left;
          // equal ones in order: a warp has a run of them, as above
          const int run_c = ((eqs + 7) / 8 + 31) / 32 * 32;
          const int fc = min(warp * run_c, eqs), tc = min(fc + run_c, eqs);
          int n_eq = 0;
          for (int c = fc + lane; c < tc; c += 32) n_eq += exact[c] == edge ? 1 : 0;
          n_eq = __reduce_add_sync(0xffffffffu, n_eq);
          __syncthreads();
          if (lane == 0) s.eq[warp] = n_eq;
          __syncthreads();
          int seen = 0;
          for (int w = 0; w < warp; ++w) seen += s.eq[w];
          for (int c0 = fc; c0 < tc; c0 += 32) {
            const int c = c0 + lane;
            const bool is = c < tc && exact[c] == edge;
            const uint32_t votes = __ballot_sync(0xffffffffu, is);
            if (c < tc)
              keys[band[c]] = exact[c] > edge ||
                                      (is && seen + __popc(votes & ((1u << lane) - 1u)) < left)
                                  ? ~0u : 0u;
            seen += __popc(votes);
          }
          __syncthreads();
        }
        // taken ones are above now, and nothing is between
        above = min(above, ~0u - 1u);
        least = ~0u;
        gt = 0;
        for (int i = from + lane; i < to; i += 32) gt += keys[i] > above ? 1 : 0;
        gt = __reduce_add_sync(0xffffffffu, gt);
        __syncthreads();
        if (lane == 0) s.gt[warp] = gt;
        __syncthreads();
        gt_before = 0;
        for (int w = 0; w < warp; ++w) gt_before += s.gt[w];
        eq_before = 0;
        ties = 0;
      }
      // taken ones in order
      int seen = eq_before, at = gt_before + min(eq_before, ties);
      for (int i0 = from; i0 < to; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t key = i < to ? keys[i] : 0u;
        const bool is_eq = ties > 0 && i < to && key >= least && key <= above;
        const uint32_t votes = __ballot_sync(0xffffffffu, is_eq), below = (1u << lane) - 1u;
        const bool take = i < to && (key > above || (is_eq && seen + __popc(votes & below) < ties));
        const uint32_t takes = __ballot_sync(0xffffffffu, take);
        if (take) out[p.keep_first + at + __popc(takes & below)] = p.keep_first + i;
        seen += __popc(votes);
        at += __popc(takes);
      }
      __syncthreads();
    }
    t0 = t1;
  }
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

int fk_select_blocks(const void* q, int64_t q_stride_token, const void* bounds, int64_t num_pages,
                     int page_size, int block, const int32_t* context_lens,
                     const int32_t* table_rows, const int32_t* block_tables,
                     int64_t block_table_stride, int64_t block_table_cols, int num_tables,
                     int num_tokens, int num_q_heads, int num_kv_heads, int head_dim, int count,
                     int keep_first, int keep_last, int32_t* selected, int32_t* status,
                     fk_stream_t stream) {
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
  // Tokens that may have one table share the scores' products, as far as their query heads fill the
  // 16 rows and 32 KiB of scores leave several CTAs on an SM.
  p.together = 1;
  if (table_rows != nullptr && (p.g & (p.g - 1)) == 0)
    while (p.together * 2 * p.g <= 16 && p.together * 2 * most * 4 <= 32768) p.together *= 2;
  p.selected = selected;
  p.status = status;
  const int64_t ctas = ((int64_t)num_tokens + p.together - 1) / p.together;
  const size_t smem = (size_t)most * (8 + 4 * (size_t)p.together + 2) + 16;
  static PerDeviceOnce once;
  FK_CUDA_OK(set_max_dynamic_smem(once, select_blocks_kernel, SEL_MAX_BLOCKS * 14 + 16));
  FK_CUDA_OK(launch_kernel(select_blocks_kernel, dim3((unsigned)ctas, (unsigned)num_kv_heads),
                           dim3(SEL_THREADS), smem, static_cast<cudaStream_t>(stream), p));
  count_launch(1);
  return FK_OK;
}

}  // extern "C"
