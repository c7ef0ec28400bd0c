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
  int num_tables, num_pages, page, block, hkv, g;
  int count, keep_first, keep_last;
  int32_t* selected;                  // [tokens, hkv, count]
  int32_t* status;
};

// Doubles in an order of whole numbers: equal values (both zeros) alike, no-number above all.
__device__ __forceinline__ uint64_t order_of(double v) {
  if (v != v) return ~0ull;
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b >> 63 ? ~b : b | (1ull << 63);
}

// One CTA per (token, KV head).  Scores are sums in 64 bits: products of two bf16 are exact in
// fp32, and 128 of them all but always in a 64-bit sum, so that the choice between two blocks does
// not hang on the order of additions.
__global__ void __launch_bounds__(SEL_THREADS) select_blocks_kernel(const SelectParams p) {
  extern __shared__ uint64_t keys[];         // of the blocks between the kept ends
  __shared__ float qs[SEL_MAX_G][SEL_D];
  __shared__ int hist[256];
  __shared__ int s_digit, s_left, s_eq[8], s_gt[8];
  pdl_launch_dependents();
  pdl_wait();
  const int token = blockIdx.x, kvh = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int32_t* out = p.selected + ((int64_t)token * p.hkv + kvh) * p.count;
  int64_t len = p.context_lens[token];
  const int row = p.rows ? p.rows[token] : token;
  bool bad = len > p.capacity;
  if (len < 0) len = 0;
  if (len > p.capacity) len = p.capacity;
  if (row < 0 || row >= p.num_tables) { len = 0; bad = true; }
  if (bad && tid == 0 && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
  const int n = (int)((len + p.block - 1) / p.block);
  if (n <= p.count) {
    for (int i = tid; i < p.count; i += SEL_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const int32_t* table = p.tables + (int64_t)row * p.table_stride;
  const int middle = n - p.keep_first - p.keep_last;
  const int want = p.count - p.keep_first - p.keep_last;     // of the middle ones
  const int per = p.page / p.block;
  for (int i = tid; i < p.g * SEL_D; i += SEL_THREADS)
    qs[i / SEL_D][i % SEL_D] =
        bf16_bits_to_float(p.q[(int64_t)token * p.q_stride + (int64_t)kvh * p.g * SEL_D + i]);
  __syncthreads();
  for (int i = warp; i < middle; i += SEL_THREADS / 32) {
    const int b = p.keep_first + i;
    int page = table[b / per];
    if (page < 0 || page >= p.num_pages) {
      if (lane == 0 && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
      if (lane == 0) keys[i] = 0ull;          // the last to be taken
      continue;
    }
    const uint16_t* at = p.bounds +
                         (((int64_t)page * p.hkv + kvh) * per + b % per) * 2 * SEL_D + lane * 4;
    const uint2 lo = *reinterpret_cast<const uint2*>(at);
    const uint2 hi = *reinterpret_cast<const uint2*>(at + SEL_D);
    const double l[4] = {bf16lo(lo.x), bf16hi(lo.x), bf16lo(lo.y), bf16hi(lo.y)};
    const double u[4] = {bf16lo(hi.x), bf16hi(hi.x), bf16lo(hi.y), bf16hi(hi.y)};
    double best = -INFINITY;
    bool nan = false;
    for (int h = 0; h < p.g; ++h) {
      double sum = 0.0;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const double q = qs[h][lane * 4 + d];
        const double a = q * l[d], c = q * u[d];
        sum += a != a || c != c ? a + c : fmax(a, c);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      nan |= sum != sum;
      best = fmax(best, sum);
    }
    if (lane == 0) keys[i] = nan ? ~0ull : order_of(best);
  }
  if (tid == 0) s_left = want;
  uint64_t border = 0;                       // digits of the want-th largest key found so far
  for (int shift = 56; shift >= 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    const uint64_t mask = shift == 56 ? 0ull : ~0ull << (shift + 8);
    for (int i = tid; i < middle; i += SEL_THREADS)
      if ((keys[i] & mask) == border) atomicAdd(&hist[(keys[i] >> shift) & 255], 1);
    __syncthreads();
    if (warp == 0) {
      // digits from the largest down, eight a lane
      int own[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += own[j] = hist[255 - lane * 8 - j];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const int left = s_left;
      int before = upto - sum;
      __syncwarp();
      if (before < left && left <= upto) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (before < left && left <= before + own[j]) {
            s_digit = 255 - lane * 8 - j;
            s_left = left - before;
          }
          before += own[j];
        }
      }
    }
    __syncthreads();
    if (want > 0) border |= (uint64_t)s_digit << shift;
  }
  // `s_left` of the blocks at the border are taken, the first ones.  Each warp has a run of blocks.
  const int run = ((middle + 7) / 8 + 31) / 32 * 32;
  const int from = min(warp * run, middle), to = min(from + run, middle);
  int eq = 0, gt = 0;
  for (int i = from + lane; i < to; i += 32) {
    eq += keys[i] == border ? 1 : 0;
    gt += keys[i] > border ? 1 : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    eq += __shfl_xor_sync(0xffffffffu, eq, o);
    gt += __shfl_xor_sync(0xffffffffu, gt, o);
  }
  if (lane == 0) { s_eq[warp] = eq; s_gt[warp] = gt; }
  __syncthreads();
  const int ties = want > 0 ? s_left : 0;
  int seen = 0, at = 0;                      // at the border, and taken, ahead of this warp's run
  for (int w = 0; w < warp; ++w) { seen += s_eq[w]; at += s_gt[w]; }
  at += min(seen, ties);
  if (want > 0) {
    for (int i0 = from; i0 < to; i0 += 32) {
      const int i = i0 + lane;
      const uint64_t key = i < to ? keys[i] : 0ull;
      const bool is_eq = i < to && key == border;
      const uint32_t eqs = __ballot_sync(0xffffffffu, is_eq), below = (1u << lane) - 1u;
      const bool take = i < to && (key > border ||
                                   (is_eq && seen + __popc(eqs & below) < ties));
      const uint32_t takes = __ballot_sync(0xffffffffu, take);
      if (take) out[p.keep_first + at + __popc(takes & below)] = p.keep_first + i;
      seen += __popc(eqs);
      at += __popc(takes);
    }
  }
  for (int i = tid; i < p.keep_first; i += SEL_THREADS) out[i] = i;
  for (int i = tid; i < p.keep_last; i += SEL_THREADS)
    out[p.count - p.keep_last + i] = n - p.keep_last + i;
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
  p.num_tables = num_tables; p.num_pages = (int)num_pages; p.page = page_size; p.block = block;
  p.hkv = num_kv_heads; p.g = num_q_heads / num_kv_heads;
  p.count = count; p.keep_first = keep_first; p.keep_last = keep_last;
  p.selected = selected;
  p.status = status;
  static PerDeviceOnce once;
  FK_CUDA_OK(set_max_dynamic_smem(once, select_blocks_kernel, SEL_MAX_BLOCKS * 8));
  FK_CUDA_OK(launch_kernel(select_blocks_kernel,
                           dim3((unsigned)num_tokens, (unsigned)num_kv_heads),
                           dim3(SEL_THREADS), (size_t)(most < 1 ? 8 : most * 8),
                           static_cast<cudaStream_t>(stream), p));
  count_launch(1);
  return FK_OK;
}

}  // extern "C"
