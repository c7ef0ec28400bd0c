// Tokens leave a paged KV cache: per sequence and KV head the first `first` and the last `last` tokens
// stay, and of those between the ones with the largest sums of softmax weights, `budget` in all.
//
// What attention computes does not depend on the order of its keys, so only as many rows move as have
// to.  With M = budget - last: stayers below M stay where they are; the i-th stayer of [M, n - last)
// goes to the i-th place below M that has become free; the last ones follow, in order, to M ..
// budget - 1.  Sources of the first kind of move lie behind all of its destinations, so these moves
// run side by side; those of the second kind run in ascending tiles, read before written.
//
// One CTA has a sequence and KV head.  The border weight is found by counting: the range of keys
// (weights as integers of the same order) is cut into 2048 parts, the part with the border into 2048
// again, so that two or three passes over the keys suffice whatever their distribution; ties go to
// the lowest places.  The keys of the first tokens are kept in shared memory, those beyond are
// read again.  Bound by latency (a chain of about ten passes and barriers) until there are rows
// enough to move; the bytes are 4 a token to decide and each moved row twice.
#include "fk_q4.cuh"

namespace fk {

constexpr int EV_THREADS = 512;
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_BINS = 2048;
constexpr int EV_KEYS = 12288;               // tokens whose keys are kept
constexpr int EV_LIST = 2048;                // moves of a round
constexpr int EV_ROWS = 4;                   // rows that 16 lanes move at a time
constexpr int EV_TILE = EV_THREADS / 16 * EV_ROWS;

struct EvictParams {
  uint8_t* k;                 // bf16 keys, or the 4-bit pool
  uint8_t* v;
  int64_t page_bytes, token_bytes, head_bytes;   // bf16
  int group_pairs;            // 4-bit: pairs of a row; 0: bf16
  float* weights;             // [pages, hkv, page]
  const int32_t* lens;
  int32_t* new_lens;
  const int32_t* tables; int64_t table_stride;
  int64_t capacity;
  int num_pages, page, page_shift, hkv;
  int budget, first, last;
  int keys;                   // kept in shared memory
  int32_t* status;
};

// Order of the weights; no number counts as the smallest.
__device__ __forceinline__ uint32_t ev_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);            // -0 is 0
  return u >> 31 ? ~u : u | 0x80000000u;
}

// Place of a token: its page, checked, and the place in it.
__device__ __forceinline__ int ev_page(const EvictParams& p, const int32_t* table, int token,
                                       int* at) {
  const int i = p.page_shift >= 0 ? token >> p.page_shift : token / p.page;
  *at = token - i * p.page;
  const int page = table[i];
  if (page >= 0 && page < p.num_pages) return page;
  if (p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
  return -1;
}

// What one of the 16 lanes of a row moves of it.
struct EvPiece {
  uint4 a, b;
  float w;
};

template <bool Q4>
struct EvRow {
  uint8_t* a;        // 16 bytes; 4-bit: lanes 0-3 keys, 4-7 values
  uint8_t* b;        // bf16: the value's; 4-bit: lanes 8, 9 the pairs of the key, the value
  float* w;          // lane 0 (bf16), 10
  __device__ __forceinline__ EvRow(const EvictParams& p, const int32_t* table, int head, int token,
                                   bool live) {
    const int lane = threadIdx.x & 15;
    a = b = nullptr;
    w = nullptr;
    if (!live) return;
    int at;
    const int64_t page = ev_page(p, table, token, &at);
    if (page < 0) return;
    if constexpr (Q4) {
      const int ng = p.group_pairs;
      uint8_t* unit = p.k + ((page * p.hkv + head) * (p.page / Q4_UNIT) + at / Q4_UNIT) *
                                q4_unit_bytes(ng);
      const int t = at % Q4_UNIT;
      if (lane < 8) a = unit + (lane >> 2) * Q4_VALUES + t * Q4_ROW + (lane & 3) * 16;
      else if (lane < 10) b = unit + Q4_PAIRS + ((lane - 8) * Q4_UNIT + t) * 4 * ng;
      if (lane == 10) w = p.weights + (page * p.hkv + head) * p.page + at;
    } else {
      const int64_t off = page * p.page_bytes + at * p.token_bytes + head * p.head_bytes + lane * 16;
      a = p.k + off;
      b = p.v + off;
      if (lane == 0) w = p.weights + (page * p.hkv + head) * p.page + at;
    }
  }
  __device__ __forceinline__ void load(const EvictParams& p, EvPiece& x) const {
    if (a) x.a = *reinterpret_cast<const uint4*>(a);
    if (b) {
      if constexpr (!Q4) x.b = *reinterpret_cast<const uint4*>(b);
      else if (p.group_pairs == 2) *reinterpret_cast<uint2*>(&x.b) = *reinterpret_cast<const uint2*>(b);
      else x.b.x = *reinterpret_cast<const uint32_t*>(b);
    }
    if (w) x.w = *w;
  }
  __device__ __forceinline__ void store(const EvictParams& p, const EvPiece& x) const {
    if (a) *reinterpret_cast<uint4*>(a) = x.a;
    if (b) {
      if constexpr (!Q4) *reinterpret_cast<uint4*>(b) = x.b;
      else if (p.group_pairs == 2) *reinterpret_cast<uint2*>(b) = make_uint2(x.b.x, x.b.y);
      else *reinterpret_cast<uint32_t*>(b) = x.b.x;
    }
    if (w) *w = x.w;
  }
};

// Sum over the CTA before this thread, and the total; `red` holds EV_WARPS words.
__device__ __forceinline__ int ev_scan(int v, int* red, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) red[warp] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < EV_WARPS; ++w) {
    if (w < warp) before += red[w];
    all += red[w];
  }
  __syncthreads();
  *total = all;
  return before + incl - v;
}

template <bool Q4>
__global__ void __launch_bounds__(EV_THREADS) evict_kernel(const EvictParams p) {
  extern __shared__ uint32_t kept[];                      // keys of tokens 0 .. p.keys - 1
  __shared__ int bins[EV_BINS];
  __shared__ int from_list[EV_LIST], to_list[EV_LIST];
  __shared__ int red[EV_WARPS];
  __shared__ uint32_t range[2 * EV_WARPS];
  __shared__ int pick[3];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seq = blockIdx.x / p.hkv, head = blockIdx.x - seq * p.hkv;
  const int64_t len = p.lens[seq];
  const int n = len < 0 ? 0 : len > p.capacity ? (int)p.capacity : (int)len;
  if (head == 0 && threadIdx.x == 0) {
    p.new_lens[seq] = min(n, p.budget);
    if (len > p.capacity && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
  }
  if (n <= p.budget) return;
  const int32_t* table = p.tables + (int64_t)seq * p.table_stride;
  const int M = p.budget - p.last, end = n - p.last;      // candidates: first .. end - 1
  auto read_key = [&](int i) -> uint32_t {
    int at;
    const int64_t page = ev_page(p, table, i, &at);
    return page < 0 ? 0u : ev_key(p.weights[(page * p.hkv + head) * p.page + at]);
  };
  auto key = [&](int i) -> uint32_t { return i < p.keys ? kept[i] : read_key(i); };

  // ---- keys, and their range ----
  uint32_t lo = ~0u, hi = 0u;
  for (int i = p.first + threadIdx.x; i < end; i += EV_THREADS) {
    const uint32_t k = read_key(i);
    if (i < p.keys) kept[i] = k;
    lo = min(lo, k);
    hi = max(hi, k);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) {
    range[warp] = lo;
    range[EV_WARPS + warp] = hi;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < EV_WARPS; ++w) {
    lo = min(lo, range[w]);
    hi = max(hi, range[EV_WARPS + w]);
  }

  // ---- the border: `want` of the keys at it stay, all above, none below ----
  int want = M - p.first;
  uint32_t border = hi;
  if (want > 0) {
    for (int pass = 0; pass < 3; ++pass) {                 // 32 bits in parts of 11
      const int bits = 32 - __clz(hi - lo);                // 0 when all are one key
      const int shift = bits > 11 ? bits - 11 : 0;
      for (int i = threadIdx.x; i < EV_BINS; i += EV_THREADS) bins[i] = 0;
      __syncthreads();
      for (int i = p.first + threadIdx.x; i < end; i += EV_THREADS) {
        const uint32_t k = key(i);
        if (k >= lo && k <= hi) atomicAdd(&bins[(k - lo) >> shift], 1);
      }
      __syncthreads();
      // from the top: the bin in which the sum reaches `want`
      constexpr int PER = EV_BINS / EV_THREADS;
      int mine[PER], sum = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += mine[i] = bins[EV_BINS - 1 - (threadIdx.x * PER + i)];
      int all;
      int above = ev_scan(sum, red, &all);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (above < want && above + mine[i] >= want) {
          pick[0] = EV_BINS - 1 - (threadIdx.x * PER + i);
          pick[1] = want - above;
          pick[2] = mine[i];
        }
        above += mine[i];
      }
      __syncthreads();
      want = pick[1];
      const int in_bin = pick[2];
      const uint32_t at = lo + ((uint32_t)pick[0] << shift);
      __syncthreads();
      if (shift == 0 || in_bin == want) {
        // one key, or the whole bin stays: from its lowest key on
        border = at;
        if (shift != 0) want = 0x7fffffff;
        break;
      }
      lo = at;
      const uint32_t top = at + ((1u << shift) - 1u);
      hi = top < hi && top >= at ? top : hi;
    }
  }
  // A bin that stays whole: everything from `border` on.  Else keys above it, and `want` at it.
  const bool whole = want == 0x7fffffff;

  // ---- moves: each warp a stretch of the tokens, in order ----
  const int stretch = ((end + EV_WARPS - 1) / EV_WARPS + 31) & ~31;
  const int w0 = min(warp * stretch, end), w1 = min(w0 + stretch, end);
  int ties = 0;
  if (!whole) {
    for (int i = w0; i < w1; i += 32) {
      const int t = i + lane;
      ties += __popc(__ballot_sync(0xffffffffu, t >= p.first && t < w1 && key(t) == border));
    }
    if (lane == 0) red[warp] = ties;
    __syncthreads();
    ties = 0;
    for (int w = 0; w < warp; ++w) ties += red[w];
    __syncthreads();
  }
  // stayers of a stretch of 32, given the ties before it
  auto stays = [&](int i, int& tied) -> uint32_t {
    const int t = i + lane;
    bool s = false, tie = false;
    if (t < w1) {
      if (t < p.first) {
        s = true;
      } else {
        const uint32_t k = key(t);
        s = whole ? k >= border : k > border;
        tie = !whole && k == border;
      }
    }
    if (!whole) {
      const uint32_t at = __ballot_sync(0xffffffffu, tie);
      if (tie) s = tied + __popc(at & ((1u << lane) - 1u)) < want;
      tied += __popc(at);
    }
    return __ballot_sync(0xffffffffu, s);
  };
  int free_here = 0, move_here = 0;
  {
    int tied = ties;
    for (int i = w0; i < w1; i += 32) {
      const uint32_t s = stays(i, tied);
      const int t = i + lane;
      free_here += __popc(__ballot_sync(0xffffffffu, t < min(w1, M) && !(s >> lane & 1u)));
      move_here += __popc(__ballot_sync(0xffffffffu, t < w1 && t >= M && (s >> lane & 1u)));
    }
  }
  int moves, frees;
  const int free_before = ev_scan(lane == 0 ? free_here : 0, red, &frees);
  const int move_before = ev_scan(lane == 0 ? move_here : 0, red, &moves);
  moves = min(moves, frees);                               // they are equal
  const int half = threadIdx.x >> 4;
  for (int r0 = 0; r0 < moves; r0 += EV_LIST) {
    int f = __shfl_sync(0xffffffffu, free_before, 0) - r0;
    int m = __shfl_sync(0xffffffffu, move_before, 0) - r0;
    int tied = ties;
    for (int i = w0; i < w1; i += 32) {
      const uint32_t s = stays(i, tied);
      const int t = i + lane;
      const uint32_t below = (1u << lane) - 1u;
      const uint32_t fr = __ballot_sync(0xffffffffu, t < min(w1, M) && !(s >> lane & 1u));
      const uint32_t mv = __ballot_sync(0xffffffffu, t < w1 && t >= M && (s >> lane & 1u));
      const int fi = f + __popc(fr & below), mi = m + __popc(mv & below);
      if ((fr >> lane & 1u) && fi >= 0 && fi < EV_LIST) to_list[fi] = t;
      if ((mv >> lane & 1u) && mi >= 0 && mi < EV_LIST) from_list[mi] = t;
      f += __popc(fr);
      m += __popc(mv);
    }
    __syncthreads();
    const int count = min(EV_LIST, moves - r0);
    for (int j0 = 0; j0 < count; j0 += EV_TILE) {
      EvPiece x[EV_ROWS];
#pragma unroll
      for (int u = 0; u < EV_ROWS; ++u) {
        const int j = j0 + u * (EV_THREADS / 16) + half;
        const int t = j < count ? from_list[j] : -1;
        EvRow<Q4>(p, table, head, t, (unsigned)t < (unsigned)n).load(p, x[u]);
      }
#pragma unroll
      for (int u = 0; u < EV_ROWS; ++u) {
        const int j = j0 + u * (EV_THREADS / 16) + half;
        const int t = j < count ? to_list[j] : -1;
        EvRow<Q4>(p, table, head, t, (unsigned)t < (unsigned)n).store(p, x[u]);
      }
    }
    __syncthreads();
  }
  // ---- the newest ----
  for (int j0 = 0; j0 < p.last; j0 += EV_TILE) {
    EvPiece x[EV_ROWS];
#pragma unroll
    for (int u = 0; u < EV_ROWS; ++u) {
      const int j = j0 + u * (EV_THREADS / 16) + half;
      EvRow<Q4>(p, table, head, end + j, j < p.last).load(p, x[u]);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < EV_ROWS; ++u) {
      const int j = j0 + u * (EV_THREADS / 16) + half;
      EvRow<Q4>(p, table, head, M + j, j < p.last).store(p, x[u]);
    }
  }
}

static int evict(const char* what, EvictParams& p, bool q4, int64_t num_pages, int page,
                 const int32_t* lens, int32_t* new_lens, const int32_t* tables,
                 int64_t table_stride, int64_t table_cols, int num_seqs, int hkv, float* weights,
                 int budget, int first, int last, int32_t* status, cudaStream_t s) {
  FK_REQUIRE(num_seqs >= 0, FK_ERR_INVALID_ARG, "%s: negative size", what);
  FK_REQUIRE(budget >= 1 && first >= 0 && last >= 0 && first <= budget && last <= budget - first,
             FK_ERR_INVALID_ARG, "%s: of a budget of %d the first %d and the last %d stay", what,
             budget, first, last);
  if (num_seqs == 0) return FK_OK;
  FK_REQUIRE(weights && lens && new_lens && tables, FK_ERR_INVALID_ARG, "%s: null pointer", what);
  FK_REQUIRE(lens != new_lens, FK_ERR_INVALID_ARG, "%s: the new lengths need a place of their own",
             what);
  FK_REQUIRE(table_cols > 0 && table_stride >= 0, FK_ERR_INVALID_ARG, "%s: bad sizes", what);
  FK_REQUIRE((int64_t)num_seqs * hkv < (1ll << 31), FK_ERR_UNSUPPORTED, "%s: too many sequences",
             what);
  p.weights = weights; p.lens = lens; p.new_lens = new_lens;
  p.tables = tables; p.table_stride = table_stride;
  const int64_t longest = 1ll << 30;
  p.capacity = table_cols < longest / page ? table_cols * page : longest;
  p.num_pages = (int)num_pages; p.page = page; p.hkv = hkv;
  p.page_shift = (page & (page - 1)) == 0 ? __builtin_ctz(page) : -1;
  p.budget = budget; p.first = first; p.last = last;
  p.keys = (int)(p.capacity < EV_KEYS ? p.capacity : EV_KEYS);
  p.status = status;
  static PerDeviceOnce once[2];
  auto kernel = q4 ? evict_kernel<true> : evict_kernel<false>;
  FK_CUDA_OK(set_max_dynamic_smem(once[q4 ? 1 : 0], kernel, EV_KEYS * 4));
  FK_CUDA_OK(launch_kernel(kernel, dim3((unsigned)(num_seqs * hkv)), dim3(EV_THREADS),
                           (size_t)p.keys * 4, s, p));
  count_launch(1);
  return FK_OK;
}

}  // namespace fk

using namespace fk;

extern "C" {

int fk_evict_kvcache(void* k_cache, void* v_cache, int64_t num_pages, int page_size,
                     int64_t kv_page_stride, int kv_layout, int num_kv_heads, int head_dim,
                     float* weights, const int32_t* context_lens, int32_t* new_context_lens,
                     const int32_t* block_tables, int64_t block_table_stride,
                     int64_t block_table_cols, int num_seqs, int budget, int keep_first,
                     int keep_last, int32_t* status, fk_stream_t stream) {
  static const char* what = "fk_evict_kvcache";
  FK_REQUIRE(k_cache && v_cache, FK_ERR_INVALID_ARG, "%s: null pointer", what);
  FK_REQUIRE(head_dim == Q4_D, FK_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (128 only)", what,
             head_dim);
  FK_REQUIRE(kv_layout == 0 || kv_layout == 1, FK_ERR_INVALID_ARG,
             "%s: kv_layout must be 0 (NHD) or 1 (HND)", what);
  FK_REQUIRE(page_size > 0 && num_kv_heads > 0 && num_pages > 0 && num_pages < (1ll << 31) &&
                 (int64_t)page_size * num_kv_heads < (1ll << 31),
             FK_ERR_INVALID_ARG, "%s: bad sizes", what);
  FK_REQUIRE(kv_page_stride >= (int64_t)page_size * num_kv_heads * head_dim, FK_ERR_INVALID_ARG,
             "%s: kv_page_stride too small", what);
  FK_REQUIRE(aligned16(k_cache) && aligned16(v_cache) && kv_page_stride % 8 == 0, FK_ERR_ALIGNMENT,
             "%s: 16-byte alignment required", what);
  EvictParams p{};
  p.k = static_cast<uint8_t*>(k_cache);
  p.v = static_cast<uint8_t*>(v_cache);
  p.page_bytes = kv_page_stride * 2;
  p.token_bytes = kv_layout ? Q4_D * 2 : (int64_t)num_kv_heads * Q4_D * 2;
  p.head_bytes = kv_layout ? (int64_t)page_size * Q4_D * 2 : Q4_D * 2;
  return evict(what, p, false, num_pages, page_size, context_lens, new_context_lens, block_tables,
               block_table_stride, block_table_cols, num_seqs, num_kv_heads, weights, budget,
               keep_first, keep_last, status, static_cast<cudaStream_t>(stream));
}

int fk_evict_kvcache_q4(void* cache, int64_t num_pages, int page_size, int num_kv_heads,
                        int head_dim, int group, float* weights, const int32_t* context_lens,
                        int32_t* new_context_lens, const int32_t* block_tables,
                        int64_t block_table_stride, int64_t block_table_cols, int num_seqs,
                        int budget, int keep_first, int keep_last, int32_t* status,
                        fk_stream_t stream) {
  static const char* what = "fk_evict_kvcache_q4";
  const int rc = q4_check_pool(what, cache, num_pages, page_size, num_kv_heads, head_dim, group);
  if (rc != FK_OK) return rc;
  EvictParams p{};
  p.k = static_cast<uint8_t*>(cache);
  p.group_pairs = Q4_D / group;
  return evict(what, p, true, num_pages, page_size, context_lens, new_context_lens, block_tables,
               block_table_stride, block_table_cols, num_seqs, num_kv_heads, weights, budget,
               keep_first, keep_last, status, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
