// Decode attention that reads less of the paged cache:
//
//   fk_selected_attn       attention over selected blocks of each query token and KV head
//   fk_shared_prefix_attn  attention of a batch whose sequences begin with the same pages in groups
//
// Both are one softmax per query head over a set of keys, out = sum_t e^(s q.k_t) v_t / sum_t
// e^(s q.k_t), cut into parts that are joined by their maxima and sums.  Selected blocks, and what the
// rows of a group have for themselves, go through the decode attention kernel (fk_attn.cu).  What
// the rows have in common goes through prefix_attn_kernel: with n rows of G query heads per KV head,
// every key and value is used by n G query rows, which makes a matrix product of it.
//
// Four launches of fk_shared_prefix_attn: shared_plan_kernel (schedule of both parts, 1 CTA),
// prefix_attn_kernel and beside it attn_decode_kernel, shared_join_kernel.
#include "fk_attn.cuh"
#include "fk_tcgen05.cuh"
#include "fk_types.cuh"

#include <mutex>
#include <unordered_map>

namespace fk {

constexpr int SH_D = 128;
constexpr int SH_MAX_G = 16;

// Checked arguments that both calls have.
struct RowsParams {
  const uint16_t* q; int64_t q_stride;
  uint16_t* out; int64_t out_stride;
  int64_t capacity;                    // tokens that a table's row has pages for
  int g;
  float scale_log2;
};

// ---------------------------------------------------------------------------
// splits of a token and head joined: out = sum_s O_s 2^(m_s - M) / sum_s l_s 2^(m_s - M)
// ---------------------------------------------------------------------------
// A lane has the (max, sum) of splits lane, lane + 32, ..., so all of them are one round of loads, and
// four partial rows are on the way at a time.  A split without keys has a sum of zero; its row was
// not written and is not read.  (One whose sum is no number counts.)
struct JoinRow {
  float4 acc;
  float l;
};
// ml(s) gives (max, sum) of split s, row(s) this lane's four channels of it
template <typename ML>
__device__ __forceinline__ float join_max(const ML& ml, int n, int lane) {
  float m = -INFINITY;
  for (int s = lane; s < n; s += 32) m = fmaxf(m, ml(s).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
template <typename ML, typename ROW>
__device__ __forceinline__ void join_add(JoinRow& r, const ML& ml, const ROW& row, int n, float top,
                                         int lane) {
  for (int s0 = 0; s0 < n; s0 += 32) {
    const float2 mlv = s0 + lane < n ? ml(s0 + lane) : make_float2(-INFINITY, 0.f);
    const float fl = mlv.y != 0.f ? fast_exp2(mlv.x - top) : 0.f;
    const int cnt = min(32, n - s0);
    for (int s = 0; s < cnt; s += 4) {
      float4 v[4];
      float f[4], l[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[i] = __shfl_sync(0xffffffffu, fl, (s + i) & 31);
        l[i] = s + i < cnt ? __shfl_sync(0xffffffffu, mlv.y, (s + i) & 31) : 0.f;
        v[i] = l[i] != 0.f ? *row(s0 + s + i) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r.l = fmaf(l[i], f[i], r.l);
        r.acc = r.acc + v[i] * f[i];
      }
    }
  }
}

// a warp per (token, query head)
__global__ void __launch_bounds__(256) selected_join_kernel(const AttnParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t gw = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (gw >= (int64_t)p.batch * p.hq) return;
  const int token = (int)(gw / p.hq), head = (int)(gw - (int64_t)token * p.hq);
  int first, last;
  selected_ctas((int64_t)token * p.hkv + head / p.g, p.tiles, p.unit, &first, &last);
  const int n = last - first + 1;
  if (n == 1) return;                        // written by the attention kernel
  auto ml = [&](int s) { return p.part_ml[gw * p.max_splits + s]; };
  auto part = [&](int s) {
    return reinterpret_cast<const float4*>(p.part_o + (gw * p.max_splits + s) * SH_D) + lane;
  };
  const float top = join_max(ml, n, lane);
  JoinRow r{make_float4(0.f, 0.f, 0.f, 0.f), 0.f};
  join_add(r, ml, part, n, top == -INFINITY ? 0.f : top, lane);
  Elem<uint16_t>::store4(p.out + (int64_t)token * p.out_stride + (int64_t)head * SH_D + lane * 4,
                         r.acc * (r.l > 0.f ? 1.0f / r.l : 0.f));
}

// How the tiles of all tokens and KV heads fall on CTAs.
struct SelectedSchedule {
  int tiles, splits, grid;
  int64_t unit;
};
static SelectedSchedule selected_schedule(int64_t items, int count, int block) {
  SelectedSchedule s;
  const int sms = sm_count();
  s.tiles = (int)(((int64_t)count * block + ATT_TILE - 1) / ATT_TILE);
  const int64_t total = items * s.tiles;
  s.unit = (total + sms - 1) / sms;
  // many items: whole ones, at most an eighth more on some CTAs than on others
  if (items >= 8ll * sms) s.unit = (items + sms - 1) / sms * s.tiles;
  s.grid = (int)((total + s.unit - 1) / s.unit);
  // an item's tiles lie in at most this many runs
  const bool whole = s.unit % s.tiles == 0;
  s.splits = whole ? 1 : (int)((s.tiles - 2 + s.unit) / s.unit) + 1;
  return s;
}

// ---------------------------------------------------------------------------
// schedule of a batch with common prefixes
// ---------------------------------------------------------------------------
// Up to two tiles of 128 query rows share the keys of an item.
struct PrefixItem {
  int row0, rows;      // batch rows
  int table;           // the row whose table is read: the one with the longest context
  int keys;            // whole pages, all of them below that row's context
  int start;           // its first tile of 128 keys among those of all items and KV heads
  int tiles;           // per KV head
  int pad0, pad1;
};

enum : int { PLAN_CHUNKS = 0, PLAN_COUNTER = 2, PLAN_ITEMS = 4, PLAN_TILES = 5, PLAN_UNIT = 6,
             PLAN_SIGN = 7, PLAN_HDR = 8 };

struct SharedPlan {
  int* hdr;            // see above; chunk_start[batch + 1] behind it, as the decode kernel has it
  int4* row_part;      // [batch] start and tiles of the item that holds a row, item * hkv, its
                       // number among the item's rows; tiles 0: none
  int* cta_item;       // [ctas] item of a CTA's first tile
  PrefixItem* items;
  int4* chunks;        // chunks of what each row has for itself
};

struct SharedPlanParams {
  const int32_t* lens; const int32_t* starts; const int32_t* prefix;
  int batch, groups, hkv, page, per_tile, max_splits, ctas, min_unit;
  int sign;            // of the sizes, by which a planned call knows a schedule that is not for it
  int beside;          // the decode kernel may run beside the common part's
  int64_t capacity;
  SharedPlan plan;
  int32_t* status;
};

constexpr int PLAN_MAX_BATCH = 16384;
constexpr int64_t PLAN_MAX_TOKENS = 1ll << 30;    // of a row: positions and sums of chunks in 32 bits
constexpr int PLAN_THREADS = 512;
constexpr int PLAN_WARPS = PLAN_THREADS / 32;

// Sum of the threads before this one, and of all.
__device__ __forceinline__ int64_t plan_before(int64_t v, int64_t* red, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t upto = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  __syncthreads();
  if (lane == 31) red[warp] = upto;
  __syncthreads();
  int64_t before = upto - v, all = 0;
#pragma unroll
  for (int w = 0; w < PLAN_WARPS; ++w) {
    if (w < warp) before += red[w];
    all += red[w];
  }
  *total = all;
  return before;
}

// How many of the SMs take the common part: of its tiles and of those that rows have for themselves
// (128 keys of a KV head each) one of the first takes an SM 2.2 us, one of the second 0.8 us where
// memory does not bound it.  The other SMs start with the second kind, and take it over together
// when the common part is through.
constexpr int PLAN_COMMON_COST = 22, PLAN_OWN_COST = 8;

__global__ void __launch_bounds__(PLAN_THREADS) shared_plan_kernel(const SharedPlanParams p) {
  extern __shared__ int plan_smem[];
  int* s_len = plan_smem;                      // [batch] tokens of a row
  int* s_from = plan_smem + p.batch;           // [batch] of them in its item
  __shared__ int64_t red[PLAN_WARPS];
  __shared__ int s_keys[PLAN_THREADS], s_table[PLAN_THREADS], s_item[PLAN_THREADS],
      s_start[PLAN_THREADS], s_count[6];
  __shared__ int s_first[PLAN_THREADS + 1], s_prefix[PLAN_THREADS];   // of a round's groups
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  pdl_wait();
  bool cut = false, odd = false;
  // a round of groups: their first rows, one more, and their prefixes
  auto fetch = [&](int g0, int here) {
    if (tid < here) {
      s_first[tid] = p.starts[g0 + tid];
      if (tid == here - 1) s_first[here] = p.starts[g0 + here];
      s_prefix[tid] = p.prefix[g0 + tid];
    }
  };
  fetch(0, min(PLAN_THREADS, p.groups));
  for (int i = tid; i < p.batch; i += PLAN_THREADS) {
    const int64_t len = p.lens[i];
    cut |= len > p.capacity;
    s_len[i] = len < 0 ? 0 : (int)(len > p.capacity ? p.capacity : len);
    s_from[i] = 0;
    p.plan.row_part[i] = make_int4(0, 0, 0, 0);
  }
  if (cut && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
  if (tid < 6) s_count[tid] = 0;

  // Groups into items, a round of them at a time: a warp looks for the longest row of a group, a
  // thread per group adds up, a warp per group writes.  Starts that do not ascend within the batch:
  // nobody has anything in common then.
  for (int g = tid; g < p.groups; g += PLAN_THREADS)
    odd |= p.starts[g] < 0 || p.starts[g + 1] < p.starts[g] || p.starts[g + 1] > p.batch;
  odd = __syncthreads_or(odd);
  if (odd && tid == 0 && p.status) atomicOr(p.status, FK_DEV_BAD_POSITION);
  const int groups = odd ? 0 : p.groups;
  const int span = 2 * p.per_tile;
  int items = 0, tiles = 0;                    // of the groups before
  for (int g0 = 0; g0 < groups; g0 += PLAN_THREADS) {
    const int here = min(PLAN_THREADS, groups - g0);
    if (g0 > 0) {
      fetch(g0, here);
      __syncthreads();
    }
    for (int i = warp; i < here; i += PLAN_WARPS) {
      const int a = s_first[i], b = s_first[i + 1], prefix = s_prefix[i];
      int longest = 0, shortest = 0x7fffffff, table = a;
      for (int r = a + lane; r < b; r += 32) {
        const int n = s_len[r];
        if (n > longest) { longest = n; table = r; }
        if (n > 0) shortest = min(shortest, n);
      }
      const int most = __reduce_max_sync(0xffffffffu, longest);
      shortest = __reduce_min_sync(0xffffffffu, shortest);
      table = __reduce_min_sync(0xffffffffu, longest == most ? table : 0x7fffffff);
      // Rows either see all keys of their item or have them for themselves, so that what a row does not
      // see is not multiplied by its zeros.  The item ends where the shortest row does, unless that
      // would leave most of the prefix to every row.
      const int full = max(0, min(prefix, most)) / p.page * p.page;
      const int all = min(full, shortest / p.page * p.page);
      const int keys = all >= full / 2 ? all : full;
      int sharing = 0;
      for (int r = a + lane; r < b; r += 32) sharing += s_len[r] >= keys ? 1 : 0;
      sharing = __reduce_add_sync(0xffffffffu, sharing);
      if (lane == 0) {
        s_keys[i] = sharing < 2 ? 0 : keys;
        s_table[i] = table;
      }
    }
    __syncthreads();
    const int keys = tid < here ? s_keys[tid] : 0;
    const int mine = keys > 0 ? (s_first[tid + 1] - s_first[tid] + span - 1) / span : 0;
    const int per_item = (keys + ATT_TILE - 1) / ATT_TILE;
    // both sums at once: items in the upper half, tiles in the lower
    int64_t all;
    const int64_t before =
        plan_before(((int64_t)mine << 32) + (int64_t)mine * per_item * p.hkv, red, &all);
    s_item[tid] = items + (int)(before >> 32);
    s_start[tid] = tiles + (int)(before & 0xffffffffll);
    items += (int)(all >> 32);
    tiles += (int)(all & 0xffffffffll);
    __syncthreads();
    for (int i = warp; i < here; i += PLAN_WARPS) {
      const int keys_i = s_keys[i];
      if (keys_i == 0) continue;
      // the rows of a group evenly over its items
      const int a = s_first[i], n = s_first[i + 1] - a;
      const int m = (n + span - 1) / span, each = (n + m - 1) / m;
      const int tiles_i = (keys_i + ATT_TILE - 1) / ATT_TILE;
      for (int j = lane; j < m; j += 32)
        p.plan.items[s_item[i] + j] =
            PrefixItem{a + j * each, min(each, n - j * each), s_table[i], keys_i,
                       s_start[i] + j * tiles_i * p.hkv, tiles_i, 0, 0};
      for (int r = lane; r < n; r += 32) {
        if (s_len[a + r] < keys_i) continue;
        const int j = r / each;
        p.plan.row_part[a + r] = make_int4(s_start[i] + j * tiles_i * p.hkv, tiles_i,
                                           (s_item[i] + j) * p.hkv, r - j * each);
        s_from[a + r] = keys_i;
      }
    }
    __syncthreads();
  }

  // What each row has for itself, in chunks of one length: long ones, but enough of them for every
  // CTA, and at most max_splits a row.  Chunks of 1024, 512, 256 and 128 are counted together.
  {
    int longest = 0, n[4] = {0, 0, 0, 0};
    for (int i = tid; i < p.batch; i += PLAN_THREADS) {
      const int rest = max(0, s_len[i] - s_from[i]);
      longest = max(longest, rest);
#pragma unroll
      for (int k = 0; k < 4; ++k) n[k] += (rest + (1024 >> k) - 1) >> (10 - k);
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0 && longest > 0) atomicMax(&s_count[4], longest);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      n[k] = __reduce_add_sync(0xffffffffu, n[k]);
      if (lane == 0 && n[k] > 0) atomicAdd(&s_count[k], n[k]);
    }
    __syncthreads();
  }
  int chunk = 1024;
  int64_t least = ATT_TILE;
  while (least * p.max_splits < s_count[4]) least <<= 1;
  if (least > chunk) chunk = (int)least;
  for (int k = 0; k < 3 && chunk > least && (int64_t)s_count[k] * p.hkv < 4ll * p.ctas; ++k)
    chunk >>= 1;
  const float own = (float)s_count[3] * (float)(p.hkv * PLAN_OWN_COST);
  const float common = (float)tiles * (float)PLAN_COMMON_COST;
  // SMs for the common part; its CTAs take `unit` tiles each
  int ctas = p.ctas;
  if (p.beside && own > 0.f && common > 0.f)
    ctas = max(p.ctas / 8, min(p.ctas, (int)((float)p.ctas * common / (common + own)) + 1));
  const int unit = max(p.min_unit, (tiles + ctas - 1) / max(ctas, 1));
  // CTAs whose first tile is in an item
  for (int i = warp; i < items; i += PLAN_WARPS) {
    const PrefixItem it = p.plan.items[i];
    const int end = it.start + it.tiles * p.hkv;
    for (int c = (it.start + unit - 1) / unit + lane; c < p.ctas && (int64_t)c * unit < end; c += 32)
      p.plan.cta_item[c] = i;
  }
  int* chunk_start = p.plan.hdr + PLAN_HDR;
  int run = 0;
  for (int i0 = 0; i0 < p.batch; i0 += PLAN_THREADS) {
    const int i = i0 + tid;
    const int from = i < p.batch ? s_from[i] : 0;
    const int len = i < p.batch ? s_len[i] : 0;
    const int n = (max(0, len - from) + chunk - 1) / chunk;
    int64_t all;
    const int at = run + (int)plan_before(n, red, &all);
    run += (int)all;
    if (i >= p.batch) continue;
    chunk_start[i] = at;
    // one chunk and nothing before it: the decode kernel writes the result itself
    const int parts = n + (from > 0 ? 2 : 0);
    for (int c = 0; c < n; ++c)
      p.plan.chunks[at + c] = make_int4(i, c | parts << 16, from + c * chunk,
                                        min(len, from + (c + 1) * chunk));
  }
  if (tid == 0) {
    chunk_start[p.batch] = run;
    p.plan.hdr[PLAN_CHUNKS] = run;
    p.plan.hdr[PLAN_COUNTER] = 0;
    p.plan.hdr[PLAN_ITEMS] = items;
    p.plan.hdr[PLAN_TILES] = tiles;
    p.plan.hdr[PLAN_UNIT] = unit;
    p.plan.hdr[PLAN_SIGN] = p.sign;
  }
}

// ---------------------------------------------------------------------------
// the common part
// ---------------------------------------------------------------------------
// One persistent CTA per SM takes a run of `unit` tiles of 128 keys from the items' tiles, one after
// another; each item and KV head in it is a split.  Rows of an item are (batch row, query head of the
// KV head): 128 / G batch rows make a tile of query rows, and an item has one or two.
//
//   warps 0-7, 8-15  softmax of tile 0 and 1, two threads per query row with 64 keys each: maximum
//                 (exchanged), exponentials, sum.  Weights are rounded to bf16 for the product with
//                 the values (their sum is of what was before): results have a relative error of
//                 0.0024 against 64 bits, and 0.0017 where weights stay in fp32.  O is scaled when a
//                 maximum grew by more than 2^8.
//   warp 16       TMA: query tiles, then K_0 V_0 K_1 V_1 ... through a ring of five 32 KiB slots
//   warp 17       tensor memory and products: S_t = Q_t K_j^T into columns [128 t, 128 t + 128),
//                 O_t += P_t V_j into [256 + 128 t, ...); P_t is read from where each half of the
//                 keys had its S_t.  The two tiles take turns, so that the softmax of one runs
//                 beside the products of the other.
//
// A tile's step is softmax (1850 clocks for 128 keys, 1024 of them its exponentials), P V and the next S
// (1024, and 600 until either side has seen the other's barrier); the two tiles are in turn, so that
// 256 rows by 128 keys take 3700 clocks: 16384 keys for 256 rows of 64/4 heads 146 us, 0.57 of the
// measured bf16 rate.  Tried: one thread a row (154 us); scores of 64 keys in two buffers a tile, so
// that the softmax never waits (195 us: a product of 64 columns takes as long as one of 128).
// Results leave through shared memory (where the query tile was) in bulk copies of 4 KiB: 32 rows of
// 32 channels, 16-byte pieces of a row exchanged by its number so that writing them is free of
// conflicts.
//
// Bounds: the bytes of the common part up to some 250 query rows a KV head, the products and
// exponentials beyond.  Waits end after two seconds, as in the other attention kernels.
constexpr int PX_SLOTS = 5;
constexpr int PX_HALF_BYTES = 128 * 128;
constexpr int PX_TILE_BYTES = 2 * PX_HALF_BYTES;
constexpr int PX_THREADS = 576;
constexpr int PX_WARP_TMA = 16, PX_WARP_MMA = 17;
constexpr int PX_OFF_Q = 0;
constexpr int PX_OFF_KV = 2 * PX_TILE_BYTES;
constexpr int PX_OFF_BAR = PX_OFF_KV + PX_SLOTS * PX_TILE_BYTES;
constexpr int PX_OFF_MAX = PX_OFF_BAR + 256;
constexpr int PX_SMEM_BASE = 256;                 // alignment of what a launch gets, by its declaration
constexpr int PX_SMEM_ALLOC = PX_OFF_MAX + 2 * 2 * 128 * 4 + 1024 - PX_SMEM_BASE;
constexpr int PX_TMEM_COLS = 512;
constexpr float PX_RESCALE_LOG2 = 8.0f;
constexpr int PX_SLOT_FLOATS = 2 * 128 * SH_D;   // partial rows of a split
static_assert(PX_SMEM_ALLOC <= 232448, "shared memory budget");
static_assert(tmem_alone(PX_SMEM_ALLOC), "two CTAs could wait for one another's tensor memory");

struct PrefixParams {
  int sign;
  const int* hdr; const int* cta_item; const PrefixItem* items;
  const int32_t* lens;
  const int32_t* tables; int64_t table_stride;
  int hq, hkv, g, per_tile;            // batch rows of a query tile
  int hnd, block_size, sub_tokens, num_blocks;
  float scale_log2;
  // Of the split with CTA c and item and head i at c + i, which is another for every split: partial
  // rows [2 tiles][4 x 32 rows][2 x 64 channels][2 x 32][32 rows][32], and (maximum, sum) of both
  // halves of the keys [2][2][128].
  float* part_o; float2* part_ml;
  int32_t* status;
};

__device__ __forceinline__ uint64_t px_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool px_poll(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                        int32_t* status) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = px_ns();
  for (;;) {
    for (int i = 0; i < 128; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (px_ns() - t0 > 2000000000ull) {
      *abort_flag = 1;
      if (status) atomicOr(status, FK_DEV_WAIT_TIMEOUT);
      return false;
    }
  }
}
// By whole warps: one answer for all lanes.
__device__ __forceinline__ bool px_wait_warp(uint64_t* bar, uint32_t parity,
                                             volatile int* abort_flag, int32_t* status) {
  return __all_sync(0xffffffffu, px_poll(bar, parity, abort_flag, status) ? 1 : 0) != 0;
}

// 32 lanes x 8 columns of tensor memory
__device__ __forceinline__ void px_ld8(uint32_t taddr, uint32_t (&v)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7])
      : "r"(taddr));
}
__device__ __forceinline__ void px_st8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
      : "memory");
}

// packed fp32 pairs and the three-input maximum
__device__ __forceinline__ uint64_t px_pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void px_unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t px_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t px_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float px_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The splits of a CTA, one after another: tiles t0 .. t1 - 1 of an item and KV head.  Little of it
// stays in registers from one to the next.
struct PrefixSeg {
  PrefixItem it;
  int kvh, t0, t1, slot, two;
};
struct PrefixWalk {
  int item, at, end;
  __device__ __forceinline__ bool next(const PrefixParams& p, PrefixSeg& s) {
    if (at >= end) return false;
    if (item < 0) item = p.cta_item[blockIdx.x];
    s.it = p.items[item];
    if (at >= s.it.start + s.it.tiles * p.hkv) s.it = p.items[++item];
    const int in = at - s.it.start;
    s.kvh = in / s.it.tiles;
    s.t0 = in - s.kvh * s.it.tiles;
    s.t1 = min(s.it.tiles, s.t0 + end - at);
    s.slot = (int)blockIdx.x + item * p.hkv + s.kvh;
    s.two = s.it.rows > p.per_tile ? 1 : 0;
    at += s.t1 - s.t0;
    return true;
  }
};

__global__ void __launch_bounds__(PX_THREADS, 1)
prefix_attn_kernel(const __grid_constant__ CUtensorMap tmap_q,
                   const __grid_constant__ CUtensorMap tmap_k,
                   const __grid_constant__ CUtensorMap tmap_v, const PrefixParams p) {
  extern __shared__ __align__(PX_SMEM_BASE) uint8_t px_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(px_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + PX_OFF_BAR);
  uint64_t* q_empty = q_full + 1;                    // the last S product of a split has been read
  uint64_t* slot_full = q_full + 2;
  uint64_t* slot_empty = slot_full + PX_SLOTS;
  uint64_t* s_full = slot_empty + PX_SLOTS;          // [2]
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* o_empty = o_full + 2;
  uint64_t* staged = o_empty + 2;                    // results have left the query tile's place
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(staged + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(staged + 3);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < PX_SLOTS; ++i) {
      mbar_init(&slot_full[i], 1);
      mbar_init(&slot_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 8);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_empty[t], 8);
      mbar_init(&staged[t], 8);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == PX_WARP_TMA && lane == 0) {
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == PX_WARP_MMA) tmem_alloc(tmem_slot, PX_TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // all 512 columns: they start at column 0
  const uint32_t tmem_got = *tmem_slot;
  constexpr uint32_t tmem_base = 0;
  pdl_wait();     // the schedule, q and the cache may come from earlier kernels
  // The decode kernel starts from here on, on the SMs that have no tiles of the common part, and
  // reads what the kernels before this one have written.
  pdl_launch_dependents();
  // A workspace without a schedule of these sizes holds any words: none of them is used.
  const bool known = p.hdr[PLAN_SIGN] == p.sign;
  const int unit = known ? p.hdr[PLAN_UNIT] : 1, total = known ? p.hdr[PLAN_TILES] : 0;
  const int64_t from = (int64_t)blockIdx.x * unit;
  const int begin = (int)(from < total ? from : total);
  const int end = tmem_got != 0 ? begin : min(total - begin, unit) + begin;
  if (tmem_got != 0 && threadIdx.x == 0 && p.status) atomicOr(p.status, FK_DEV_TMEM_BASE);
  PrefixWalk walk{-1, begin, end};

  if (warp == PX_WARP_TMA) {
    const int st = p.sub_tokens, npieces = 128 / st;
    int kv_idx = 0, segs = 0, before = 0;
    uint32_t uses[2] = {0, 0};                 // splits that had query tile t
    bool ok = true;
    PrefixSeg w;
    while (ok && walk.next(p, w)) {
      int pass = 1;
      if (lane == 0) {
        if (segs > 0) {
          pass = px_poll(q_empty, (uint32_t)(segs - 1) & 1u, abort_flag, p.status) ? 1 : 0;
          for (int t = 0; t <= before && pass; ++t)
            pass = px_poll(&staged[t], (uses[t] - 1) & 1u, abort_flag, p.status) ? 1 : 0;
        }
        if (pass) {
          mbar_arrive_expect_tx(q_full, (uint32_t)(1 + w.two) * 2u * 128u *
                                            (uint32_t)(p.g * p.per_tile));
          for (int t = 0; t <= w.two; ++t)
            for (int dh = 0; dh < 2; ++dh)
              tma_load_4d(smem + PX_OFF_Q + t * PX_TILE_BYTES + dh * PX_HALF_BYTES, &tmap_q, q_full,
                          dh * 64, w.kvh * p.g, w.it.row0 + t * p.per_tile, 0);
        }
      }
      pass = __shfl_sync(0xffffffffu, pass, 0);
      if (!pass) { ok = false; break; }
      ++segs;
      ++uses[0];
      if (w.two) ++uses[1];
      before = w.two;
      const int32_t* bt = p.tables + (int64_t)w.it.table * p.table_stride;
      for (int i = 2 * w.t0; i < 2 * w.t1; ++i, ++kv_idx) {
        const int slot = kv_idx % PX_SLOTS;
        const uint32_t lap = (uint32_t)(kv_idx / PX_SLOTS) & 1u;
        const int tok = (i >> 1) * 128 + lane * st;
        int page = p.num_blocks;               // past the end: the copy reads the zero fill
        if (lane < npieces && tok < w.it.keys) {
          page = bt[tok / p.block_size];
          if (page < 0 || page >= p.num_blocks) {
            page = p.num_blocks;
            if (p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
          }
        }
        pass = 1;
        if (lane == 0) pass = px_poll(&slot_empty[slot], lap ^ 1, abort_flag, p.status) ? 1 : 0;
        pass = __shfl_sync(0xffffffffu, pass, 0);
        if (!pass) { ok = false; break; }
        if (lane == 0) mbar_arrive_expect_tx(&slot_full[slot], PX_TILE_BYTES);
        __syncwarp();
        if (lane < npieces) {
          uint8_t* dst = smem + PX_OFF_KV + slot * PX_TILE_BYTES + lane * st * 128;
          const CUtensorMap* map = i & 1 ? &tmap_v : &tmap_k;
          const int off = tok % p.block_size;
          const int c1 = p.hnd ? off : w.kvh, c2 = p.hnd ? w.kvh : off;
          tma_load_4d(dst, map, &slot_full[slot], 0, c1, c2, page);
          tma_load_4d(dst + PX_HALF_BYTES, map, &slot_full[slot], 64, c1, c2, page);
        }
      }
    }
    if (!ok && lane == 0) {
      // given up: copies under way must land before the CTA's memory is another's
      if (segs > 0) (void)mbar_wait(q_full, (uint32_t)(segs - 1) & 1u, 1u << 20);
      for (int s = 0; s < PX_SLOTS && s < kv_idx; ++s) {
        const int uses_s = (kv_idx - 1 - s) / PX_SLOTS;      // of slot s before its last one
        (void)mbar_wait(&slot_full[s], (uint32_t)uses_s & 1u, 1u << 20);
      }
    }
    __syncwarp();
  } else if (warp == PX_WARP_MMA) {
    constexpr uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(128 >> 3) << 17) |
                                 ((uint32_t)(128 >> 4) << 24);
    constexpr uint32_t idesc_pv = idesc_s | (1u << 16);   // B (= V) is MN-major
    const uint32_t q_addr = smem_u32(smem + PX_OFF_Q);
    const uint32_t kv_addr = smem_u32(smem + PX_OFF_KV);
    auto issue_s = [&](int t, int slot) {
      const uint32_t a = q_addr + t * PX_TILE_BYTES;
      const uint32_t b = kv_addr + slot * PX_TILE_BYTES;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < SH_D / 16; ++kk) {
          const uint32_t o = (kk >> 2) * PX_HALF_BYTES + (kk & 3) * 32;
          tc_mma_bf16(tmem_base + t * 128, smem_desc_sw128(a + o), smem_desc_sw128(b + o), idesc_s,
                      kk > 0 ? 1u : 0u);
        }
      }
      __syncwarp();
    };
    auto issue_pv = [&](int t, int slot, bool acc) {
      // weights of keys 0 .. 63 in columns 0 .. 31 of S_t, of the others in columns 64 .. 95
      const uint32_t a = tmem_base + t * 128;
      const uint32_t b = kv_addr + slot * PX_TILE_BYTES;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          tc_mma_bf16_ts(tmem_base + 256 + t * SH_D, a + (kk >> 2) * 64 + (kk & 3) * 8,
                         smem_desc_sw128_mn(b + kk * 2048, PX_HALF_BYTES, 1024), idesc_pv,
                         (acc || kk > 0) ? 1u : 0u);
      }
      __syncwarp();
    };
    int kv_base = 0, segs = 0;
    uint32_t n_sp[2] = {0, 0}, n_o[2] = {0, 0};   // hand-overs and splits per query tile so far
    bool ok = true;
    PrefixSeg w;
    while (ok && walk.next(p, w)) {
      const int n = w.t1 - w.t0, qt = 1 + w.two;
      ok = px_wait_warp(q_full, (uint32_t)segs & 1u, abort_flag, p.status) &&
           px_wait_warp(&slot_full[kv_base % PX_SLOTS], (uint32_t)(kv_base / PX_SLOTS) & 1u,
                        abort_flag, p.status);
      if (!ok) break;
      tc_fence_after();
      for (int t = 0; t < qt; ++t) {
        issue_s(t, kv_base % PX_SLOTS);
        tc_commit_elect(&s_full[t]);
      }
      tc_commit_elect(&slot_empty[kv_base % PX_SLOTS]);
      if (n == 1) tc_commit_elect(q_empty);
      for (int j = 0; j < n && ok; ++j) {
        const int vi = kv_base + 2 * j + 1, ki = vi + 1;
        const int vslot = vi % PX_SLOTS, kslot = ki % PX_SLOTS;
        // both tiles of this step ahead of the weights, so that P V and the next S go out together
        ok = px_wait_warp(&slot_full[vslot], (uint32_t)(vi / PX_SLOTS) & 1u, abort_flag, p.status);
        const bool more = j + 1 < n;
        if (ok && more)
          ok = px_wait_warp(&slot_full[kslot], (uint32_t)(ki / PX_SLOTS) & 1u, abort_flag, p.status);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok || t >= qt) break;
          if (j == 0 && n_o[t] > 0) {
            // O_t holds the split before until its rows have been read
            ok = px_wait_warp(&o_empty[t], (n_o[t] - 1) & 1u, abort_flag, p.status);
            if (!ok) break;
          }
          ok = px_wait_warp(&p_full[t], (n_sp[t] + (uint32_t)j) & 1u, abort_flag, p.status);
          if (!ok) break;
          tc_fence_after();
          issue_pv(t, vslot, j > 0);
          if (j == n - 1) tc_commit_elect(&o_full[t]);
          if (more) {
            issue_s(t, kslot);
            tc_commit_elect(&s_full[t]);
          }
        }
        if (!ok) break;
        tc_commit_elect(&slot_empty[vslot]);
        if (more) tc_commit_elect(&slot_empty[kslot]);
        if (j + 2 == n) tc_commit_elect(q_empty);   // the last S products have been issued
      }
      kv_base += 2 * n;
      ++segs;
      for (int t = 0; t < qt; ++t) {
        n_sp[t] += (uint32_t)n;
        ++n_o[t];
      }
    }
  } else {
    const int t = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3;
    const uint32_t s_addr = tmem_base + ((uint32_t)(quad * 32) << 16) + t * 128 + half * 64;
    const uint32_t o_addr = s_addr + 256;
    // maxima of the two threads of a row.  In fp32: a reference value that is off by a part of the
    // maximum, as a rounded one is, puts all exponentials of scores past some 10^5 below fp32's range.
    const uint32_t max_at = smem_u32(smem + PX_OFF_MAX) + t * 1024 + (quad * 32 + lane) * 4;
    constexpr uint32_t kGone = 0x7fffffffu;    // no number: this warp's wait has run out
    uint32_t n_sp = 0, n_o = 0;
    bool ok = true;
    for (;;) {
      int n, kpos, lim = 0, slot;
      {
        PrefixSeg w;
        if (!walk.next(p, w)) break;
        if (t > w.two) continue;
        n = w.t1 - w.t0;
        kpos = w.t0 * 128 + half * 64;
        slot = w.slot;
        const int in_tile = (quad * 32 + lane) / p.g, i = t * p.per_tile + in_tile;
        if (in_tile < p.per_tile && i < w.it.rows) {
          const int64_t len = p.lens[w.it.row0 + i];
          lim = len >= w.it.keys ? w.it.keys : 0;
        }
      }
      // 32 rows without one that sees keys (behind the last of an item) have nothing to do: what is
      // in their columns stays in their rows of the products
      const bool some = __any_sync(0xffffffffu, lim > 0);
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j, kpos += 128) {
        // Two warps have a row between them and meet at a barrier in every step: one whose wait has
        // run out says so there, and both leave.
        ok = ok && px_wait_warp(&s_full[t], (n_sp + (uint32_t)j) & 1u, abort_flag, p.status);
        if (!some) {
          if (!ok) break;
          if (lane == 0) mbar_arrive(&p_full[t]);
          __syncwarp();
          continue;
        }
        // (scores of a step whose wait ran out are not used)
        tc_fence_after();
        uint32_t v[64];                        // scores, then weights two a word
        float sum;
        // With the reference value that the row has, and again only if a maximum is far above it, as
        // in the first step: the exponentials need not wait for the other half's maximum.
        for (int pass = 0; pass < 2; ++pass) {
          tc_ld32(s_addr, v);
          tc_ld32(s_addr + 32, v + 32);
          tc_wait_ld();
          if (kpos + 64 > lim) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (kpos + i >= lim) v[i] = 0xff800000u;   // -inf
          }
          const float neg_mu = m_used == -INFINITY ? 0.f : -m_used;
          const uint64_t nm2 = px_pack2(neg_mu, neg_mu),
                         sc2 = px_pack2(p.scale_log2, p.scale_log2);
          uint64_t sum2[2] = {0ull, 0ull};
          float mx = -INFINITY, m2 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            mx = px_max3(mx, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
            m2 = px_max3(m2, __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
            float t0, t1, t2, t3;
            px_unpack2(px_fma2(px_pack2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), sc2, nm2),
                       t0, t1);
            px_unpack2(px_fma2(px_pack2(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])), sc2,
                               nm2), t2, t3);
            const float e0 = fast_exp2(t0), e1 = fast_exp2(t1);
            const float e2 = fast_exp2(t2), e3 = fast_exp2(t3);
            sum2[0] = px_add2(sum2[0], px_pack2(e0, e1));
            sum2[1] = px_add2(sum2[1], px_pack2(e2, e3));
            v[i / 2] = pack_bf16(e0, e1);
            v[i / 2 + 1] = pack_bf16(e2, e3);
          }
          {
            float a0, a1, a2, a3;
            px_unpack2(sum2[0], a0, a1);
            px_unpack2(sum2[1], a2, a3);
            sum = (a0 + a1) + (a2 + a3);
          }
          if (pass) break;
          {
            // (a maximum is a number: it begins at -infinity, and no-number scores are passed over)
            const uint32_t a = ok ? __float_as_uint(fmaxf(mx, m2)) : kGone;
            uint32_t b;
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(max_at + half * 512), "r"(a) : "memory");
            named_bar_sync(1 + t * 4 + quad, 64);
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(b) : "r"(max_at + (half ^ 1) * 512)
                         : "memory");
            ok = a != kGone && b != kGone;     // the same for both warps: one flag for all lanes
            mx = fmaxf(__uint_as_float(a), __uint_as_float(b)) * p.scale_log2;
          }
          if (!ok) break;
          const bool grow = mx > m_used + PX_RESCALE_LOG2;
          if (!__any_sync(0xffffffffu, grow)) break;
          const float alpha = grow ? fast_exp2(m_used - mx) : 1.0f;
          if (j > 0) {
            // eight columns at a time: few registers
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t o[8];
              px_ld8(o_addr + c * 8, o);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              px_st8(o_addr + c * 8, o);
            }
            tc_wait_st();
          }
          if (grow) {
            l *= alpha;
            m_used = mx;
          }
        }
        if (!ok) break;
        l += sum;
        __syncwarp();
        tc_st32(s_addr, v);                    // over what this warp has read
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      // a warp whose wait runs out here goes on to the next step's barrier, and says so there
      ok = px_wait_warp(&o_full[t], n_o & 1u, abort_flag, p.status);
      n_sp += (uint32_t)n;
      ++n_o;
      if (!ok) continue;
      tc_fence_after();
      float* dst = p.part_o + (int64_t)slot * PX_SLOT_FLOATS + ((t * 4 + quad) * 2 + half) * 2048;
      uint8_t* stage = smem + PX_OFF_Q + t * PX_TILE_BYTES + (half * 4 + quad) * 4096;
      if (!some) {
        tc_fence_before();
        if (lane == 0) mbar_arrive(&o_empty[t]);
      }
#pragma unroll
      for (int c = 0; c < 2 && some; ++c) {
        uint32_t o[32];
        tc_ld32(o_addr + c * 32, o);
        tc_wait_ld();
        if (c == 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&o_empty[t]);
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          }
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) =
              make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                           dst + c * 1024),
                       "r"(smem_u32(stage)), "r"(4096)
                       : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        __syncwarp();
      }
      p.part_ml[(int64_t)slot * 512 + (t * 2 + half) * 128 + quad * 32 + lane] =
          make_float2(m_used, l);
      if (lane == 0) {
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        mbar_arrive(&staged[t]);
      }
      __syncwarp();
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == PX_WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem_got, PX_TMEM_COLS);
  }
}

// a warp per (row, query head): the splits of its common part, then its own
struct SharedJoinParams {
  const int* hdr; const int4* row_part;
  int* counter;
  uint16_t* out; int64_t out_stride;
  const float* pre_o; const float2* pre_ml;
  const float* own_o; const float2* own_ml; int own_splits;
  int batch, hq, hkv, g, per_tile;
  int sign;
  int32_t* status;
};
__global__ void __launch_bounds__(256) shared_join_kernel(const SharedJoinParams p) {
  pdl_launch_dependents();
  pdl_wait();
  // the decode kernel has ended: its work counter is ready for the next layer
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.counter = 0;
  const int64_t gw = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (gw >= (int64_t)p.batch * p.hq) return;
  const int row = (int)(gw / p.hq), head = (int)(gw - (int64_t)row * p.hq);
  const int* chunk_start = p.hdr + PLAN_HDR;
  int n_own = chunk_start[row + 1] - chunk_start[row];
  int4 in = p.row_part[row];
  const int unit = p.hdr[PLAN_UNIT];
  if (p.hdr[PLAN_SIGN] != p.sign) {            // no schedule of these sizes: nothing was computed
    n_own = in.y = 0;
    if (gw == 0 && lane == 0 && p.status) atomicOr(p.status, FK_DEV_BAD_POSITION);
  }
  int n_pre = 0;
  int64_t slot = 0;                            // of the first split
  int at = 0;                                  // row among the two tiles of a split
  if (in.y > 0) {
    const int kvh = head / p.g, first = in.x + kvh * in.y;
    const int cta = first / unit;
    n_pre = (first + in.y - 1) / unit - cta + 1;
    slot = cta + in.z + kvh;
    const int t = in.w / p.per_tile;
    at = t * 128 + (in.w - t * p.per_tile) * p.g + head - kvh * p.g;
  }
  if (n_pre == 0 && n_own == 1) return;        // written by the decode kernel
  // the sum of a row over both halves of the keys, and this lane's piece of its channels
  const int64_t ml_at = slot * 512 + (at >> 7) * 256 + (at & 127);
  auto pre_ml = [&](int s) {
    const float2 a = p.pre_ml[ml_at + (int64_t)s * 512], b = p.pre_ml[ml_at + (int64_t)s * 512 + 128];
    return make_float2(a.x, a.y + b.y);
  };
  const float* pre_at = p.pre_o + slot * PX_SLOT_FLOATS + (at >> 5) * 4096 + (lane >> 3) * 1024 +
                        (at & 31) * 32 + (((lane ^ at) & 7) << 2);
  auto pre_row = [&](int s) {
    return reinterpret_cast<const float4*>(pre_at + (int64_t)s * PX_SLOT_FLOATS);
  };
  auto own_ml = [&](int s) { return p.own_ml[gw * p.own_splits + s]; };
  auto own_row = [&](int s) {
    return reinterpret_cast<const float4*>(p.own_o + (gw * p.own_splits + s) * SH_D) + lane;
  };
  float top = fmaxf(join_max(pre_ml, n_pre, lane), join_max(own_ml, n_own, lane));
  if (top == -INFINITY) top = 0.f;
  JoinRow r{make_float4(0.f, 0.f, 0.f, 0.f), 0.f};
  join_add(r, pre_ml, pre_row, n_pre, top, lane);
  join_add(r, own_ml, own_row, n_own, top, lane);
  Elem<uint16_t>::store4(p.out + (int64_t)row * p.out_stride + (int64_t)head * SH_D + lane * 4,
                         r.acc * (r.l > 0.f ? 1.0f / r.l : 0.f));
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// Tensor map of q for query tiles: (64 channels, g heads, per_tile batch rows) a copy.
struct QMapKey {
  const void* q; int64_t stride; int batch, hq, g, per_tile;
  bool operator==(const QMapKey& o) const {
    return q == o.q && stride == o.stride && batch == o.batch && hq == o.hq && g == o.g &&
           per_tile == o.per_tile;
  }
};
struct QMapHash {
  size_t operator()(const QMapKey& k) const {
    return std::hash<const void*>()(k.q) ^
           std::hash<int64_t>()(k.stride * 31 + k.batch * 1000003ll + k.hq * 97ll + k.g);
  }
};
static int get_q_map(const QMapKey& key, CUtensorMap* out) {
  static std::mutex mu;
  static std::unordered_map<QMapKey, CUtensorMap, QMapHash> maps;
  std::lock_guard<std::mutex> lk(mu);
  auto it = maps.find(key);
  if (it != maps.end()) {
    *out = it->second;
    return FK_OK;
  }
  tensormap_encode_fn enc = get_tensormap_encode();
  FK_REQUIRE(enc != nullptr, FK_ERR_CUDA, "cuTensorMapEncodeTiled not available from the driver");
  const cuuint64_t dims[4] = {SH_D, (cuuint64_t)key.hq, (cuuint64_t)key.batch, 1};
  const cuuint64_t strides[3] = {SH_D * 2, (cuuint64_t)key.stride * 2,
                                 (cuuint64_t)key.stride * 2 * (cuuint64_t)key.batch};
  const cuuint32_t box[4] = {64, (cuuint32_t)key.g, (cuuint32_t)key.per_tile, 1};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(key.q), dims,
                         strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  FK_REQUIRE(r == CUDA_SUCCESS, FK_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
  if (maps.size() > 4096) maps.clear();
  maps.emplace(key, *out);
  return FK_OK;
}

// longest tables of a call that is one launch
constexpr int SHARED_DIRECT_TOKENS = 2048;
// fewest 128-key tiles of the common part that a CTA takes: 16 rows of 4096 common keys take 28.4 us
// with 4, 31.7 with 2 and 34.3 with 8; of 2048 common keys 27.5, 28.0 and 33.7; 4 rows of 32768 take
// 62.1 with 4 and 65.8 with 2
constexpr int PREFIX_MIN_UNIT = 4;

struct SharedLayout {
  size_t row_part, cta_item, items, chunks, pre_o, pre_ml, own_o, own_ml, total;
};
static SharedLayout shared_layout(int64_t batch, int groups, int hq, int hkv, int max_splits) {
  SharedLayout s;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at = (at + bytes + 255) & ~size_t(255);
    return here;
  };
  // an item has at least one full group's rest, or the rows of two query tiles
  const int64_t span = 2 * (128 / (hq / hkv));
  const int64_t items = groups < 1 ? 0 : groups + batch / span < batch ? groups + batch / span : batch;
  const int64_t slots = items == 0 ? 0 : sm_count() + items * hkv;
  take((PLAN_HDR + batch + 1) * sizeof(int));
  s.row_part = take(batch * sizeof(int4));
  s.cta_item = take(sm_count() * sizeof(int));
  s.items = take(items * sizeof(PrefixItem));
  s.chunks = take((size_t)batch * max_splits * sizeof(int4));
  s.pre_o = take((size_t)slots * PX_SLOT_FLOATS * sizeof(float));
  s.pre_ml = take((size_t)slots * 512 * sizeof(float2));
  const size_t rows = (size_t)batch * hq;
  s.own_o = take(rows * max_splits * SH_D * sizeof(float));
  s.own_ml = take(rows * max_splits * sizeof(float2));
  s.total = at;
  return s;
}

static int rows_args(const char* what, RowsParams& p, const void* q, int64_t q_stride, void* out,
                     int64_t out_stride, const void* k, const void* v, int64_t num_pages, int page,
                     int64_t page_stride, int layout, const int32_t* lens, const int32_t* tables,
                     int64_t table_stride, int64_t table_cols, int hq, int hkv, int d,
                     float scale) {
  FK_REQUIRE(q && out && k && v && lens && tables, FK_ERR_INVALID_ARG, "%s: null pointer", what);
  FK_REQUIRE(d == SH_D, FK_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (128 only)", what, d);
  FK_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0, FK_ERR_INVALID_ARG,
             "%s: num_q_heads must be a multiple of num_kv_heads", what);
  FK_REQUIRE(hq / hkv <= SH_MAX_G, FK_ERR_UNSUPPORTED, "%s: more than %d query heads per KV head",
             what, SH_MAX_G);
  FK_REQUIRE(page == 16 || page == 32 || (page >= 64 && page % 64 == 0), FK_ERR_UNSUPPORTED,
             "%s: block_size %d must be 16, 32 or a multiple of 64", what, page);
  FK_REQUIRE(layout == 0 || layout == 1, FK_ERR_INVALID_ARG,
             "%s: kv_layout must be 0 (NHD) or 1 (HND)", what);
  FK_REQUIRE(num_pages > 0 && num_pages < (1ll << 31) && table_cols > 0 && hkv <= 65535,
             FK_ERR_INVALID_ARG, "%s: bad sizes", what);
  FK_REQUIRE(page_stride >= (int64_t)page * hkv * d && table_stride >= 0 &&
                 q_stride >= (int64_t)hq * d && out_stride >= (int64_t)hq * d,
             FK_ERR_INVALID_ARG, "%s: stride too small", what);
  FK_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k) && aligned16(v) && q_stride % 8 == 0 &&
                 out_stride % 8 == 0 && page_stride % 8 == 0,
             FK_ERR_ALIGNMENT, "%s: 16-byte alignment required", what);
  p.q = static_cast<const uint16_t*>(q); p.q_stride = q_stride;
  p.out = static_cast<uint16_t*>(out); p.out_stride = out_stride;
  p.capacity = table_cols * page;
  p.g = hq / hkv;
  p.scale_log2 = scale * 1.4426950408889634f;
  return FK_OK;
}

}  // namespace fk

using namespace fk;

extern "C" {

size_t fk_selected_attn_workspace_bytes(int num_tokens, int num_q_heads, int num_kv_heads,
                                        int head_dim, int count, int block) {
  if (num_tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || count <= 0 ||
      block <= 0)
    return 0;
  const SelectedSchedule s = selected_schedule((int64_t)num_tokens * num_kv_heads, count, block);
  if (s.splits == 1) return 0;
  return (size_t)num_tokens * num_q_heads * s.splits * (head_dim * sizeof(float) + sizeof(float2));
}

int fk_selected_attn(const void* q, int64_t q_stride_token, void* out, int64_t out_stride_token,
                     const void* k_cache, const void* v_cache, int64_t num_pages, int page_size,
                     int64_t kv_page_stride, int kv_layout, const int32_t* context_lens,
                     const int32_t* table_rows, const int32_t* block_tables,
                     int64_t block_table_stride, int64_t block_table_cols, int num_tables,
                     const int32_t* selected, int count, int block, int num_tokens,
                     int num_q_heads, int num_kv_heads, int head_dim, float softmax_scale,
                     void* workspace, size_t workspace_bytes, int32_t* status,
                     fk_stream_t stream) {
  FK_REQUIRE(num_tokens >= 0 && count >= 0, FK_ERR_INVALID_ARG, "fk_selected_attn: negative size");
  if (num_tokens == 0) return FK_OK;
  RowsParams p{};
  const int rc = rows_args("fk_selected_attn", p, q, q_stride_token, out, out_stride_token, k_cache,
                           v_cache, num_pages, page_size, kv_page_stride, kv_layout, context_lens,
                           block_tables, block_table_stride, block_table_cols, num_q_heads,
                           num_kv_heads, head_dim, softmax_scale);
  if (rc != FK_OK) return rc;
  FK_REQUIRE(selected != nullptr && count > 0, FK_ERR_INVALID_ARG,
             "fk_selected_attn: no selected blocks");
  FK_REQUIRE(block == 16 || block == 32 || (block >= 64 && block % 64 == 0), FK_ERR_UNSUPPORTED,
             "fk_selected_attn: block %d must be 16, 32 or a multiple of 64", block);
  FK_REQUIRE(page_size % block == 0, FK_ERR_INVALID_ARG,
             "fk_selected_attn: a page of %d tokens is not a whole number of blocks of %d",
             page_size, block);
  FK_REQUIRE(table_rows != nullptr || num_tables >= num_tokens, FK_ERR_INVALID_ARG,
             "fk_selected_attn: %d tables for %d tokens", num_tables, num_tokens);
  FK_REQUIRE((int64_t)count * block <= (1 << 30), FK_ERR_UNSUPPORTED,
             "fk_selected_attn: %d blocks of %d tokens", count, block);
  const size_t need = fk_selected_attn_workspace_bytes(num_tokens, num_q_heads, num_kv_heads,
                                                       head_dim, count, block);
  FK_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need &&
                           (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0),
             FK_ERR_WORKSPACE,
             "fk_selected_attn: workspace needs %zu bytes, 256-byte aligned (got %zu)", need,
             workspace_bytes);
  const SelectedSchedule s = selected_schedule((int64_t)num_tokens * num_kv_heads, count, block);
  AttnParams a{};
  a.q = p.q; a.q_stride = p.q_stride;
  a.out = p.out; a.out_stride = p.out_stride;
  a.context_lens = context_lens;
  a.block_tables = block_tables; a.bt_stride = block_table_stride;
  a.batch = num_tokens; a.hq = num_q_heads; a.hkv = num_kv_heads; a.g = p.g;
  a.block_size = page_size; a.num_blocks = (int)num_pages;
  a.sub_tokens = block < ATT_BOX ? block : ATT_BOX;
  a.fused16 = block == 16;
  a.bs_shift = -1;
  a.hnd = kv_layout;
  a.scale_log2 = p.scale_log2;
  a.max_splits = s.splits;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)num_tokens * num_q_heads * s.splits *
                                                       head_dim);
  a.status = status;
  a.selected = selected; a.rows = table_rows;
  a.count = count; a.sel_block = block; a.num_tables = num_tables;
  a.capacity = p.capacity;
  a.tiles = s.tiles; a.unit = s.unit;
  CUtensorMap mk, mv;
  int rc2 = get_kv_map(k_cache, num_pages, page_size, num_kv_heads, kv_page_stride, kv_layout,
                       a.sub_tokens, a.fused16, &mk);
  if (rc2 == FK_OK)
    rc2 = get_kv_map(v_cache, num_pages, page_size, num_kv_heads, kv_page_stride, kv_layout,
                     a.sub_tokens, a.fused16, &mv);
  if (rc2 != FK_OK) return rc2;
  // (weights in one bf16 part: relative error 0.0023 against 64 bits, 0.0017 with fp32 weights; two
  // parts took 1 to 2 % longer)
  FK_CUDA_OK(launch_decode(p.g > 8, false, true, s.grid, mk, mv, a,
                           static_cast<cudaStream_t>(stream)));
  count_launch(1);
  if (s.splits > 1) {
    const int64_t warps = (int64_t)num_tokens * num_q_heads;
    FK_CUDA_OK(launch_kernel(selected_join_kernel, dim3((unsigned)((warps + 7) / 8)), dim3(256),
                             (size_t)0, static_cast<cudaStream_t>(stream), a));
    count_launch(1);
  }
  return FK_OK;
}

size_t fk_shared_prefix_workspace_bytes(int batch, int num_groups, int num_q_heads,
                                        int num_kv_heads, int head_dim, int max_splits) {
  if (batch <= 0 || num_groups < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      max_splits <= 0 || num_q_heads < num_kv_heads || num_q_heads / num_kv_heads > SH_MAX_G)
    return 0;
  return shared_layout(batch, num_groups, num_q_heads, num_kv_heads, max_splits).total;
}

// mode 0: schedule and attention, 1: the schedule only, 2: by the schedule in the workspace
static int shared_impl(int mode, const void* q, int64_t q_stride_token, void* out,
                       int64_t out_stride_token, const void* k_cache, const void* v_cache,
                       int64_t num_pages, int page_size, int64_t kv_page_stride, int kv_layout,
                       const int32_t* context_lens, const int32_t* block_tables,
                       int64_t block_table_stride, int64_t block_table_cols,
                       const int32_t* group_starts, const int32_t* prefix_lens, int num_groups,
                       int batch, int num_q_heads, int num_kv_heads, int head_dim,
                       float softmax_scale, int max_splits, void* workspace,
                       size_t workspace_bytes, int32_t* status, fk_stream_t stream) {
  FK_REQUIRE(batch >= 0 && num_groups >= 0, FK_ERR_INVALID_ARG,
             "fk_shared_prefix_attn: negative size");
  if (batch == 0) return FK_OK;
  RowsParams r{};
  // a schedule has no tensors to check
  const void* const none = workspace;
  int rc = rows_args("fk_shared_prefix_attn", r, mode == 1 ? none : q, q_stride_token,
                     mode == 1 ? workspace : out, out_stride_token, mode == 1 ? none : k_cache,
                     mode == 1 ? none : v_cache, num_pages, page_size, kv_page_stride, kv_layout, context_lens,
                     block_tables, block_table_stride, block_table_cols, num_q_heads, num_kv_heads,
                     head_dim, softmax_scale);
  if (rc != FK_OK) return rc;
  FK_REQUIRE(num_groups == 0 || (group_starts && prefix_lens), FK_ERR_INVALID_ARG,
             "fk_shared_prefix_attn: null pointer");
  FK_REQUIRE(max_splits > 0 && max_splits < (1 << 14), FK_ERR_INVALID_ARG,
             "fk_shared_prefix_attn: %d splits", max_splits);
  FK_REQUIRE(softmax_scale > 0.f, FK_ERR_INVALID_ARG,
             "fk_shared_prefix_attn: softmax_scale must be above zero");
  FK_REQUIRE((int64_t)batch * num_kv_heads * ((r.capacity + ATT_TILE - 1) / ATT_TILE) <
                 (1ll << 31) - (1 << 20),
             FK_ERR_UNSUPPORTED, "fk_shared_prefix_attn: batch and tables too large");
  FK_REQUIRE(batch <= PLAN_MAX_BATCH, FK_ERR_UNSUPPORTED, "fk_shared_prefix_attn: more than %d rows",
             PLAN_MAX_BATCH);
  const SharedLayout w = shared_layout(batch, num_groups, num_q_heads, num_kv_heads,
                                       max_splits);
  FK_REQUIRE(workspace != nullptr && workspace_bytes >= w.total &&
                 (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0,
             FK_ERR_WORKSPACE,
             "fk_shared_prefix_attn: workspace needs %zu bytes, 256-byte aligned (got %zu)",
             w.total, workspace_bytes);
  if (r.capacity > PLAN_MAX_TOKENS) r.capacity = PLAN_MAX_TOKENS;
  const int g = r.g, sms = sm_count(), per_tile = 128 / g;
  // Small calls as fk_paged_decode_attn has them: a CTA per row and KV head, which read the common part
  // from L2, in one launch instead of four that wait for one another (8 rows of 512 common tokens
  // and up to 200 of their own, 32/8 heads: 30.6 -> 9.9 us).
  const bool direct = (int64_t)batch * num_kv_heads <= sms && r.capacity <= SHARED_DIRECT_TOKENS;
  if (direct && mode == 1) return FK_OK;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);

  SharedPlanParams pl{};
  pl.lens = context_lens; pl.starts = group_starts; pl.prefix = prefix_lens;
  pl.batch = batch; pl.groups = num_groups; pl.hkv = num_kv_heads; pl.page = page_size;
  pl.per_tile = per_tile; pl.max_splits = max_splits; pl.ctas = sms;
  pl.min_unit = PREFIX_MIN_UNIT;
  uint32_t sign = 2166136261u;
  for (const int64_t v : {(int64_t)batch, (int64_t)num_groups, (int64_t)num_q_heads,
                          (int64_t)num_kv_heads, (int64_t)page_size, r.capacity,
                          (int64_t)max_splits, (int64_t)sms})
    sign = (sign ^ (uint32_t)v ^ (uint32_t)(v >> 32) * 31u) * 16777619u;
  pl.sign = (int)(sign | 1u);
  pl.beside = pdl_enabled();
  pl.capacity = r.capacity;
  pl.plan.hdr = reinterpret_cast<int*>(ws);
  pl.plan.row_part = reinterpret_cast<int4*>(ws + w.row_part);
  pl.plan.cta_item = reinterpret_cast<int*>(ws + w.cta_item);
  pl.plan.items = reinterpret_cast<PrefixItem*>(ws + w.items);
  pl.plan.chunks = reinterpret_cast<int4*>(ws + w.chunks);
  pl.status = status;

  if (mode != 2 && !direct) {
    static PerDeviceOnce plan_once;
    FK_CUDA_OK(set_max_dynamic_smem(plan_once, shared_plan_kernel, PLAN_MAX_BATCH * 8));
    FK_CUDA_OK(launch_kernel(shared_plan_kernel, dim3(1), dim3(PLAN_THREADS), (size_t)batch * 8, s,
                             pl));
    count_launch(1);
  }
  if (mode == 1) return FK_OK;

  const int sub = page_size < ATT_BOX ? page_size : ATT_BOX;
  const int fused16 = page_size == 16;
  CUtensorMap mq, mk, mv, dk, dv;
  rc = get_q_map(QMapKey{q, q_stride_token, batch, num_q_heads, g, per_tile}, &mq);
  if (rc == FK_OK)
    rc = get_kv_map(k_cache, num_pages, page_size, num_kv_heads, kv_page_stride, kv_layout, sub, 0,
                    &mk);
  if (rc == FK_OK)
    rc = get_kv_map(v_cache, num_pages, page_size, num_kv_heads, kv_page_stride, kv_layout, sub, 0,
                    &mv);
  dk = mk; dv = mv;
  if (rc == FK_OK && fused16) {
    rc = get_kv_map(k_cache, num_pages, page_size, num_kv_heads, kv_page_stride, kv_layout, sub, 1,
                    &dk);
    if (rc == FK_OK)
      rc = get_kv_map(v_cache, num_pages, page_size, num_kv_heads, kv_page_stride, kv_layout, sub,
                      1, &dv);
  }
  if (rc != FK_OK) return rc;

  PrefixParams px{};
  px.sign = pl.sign;
  px.hdr = pl.plan.hdr; px.cta_item = pl.plan.cta_item; px.items = pl.plan.items;
  px.lens = context_lens;
  px.tables = block_tables; px.table_stride = block_table_stride;
  px.hq = num_q_heads; px.hkv = num_kv_heads; px.g = g; px.per_tile = per_tile;
  px.hnd = kv_layout; px.block_size = page_size; px.sub_tokens = sub;
  px.num_blocks = (int)num_pages;
  px.scale_log2 = r.scale_log2;
  px.part_o = reinterpret_cast<float*>(ws + w.pre_o);
  px.part_ml = reinterpret_cast<float2*>(ws + w.pre_ml);
  px.status = status;

  AttnParams a{};
  a.q = r.q; a.q_stride = r.q_stride;
  a.out = r.out; a.out_stride = r.out_stride;
  a.context_lens = context_lens;
  a.block_tables = block_tables; a.bt_stride = block_table_stride;
  a.batch = batch; a.hq = num_q_heads; a.hkv = num_kv_heads; a.g = g;
  a.block_size = page_size; a.num_blocks = (int)num_pages;
  a.sub_tokens = sub;
  a.fused16 = fused16;
  a.hnd = kv_layout;
  a.bs_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  a.scale_log2 = r.scale_log2;
  a.max_splits = max_splits;
  a.plan = pl.plan.hdr; a.sign = pl.sign;
  a.chunk_info = pl.plan.chunks;
  a.part_o = reinterpret_cast<float*>(ws + w.own_o);
  a.part_ml = reinterpret_cast<float2*>(ws + w.own_ml);
  a.status = status;

  if (direct) {
    a.direct = 1; a.sign = 0;
    a.capacity = r.capacity;
    a.starts = group_starts; a.groups = num_groups;
    FK_CUDA_OK(launch_decode(g > 8, false, false, batch * num_kv_heads, dk, dv, a, s));
    count_launch(1);
    return FK_OK;
  }

  SharedJoinParams jn{};
  jn.hdr = pl.plan.hdr; jn.row_part = pl.plan.row_part; jn.sign = pl.sign; jn.status = status;
  jn.counter = pl.plan.hdr + PLAN_COUNTER;
  jn.out = r.out; jn.out_stride = r.out_stride;
  jn.pre_o = px.part_o; jn.pre_ml = px.part_ml;
  jn.own_o = a.part_o; jn.own_ml = a.part_ml; jn.own_splits = max_splits;
  a.beside = num_groups > 0;
  jn.batch = batch; jn.hq = num_q_heads; jn.hkv = num_kv_heads; jn.g = g; jn.per_tile = per_tile;

  if (num_groups > 0) {
    static PerDeviceOnce once;
    FK_CUDA_OK(set_max_dynamic_smem(once, prefix_attn_kernel, PX_SMEM_ALLOC));
    FK_CUDA_OK(launch_kernel(prefix_attn_kernel, dim3((unsigned)sms), dim3(PX_THREADS),
                             (size_t)PX_SMEM_ALLOC, s, mq, mk, mv, px));
    count_launch(1);
  }
  // (weights in one part, as the common part has them)
  FK_CUDA_OK(launch_decode(g > 8, false, false, sms, dk, dv, a, s));
  const int64_t warps = (int64_t)batch * num_q_heads;
  FK_CUDA_OK(launch_kernel(shared_join_kernel, dim3((unsigned)((warps + 7) / 8)), dim3(256),
                           (size_t)0, s, jn));
  count_launch(2);
  return FK_OK;
}

int fk_shared_prefix_attn(int planned, const void* q, int64_t q_stride_token, void* out,
                          int64_t out_stride_token, const void* k_cache, const void* v_cache,
                          int64_t num_pages, int page_size, int64_t kv_page_stride, int kv_layout,
                          const int32_t* context_lens, const int32_t* block_tables,
                          int64_t block_table_stride, int64_t block_table_cols,
                          const int32_t* group_starts, const int32_t* prefix_lens, int num_groups,
                          int batch, int num_q_heads, int num_kv_heads, int head_dim,
                          float softmax_scale, int max_splits, void* workspace,
                          size_t workspace_bytes, int32_t* status, fk_stream_t stream) {
  return shared_impl(planned ? 2 : 0, q, q_stride_token, out, out_stride_token, k_cache, v_cache,
                     num_pages, page_size, kv_page_stride, kv_layout, context_lens, block_tables,
                     block_table_stride, block_table_cols, group_starts, prefix_lens, num_groups,
                     batch, num_q_heads, num_kv_heads, head_dim, softmax_scale, max_splits,
                     workspace, workspace_bytes, status, stream);
}

int fk_shared_prefix_plan(const int32_t* context_lens, int page_size, int64_t block_table_cols,
                          const int32_t* group_starts, const int32_t* prefix_lens, int num_groups,
                          int batch, int num_q_heads, int num_kv_heads, int head_dim,
                          int max_splits, void* workspace, size_t workspace_bytes, int32_t* status,
                          fk_stream_t stream) {
  const int64_t row = (int64_t)num_q_heads * head_dim;
  return shared_impl(1, nullptr, row, nullptr, row, nullptr, nullptr, 1, page_size,
                     (int64_t)page_size * num_kv_heads * head_dim, 0, context_lens, context_lens, 0,
                     block_table_cols, group_starts, prefix_lens, num_groups, batch, num_q_heads,
                     num_kv_heads, head_dim, 1.0f, max_splits, workspace, workspace_bytes, status,
                     stream);
}

}  // extern "C"
