// Tokens leave a paged KV cache: per sequence and KV head the first `first` and the last `last` tokens
// stay, and of those between the ones with the largest sums of softmax weights, `budget` in all.
//
// What attention computes does not depend on the order of its keys, so only as many rows move as have
// to.  With M = budget - last: stayers below M stay where they are; the i-th stayer of [M, n - last)
// goes to the i-th place below M that has become free; the last ones follow, in order, to M ..
// budget - 1.  Sources of the first kind of move lie behind all of its destinations, so these moves
// run side by side; those of the second kind run in ascending tiles, read before written.
//
// One CTA has a sequence and KV head; its warps have a stretch of the tokens each, a lane every
// 32nd.  Keys (weights as integers of the same order) stay in shared memory as far as there is room,
// others are read again.  The border weight is found by counting: the range of keys is cut into
// 2048 parts, the part with the border into 2048 again, so that two or three passes suffice whatever
// their distribution; ties go to the lowest places.  Bound by latency (a chain of loads, passes and
// barriers, 11 us for 1100 tokens, then 1 us for 1024 more) until there are rows enough to move; the
// bytes are 4 a token to decide and each moved row twice.
//
// Where there are fewer pairs than half the SMs a cluster of up to 8 CTAs has one: counts, sums and
// lists go between them by their shared memory, and rows are moved by all.  8 pairs of 12 000 tokens of
// a 4-bit cache cut to 1024 take 20.7 us (one CTA each 22.7), of bf16 21.6; bf16 of 40 000 24.4 (52), of
// 100 000 cut to 4096 36.6 (282).  Barriers and peers' loads cost some 6 us.
#include <type_traits>

#include "fk_q4.cuh"
#include "fk_tcgen05.cuh"

namespace fk {

constexpr int EV_BINS = 2048;
constexpr int EV_LIST = 2048;                // moves of a round
constexpr int EV_ROWS = 4;                   // rows that 16 lanes move at a time
constexpr int EV_RANKS = 8;                  // CTAs of a sequence and head, at most
// Up to so many CTAs each reads the counts of all; of more, each adds up a part and gives it to all.  4-bit
// caches of 12 000 tokens cut to 1024: 3 CTAs (40 pairs) 21.8 us by reading all and 22.8 by parts, 8 CTAs
// (8 pairs) 24.7 and 20.7.
constexpr int EV_GATHER = 4;
// Tokens up to which one CTA of a cluster has them all, and that tables have to hold for clusters, whose
// launch costs 2.5 us more.  8 pairs of a 4-bit cache, one CTA each and 8: 8000 tokens 18.2 us and 19.4,
// 10 000 20.7 and 20.7, 12 000 22.7 and 20.7; under tables that hold 12 800, one CTA of a cluster and all:
// 5000 tokens 17.7 us and 19.2, 6000 18.9 and 19.3, 7000 by all 19.4.
constexpr int EV_ALONE = 6144, EV_CLUSTER = 10240;
// Tokens whose keys a CTA keeps: two CTAs of 512 threads are on an SM, or one of 1024.
__host__ __device__ constexpr int ev_keys(int threads) { return threads == 512 ? 14336 : 43008; }

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
  int keys;                   // of a CTA's tokens kept in shared memory
  int ranks;                  // CTAs of a sequence and head: a cluster
  int32_t* status;
};

// Order of the weights; no number counts as the smallest.
__device__ __forceinline__ uint32_t ev_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);            // -0 is 0
  return u >> 31 ? ~u : u | 0x80000000u;
}

// (page, place in it) of a token; page -1 if its id is bad.
__device__ __forceinline__ int2 ev_place(const EvictParams& p, const int32_t* table, int token) {
  const int i = p.page_shift >= 0 ? token >> p.page_shift : token / p.page;
  const int page = table[i];
  if (page >= 0 && page < p.num_pages) return make_int2(page, token - i * p.page);
  if (p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
  return make_int2(-1, 0);
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
  __device__ __forceinline__ EvRow(const EvictParams& p, int head, int2 place) {
    const int lane = threadIdx.x & 15;
    a = b = nullptr;
    w = nullptr;
    if (place.x < 0) return;
    const int at = place.y;
    if constexpr (Q4) {
      const int ng = p.group_pairs;
      uint8_t* unit = p.k + ((int64_t)(place.x * p.hkv + head) * (p.page / Q4_UNIT) + at / Q4_UNIT) *
                                q4_unit_bytes(ng);
      const int t = at % Q4_UNIT;
      if (lane < 8) a = unit + (lane >> 2) * Q4_VALUES + t * Q4_ROW + (lane & 3) * 16;
      else if (lane < 10) b = unit + Q4_PAIRS + ((lane - 8) * Q4_UNIT + t) * 4 * ng;
      if (lane == 10) w = p.weights + (int64_t)(place.x * p.hkv + head) * p.page + at;
    } else {
      const int64_t off = place.x * p.page_bytes + at * p.token_bytes + head * p.head_bytes + lane * 16;
      a = p.k + off;
      b = p.v + off;
      if (lane == 0) w = p.weights + (int64_t)(place.x * p.hkv + head) * p.page + at;
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

__device__ __forceinline__ uint32_t ev_peer(const void* x, int rank) {
  return cluster_map(smem_u32(x), (uint32_t)rank);
}
// (no memory clobber: loads of several peers are on their way together; barriers have one)
__device__ __forceinline__ int2 ev_peer_load(const int2* x, int rank) {
  int2 v;
  asm volatile("ld.shared::cluster.v2.b32 {%0, %1}, [%2];"
               : "=r"(v.x), "=r"(v.y)
               : "r"(ev_peer(x, rank)));
  return v;
}
__device__ __forceinline__ void ev_peer_store(void* x, int rank, int v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(ev_peer(x, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void ev_peer_store(void* x, int rank, int2 v) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(ev_peer(x, rank)), "r"(v.x),
               "r"(v.y)
               : "memory");
}

// `red` and `red_of` are used in turn, with a barrier in each turn: what one holds is read before it is
// written again.  The same holds for `bins` and, of few CTAs, `sums`.
template <int THREADS, bool CLUSTER>
struct EvShared {
  static constexpr int LIST = CLUSTER ? EV_LIST / 2 : EV_LIST;
  alignas(8) int bins[EV_BINS];                // of this CTA's keys
  alignas(8) int sums[CLUSTER ? EV_BINS : 2];  // of all CTAs', each written by one; of every other pass
  int2 from[LIST], to[LIST];                   // (page, place)
  int2 red[2][THREADS / 32];
  int2 range[THREADS / 32];
  int2 red_of[2][EV_RANKS], range_of[EV_RANKS];            // of each CTA, written by it
  int pick[3];
  int next_turn[2];            // behind the last place of the lists before, and of these
};

template <bool Q4, int THREADS, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) evict_kernel(const EvictParams p) {
  extern __shared__ uint32_t kept[];                       // keys of this CTA's first p.keys tokens
  __shared__ EvShared<THREADS, CLUSTER> sh;
  pdl_launch_dependents();
  pdl_wait();
  const int pair = CLUSTER ? blockIdx.x / p.ranks : blockIdx.x;
  const int rank = CLUSTER ? blockIdx.x - pair * p.ranks : 0;
  const int seq = pair / p.hkv, head = pair - seq * p.hkv;
  const int64_t len = p.lens[seq];
  const int n = len < 0 ? 0 : len > p.capacity ? (int)p.capacity : (int)len;
  if (head == 0 && rank == 0 && threadIdx.x == 0) {
    p.new_lens[seq] = min(n, p.budget);
    if (len > p.capacity && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
  }
  const int ranks = CLUSTER && n > EV_ALONE ? p.ranks : 1;
  if (n <= p.budget || rank >= ranks) return;
  if (CLUSTER && ranks > 1) {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  const int32_t* table = p.tables + (int64_t)seq * p.table_stride;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int WARPS = THREADS / 32;
  static_assert(!CLUSTER || WARPS == 32, "a lane reads a warp's entry of each CTA");
  const int M = p.budget - p.last, end = n - p.last;       // candidates: first .. end - 1
  const int stretch = ((end + ranks * WARPS - 1) / (ranks * WARPS) + 31) & ~31;
  const int base = rank * WARPS * stretch;
  const int w0 = min(base + warp * stretch, end), w1 = min(w0 + stretch, end);
  auto sync = [&] {
    if (CLUSTER && ranks > 1) {
      __syncwarp();
      cluster_barrier_sync();
    } else {
      __syncthreads();
    }
  };
  // Sums, over the pair's (or only `here` this CTA's) warps before this one, of two numbers that a
  // warp's lanes agree on, and the totals.
  int turn = 0;
  auto before_me = [&](int a, int b, int2* all, bool here) {
    turn ^= 1;
    if (lane == 0) sh.red[turn][warp] = make_int2(a, b);
    __syncthreads();
    int2 v = lane < WARPS ? sh.red[turn][lane] : make_int2(0, 0);
    auto add = [&](bool which) {
      return make_int2(__reduce_add_sync(0xffffffffu, which ? v.x : 0),
                       __reduce_add_sync(0xffffffffu, which ? v.y : 0));
    };
    int2 before = add(lane < warp);
    *all = add(true);
    if (CLUSTER && !here && ranks > 1) {
      if (warp == 0 && lane < ranks) ev_peer_store(&sh.red_of[turn][rank], lane, *all);
      sync();
      v = lane < ranks ? sh.red_of[turn][lane] : make_int2(0, 0);
      const int2 more = add(lane < rank);
      before = make_int2(before.x + more.x, before.y + more.y);
      *all = add(true);
    }
    return before;
  };
  const float* weights = p.weights + (int64_t)head * p.page;
  auto read_key = [&](int t) -> uint32_t {
    if (t < p.first || t >= w1) return 0u;
    const int i = p.page_shift >= 0 ? t >> p.page_shift : t / p.page;
    const int page = table[i];
    if (page < 0 || page >= p.num_pages) {
      if (p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
      return 0u;
    }
    return ev_key(weights[(int64_t)page * p.hkv * p.page + (t - i * p.page)]);
  };
  // every 32 tokens of the stretch, with this lane's token and key
  auto each_read = [&](auto f) {
#pragma unroll 4
    for (int i = w0; i < w1; i += 32) f(i + lane, read_key(i + lane));
  };
  auto each = [&](auto f) {
    const int w = min(w1, max(w0, base + p.keys));
#pragma unroll 4
    for (int i = w0; i < w; i += 32) f(i + lane, kept[i - base + lane]);
#pragma unroll 1
    for (int i = w; i < w1; i += 32) f(i + lane, read_key(i + lane));
  };

  // ---- the range of the candidates' keys ----
  uint32_t lo = ~0u, hi = 0u;
#pragma unroll 8
  for (int i = w0; i < w1; i += 32) {
    const int t = i + lane;
    const uint32_t k = read_key(t);
    if (i + 32 <= base + p.keys) kept[t - base] = k;
    if (t < p.first || t >= w1) continue;
    lo = min(lo, k);
    hi = max(hi, k);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) sh.range[warp] = make_int2((int)lo, (int)hi);
  for (int i = threadIdx.x; i < EV_BINS; i += THREADS) sh.bins[i] = 0;
  __syncthreads();
  auto widest = [&](int2 v) {
    lo = __reduce_min_sync(0xffffffffu, (uint32_t)v.x);
    hi = __reduce_max_sync(0xffffffffu, (uint32_t)v.y);
  };
  widest(lane < WARPS ? sh.range[lane] : make_int2(-1, 0));
  if (CLUSTER && ranks > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // all have begun
    if (warp == 0 && lane < ranks) ev_peer_store(&sh.range_of[rank], lane, make_int2((int)lo, (int)hi));
    sync();
    widest(lane < ranks ? sh.range_of[lane] : make_int2(-1, 0));
  }

  // ---- the border: `want` of the keys at it stay, all above, none below ----
  int want = M - p.first;
  uint32_t border = hi;
  bool whole = false;            // all at the border and above stay
  if (want > 0) {
    for (int pass = 0; pass < 3; ++pass) {                 // 32 bits in parts of 11
      const int bits = 32 - __clz(hi - lo);                // 0 when all are one key
      const int shift = bits > 11 ? bits - 11 : 0;
      const bool gather = CLUSTER && ranks <= EV_GATHER;
      int* bins = gather && (pass & 1) ? sh.sums : sh.bins;
      if (pass > 0) {
        for (int i = threadIdx.x; i < EV_BINS; i += THREADS) bins[i] = 0;
        __syncthreads();
      }
      each([&](int t, uint32_t k) {
        if (t >= p.first && t < w1 && k >= lo && k <= hi) atomicAdd(&bins[(k - lo) >> shift], 1);
      });
      sync();
      // from the top: the bin in which the sum reaches `want`
      constexpr int PER = EV_BINS / THREADS;
      int mine[PER], sum = 0;
      const int at = EV_BINS - (threadIdx.x + 1) * PER;
      if constexpr (CLUSTER) {
        // of few CTAs each adds up all bins, two a thread; of more a part that it gives to all
        const int part = gather ? THREADS : (EV_BINS / 2 + ranks - 1) / ranks;
        const int q = gather ? at / 2 : rank * part + threadIdx.x;
        int2 v[EV_RANKS];
        if (threadIdx.x < part && q < EV_BINS / 2) {
#pragma unroll
          for (int r = 0; r < EV_RANKS; ++r)
            v[r] = r < ranks && ranks > 1
                       ? ev_peer_load(reinterpret_cast<const int2*>(bins) + q, r)
                       : make_int2(0, 0);
          if (ranks == 1) v[0] = reinterpret_cast<const int2*>(bins)[q];
#pragma unroll
          for (int r = 1; r < EV_RANKS; ++r) {
            v[0].x += v[r].x;
            v[0].y += v[r].y;
          }
          if (!gather)
            for (int r = 0; r < ranks; ++r)
              ev_peer_store(reinterpret_cast<int2*>(sh.sums) + q, r, v[0]);
        }
        if (!gather) {
          sync();
          v[0] = *reinterpret_cast<const int2*>(&sh.sums[at]);
        }
        static_assert(!CLUSTER || PER == 2, "two bins a thread");
        mine[0] = v[0].y;
        mine[1] = v[0].x;
        sum = v[0].x + v[0].y;
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += mine[i] = bins[at + PER - 1 - i];
      }
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      int2 all;
      int above = before_me(__shfl_sync(0xffffffffu, incl, 31), 0, &all, true).x + incl - sum;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (above < want && above + mine[i] >= want) {
          sh.pick[0] = EV_BINS - 1 - (threadIdx.x * PER + i);
          sh.pick[1] = want - above;
          sh.pick[2] = mine[i];
        }
        above += mine[i];
      }
      __syncthreads();
      want = sh.pick[1];
      border = lo + ((uint32_t)sh.pick[0] << shift);
      whole = sh.pick[2] == want;
      if (shift == 0 || whole) break;
      lo = border;
      const uint32_t top = border + ((1u << shift) - 1u);
      hi = top < hi && top >= border ? top : hi;
    }
  }

  // ---- of the keys at the border those of the first `want` places stay, those below `cut` ----
  int cut = whole ? 0x7fffffff : 0;
  int2 all;
  if (!whole && want > 0) {
    int here = 0;
    each([&](int t, uint32_t k) {
      here += __popc(__ballot_sync(0xffffffffu, t >= p.first && t < w1 && k == border));
    });
    int before = before_me(here, 0, &all, false).x;
    if (before < want && before + here >= want) {
      each([&](int t, uint32_t k) {
        const uint32_t at = __ballot_sync(0xffffffffu, t >= p.first && t < w1 && k == border);
        if ((at >> lane & 1u) && before + __popc(at & ((1u << lane) - 1u)) == want - 1)
          for (int r = 0; r < ranks; ++r) {
            if (CLUSTER) ev_peer_store(&sh.pick[0], r, t + 1);
            else sh.pick[0] = t + 1;
          }
        before += __popc(at);
      });
    }
    sync();
    cut = sh.pick[0];
  }
  auto stays = [&](int t, uint32_t k) {
    return t < p.first || k > border || (k == border && t < cut);
  };
  // Places whose turn has been are not looked at again: a moved token's weight is there now, or, where a
  // page id is bad, the old one.
  auto freed = [&](int t, uint32_t k, auto later) {
    bool turn = t < min(w1, M) && !stays(t, k);
    if constexpr (later) turn = turn && t >= sh.next_turn[0];
    return __ballot_sync(0xffffffffu, turn);
  };
  auto moved = [&](int t, uint32_t k) {
    return __ballot_sync(0xffffffffu, t < w1 && t >= M && stays(t, k));
  };

  // ---- moves, in order: lists of them, a CTA every ranks-th tile, then the rows ----
  const int half = threadIdx.x >> 4;
  constexpr int TILE = THREADS / 16 * EV_ROWS;
  const int2 none = make_int2(-1, 0);
  const int most = EvShared<THREADS, CLUSTER>::LIST * ranks;
  auto list = [&](int2* at, int i, int t) {
    const int2 place = ev_place(p, table, t);
    if (CLUSTER && ranks > 1) {
      const int tile = i / TILE, turns = tile / ranks;
      ev_peer_store(&at[turns * TILE + i % TILE], tile - turns * ranks, place);
    } else {
      at[i] = place;
    }
  };
  auto round = [&](int done, auto over, auto later) {
    int2 here = make_int2(0, 0);
    over([&](int t, uint32_t k) {
      here.x += __popc(freed(t, k, later));
      here.y += __popc(moved(t, k));
    });
    here = before_me(here.x, here.y, &all, false);
    here.y -= done;
    over([&](int t, uint32_t k) {
      const uint32_t fr = freed(t, k, later), mv = moved(t, k), below = (1u << lane) - 1u;
      const int fi = here.x + __popc(fr & below), mi = here.y + __popc(mv & below);
      if ((fr >> lane & 1u) && fi < most) {
        list(sh.to, fi, t);
        if (fi == most - 1)
          for (int r = 0; r < ranks; ++r) {
            if (CLUSTER) ev_peer_store(&sh.next_turn[1], r, t + 1);
            else sh.next_turn[1] = t + 1;
          }
      }
      if ((mv >> lane & 1u) && mi >= 0 && mi < most) list(sh.from, mi, t);
      here.x += __popc(fr);
      here.y += __popc(mv);
    });
    sync();                                  // all have decided, and their lists are here
    const int count = min(most, min(all.x, all.y - done));
    for (int mine = 0, j0 = rank * TILE; j0 < count; mine += TILE, j0 += TILE * ranks) {
      EvPiece x[EV_ROWS];
#pragma unroll
      for (int u = 0; u < EV_ROWS; ++u) {
        const int j = u * (THREADS / 16) + half;
        EvRow<Q4>(p, head, j0 + j < count ? sh.from[mine + j] : none).load(p, x[u]);
      }
#pragma unroll
      for (int u = 0; u < EV_ROWS; ++u) {
        const int j = u * (THREADS / 16) + half;
        const bool moves = j0 + j < count && sh.from[mine + j].x >= 0;
        EvRow<Q4>(p, head, moves ? sh.to[mine + j] : none).store(p, x[u]);
      }
    }
    sync();
    return all.y;
  };
  const int moves = round(0, each, std::false_type{});
  for (int done = most; done < moves; done += most) {
    if (threadIdx.x == 0) sh.next_turn[0] = sh.next_turn[1];
    __syncthreads();
    round(done, each_read, std::true_type{});
  }
  // ---- the newest ----
  const bool apart = n - p.budget >= p.last;               // places and sources are
  if (!apart && rank > 0) return;
  const int by = apart ? TILE * ranks : TILE;
  for (int j0 = rank * TILE; j0 < p.last; j0 += by) {
    EvPiece x[EV_ROWS];
    int2 from[EV_ROWS], to[EV_ROWS];
#pragma unroll
    for (int u = 0; u < EV_ROWS; ++u) {
      const int j = j0 + u * (THREADS / 16) + half;
      from[u] = j < p.last ? ev_place(p, table, end + j) : none;
      to[u] = from[u].x >= 0 ? ev_place(p, table, M + j) : none;
    }
#pragma unroll
    for (int u = 0; u < EV_ROWS; ++u) EvRow<Q4>(p, head, from[u]).load(p, x[u]);
    if (!apart) __syncthreads();
#pragma unroll
    for (int u = 0; u < EV_ROWS; ++u) EvRow<Q4>(p, head, to[u]).store(p, x[u]);
  }
}

template <bool Q4, int THREADS, bool CLUSTER>
static cudaError_t ev_launch(EvictParams p, int64_t pairs, cudaStream_t s) {
  static PerDeviceOnce once;
  auto kernel = evict_kernel<Q4, THREADS, CLUSTER>;
  const cudaError_t e = set_max_dynamic_smem(once, kernel, ev_keys(THREADS) * 4);
  if (e != cudaSuccess) return e;
  // what a CTA can have of the tables' tokens: its warps' stretches are whole rounds of 32
  const int64_t alone = p.capacity < EV_ALONE ? p.capacity : EV_ALONE, part = p.capacity / p.ranks;
  const int64_t most = (part > alone ? part : alone) + THREADS;
  p.keys = (int)(most < ev_keys(THREADS) ? most & ~31 : ev_keys(THREADS));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(pairs * p.ranks));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = (size_t)p.keys * 4;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (CLUSTER) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)p.ranks;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}
template <bool Q4>
static cudaError_t ev_launch(const EvictParams& p, int64_t pairs, cudaStream_t s) {
  if (p.ranks > 1) return ev_launch<Q4, 1024, true>(p, pairs, s);
  return pairs <= sm_count() ? ev_launch<Q4, 1024, false>(p, pairs, s)
                             : ev_launch<Q4, 512, false>(p, pairs, s);
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
  FK_REQUIRE(lens + num_seqs <= new_lens || new_lens + num_seqs <= lens, FK_ERR_INVALID_ARG,
             "%s: the new lengths need a place of their own", what);
  FK_REQUIRE(table_cols > 0 && table_stride >= 0, FK_ERR_INVALID_ARG, "%s: bad sizes", what);
  FK_REQUIRE((int64_t)num_seqs * hkv < (1ll << 31), FK_ERR_UNSUPPORTED, "%s: too many sequences",
             what);
  FK_REQUIRE(num_pages * hkv < (1ll << 31), FK_ERR_UNSUPPORTED, "%s: pool too large", what);
  p.weights = weights; p.lens = lens; p.new_lens = new_lens;
  p.tables = tables; p.table_stride = table_stride;
  const int64_t longest = 1ll << 30;
  p.capacity = table_cols < longest / page ? table_cols * page : longest;
  p.num_pages = (int)num_pages; p.page = page; p.hkv = hkv;
  p.page_shift = (page & (page - 1)) == 0 ? __builtin_ctz(page) : -1;
  p.budget = budget; p.first = first; p.last = last;
  p.status = status;
  const int64_t pairs = (int64_t)num_seqs * hkv;
  // (clusters find room where an eighth of the SMs may stay empty)
  const int64_t ranks = sm_count() * 7 / 8 / pairs;
  p.ranks = p.capacity <= EV_CLUSTER || ranks < 2 ? 1 : (int)(ranks < EV_RANKS ? ranks : EV_RANKS);
  FK_CUDA_OK(q4 ? ev_launch<true>(p, pairs, s) : ev_launch<false>(p, pairs, s));
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
