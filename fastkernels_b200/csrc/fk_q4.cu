// Tokens into a paged KV cache of 4 bits a value, and back.
//
// Of each row's groups of G channels (64 or 128), in real numbers but where a rounding is named:
//   lo = min x,  hi = max x,  s = bf16(fp32(hi / 2 - lo / 2) / 7.5)
//   c  = min(15, nearest integer of (x - lo) / s, the even one of two), 0 where s = 0
//   x' = lo + s c
// lo is one of the bf16 inputs, so that it is kept exactly; the halves keep the difference of the
// largest values finite.  A group with a value that is no finite number has no scale either (NaN),
// and reads back as NaN.
//
// Both kernels move 512 B of bf16 per token and head against 136 to 144 B packed.  16 lanes have a
// row, a 16-byte load and one word of codes each; CTAs have 16 tokens of some heads, as a unit has.
// Loading is near its bytes; storing is bound by its instructions (some 180 for 32 lanes' words, 0.68
// of the issue slots): smallest and largest value, quotients two at a time, and for the third of
// the warps that meet an exact half its side.  5 prompts of 16 309 tokens, 8 heads: stored and loaded
// again in 46 us, 3.7 TB/s.
#include "fk_q4.cuh"

namespace fk {

struct Q4MoveParams {
  const uint4* k; int64_t k_stride;       // 16-byte pieces of a token
  const uint4* v; int64_t v_stride;
  uint4* k_out; uint4* v_out;
  uint8_t* pool;
  const void* slots; int slots64;
  int64_t rows, num_slots;
  int hkv, page, page_shift;
  int32_t* status;
};

__device__ __forceinline__ uint32_t max_nan2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t min_nan2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Unit of a slot's token for a head, and the token's place in it; null where there is none.
__device__ __forceinline__ uint8_t* q4_unit(const Q4MoveParams& p, int64_t row, int head,
                                            int unit_bytes, int* token) {
  const int64_t slot = p.slots64 ? static_cast<const int64_t*>(p.slots)[row]
                                 : static_cast<const int32_t*>(p.slots)[row];
  if (slot < 0) return nullptr;
  if (slot >= p.num_slots) {
    if (p.status) atomicOr(p.status, FK_DEV_BAD_SLOT);
    return nullptr;
  }
  const int64_t page = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page;
  const int at = (int)(slot - page * p.page);
  *token = at % Q4_UNIT;
  return p.pool + ((page * p.hkv + head) * (p.page / Q4_UNIT) + at / Q4_UNIT) * unit_bytes;
}

// The code of x in a group whose step is near the ends of fp32's range, where 1 / s or x - lo may
// not be a number: from halves, by division.  Only such groups come here.
__device__ __noinline__ uint32_t q4_code_far(float x, float lo, float s) {
  const float h = s * 0.5f, d = fmaf(x, 0.5f, -lo * 0.5f);
  const float y = fminf(d / h, 15.f), k = floorf(y);
  const float back = d - x * 0.5f;                   // two-sum: x / 2 - lo / 2 = d + e
  const float e = (x * 0.5f - (d - back)) + (-lo * 0.5f - back);
  // (near a half the products and differences are exact)
  const float over = fabsf(y - k - 0.5f) < 0.000244140625f ? (d - (k + 0.5f) * h) + e : y - k - 0.5f;
  return (uint32_t)k + (over > 0.f || (over == 0.f && ((int)k & 1)));
}

// One row: the lane's 8 channels into a word, with the pair of its group.
template <int NG>
__device__ __forceinline__ uint32_t q4_pack(const uint4& x, uint32_t* pair) {
  uint32_t hi2 = max_nan2(max_nan2(x.x, x.y), max_nan2(x.z, x.w));
  uint32_t lo2 = min_nan2(min_nan2(x.x, x.y), min_nan2(x.z, x.w));
#pragma unroll
  for (int o = 1; o < 16 / NG; o <<= 1) {
    hi2 = max_nan2(hi2, __shfl_xor_sync(0xffffffffu, hi2, o));
    lo2 = min_nan2(lo2, __shfl_xor_sync(0xffffffffu, lo2, o));
  }
  hi2 = max_nan2(hi2, hi2 >> 16 | hi2 << 16);
  lo2 = min_nan2(lo2, lo2 >> 16 | lo2 << 16);
  const float hi = bf16lo(hi2), lo = bf16lo(lo2);
  const float s = round_bf16((hi * 0.5f - lo * 0.5f) / 7.5f);
  if (!(s < INFINITY)) {                             // a number that is not finite, or none
    *pair = 0x7fc07fc0u;
    return 0u;
  }
  *pair = (__float_as_uint(s) >> 16) | (__float_as_uint(lo) & 0xffff0000u);
  if (s == 0.f) return 0u;
  // The plain way, where 1 / s is a number and x - lo too, two channels at a time: three roundings
  // and the reciprocal's put the quotient less than 2^-18 off, so that one that is 2^-17 from a
  // half is on the right side of it.
  constexpr float kWhole = 8388608.f;                // its sum with a code is a whole number
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  const float inv = rcp_approx(s);
  const uint64_t inv2 = pair_of(inv, inv), low2 = pair_of(-lo, -lo);
  const uint64_t up = pair_of(kWhole, kWhole), down = pair_of(-kWhole, -kWhole);
  const uint64_t one = pair_of(-1.f, -1.f);
  float far = s > 1e-30f && s < 1e30f ? 0.f : 1.f;   // largest distance from a code
  float2 r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t d = add2(pair_of(bf16lo(w[i]), bf16hi(w[i])), low2);
    const uint64_t c = add2(fma2(d, inv2, up), down);          // to nearest, even on ties
    const float2 e = both_of(fma2(d, inv2, fma2(c, one, 0ull)));
    far = fmaxf(far, fmaxf(fabsf(e.x), fabsf(e.y)));
    r[i] = both_of(c);
  }
  // 16 bits of four codes, a number that fp32 holds
  const float half0 = fmaf(r[1].y, 4096.f, fmaf(r[1].x, 256.f, fmaf(r[0].y, 16.f, r[0].x)));
  const float half1 = fmaf(r[3].y, 4096.f, fmaf(r[3].x, 256.f, fmaf(r[2].y, 16.f, r[2].x)));
  uint32_t word = __byte_perm(__float_as_uint(half0 + kWhole), __float_as_uint(half1 + kWhole), 0x5410);
  if (far >= 0.5f - 7.62939453125e-06f) {
    // Closer: what is left of x - lo = d + e (two-sum) beyond code c is exact, and compared with
    // s / 2.  Halves are frequent: keys and values are bf16, as is s.
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = i & 1 ? bf16hi(w[i >> 1]) : bf16lo(w[i >> 1]);
      if (far == 1.f) {
        word = (word & ~(15u << (4 * i))) | q4_code_far(v, lo, s) << (4 * i);
        continue;
      }
      const float c = i & 1 ? r[i >> 1].y : r[i >> 1].x;
      const float d = v - lo, left = fmaf(-c, s, d), over = fabsf(left) - 0.5f * s;
      if (over < s * -7.62939453125e-06f) continue;
      const float back = d - v, e = (v - (d - back)) + (-lo - back);
      const float more = over + (left > 0.f ? e : -e);
      if (more > 0.f || (more == 0.f && ((word >> (4 * i)) & 1u)))
        word += left > 0.f ? 1u << (4 * i) : ~0u << (4 * i);
    }
  }
  return word;
}

__device__ __forceinline__ uint4 q4_unpack(uint32_t word, uint32_t pair) {
  const float s = bf16lo(pair), lo = bf16hi(pair);
  const uint64_t s2 = pair_of(s, s), lo2 = pair_of(lo, lo), down = pair_of(-8388608.f, -8388608.f);
  const uint32_t even = word & 0x0f0f0f0fu, odd = word >> 4 & 0x0f0f0f0fu;
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // 2^23 + code
    const float a = __uint_as_float(__byte_perm(even, 0x4b000000u, 0x7440 + i));
    const float b = __uint_as_float(__byte_perm(odd, 0x4b000000u, 0x7440 + i));
    const float2 v = both_of(fma2(s2, add2(pair_of(a, b), down), lo2));
    out[i] = pack_bf16(v.x, v.y);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

constexpr int Q4_MOVE_THREADS = 256;
constexpr int Q4_MOVE_HEADS = 2;             // heads of a lane's token, key and value each

// A CTA takes Q4_MOVE_HEADS heads of 16 tokens, so that successive tokens fill a unit from one place.
struct Q4Place {
  int64_t row;
  int head, heads;             // the first of so many; none: no row
  uint8_t* unit;               // of the first head; null: no slot
  int64_t next;                // bytes to the next head's
  int token;
  __device__ __forceinline__ Q4Place(const Q4MoveParams& p, int unit_bytes) {
    const int groups = (p.hkv + Q4_MOVE_HEADS - 1) / Q4_MOVE_HEADS;
    const int tile = blockIdx.x / groups;
    row = (int64_t)tile * 16 + (threadIdx.x >> 4);
    head = (int)(blockIdx.x - tile * groups) * Q4_MOVE_HEADS;
    heads = row < p.rows ? min(Q4_MOVE_HEADS, p.hkv - head) : 0;
    next = (int64_t)(p.page / Q4_UNIT) * unit_bytes;
    unit = heads > 0 ? q4_unit(p, row, head, unit_bytes, &token) : nullptr;
  }
};

template <int NG>
__global__ void __launch_bounds__(Q4_MOVE_THREADS) q4_store_kernel(const Q4MoveParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 15;
  const Q4Place at(p, q4_unit_bytes(NG));
  uint4 x[Q4_MOVE_HEADS][2];
#pragma unroll
  for (int u = 0; u < Q4_MOVE_HEADS; ++u) {
    x[u][0] = x[u][1] = make_uint4(0u, 0u, 0u, 0u);
    if (u < at.heads) {
      x[u][0] = p.k[at.row * p.k_stride + (at.head + u) * 16 + lane];
      x[u][1] = p.v[at.row * p.v_stride + (at.head + u) * 16 + lane];
    }
  }
#pragma unroll
  for (int u = 0; u < Q4_MOVE_HEADS; ++u)
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint32_t pair;
      const uint32_t word = q4_pack<NG>(x[u][kv], &pair);
      if (!at.unit || u >= at.heads) continue;
      uint8_t* unit = at.unit + u * at.next;
      const int place = kv ? q4_value_place(lane) : q4_key_place(lane);
      reinterpret_cast<uint32_t*>(unit + kv * Q4_VALUES + at.token * Q4_ROW)[place] = word;
      if (lane % (16 / NG) == 0)
        reinterpret_cast<uint32_t*>(unit + Q4_PAIRS)[(kv * Q4_UNIT + at.token) * NG +
                                                     lane / (16 / NG)] = pair;
    }
}

template <int NG>
__global__ void __launch_bounds__(Q4_MOVE_THREADS) q4_load_kernel(const Q4MoveParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 15;
  const Q4Place at(p, q4_unit_bytes(NG));
  uint32_t word[Q4_MOVE_HEADS][2], pair[Q4_MOVE_HEADS][2];
#pragma unroll
  for (int u = 0; u < Q4_MOVE_HEADS; ++u)
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      word[u][kv] = pair[u][kv] = 0u;
      if (!at.unit || u >= at.heads) continue;
      const uint8_t* unit = at.unit + u * at.next;
      const int place = kv ? q4_value_place(lane) : q4_key_place(lane);
      word[u][kv] = reinterpret_cast<const uint32_t*>(unit + kv * Q4_VALUES +
                                                      at.token * Q4_ROW)[place];
      pair[u][kv] = reinterpret_cast<const uint32_t*>(
          unit + Q4_PAIRS)[(kv * Q4_UNIT + at.token) * NG + lane / (16 / NG)];
    }
#pragma unroll
  for (int u = 0; u < Q4_MOVE_HEADS; ++u) {
    if (u >= at.heads) break;
    const int64_t i = at.row * p.hkv + at.head + u;
    p.k_out[i * 16 + lane] = q4_unpack(word[u][0], pair[u][0]);
    p.v_out[i * 16 + lane] = q4_unpack(word[u][1], pair[u][1]);
  }
}

static int q4_move(const char* what, bool store, const void* k, int64_t k_stride, const void* v,
                   int64_t v_stride, void* k_out, void* v_out, void* cache, int64_t num_pages,
                   int page, int hkv, int head_dim, int group, const void* slots, int slots64,
                   int64_t rows, int32_t* status, cudaStream_t s) {
  FK_REQUIRE(rows >= 0, FK_ERR_INVALID_ARG, "%s: negative size", what);
  const int rc = q4_check_pool(what, cache, num_pages, page, hkv, head_dim, group);
  if (rc != FK_OK) return rc;
  if (rows == 0) return FK_OK;
  FK_REQUIRE(slots && (store ? k && v : k_out && v_out), FK_ERR_INVALID_ARG, "%s: null pointer",
             what);
  FK_REQUIRE(slots64 == 0 || slots64 == 1, FK_ERR_INVALID_ARG, "%s: slots of 32 or 64 bits", what);
  FK_REQUIRE(!store || (k_stride >= (int64_t)hkv * head_dim && v_stride >= (int64_t)hkv * head_dim),
             FK_ERR_INVALID_ARG, "%s: token stride too small", what);
  FK_REQUIRE(store ? aligned16(k) && aligned16(v) && k_stride % 8 == 0 && v_stride % 8 == 0
                   : aligned16(k_out) && aligned16(v_out),
             FK_ERR_ALIGNMENT, "%s: 16-byte alignment required", what);
  const int64_t blocks = (rows + 15) / 16 * ((hkv + Q4_MOVE_HEADS - 1) / Q4_MOVE_HEADS);
  FK_REQUIRE(rows < (1ll << 31) && blocks < (1ll << 31), FK_ERR_UNSUPPORTED, "%s: too many tokens",
             what);
  Q4MoveParams p{};
  p.k = static_cast<const uint4*>(k); p.k_stride = k_stride / 8;
  p.v = static_cast<const uint4*>(v); p.v_stride = v_stride / 8;
  p.k_out = static_cast<uint4*>(k_out); p.v_out = static_cast<uint4*>(v_out);
  p.pool = static_cast<uint8_t*>(cache);
  p.slots = slots; p.slots64 = slots64;
  p.rows = rows; p.num_slots = num_pages * page;
  p.hkv = hkv; p.page = page;
  p.page_shift = (page & (page - 1)) == 0 ? __builtin_ctz(page) : -1;
  p.status = status;
  const dim3 grid((unsigned)blocks);
  auto kernel = store ? group == 64 ? q4_store_kernel<2> : q4_store_kernel<1>
                      : group == 64 ? q4_load_kernel<2> : q4_load_kernel<1>;
  FK_CUDA_OK(launch_kernel(kernel, grid, dim3(Q4_MOVE_THREADS), (size_t)0, s, p));
  count_launch(1);
  return FK_OK;
}

}  // namespace fk

using namespace fk;

extern "C" {

int64_t fk_q4_unit_bytes(int head_dim, int group) {
  if (head_dim != Q4_D || (group != 64 && group != 128)) return 0;
  return q4_unit_bytes(Q4_D / group);
}

int fk_store_kvcache_q4(const void* k, int64_t k_stride_token, const void* v,
                        int64_t v_stride_token, void* cache, int64_t num_pages, int page_size,
                        int num_kv_heads, int head_dim, int group, const void* slot_mapping,
                        int slots_are_int64, int64_t num_tokens, int32_t* status,
                        fk_stream_t stream) {
  return q4_move("fk_store_kvcache_q4", true, k, k_stride_token, v, v_stride_token, nullptr,
                 nullptr, cache, num_pages, page_size, num_kv_heads, head_dim, group, slot_mapping,
                 slots_are_int64, num_tokens, status, static_cast<cudaStream_t>(stream));
}

int fk_load_kvcache_q4(void* k, void* v, const void* cache, int64_t num_pages, int page_size,
                       int num_kv_heads, int head_dim, int group, const void* slot_mapping,
                       int slots_are_int64, int64_t num_tokens, int32_t* status,
                       fk_stream_t stream) {
  return q4_move("fk_load_kvcache_q4", false, nullptr, 0, nullptr, 0, k, v,
                 const_cast<void*>(cache), num_pages, page_size, num_kv_heads, head_dim, group,
                 slot_mapping, slots_are_int64, num_tokens, status,
                 static_cast<cudaStream_t>(stream));
}

}  // extern "C"
