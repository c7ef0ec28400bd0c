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
// Both kernels are bound by memory: 512 B of bf16 per token and head against 136 to 144 B packed.
// 16 lanes have a row, a 16-byte load and one word of codes each.
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

// Nearest integer of (x - lo) / s to 15, exactly, from halves of lo and s (exact, and no difference
// of finite values overflows).  The quotient's own error (three roundings, below 2^-18 of 16) is
// far below 2^-12, so a quotient that is not that close to a half is on the right side of it; others
// are compared with (k + 1/2) s, which fp32 holds exactly, as is the difference of two numbers that
// close, and the rounding of x - lo is made up for.
__device__ __forceinline__ uint32_t q4_code(float x, float lo_half, float s_half, float inv,
                                            bool tiny) {
  const float d = fmaf(x, 0.5f, -lo_half);
  const float y = fminf(tiny ? d / s_half : d * inv, 15.f);
  const float k = floorf(y);
  if (fabsf(y - k - 0.5f) < 0.000244140625f) {
    const float x_half = x * 0.5f;
    const float back = d - x_half;                   // two-sum: x / 2 - lo / 2 = d + e
    const float e = (x_half - (d - back)) + (-lo_half - back);
    const float over = (d - (k + 0.5f) * s_half) + e;
    const int ki = (int)k;
    return (uint32_t)(over > 0.f || (over == 0.f && (ki & 1)) ? ki + 1 : ki);
  }
  return __float_as_uint(y + 8388608.f) & 15u;       // to nearest
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
  const bool tiny = s < 1e-30f;                      // 1 / s might not be finite
  const float lo_half = lo * 0.5f, s_half = s * 0.5f;
  const float inv = tiny ? 0.f : 1.0f / s_half;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t word = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    word |= q4_code(bf16lo(w[i]), lo_half, s_half, inv, tiny) << (8 * i);
    word |= q4_code(bf16hi(w[i]), lo_half, s_half, inv, tiny) << (8 * i + 4);
  }
  return word;
}

template <int NG>
__device__ __forceinline__ uint4 q4_unpack(uint32_t word, uint32_t pair) {
  const float s = bf16lo(pair), lo = bf16hi(pair);
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    out[i] = pack_bf16(fmaf(s, (float)(word >> (8 * i) & 15u), lo),
                       fmaf(s, (float)(word >> (8 * i + 4) & 15u), lo));
  return make_uint4(out[0], out[1], out[2], out[3]);
}

constexpr int Q4_MOVE_THREADS = 256;
constexpr int Q4_MOVE_HEADS = 2;             // (token, head) pairs of a lane, key and value each

template <int NG>
__global__ void __launch_bounds__(Q4_MOVE_THREADS) q4_store_kernel(const Q4MoveParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 15;
  const int64_t total = p.rows * p.hkv;
  const int64_t first = (int64_t)blockIdx.x * (Q4_MOVE_THREADS / 16) * Q4_MOVE_HEADS +
                        (threadIdx.x >> 4);
  uint4 x[Q4_MOVE_HEADS][2];
  uint8_t* unit[Q4_MOVE_HEADS];
  int token[Q4_MOVE_HEADS];
#pragma unroll
  for (int u = 0; u < Q4_MOVE_HEADS; ++u) {
    const int64_t i = first + u * (Q4_MOVE_THREADS / 16);
    unit[u] = nullptr;
    x[u][0] = x[u][1] = make_uint4(0u, 0u, 0u, 0u);
    if (i < total) {
      const int64_t row = i / p.hkv;
      const int head = (int)(i - row * p.hkv);
      x[u][0] = p.k[row * p.k_stride + head * 16 + lane];
      x[u][1] = p.v[row * p.v_stride + head * 16 + lane];
      unit[u] = q4_unit(p, row, head, q4_unit_bytes(NG), &token[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < Q4_MOVE_HEADS; ++u)
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint32_t pair;
      const uint32_t word = q4_pack<NG>(x[u][kv], &pair);
      if (!unit[u]) continue;
      const int place = kv ? q4_value_place(lane) : q4_key_place(lane);
      reinterpret_cast<uint32_t*>(unit[u] + kv * Q4_VALUES + token[u] * Q4_ROW)[place] = word;
      if (lane % (16 / NG) == 0)
        reinterpret_cast<uint32_t*>(unit[u] + Q4_PAIRS)[(kv * Q4_UNIT + token[u]) * NG +
                                                        lane / (16 / NG)] = pair;
    }
}

template <int NG>
__global__ void __launch_bounds__(Q4_MOVE_THREADS) q4_load_kernel(const Q4MoveParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 15;
  const int64_t total = p.rows * p.hkv;
  const int64_t first = (int64_t)blockIdx.x * (Q4_MOVE_THREADS / 16) * Q4_MOVE_HEADS +
                        (threadIdx.x >> 4);
  uint32_t word[Q4_MOVE_HEADS][2], pair[Q4_MOVE_HEADS][2];
#pragma unroll
  for (int u = 0; u < Q4_MOVE_HEADS; ++u) {
    const int64_t i = first + u * (Q4_MOVE_THREADS / 16);
    word[u][0] = word[u][1] = pair[u][0] = pair[u][1] = 0u;
    if (i < total) {
      const int64_t row = i / p.hkv;
      int token;
      const uint8_t* unit = q4_unit(p, row, (int)(i - row * p.hkv), q4_unit_bytes(NG), &token);
      if (unit)
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int place = kv ? q4_value_place(lane) : q4_key_place(lane);
          word[u][kv] = reinterpret_cast<const uint32_t*>(unit + kv * Q4_VALUES +
                                                          token * Q4_ROW)[place];
          pair[u][kv] = reinterpret_cast<const uint32_t*>(
              unit + Q4_PAIRS)[(kv * Q4_UNIT + token) * NG + lane / (16 / NG)];
        }
    }
  }
#pragma unroll
  for (int u = 0; u < Q4_MOVE_HEADS; ++u) {
    const int64_t i = first + u * (Q4_MOVE_THREADS / 16);
    if (i >= total) break;
    p.k_out[i * 16 + lane] = q4_unpack<NG>(word[u][0], pair[u][0]);
    p.v_out[i * 16 + lane] = q4_unpack<NG>(word[u][1], pair[u][1]);
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
  const int64_t per = (Q4_MOVE_THREADS / 16) * Q4_MOVE_HEADS;
  FK_REQUIRE(rows < (1ll << 31) && (rows * hkv + per - 1) / per < (1ll << 31), FK_ERR_UNSUPPORTED,
             "%s: too many tokens", what);
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
  const dim3 grid((unsigned)((rows * hkv + per - 1) / per));
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
