// The paged KV cache of 4 bits a value, as its kernels and the eviction's see it.
//
//   pool   [pages, KV heads, page / 16] units of 16 tokens
//   unit   16 x 64 B  codes of the keys     (row of a token: 16 words of 8 channels)
//          16 x 64 B  codes of the values
//          16 x NG    (scale, lowest) of the keys, bf16 pairs; NG = 128 / group
//          16 x NG    (scale, lowest) of the values
//
// Word w holds channels 8 w .. 8 w + 7, four bits each, the lowest channel in the lowest bits.
// Key word w lies at place w % 4 * 4 + w / 4 of its row and value word w at w % 8 * 2 + w / 8, so
// that what a lane of the attention kernel needs of a row is one 16-byte (8-byte) load.  A whole
// unit, and so any run of units of one page, is one contiguous copy.
#pragma once

#include "fk_common.cuh"

namespace fk {

constexpr int Q4_D = 128;                    // channels of a head
constexpr int Q4_UNIT = 16;                  // tokens of a unit
constexpr int Q4_ROW = Q4_D / 2;             // bytes of a token's codes
constexpr int Q4_VALUES = Q4_UNIT * Q4_ROW;  // offset of the values' codes
constexpr int Q4_PAIRS = 2 * Q4_VALUES;      // offset of the keys' (scale, lowest)

__host__ __device__ constexpr int q4_unit_bytes(int ng) { return Q4_PAIRS + 2 * Q4_UNIT * 4 * ng; }

// place of channel word w in a row
__host__ __device__ constexpr int q4_key_place(int w) { return w % 4 * 4 + w / 4; }
__host__ __device__ constexpr int q4_value_place(int w) { return w % 8 * 2 + w / 8; }

// What the entry points check of a pool.
inline int q4_check_pool(const char* what, const void* cache, int64_t num_pages, int page, int hkv,
                         int head_dim, int group) {
  FK_REQUIRE(cache != nullptr, FK_ERR_INVALID_ARG, "%s: null pointer", what);
  FK_REQUIRE(head_dim == Q4_D, FK_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (128 only)", what,
             head_dim);
  FK_REQUIRE(group == 64 || group == 128, FK_ERR_UNSUPPORTED,
             "%s: groups of %d channels unsupported (64 or 128)", what, group);
  FK_REQUIRE(page == 16 || page == 32 || (page >= 64 && page % 64 == 0), FK_ERR_UNSUPPORTED,
             "%s: page of %d tokens unsupported (16, 32 or a multiple of 64)", what, page);
  FK_REQUIRE(num_pages > 0 && num_pages < (1ll << 31) && hkv > 0, FK_ERR_INVALID_ARG,
             "%s: bad sizes", what);
  FK_REQUIRE(num_pages * page < (1ll << 40) && (int64_t)hkv * page < (1ll << 31),
             FK_ERR_UNSUPPORTED, "%s: pool too large", what);
  FK_REQUIRE(aligned16(cache), FK_ERR_ALIGNMENT, "%s: 16-byte alignment required", what);
  return FK_OK;
}

#ifdef __CUDACC__
// Two fp32 side by side.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t pair_of(float a) { return pair_of(a, a); }
__device__ __forceinline__ float2 both_of(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
#endif

}  // namespace fk
