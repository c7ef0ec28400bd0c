// Decode attention that reads less of the paged cache:
//
//   fk_selected_attn       attention over selected blocks of each query token and KV head
//   fk_shared_prefix_attn  attention of a batch whose sequences begin with the same pages in groups
//
// Both are one softmax per query head over a set of keys, out = sum_t e^(s q.k_t) v_t / sum_t
// e^(s q.k_t).
#include "fk_common.cuh"
#include "fk_types.cuh"

namespace fk {

constexpr int SH_D = 128;
constexpr int SH_MAX_G = 16;
constexpr int SH_THREADS = 256;

struct RowsParams {
  const uint16_t* q; int64_t q_stride;
  uint16_t* out; int64_t out_stride;
  const uint16_t* k; const uint16_t* v; int64_t page_stride;
  const int32_t* context_lens;
  const int32_t* rows;
  const int32_t* tables; int64_t table_stride;
  int64_t capacity;
  const int32_t* selected; int count;      // null: all blocks
  int num_tables, num_pages, page, block, hkv, g, hnd;
  float scale_log2;
  int32_t* status;
};

// One CTA per (token, KV head); its warps take blocks in turn, a lane has four channels, and every
// warp keeps a running maximum and sum of its own, which are joined at the end.
__global__ void __launch_bounds__(SH_THREADS) attn_rows_kernel(const RowsParams p) {
  __shared__ float o_part[SH_D];
  __shared__ float m_part[8], l_part[8];
  pdl_launch_dependents();
  pdl_wait();
  const int token = blockIdx.x, kvh = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t len = p.context_lens[token];
  const int row = p.rows ? p.rows[token] : token;
  bool bad = len > p.capacity;
  if (len < 0) len = 0;
  if (len > p.capacity) len = p.capacity;
  if (row < 0 || row >= p.num_tables) { len = 0; bad = true; }
  if (bad && threadIdx.x == 0 && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
  const int n = (int)((len + p.block - 1) / p.block);
  const int units = p.selected ? p.count : n;
  const int32_t* sel = p.selected ? p.selected + ((int64_t)token * p.hkv + kvh) * p.count : nullptr;
  const int32_t* table = p.tables + (int64_t)row * p.table_stride;
  for (int h = 0; h < p.g; ++h) {
    const int64_t at = (int64_t)(kvh * p.g + h) * SH_D;
    const float4 q = Elem<uint16_t>::load4(p.q + (int64_t)token * p.q_stride + at + lane * 4);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    for (int u = warp; u < units; u += SH_THREADS / 32) {
      const int b = sel ? sel[u] : u;
      if (b < 0 || b >= n) continue;
      const int64_t pos = (int64_t)b * p.block;
      const int page = table[pos / p.page];
      if (page < 0 || page >= p.num_pages) {
        if (lane == 0 && p.status) atomicOr(p.status, FK_DEV_BAD_PAGE);
        continue;
      }
      const int off = (int)(pos % p.page);
      const int keys = (int)(len - pos < p.block ? len - pos : p.block);
      const int64_t step = p.hnd ? SH_D : (int64_t)p.hkv * SH_D;
      const int64_t base = (int64_t)page * p.page_stride + lane * 4 +
                           (p.hnd ? ((int64_t)kvh * p.page + off) * SH_D
                                  : (int64_t)off * p.hkv * SH_D + (int64_t)kvh * SH_D);
      for (int t = 0; t < keys; ++t) {
        const float4 k = Elem<uint16_t>::load4(p.k + base + t * step);
        const float s = warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w) * p.scale_log2;
        const float4 v = Elem<uint16_t>::load4(p.v + base + t * step);
        const float mn = fmaxf(m, s);
        const float keep = m == -INFINITY ? 0.f : exp2f(m - mn);
        const float e = mn == -INFINITY ? 0.f : exp2f(s - mn);
        m = mn;
        l = l * keep + e;
        o = o * keep + v * e;
      }
    }
    if (lane == 0) { m_part[warp] = m; l_part[warp] = l; }
    if (threadIdx.x < SH_D) o_part[threadIdx.x] = 0.f;
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < 8; ++w) top = fmaxf(top, m_part[w]);
    for (int w = 0; w < 8; ++w)
      sum += m_part[w] == -INFINITY ? 0.f : l_part[w] * exp2f(m_part[w] - top);
    const float f = m == -INFINITY ? 0.f : exp2f(m - top);
    for (int w = 0; w < 8; ++w) {              // in order
      if (w == warp) {
        float4* d = reinterpret_cast<float4*>(o_part) + lane;
        *d = *d + o * f;
      }
      __syncthreads();
    }
    if (warp == 0) {
      const float inv = sum > 0.f ? 1.0f / sum : 0.f;
      Elem<uint16_t>::store4(p.out + (int64_t)token * p.out_stride + at + lane * 4,
                             reinterpret_cast<float4*>(o_part)[lane] * inv);
    }
    __syncthreads();
  }
}

static int rows_args(const char* what, RowsParams& p, const void* q, int64_t q_stride, void* out,
                     int64_t out_stride, const void* k, const void* v, int64_t num_pages, int page,
                     int64_t page_stride, int layout, const int32_t* lens, const int32_t* tables,
                     int64_t table_stride, int64_t table_cols, int hq, int hkv, int d, int block,
                     float scale, int32_t* status) {
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
  p.k = static_cast<const uint16_t*>(k); p.v = static_cast<const uint16_t*>(v);
  p.page_stride = page_stride;
  p.context_lens = lens;
  p.tables = tables; p.table_stride = table_stride; p.capacity = table_cols * page;
  p.num_pages = (int)num_pages; p.page = page; p.block = block; p.hkv = hkv; p.g = hq / hkv;
  p.hnd = layout;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = status;
  return FK_OK;
}

}  // namespace fk

using namespace fk;

extern "C" {

size_t fk_selected_attn_workspace_bytes(int num_tokens, int num_q_heads, int num_kv_heads,
                                        int head_dim, int count, int block) {
  return num_tokens > 0 && num_q_heads > 0 && num_kv_heads > 0 && head_dim > 0 && count > 0 &&
                 block > 0
             ? 256
             : 0;
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
                           num_kv_heads, head_dim, block, softmax_scale, status);
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
  const size_t need = fk_selected_attn_workspace_bytes(num_tokens, num_q_heads, num_kv_heads,
                                                       head_dim, count, block);
  FK_REQUIRE(workspace != nullptr && workspace_bytes >= need &&
                 (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0,
             FK_ERR_WORKSPACE,
             "fk_selected_attn: workspace needs %zu bytes, 256-byte aligned (got %zu)", need,
             workspace_bytes);
  p.rows = table_rows; p.num_tables = num_tables;
  p.selected = selected; p.count = count;
  FK_CUDA_OK(launch_kernel(attn_rows_kernel, dim3((unsigned)num_tokens, (unsigned)num_kv_heads),
                           dim3(SH_THREADS), (size_t)0, static_cast<cudaStream_t>(stream), p));
  count_launch(1);
  return FK_OK;
}

size_t fk_shared_prefix_workspace_bytes(int batch, int num_groups, int num_q_heads,
                                        int num_kv_heads, int head_dim, int max_splits) {
  return batch > 0 && num_groups >= 0 && num_q_heads > 0 && num_kv_heads > 0 && head_dim > 0 &&
                 max_splits > 0
             ? 256
             : 0;
}

int fk_shared_prefix_attn(const void* q, int64_t q_stride_token, void* out,
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
  RowsParams p{};
  const int rc = rows_args("fk_shared_prefix_attn", p, q, q_stride_token, out, out_stride_token,
                           k_cache, v_cache, num_pages, page_size, kv_page_stride, kv_layout,
                           context_lens, block_tables, block_table_stride, block_table_cols,
                           num_q_heads, num_kv_heads, head_dim, page_size, softmax_scale, status);
  if (rc != FK_OK) return rc;
  FK_REQUIRE(num_groups == 0 || (group_starts && prefix_lens), FK_ERR_INVALID_ARG,
             "fk_shared_prefix_attn: null pointer");
  FK_REQUIRE(max_splits > 0, FK_ERR_INVALID_ARG, "fk_shared_prefix_attn: max_splits < 1");
  const size_t need = fk_shared_prefix_workspace_bytes(batch, num_groups, num_q_heads,
                                                       num_kv_heads, head_dim, max_splits);
  FK_REQUIRE(workspace != nullptr && workspace_bytes >= need &&
                 (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0,
             FK_ERR_WORKSPACE,
             "fk_shared_prefix_attn: workspace needs %zu bytes, 256-byte aligned (got %zu)", need,
             workspace_bytes);
  p.num_tables = batch;
  FK_CUDA_OK(launch_kernel(attn_rows_kernel, dim3((unsigned)batch, (unsigned)num_kv_heads),
                           dim3(SH_THREADS), (size_t)0, static_cast<cudaStream_t>(stream), p));
  count_launch(1);
  return FK_OK;
}

}  // extern "C"
