// sm_paged_attention: the causal form of the kernels in paged_attention.hpp.
#include "paged_attention.hpp"

namespace sm {

// Shared with the append: what a cache descriptor has to be.
int check_paged_cache(const char* who, const sm_paged_cache* c) {
  SM_REQUIRE(c, "%s: null cache", who);
  SM_REQUIRE(c->dtype == SM_BF16 || c->dtype == SM_F16 || c->dtype == SM_F8E4M3,
             "%s: cache dtype must be SM_BF16, SM_F16 or SM_F8E4M3", who);
  SM_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "%s: head_dim must be 64 or 128", who);
  SM_REQUIRE(c->pages > 0 && c->kv_heads > 0 && c->page_tokens > 0 &&
                 c->page_tokens % kBlock == 0,
             "%s: need pages and kv_heads > 0 and page_tokens a positive multiple of 16", who);
  const int64_t most = 0x7fffffff;
  SM_REQUIRE(c->pages <= most && c->kv_heads <= 65535 && c->page_tokens <= most &&
                 c->kv_heads * (c->page_tokens / kBlock) <= most / c->pages,
             "%s: a cache holds less than 2^31 blocks of 16 tokens", who);
  SM_REQUIRE(c->k && c->v, "%s: null cache pages", who);
  SM_REQUIRE(reinterpret_cast<uintptr_t>(c->k) % 16 == 0 &&
                 reinterpret_cast<uintptr_t>(c->v) % 16 == 0,
             "%s: cache pages must be 16-byte aligned", who);
  SM_REQUIRE(c->dtype != SM_F8E4M3 || (c->k_scales && c->v_scales),
             "%s: an SM_F8E4M3 cache needs k_scales and v_scales", who);
  return SM_OK;
}

}  // namespace sm

extern "C" int64_t sm_paged_attention_workspace_bytes(int64_t S, int64_t rows, int64_t max_rows,
                                                      int64_t H, int64_t KVH, int64_t head_dim,
                                                      int64_t max_tokens) {
  if (sm::check_shape("sm_paged_attention_workspace_bytes", S, rows, max_rows, H, KVH, head_dim,
                      max_tokens) != SM_OK)
    return -1;
  if (S == 0 || max_rows == 0) return 0;
  return sm::PagedPlan(S, max_rows, H / KVH, KVH, head_dim, max_tokens).bytes(rows, H, head_dim);
}

extern "C" int sm_paged_attention(const sm_paged_cache* cache, const int32_t* block_table,
                                  int64_t table_cols, const int32_t* pos0,
                                  const int32_t* row_start, int64_t S, int64_t rows,
                                  int64_t max_rows, int64_t max_tokens, const void* q, int dtype,
                                  int64_t ldq, int64_t H, void* out, float* lse, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  return sm::paged_attention<false>("sm_paged_attention", cache, block_table, table_cols, pos0,
                                    row_start, S, rows, max_rows, max_tokens, nullptr, 0, q,
                                    dtype, ldq, H, out, lse, workspace, workspace_bytes, stream);
}
