// sm_paged_tree_attention: the tree form of the kernels in paged_attention.hpp, whose rows see
// the context and those of their sequence's rows that a mask names.
#include "paged_attention.hpp"

extern "C" int64_t sm_paged_tree_attention_workspace_bytes(int64_t S, int64_t rows,
                                                           int64_t max_rows, int64_t H,
                                                           int64_t KVH, int64_t head_dim,
                                                           int64_t max_tokens) {
  if (sm::check_shape("sm_paged_tree_attention_workspace_bytes", S, rows, max_rows, H, KVH,
                      head_dim, max_tokens) != SM_OK)
    return -1;
  if (S == 0 || max_rows == 0) return 0;
  sm::PagedPlan plan(S, max_rows, H / KVH, KVH, head_dim, max_tokens);
  plan.by_length(S, KVH, max_tokens);
  return plan.bytes(rows, H, head_dim) + plan.counts(S);
}

extern "C" int sm_paged_tree_attention(const sm_paged_cache* cache, const int32_t* block_table,
                                       int64_t table_cols, const int32_t* pos0,
                                       const int32_t* row_start, int64_t S, int64_t rows,
                                       int64_t max_rows, int64_t max_tokens, const int32_t* mask,
                                       int64_t words, const void* q, int dtype, int64_t ldq,
                                       int64_t H, void* out, float* lse, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  return sm::paged_attention<true>("sm_paged_tree_attention", cache, block_table, table_cols,
                                   pos0, row_start, S, rows, max_rows, max_tokens, mask, words, q,
                                   dtype, ldq, H, out, lse, workspace, workspace_bytes, stream);
}
