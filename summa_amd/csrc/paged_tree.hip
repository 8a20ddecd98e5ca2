// sm_paged_tree_attention: the tree form of the kernels in paged_attention.hpp, whose rows see
// the context and those of their sequence's rows that a mask names.
#include "paged_attention.hpp"

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
