// The entry point of the attention of tokens drafted as trees: kernels, checks and launches are gqa_split.hpp's.
#include "gqa_split.hpp"
#include "../../include/mla_hip.h"

using namespace mlahip;

extern "C" int mlahip_gqa_tree_decode(const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t num_tokens, const void* k_cache,
                                 int64_t kc_page_stride, int64_t kc_row_stride, int64_t kc_head_stride, const void* v_cache,
                                 int64_t vc_page_stride, int64_t vc_row_stride, int64_t vc_head_stride, int64_t num_pages,
                                 int32_t page_size, const int32_t* block_table, int64_t bt_stride, int32_t max_blocks,
                                 const int32_t* seq_lens, const int32_t* query_start_loc, const uint64_t* visible, int64_t visible_stride, int32_t words,
                                 int32_t batch, int32_t max_q_len,
                                 int32_t q_heads, int32_t kv_heads, int32_t dim, int32_t dtype, int32_t cache_dtype,
                                 const float* k_scale, const float* v_scale, float scale, int32_t window, void* out,
                                 int64_t out_stride_t, int64_t out_stride_h, float* lse_out, void* workspace, size_t workspace_bytes,
                                 int32_t num_chunks, int32_t heads_per_group, int32_t rows_per_group,
                                 hipStream_t stream) {
  return gqa::run<true>("mlahip_gqa_tree_decode", q, q_stride_t, q_stride_h, num_tokens, k_cache, kc_page_stride, kc_row_stride, kc_head_stride,
                                v_cache, vc_page_stride, vc_row_stride, vc_head_stride, num_pages, page_size, block_table, bt_stride, max_blocks,
                                seq_lens, query_start_loc, batch, max_q_len, q_heads, kv_heads, dim, dtype, cache_dtype, k_scale, v_scale, scale,
                                window, out, out_stride_t, out_stride_h, lse_out, workspace, workspace_bytes, num_chunks, heads_per_group,
                                rows_per_group, visible, visible_stride, words, stream);
}
