// Paged attention over 8-bit rows: the entries; the kernels are in paged.h.
#include "paged_entry.h"
#include "../../include/ssattn_paged8.h"

extern "C" {

long long ssa_paged8_workspace_bytes(int tokens, int batch, int heads, int kv_heads, int prefix_tokens,
                                     int table_pages, int ragged, int causal, int eight, int shaped, int window) {
  return workspace_of(Sizes{0, tokens, batch, heads, kv_heads, prefix_tokens, table_pages, ragged != 0, causal != 0,
                            eight != 0, shaped != 0, window});
}

int ssa_paged8_attention(const void* q, long long q_token_stride, long long q_head_stride, const void* cache_k, const
                         void* cache_v, long long kv_page_stride, long long kv_head_stride, const void* scales, long
                         long scales_page_stride, long long scales_head_stride, const int32_t* prefix, int
                         prefix_tokens, const int32_t* table, const int32_t* lengths, const int32_t* starts, void*
                         out, long long out_token_stride, long long out_head_stride, float* lse, int tokens, int
                         batch, int heads, int kv_heads, int pages, int table_pages, float scale, int flags, void*
                         workspace, long long workspace_bytes, hipStream_t stream) {
  return attend8<false>(q, q_token_stride, q_head_stride, cache_k, cache_v, kv_page_stride, kv_head_stride, scales,
                        scales_page_stride, scales_head_stride, prefix, prefix_tokens, table, lengths, starts, out,
                        out_token_stride, out_head_stride, lse, tokens, batch, heads, kv_heads, pages, table_pages,
                        scale, 0.0f, nullptr, 0, flags, workspace, workspace_bytes, stream);
}

}  // extern "C"
