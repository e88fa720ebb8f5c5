// Paged attention over 16-bit rows with shaped scores: the entry; the kernels are in paged.h.
#include "paged_entry.h"
#include "../../include/ssattn_paged8.h"

extern "C" {

int ssa_paged_attention_shaped(const void* q, long long q_token_stride, long long q_head_stride, const void* cache_k,
                               const void* cache_v, long long kv_token_stride, long long kv_head_stride, const
                               int32_t* prefix, int prefix_tokens, const int32_t* table, const int32_t* lengths, const
                               int32_t* starts, void* out, long long out_token_stride, long long out_head_stride,
                               float* lse, int tokens, int batch, int heads, int kv_heads, int pages, int table_pages,
                               float scale, float cap, const float* slopes, int window, int flags, void* workspace,
                               long long workspace_bytes, hipStream_t stream) {
  return attend16<true>(q, q_token_stride, q_head_stride, cache_k, cache_v, kv_token_stride, kv_head_stride, prefix,
                        prefix_tokens, table, lengths, starts, out, out_token_stride, out_head_stride, lse, tokens,
                        batch, heads, kv_heads, pages, table_pages, scale, cap, slopes, window, flags, workspace,
                        workspace_bytes, stream);
}

}  // extern "C"
