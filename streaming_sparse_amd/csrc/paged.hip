// Attention of a batch of sequences behind a prefix they share, over a paged cache of
// 16-bit rows: the entries; the kernels and the plan are in paged.h.
#include "paged_entry.h"
#include "../../include/ssattn_paged.h"

extern "C" {

long long ssa_paged_attention_workspace_bytes(int tokens, int batch, int heads, int kv_heads, int prefix_tokens,
                                              int table_pages, int ragged, int causal) {
  return workspace_of(Sizes{0, tokens, batch, heads, kv_heads, prefix_tokens, table_pages, ragged != 0, causal != 0});
}

int ssa_paged_attention(const void* q, long long q_token_stride, long long q_head_stride, const void* cache_k,
                        const void* cache_v, long long kv_token_stride, long long kv_head_stride,
                        const int32_t* prefix, int prefix_tokens, const int32_t* table, const int32_t* lengths,
                        const int32_t* starts, void* out, long long out_token_stride, long long out_head_stride,
                        float* lse, int tokens, int batch, int heads, int kv_heads, int pages, int table_pages,
                        float scale, int flags, void* workspace, long long workspace_bytes, hipStream_t stream) {
  return attend16<false>(q, q_token_stride, q_head_stride, cache_k, cache_v, kv_token_stride, kv_head_stride, prefix,
                         prefix_tokens, table, lengths, starts, out, out_token_stride, out_head_stride, lse, tokens,
                         batch, heads, kv_heads, pages, table_pages, scale, 0.0f, nullptr, 0, flags, workspace,
                         workspace_bytes, stream);
}

}  // extern "C"
