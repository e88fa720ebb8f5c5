/*
 * C ABI of libssattn.so, continued: several sequences over one paged K/V
 * cache (appending, and attention behind a shared prefix).
 *
 * Conventions as in ssattn.h: device pointers, strides in elements, work
 * enqueued on `stream` of the current device, nothing allocated, no
 * synchronisation, a hipError_t as int (hipErrorInvalidValue = 1 for rejected
 * arguments, and nothing launched).  Head dimension 128; 16-bit elements, bf16
 * or (flags bit 0) fp16.  A page is 64 consecutive rows of the cache; row
 * `row` of K/V head h starts at element row * kv_token_stride + h *
 * kv_head_stride.  Rows are read and written in 16-byte pieces: pointers are
 * 16-byte aligned and strides multiples of 8.
 */
#ifndef SSATTN_PAGED_H
#define SSATTN_PAGED_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Keys and values of `tokens` new tokens into the cache, queries and keys
 * rotated by their positions on the way.
 *
 * Sequence b (of `batch`) owns the tokens [starts[b], starts[b + 1]) (starts
 * [batch + 1] int32, starts[0] = 0, not decreasing; NULL: tokens / batch each)
 * and holds held[b] tokens already; its token i becomes its row at = held[b] +
 * i, cache row 64 * table[b, at / 64] + at % 64 (table [batch, table_pages]
 * int32).  A token whose row lies outside the table, or whose page outside
 * [0, pages), is not written; tokens from starts[batch] on are left alone
 * altogether.  Two tokens of one call must not share a cache row.
 *
 * The pairs j < pairs (at most 64) of query and key rows turn by position *
 * freqs[j] (float64, radians): elements (2j, 2j + 1) with flags bit 1, else (j,
 * j + pairs), pairs then a multiple of 8.  The position is first + at (first
 * within 2^53), or positions[t, axis] (int32 [tokens, axes], axes 1..3, wanted
 * for axes > 1): the first axis0 pairs turn on axis 0, the next axis1 on axis 1,
 * the others on axis 2; with positions the counts must reach the last of fewer
 * axes: axis0 = pairs for one, axis0 + axis1 = pairs for two.  Angles are formed
 * in float64; each result is rounded once.
 *
 * q [tokens, heads, 128] goes to q_out (which may be q itself); heads = 0: no
 * queries.  k and v must not overlap the cache rows written.  tokens is at most
 * 2^26 - 4. */
int ssa_paged_append(const void* q, long long q_token_stride, long long q_head_stride, void* q_out,
                     long long out_token_stride, long long out_head_stride, const void* k, long long k_token_stride,
                     long long k_head_stride, const void* v, long long v_token_stride, long long v_head_stride,
                     void* cache_k, void* cache_v, long long kv_token_stride, long long kv_head_stride,
                     const int32_t* table, const int32_t* held, const int32_t* starts, const int32_t* positions,
                     const double* freqs, long long first, int tokens, int batch, int heads, int kv_heads, int pages,
                     int table_pages, int pairs, int axis0, int axis1, int axes, int flags, hipStream_t stream);

/* Attention of a batch behind a shared prefix.  Sequence b owns the query
 * rows [starts[b], starts[b + 1]) of q [tokens, heads, 128] (starts as above)
 * and `lengths[b]` rows of its own in the cache (row j at page table[b, j / 64],
 * row j % 64; the new tokens' rows among them); before them all sequences see
 * the prefix_tokens rows of the pages prefix[0..].  Query i of the n new ones
 * of a sequence attends the whole prefix and the sequence's rows j <
 * lengths[b], with flags bit 1 (causal) only j <= lengths[b] - n + i.  Query
 * head h reads K/V head h / (heads / kv_heads).
 *   out = softmax(scale q . k) v,  lse [tokens, heads] fp32 (or NULL) = ln sum
 * exp(scale q . k).  A query that sees no row has out 0 and lse -infinity.
 * Rows of out and lse from starts[batch] on are left as they were.  Pages
 * outside [0, pages), and those behind the table's end where a length passes
 * it, count as absent: none of their rows is seen, nor does any other row's
 * place change.  Values in
 * rows of a page that no query sees (behind a sequence's or the prefix's end)
 * may be anything, NaN included; one that some query of the call sees must be
 * finite for the others to come out finite (an infinite one may come out NaN).
 * out may be q itself.
 *
 * A probability meets V in 16 bits, in two parts (hi + lo) or in one: flags bits
 * 3 and 4 are 1 for one part in all tiles of more than 32 query rows a K/V head,
 * 2 for two parts throughout, 0 for one in those tiles where the sequences bring
 * more than 32 rows (their mean, tokens / batch * heads / kv_heads), else two.
 * Bit 2 is 0.
 *
 * workspace: 16-byte aligned, at least ssa_paged_attention_workspace_bytes of
 * the same sizes, any contents; calls that share one must not overlap. */
int ssa_paged_attention(const void* q, long long q_token_stride, long long q_head_stride, const void* cache_k,
                        const void* cache_v, long long kv_token_stride, long long kv_head_stride,
                        const int32_t* prefix, int prefix_tokens, const int32_t* table, const int32_t* lengths,
                        const int32_t* starts, void* out, long long out_token_stride, long long out_head_stride,
                        float* lse, int tokens, int batch, int heads, int kv_heads, int pages, int table_pages,
                        float scale, int flags, void* workspace, long long workspace_bytes, hipStream_t stream);

/* Bytes of that workspace (0: none needed), from sizes alone; -1 for sizes the
 * call rejects (tokens * heads >= 2^30, or more work than a grid holds).
 * ragged: whether the call gives starts; causal: whether it is. */
long long ssa_paged_attention_workspace_bytes(int tokens, int batch, int heads, int kv_heads, int prefix_tokens,
                                              int table_pages, int ragged, int causal);

#ifdef __cplusplus
}
#endif

#endif /* SSATTN_PAGED_H */
