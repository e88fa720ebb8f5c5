/*
 * C ABI of libssattn.so, continued: a paged K/V cache of 8-bit rows (appending,
 * reading back, attention), and attention with shaped scores over both caches.
 *
 * Conventions as in ssattn_paged.h.  The 8-bit cache holds a row of 128
 * elements as e4m3 values and one power of two: the 64 rows of 128 bytes of page
 * P and K/V head h lie next to each other at byte P * kv_page_stride + h *
 * kv_head_stride of cache_k and cache_v (16-byte aligned, strides multiples of
 * 16), their biased exponents, 64 of the keys and then 64 of the values, at byte
 * P * scales_page_stride + h * scales_head_stride of `scales` (4-byte aligned,
 * strides multiples of 4).  A value x with its row's byte s (1..254) stands for x
 * 2^(s - 127).  bf16 holds every value that an append writes; fp16 those of rows appended
 * as fp16.
 */
#ifndef SSATTN_PAGED8_H
#define SSATTN_PAGED8_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ssa_paged_append into an 8-bit cache, of whose rows the strides are above.  A
 * key's or value's row is rounded to its 16-bit type as there (keys turn in float64 and
 * are rounded to float32 first); its power of two is the smallest 2^e, e >= -126, with max |x| <= 448 * 2^e over its finite elements,
 * and x 2^-e is rounded to e4m3 (nearest, ties to even).  Infinities and NaN become
 * NaN; fp16 elements from 63488 on are held as 61440, bf16 ones from 1.9375 * 2^127 on as
 * 1.875 * 2^127, so that what is finite stays so. */
int ssa_paged8_append(const void* q, long long q_token_stride, long long q_head_stride, void* q_out,
                      long long out_token_stride, long long out_head_stride, const void* k, long long k_token_stride,
                      long long k_head_stride, const void* v, long long v_token_stride, long long v_head_stride,
                      void* cache_k, void* cache_v, long long kv_page_stride, long long kv_head_stride, void* scales,
                      long long scales_page_stride, long long scales_head_stride, const int32_t* table,
                      const int32_t* held, const int32_t* starts, const int32_t* positions, const double* freqs,
                      long long first, int tokens, int batch, int heads, int kv_heads, int pages, int table_pages,
                      int pairs, int axis0, int axis1, int axes, int flags, hipStream_t stream);

/* Rows of an 8-bit cache as 16-bit ones (fp16 with flags bit 0, else bf16): row i of
 * the packed rows [starts[b], starts[b + 1]) of k and v [tokens, kv_heads, 128]
 * becomes the sequence's row first[b] + i (first [batch] int32).  Rows outside the
 * table, or of pages outside [0, pages), become zeros; those from starts[batch] on
 * are left as they were. */
int ssa_paged8_read(const void* cache_k, const void* cache_v, long long kv_page_stride, long long kv_head_stride,
                    const void* scales, long long scales_page_stride, long long scales_head_stride,
                    const int32_t* table, const int32_t* first, const int32_t* starts, void* k,
                    long long k_token_stride, long long k_head_stride, void* v, long long v_token_stride,
                    long long v_head_stride, int tokens, int batch, int kv_heads, int pages, int table_pages, int flags,
                    hipStream_t stream);

/* ssa_paged_attention over an 8-bit cache.  In tiles of up to 32 rows a probability
 * meets V in two parts, whatever the flags.  Where there are two, the queries are bf16
 * and the flags do not ask for two, they may be one of fp16 instead, which carries 11
 * bits down to 2^-21 of a row's largest probability (values whose powers of two lie
 * within 2^15 of the largest of the pages walked before; rows whose byte is 1, values
 * below 2^-117, count as zeros then). */
int ssa_paged8_attention(const void* q, long long q_token_stride, long long q_head_stride, const void* cache_k,
                         const void* cache_v, long long kv_page_stride, long long kv_head_stride, const void* scales,
                         long long scales_page_stride, long long scales_head_stride, const int32_t* prefix,
                         int prefix_tokens, const int32_t* table, const int32_t* lengths, const int32_t* starts,
                         void* out, long long out_token_stride, long long out_head_stride, float* lse, int tokens,
                         int batch, int heads, int kv_heads, int pages, int table_pages, float scale, int flags,
                         void* workspace, long long workspace_bytes, hipStream_t stream);

/* ssa_paged_attention with shaped scores: of s = scale q . k,
 *   cap > 0:      s becomes cap tanh(s / cap);
 *   slopes:       s -= slopes[query head] * |distance| (float [heads], or NULL), the
 *                 distance in rows from the query's own (row lengths[b] - n + i of its
 *                 sequence for query i of n) to the key's, the prefix's rows lying
 *                 before the sequence's row 0;
 *   window > 0:   of its own sequence a query sees the rows j > lengths[b] - n + i -
 *                 window only.  Pages that no query sees may be absent, their rows
 *                 anything.
 * 0 <= cap <= 65536 (and large enough that 2 log2(e) scale / cap is a finite float), 0 <=
 * window < 2^30; slopes are finite, and so are they times the distances as floats.  A score
 * is off by up to 2^-22 of the cap, and by up to 2^-22 of what the slope takes from it
 * (distances beyond 2^24 are themselves rounded to floats). */
int ssa_paged_attention_shaped(const void* q, long long q_token_stride, long long q_head_stride, const void* cache_k,
                               const void* cache_v, long long kv_token_stride, long long kv_head_stride,
                               const int32_t* prefix, int prefix_tokens, const int32_t* table, const int32_t* lengths,
                               const int32_t* starts, void* out, long long out_token_stride, long long out_head_stride,
                               float* lse, int tokens, int batch, int heads, int kv_heads, int pages, int table_pages,
                               float scale, float cap, const float* slopes, int window, int flags, void* workspace,
                               long long workspace_bytes, hipStream_t stream);

/* The same over an 8-bit cache. */
int ssa_paged8_attention_shaped(const void* q, long long q_token_stride, long long q_head_stride, const void* cache_k,
                                const void* cache_v, long long kv_page_stride, long long kv_head_stride,
                                const void* scales, long long scales_page_stride, long long scales_head_stride,
                                const int32_t* prefix, int prefix_tokens, const int32_t* table, const int32_t* lengths,
                                const int32_t* starts, void* out, long long out_token_stride,
                                long long out_head_stride, float* lse, int tokens, int batch, int heads, int kv_heads,
                                int pages, int table_pages, float scale, float cap, const float* slopes, int window,
                                int flags, void* workspace, long long workspace_bytes, hipStream_t stream);

/* Bytes of the workspace of those three, as ssa_paged_attention_workspace_bytes: eight,
 * whether the rows are of 8 bits; shaped, whether a shaped entry is called, with what
 * window (0 for the plain one). */
long long ssa_paged8_workspace_bytes(int tokens, int batch, int heads, int kv_heads, int prefix_tokens,
                                     int table_pages, int ragged, int causal, int eight, int shaped, int window);

#ifdef __cplusplus
}
#endif

#endif /* SSATTN_PAGED8_H */
