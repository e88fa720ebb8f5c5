// What the C entries of paged attention share: their arguments as the kernels' own.
#pragma once
#include "paged.h"

namespace {

// cap 0: none; slopes null: none; window 0: none.  A score's error is 2^-22 of the cap,
// 2^-6 at the largest that is taken.
bool shape_fits(float scale, float cap, const float* slopes, int window) {
  return cap >= 0.0f && cap <= 65536.0f && (cap == 0.0f || 2.0f * kLog2e * scale / cap < INFINITY) && window >= 0 && window < (1 << 30) && !((uintptr_t)slopes & 3);
}

void set_shape(PagedParams* p, float scale, float cap, const float* slopes, int window) {
  p->cap_log2 = cap * kLog2e;
  p->cap_scale = cap > 0.0f ? 2.0f * kLog2e * scale / cap : 0.0f;
  p->slopes = slopes;
  p->window = window;
}

template <bool SHAPED>
int attend16(const void* q, long long q_token_stride, long long q_head_stride, const void* cache_k,
             const void* cache_v, long long kv_token_stride, long long kv_head_stride, const int32_t* prefix,
             int prefix_tokens, const int32_t* table, const int32_t* lengths, const int32_t* starts, void* out,
             long long out_token_stride, long long out_head_stride, float* lse, int tokens, int batch, int heads,
             int kv_heads, int pages, int table_pages, float scale, float cap, const float* slopes, int window,
             int flags, void* workspace, long long workspace_bytes, hipStream_t stream) {
  PagedParams p{};
  p.q = (const uint16_t*)q;
  p.k = cache_k;
  p.v = cache_v;
  p.out = (uint16_t*)out;
  p.lse = lse;
  p.q_tok = q_token_stride;
  p.q_head = q_head_stride;
  p.o_tok = out_token_stride;
  p.o_head = out_head_stride;
  p.kv_tok = kv_token_stride;
  p.kv_head = kv_head_stride;
  p.prefix = prefix;
  p.table = table;
  p.lengths = lengths;
  p.starts = starts;
  p.pages = pages;
  const Sizes z{0, tokens, batch, heads, kv_heads, prefix_tokens, table_pages, starts != nullptr, (flags & 2) != 0};
  // 16-byte row pieces; a page's byte offsets fit 32 bits
  if (!call_fits(p, z, scale, flags) || !shape_fits(scale, cap, slopes, window) || ((kv_token_stride | kv_head_stride) & 7) ||
      (kv_token_stride | kv_head_stride) < 0 || kv_token_stride < kHeadDim || kv_token_stride >= (1ll << 24))
    return (int)hipErrorInvalidValue;
  set_shape(&p, scale, cap, slopes, window);
  return run<false, SHAPED>(p, z, scale, flags, workspace, workspace_bytes, stream);
}

template <bool SHAPED>
int attend8(const void* q, long long q_token_stride, long long q_head_stride, const void* cache_k,
            const void* cache_v, long long kv_page_stride, long long kv_head_stride, const void* scales,
            long long scales_page_stride, long long scales_head_stride, const int32_t* prefix, int prefix_tokens,
            const int32_t* table, const int32_t* lengths, const int32_t* starts, void* out,
            long long out_token_stride, long long out_head_stride, float* lse, int tokens, int batch, int heads,
            int kv_heads, int pages, int table_pages, float scale, float cap, const float* slopes, int window,
            int flags, void* workspace, long long workspace_bytes, hipStream_t stream) {
  PagedParams p{};
  p.q = (const uint16_t*)q;
  p.k = cache_k;
  p.v = cache_v;
  p.scales = (const uint8_t*)scales;
  p.out = (uint16_t*)out;
  p.lse = lse;
  p.q_tok = q_token_stride;
  p.q_head = q_head_stride;
  p.o_tok = out_token_stride;
  p.o_head = out_head_stride;
  p.kv_tok = kv_page_stride;
  p.kv_head = kv_head_stride;
  p.s_page = scales_page_stride;
  p.s_head = scales_head_stride;
  p.prefix = prefix;
  p.table = table;
  p.lengths = lengths;
  p.starts = starts;
  p.pages = pages;
  const Sizes z{0, tokens, batch, heads, kv_heads, prefix_tokens, table_pages, starts != nullptr, (flags & 2) != 0};
  // 16-byte pieces of rows, 4-byte pieces of exponents
  if (!call_fits(p, z, scale, flags) || !shape_fits(scale, cap, slopes, window) || !scales || ((uintptr_t)scales & 3) ||
      ((scales_page_stride | scales_head_stride) & 3) || (scales_page_stride | scales_head_stride) < 0 ||
      ((kv_page_stride | kv_head_stride) & 15) || (kv_page_stride | kv_head_stride) < 0)
    return (int)hipErrorInvalidValue;
  set_shape(&p, scale, cap, slopes, window);
  return run<true, SHAPED>(p, z, scale, flags, workspace, workspace_bytes, stream);
}

}  // namespace
