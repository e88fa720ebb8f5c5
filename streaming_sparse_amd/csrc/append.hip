// New tokens of several sequences into a paged K/V cache, queries and keys
// rotated by their positions on the way.
//
// Pair j of a row turns by the angle p * freq_j, p the token's position on the
// pair's axis:
//   y1 = x1 cos - x2 sin,  y2 = x1 sin + x2 cos
// over the elements (2j, 2j + 1) (interleaved) or (j, j + pairs) (halves);
// the other elements are copied bit for bit.  The angle is formed in turns in
// float64 (three roundings, 3 x 2^-53 of it) and reduced to half a turn there, so
// that it keeps 2^-24 of a turn up to 2^27 turns, 2^-23 at the ends of int32 with one
// radian a position, and beyond what float64 holds; sine, cosine and the products
// are float32 and each result is rounded once.
//
// Bound by memory: every element is read and written once.  A wave takes one
// token: each of its 64 lanes forms the sine and cosine of one pair, once per
// token, and the lanes exchange them as their elements need them (16 lanes
// hold a row in 16-byte pieces, so a wave moves four rows per instruction and
// four of those at a time).
#include "common.h"
#include "../../include/ssattn_paged.h"

#include <algorithm>

using namespace ssa;

namespace {

constexpr int kWaves = 4;
constexpr int kRowsPerWave = 16;      // rows a wave has in flight: 4 per instruction

struct AppendParams {
  const uint16_t *q, *k, *v;
  uint16_t *q_out, *cache_k, *cache_v;
  long long q_tok, q_head, o_tok, o_head, k_tok, k_head, v_tok, v_head, kv_tok, kv_head;
  const int32_t *table, *held, *starts, *positions;
  const double* freqs;
  long long first;
  int tokens, batch, per_seq, heads, kv_heads, pages, table_pages, pairs, axis0, axis1, axes, slices;
};

template <bool F16>
__device__ __forceinline__ float lo_of(uint32_t w) {
  if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)w);
  return bf16_lo(w);
}
template <bool F16>
__device__ __forceinline__ float hi_of(uint32_t w) {
  if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
  return bf16_hi(w);
}
template <bool F16>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  if constexpr (F16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    f16x2 r;
    r[0] = (_Float16)lo;
    r[1] = (_Float16)hi;
    return __builtin_bit_cast(uint32_t, r);
  }
  return pack_bf16(lo, hi);
}

__device__ __forceinline__ float from_lane(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_ds_bpermute(lane << 2, __float_as_int(x)));
}

// INTERLEAVED: lane c of a row holds elements 8c .. 8c + 7, pairs 4c .. 4c + 3.
// Otherwise the same elements, whose partners lie pairs / 8 lanes away.
template <bool F16, bool INTERLEAVED>
__global__ __launch_bounds__(64 * kWaves) void append_kernel(AppendParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int t = (int)blockIdx.x * kWaves + wave, slice = blockIdx.y;
  if (t >= p.tokens) return;
  int b, i;
  if (p.starts) {
    // the last sequence that starts at or before t: how many of starts[1..]
    // are at most t
    b = 0;
    for (int c = 0; c < p.batch; c += 64)
      b += (int)__popcll(__ballot(c + lane < p.batch && p.starts[min(c + lane, p.batch - 1) + 1] <= t));
    if (b >= p.batch) return;             // a row behind the last sequence
    i = t - p.starts[b];
    if (i < 0) return;
  } else {
    b = t / p.per_seq;
    i = t - b * p.per_seq;
  }
  const long long at = (long long)p.held[b] + i;
  long long row = -1;                     // cache row, -1: none
  if (at >= 0 && at < 64ll * p.table_pages) {
    const int page = p.table[(long long)b * p.table_pages + (at >> 6)];
    if (page >= 0 && page < p.pages) row = 64ll * page + (at & 63);
  }
  // lane j's pair
  float cs = 1.0f, sn = 0.0f;
  if (lane < p.pairs) {
    double pos;
    if (p.positions) {
      const int axis = (lane >= p.axis0) + (lane >= p.axis0 + p.axis1);
      pos = (double)p.positions[(long long)t * p.axes + axis];
    } else {
      pos = (double)(at + p.first);
    }
    const double turns = pos * (p.freqs[lane] * 0.15915494309189535);   // 1 / (2 pi)
    const float half_turns = (float)(2.0 * (turns - __builtin_rint(turns)));
    sincospif(half_turns, &sn, &cs);
  }
  const int c = lane & 15, sub = lane >> 4;
  constexpr int kNeed = INTERLEAVED ? 4 : 8;
  // the sines and cosines of this lane's elements; in halves, the second half's
  // lanes take the negated sine: y2 = x2 cos - x1 (-sin)
  const int half_lanes = p.pairs >> 3;
  const bool second = !INTERLEAVED && c >= half_lanes;
  const int pair0 = INTERLEAVED ? 4 * c : 8 * (second ? c - half_lanes : c);
  const int partner = (lane & 48) | ((second ? c - half_lanes : c + half_lanes) & 15);
  float C[kNeed], S[kNeed];
#pragma unroll
  for (int e = 0; e < kNeed; ++e) {
    C[e] = from_lane(cs, (pair0 + e) & 63);
    S[e] = from_lane(sn, (pair0 + e) & 63);
    if (second) S[e] = -S[e];
  }
  // pairs of this lane that turn (halves: pairs is a multiple of 8, so all or none)
  const int turning = INTERLEAVED ? p.pairs - 4 * c : (c < 2 * half_lanes ? 8 : 0);

  const int rows = p.heads + 2 * p.kv_heads;
  for (int r0 = slice * kRowsPerWave; r0 < rows; r0 += kRowsPerWave * p.slices) {
    u32x4 x[4];
    uint16_t* to[4];
    bool turn[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = r0 + 4 * u + sub;
      x[u] = u32x4{};
      to[u] = nullptr;
      turn[u] = r < p.heads + p.kv_heads;
      if (r < p.heads) {
        x[u] = ldg16(p.q + (long long)t * p.q_tok + (long long)r * p.q_head + 8 * c);
        to[u] = p.q_out + (long long)t * p.o_tok + (long long)r * p.o_head + 8 * c;
      } else if (r < rows && row >= 0) {
        const bool is_v = !turn[u];
        const int h = r - p.heads - (is_v ? p.kv_heads : 0);
        const uint16_t* from = is_v ? p.v + (long long)t * p.v_tok + (long long)h * p.v_head
                                    : p.k + (long long)t * p.k_tok + (long long)h * p.k_head;
        x[u] = ldg16(from + 8 * c);
        to[u] = (is_v ? p.cache_v : p.cache_k) + row * p.kv_tok + (long long)h * p.kv_head + 8 * c;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      u32x4 y = x[u];
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = lo_of<F16>(x[u][e]), d = hi_of<F16>(x[u][e]);
          const uint32_t w = pack<F16>(a * C[e] - d * S[e], a * S[e] + d * C[e]);
          y[e] = turn[u] && e < turning ? w : y[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t o = (uint32_t)__builtin_amdgcn_ds_bpermute(partner << 2, (int)x[u][e]);
          const uint32_t w = pack<F16>(lo_of<F16>(x[u][e]) * C[2 * e] - lo_of<F16>(o) * S[2 * e],
                                       hi_of<F16>(x[u][e]) * C[2 * e + 1] - hi_of<F16>(o) * S[2 * e + 1]);
          y[e] = turn[u] && turning ? w : y[e];
        }
      }
      // past the L2, which the rows of a large call would only sweep: 36864
      // tokens x 36 rows 135.1 -> 128.9 us, ragged 7839 x 36 (fp16) 33.1 -> 23.4;
      // an attention right behind, which then reads them from further off, takes
      // as much longer where all fits the caches (append and attention of 4608
      // tokens 242.7 and 243.2 us)
      if (to[u]) __builtin_nontemporal_store(y, reinterpret_cast<u32x4*>(to[u]));
    }
  }
}

// Over how many waves a token's rows are spread: enough that about 12,000 waves
// share the work (12 a SIMD), no more than have 16 rows each.  One wave a token
// leaves a chunk of 4608 tokens x 36 rows with 4.5 a SIMD, too few to hide the
// loads' latency: 18.1 us, with three 16.0; 36864 tokens 135.1 us with one, 137.2
// with three.
int wave_slices(int tokens, int rows) {
  const int most = (rows + kRowsPerWave - 1) / kRowsPerWave;
  return std::max(1, std::min(most, (12288 + tokens - 1) / tokens));
}

}  // namespace

extern "C" int ssa_paged_append(const void* q, long long q_token_stride, long long q_head_stride, void* q_out,
                                long long out_token_stride, long long out_head_stride, const void* k,
                                long long k_token_stride, long long k_head_stride, const void* v,
                                long long v_token_stride, long long v_head_stride, void* cache_k, void* cache_v,
                                long long kv_token_stride, long long kv_head_stride, const int32_t* table,
                                const int32_t* held, const int32_t* starts, const int32_t* positions,
                                const double* freqs, long long first, int tokens, int batch, int heads, int kv_heads,
                                int pages, int table_pages, int pairs, int axis0, int axis1, int axes, int flags,
                                hipStream_t stream) {
  const bool interleaved = flags & 2;
  // a grid holds less than 2^32 threads
  constexpr int kMostTokens = kWaves * (int)(((1ll << 32) - 1) / (64 * kWaves));
  if (tokens < 0 || tokens > kMostTokens || batch <= 0 || heads < 0 || kv_heads <= 0 ||
      heads + 2ll * kv_heads > 65536 || pages <= 0 || table_pages <= 0 || (!starts && tokens % batch) || (flags & ~3))
    return (int)hipErrorInvalidValue;
  if (pairs < 0 || pairs > kHeadDim / 2 || (!interleaved && pairs % 8) || (pairs > 0 && !freqs) || axes < 1 ||
      axes > 3 || axis0 < 0 || axis1 < 0 || axis0 > pairs - axis1 || (axes > 1 && !positions && pairs > 0))
    return (int)hipErrorInvalidValue;
  // beyond, float64 does not hold every position
  if (first > 1ll << 53 || first < -(1ll << 53)) return (int)hipErrorInvalidValue;
  // pairs behind the counts turn on the next axis, which positions must hold
  if (positions && pairs > 0 && ((axes == 1 && axis0 != pairs) || (axes == 2 && axis0 + axis1 != pairs)))
    return (int)hipErrorInvalidValue;
  if (!k || !v || !cache_k || !cache_v || !table || !held || (heads > 0 && (!q || !q_out)))
    return (int)hipErrorInvalidValue;
  // 16-byte row pieces
  const long long strides = k_token_stride | k_head_stride | v_token_stride | v_head_stride | kv_token_stride |
                            kv_head_stride |
                            (heads ? q_token_stride | q_head_stride | out_token_stride | out_head_stride : 0);
  const uintptr_t ptrs = (uintptr_t)k | (uintptr_t)v | (uintptr_t)cache_k | (uintptr_t)cache_v |
                         (heads ? (uintptr_t)q | (uintptr_t)q_out : 0);
  if ((strides & 7) || strides < 0 || kv_token_stride < kHeadDim || (ptrs & 15)) return (int)hipErrorInvalidValue;
  if (tokens == 0) return (int)hipSuccess;
  AppendParams p;
  p.q = (const uint16_t*)q;
  p.k = (const uint16_t*)k;
  p.v = (const uint16_t*)v;
  p.q_out = (uint16_t*)q_out;
  p.cache_k = (uint16_t*)cache_k;
  p.cache_v = (uint16_t*)cache_v;
  p.q_tok = q_token_stride;
  p.q_head = q_head_stride;
  p.o_tok = out_token_stride;
  p.o_head = out_head_stride;
  p.k_tok = k_token_stride;
  p.k_head = k_head_stride;
  p.v_tok = v_token_stride;
  p.v_head = v_head_stride;
  p.kv_tok = kv_token_stride;
  p.kv_head = kv_head_stride;
  p.table = table;
  p.held = held;
  p.starts = starts;
  p.positions = positions;
  p.freqs = freqs;
  p.first = first;
  p.tokens = tokens;
  p.batch = batch;
  p.per_seq = starts ? 0 : tokens / batch;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.pages = pages;
  p.table_pages = table_pages;
  p.pairs = pairs;
  p.axis0 = axis0;
  p.axis1 = axis1;
  p.axes = axes;
  p.slices = wave_slices(tokens, heads + 2 * kv_heads);
  const dim3 grid((tokens - 1) / kWaves + 1, p.slices);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, stream, p); };
  if (flags & 1)
    interleaved ? launch(append_kernel<true, true>) : launch(append_kernel<true, false>);
  else
    interleaved ? launch(append_kernel<false, true>) : launch(append_kernel<false, false>);
  return (int)hipGetLastError();
}
