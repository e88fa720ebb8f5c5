// New tokens of several sequences into a paged K/V cache, queries and keys
// rotated by their positions on the way; into one of 8-bit rows, quantised too; and
// rows of such a cache read back.
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
//
// An 8-bit row is e4m3 values and one power of two: of the row as the 16-bit cache would
// hold it, the smallest 2^e (e >= -126) with max |x| <= 448 2^e; values are rounded to
// nearest, ties to even.  A larger mantissa than the format's would gain nothing from a
// finer scale: its four bits are relative, and the values down to 2^-13 of the largest
// keep all of them.  With powers of two the way back is exact.
#include "common.h"
#include "../../include/ssattn_paged.h"
#include "../../include/ssattn_paged8.h"

#include <algorithm>

using namespace ssa;

namespace {

constexpr int kWaves = 4;
constexpr int kRowsPerWave = 16;      // rows a wave has in flight: 4 per instruction

struct AppendParams {
  const uint16_t *q, *k, *v;
  uint16_t* q_out;
  void *cache_k, *cache_v;       // 8-bit rows: those of a page and head at page * kv_tok + head * kv_head bytes
  uint8_t* scales;               // and their biased exponents, 64 of K and 64 of V, at page * s_page + head * s_head
  long long s_page, s_head;
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

__device__ __forceinline__ double from_lane(double x, int lane) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  const uint32_t lo = __builtin_amdgcn_ds_bpermute(lane << 2, (int)(uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_ds_bpermute(lane << 2, (int)(uint32_t)(u >> 32));
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

// Sine and cosine of h half turns, |h| <= 1, to 2^-45: their series about the nearest
// quarter turn.
__device__ __forceinline__ void turn64(double h, double* sine, double* cosine) {
  const double quarter = __builtin_rint(2.0 * h), x = (h - 0.5 * quarter) * 3.141592653589793, t = x * x;
  const double s =
      x * (1 + t * (-1.0 / 6 + t * (1.0 / 120 + t * (-1.0 / 5040 + t * (1.0 / 362880 + t * (-1.0 / 39916800 +
                                                                                        t * (1.0 / 6227020800)))))));
  const double c =
      1 + t * (-1.0 / 2 + t * (1.0 / 24 + t * (-1.0 / 720 + t * (1.0 / 40320 + t * (-1.0 / 3628800 +
                                                                               t * (1.0 / 479001600 - t * (1.0 / 87178291200)))))));
  const int q = (int)quarter;
  const double a = q & 1 ? c : s, b = q & 1 ? s : c;
  *sine = q & 2 ? -a : a;
  *cosine = (q + 1) & 2 ? -b : b;
}

// x in float32 (the empty asm keeps the compiler from rounding it to 16 bits at once, a
// longer sequence with another result where x lies next to a border).
__device__ __forceinline__ float single(double x) {
  float y = (float)x;
  asm volatile("" : "+v"(y));
  return y;
}

// The sequence and place of packed token t among sequences that start at starts[0..] (null:
// per_seq tokens each); false: behind the last one.
__device__ __forceinline__ bool place_of(const int32_t* starts, int batch, int per_seq, int t, int lane, int* b,
                                         int* i) {
  if (starts) {
    // the last sequence that starts at or before t: how many of starts[1..] are at
    // most t
    *b = 0;
    for (int c = 0; c < batch; c += 64)
      *b += (int)__popcll(__ballot(c + lane < batch && starts[min(c + lane, batch - 1) + 1] <= t));
    if (*b >= batch) return false;
    *i = t - starts[*b];
    return *i >= 0;
  }
  *b = t / per_seq;
  *i = t - *b * per_seq;
  return true;
}

// Cache row of a sequence's row `at`, -1: outside its table or the cache.
__device__ __forceinline__ long long cache_row(const int32_t* table, int table_pages, int pages, int b, long long at) {
  if (at < 0 || at >= 64ll * table_pages) return -1;
  const int page = table[(long long)b * table_pages + (at >> 6)];
  return page >= 0 && page < pages ? 64ll * page + (at & 63) : -1;
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// The 8 values that a lane holds of a row (16 lanes) in 8 bits, and the row's biased
// exponent.  Infinities and NaN become NaN and count nothing for the exponent; values that
// would be rounded to the power of two behind the type's largest, fp16's to 65536 and
// bf16's to 2^128, become 15 / 16 of it.
template <bool F16>
__device__ __forceinline__ u32x2 quantise(u32x4 x, uint32_t* exponent) {
  // magnitudes, moved up so that those of infinities and NaN are negative
  constexpr uint16_t kUp = F16 ? 0x0400 : 0x0080;
  constexpr int16_t kLargest = (F16 ? 0x7bbf : 0x7f77) + kUp;      // of those that are not rounded up
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    i16x2 m = __builtin_bit_cast(i16x2, (u16x2)(__builtin_bit_cast(u16x2, x[e] & 0x7fff7fffu) + (u16x2){kUp, kUp}));
    m = __builtin_elementwise_min(m, (i16x2){kLargest, kLargest});
    x[e] = (x[e] & 0x80008000u) | __builtin_bit_cast(uint32_t, (u16x2)(__builtin_bit_cast(u16x2, m) - (u16x2){kUp, kUp}));
    top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(m, __builtin_bit_cast(i16x2, top)));
  }
  int most = max((int)(int16_t)top, (int)(int16_t)(top >> 16));
  most = max(most, rotate_row<0x128>(most));   // row_ror:8
  most = max(most, rotate_row<0x124>(most));   // row_ror:4
  most = max(most, rotate_row<0x122>(most));   // row_ror:2
  most = max(most, rotate_row<0x121>(most));   // row_ror:1
  most = max(most - (int)kUp, 0);
  const uint32_t bits = F16 ? __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)most)) : (uint32_t)most << 16;
  // 448 = 1.75 * 2^8: the sum carries into the exponent where the mantissa is over 1.75
  *exponent = (uint32_t)max((int)((bits + 0x1fffffu) >> 23) - 8, 1);
  const float scale = __uint_as_float(*exponent << 23);
  u32x2 r;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t x0 = x[2 * e], x1 = x[2 * e + 1];
    i16x2 w = {0, 0};
    if constexpr (F16) {
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(f16x2, x0), scale, false);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(f16x2, x1), scale, true);
    } else {
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, x0), scale, false);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, x1), scale, true);
    }
    r[e] = __builtin_bit_cast(uint32_t, w);
  }
  return r;
}

// INTERLEAVED: lane c of a row holds elements 8c .. 8c + 7, pairs 4c .. 4c + 3.
// Otherwise the same elements, whose partners lie pairs / 8 lanes away.
// EIGHT: the cache's rows are of 8 bits.
template <bool F16, bool INTERLEAVED, bool EIGHT>
__global__ __launch_bounds__(64 * kWaves) void append_kernel(AppendParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int t = (int)blockIdx.x * kWaves + wave, slice = blockIdx.y;
  if (t >= p.tokens) return;
  int b, i;
  if (!place_of(p.starts, p.batch, p.per_seq, t, lane, &b, &i)) return;      // a row behind the last sequence
  const long long at = (long long)p.held[b] + i;
  const long long row = cache_row(p.table, p.table_pages, p.pages, b, at);
  // whether this wave's rows hold keys (EIGHT)
  bool has_keys = false;
  if constexpr (EIGHT) {
    for (int r0 = slice * kRowsPerWave; r0 < p.heads + p.kv_heads; r0 += kRowsPerWave * p.slices)
      has_keys |= r0 + kRowsPerWave > p.heads;
  }
  // lane j's pair
  float cs = 1.0f, sn = 0.0f;
  double cs64 = 1.0, sn64 = 0.0;
  if (lane < p.pairs) {
    double pos;
    if (p.positions) {
      const int axis = (lane >= p.axis0) + (lane >= p.axis0 + p.axis1);
      pos = (double)p.positions[(long long)t * p.axes + axis];
    } else {
      pos = (double)(at + p.first);
    }
    const double turns = pos * (p.freqs[lane] * 0.15915494309189535);   // 1 / (2 pi)
    const double half_turns = 2.0 * (turns - __builtin_rint(turns));
    if (EIGHT && has_keys)
      turn64(half_turns, &sn64, &cs64);
    else
      sincospif((float)half_turns, &sn, &cs);
  }
  const int c = lane & 15, sub = lane >> 4;
  constexpr int kNeed = INTERLEAVED ? 4 : 8;
  // the sines and cosines of this lane's elements; in halves, the second half's
  // lanes take the negated sine: y2 = x2 cos - x1 (-sin)
  const int half_lanes = p.pairs >> 3;
  const bool second = !INTERLEAVED && c >= half_lanes;
  const int pair0 = INTERLEAVED ? 4 * c : 8 * (second ? c - half_lanes : c);
  const int partner = (lane & 48) | ((second ? c - half_lanes : c + half_lanes) & 15);
  // 8-bit keys turn in float64: a step of theirs is a sixteenth of a value, and so is what
  // a rounding to the other side of a border costs, which float32 does to one value in
  // 10^5 (36864 tokens x 36 rows 102.3 and 104.1 us, ragged 7839 x 36, fp16, 24.4 and 28.2)
  float C[kNeed], S[kNeed];
  double C64[EIGHT ? kNeed : 1], S64[EIGHT ? kNeed : 1];
  if (EIGHT && has_keys) {
#pragma unroll
    for (int e = 0; e < (EIGHT ? kNeed : 1); ++e) {
      C64[e] = from_lane(cs64, (pair0 + e) & 63);
      S64[e] = from_lane(sn64, (pair0 + e) & 63);
      if (second) S64[e] = -S64[e];
      C[e] = (float)C64[e];
      S[e] = (float)S64[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < kNeed; ++e) {
      C[e] = from_lane(cs, (pair0 + e) & 63);
      S[e] = from_lane(sn, (pair0 + e) & 63);
      if (second) S[e] = -S[e];
    }
  }
  // pairs of this lane that turn (halves: pairs is a multiple of 8, so all or none)
  const int turning = INTERLEAVED ? p.pairs - 4 * c : (c < 2 * half_lanes ? 8 : 0);

  const int rows = p.heads + 2 * p.kv_heads;
  for (int r0 = slice * kRowsPerWave; r0 < rows; r0 += kRowsPerWave * p.slices) {
    u32x4 x[4];
    uint16_t* to[4];
    uint8_t* scale_to[4];      // EIGHT: where a key's or value's exponent goes, the row's own place in `to`
    bool turn[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = r0 + 4 * u + sub;
      x[u] = u32x4{};
      to[u] = nullptr;
      scale_to[u] = nullptr;
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
        void* const cache = is_v ? p.cache_v : p.cache_k;
        if constexpr (EIGHT) {
          to[u] = (uint16_t*)((uint8_t*)cache + (row >> 6) * p.kv_tok + (long long)h * p.kv_head + (row & 63) * kHeadDim +
                              8 * c);
          scale_to[u] = p.scales + (row >> 6) * p.s_page + (long long)h * p.s_head + (is_v ? 64 : 0) + (row & 63);
        } else {
          to[u] = (uint16_t*)cache + row * p.kv_tok + (long long)h * p.kv_head + 8 * c;
        }
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
      if constexpr (EIGHT) {
        // whether some of these four rows are keys
        if (r0 + 4 * u + 3 >= p.heads && r0 + 4 * u < p.heads + p.kv_heads) {
          const bool is_key = turn[u] && r0 + 4 * u + sub >= p.heads;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const double a = lo_of<F16>(x[u][e]), d = hi_of<F16>(x[u][e]);
            uint32_t w;
            if constexpr (INTERLEAVED) {
              w = pack<F16>(single(a * C64[e] - d * S64[e]), single(a * S64[e] + d * C64[e]));
            } else {
              const uint32_t o = (uint32_t)__builtin_amdgcn_ds_bpermute(partner << 2, (int)x[u][e]);
              w = pack<F16>(single(a * C64[2 * e] - lo_of<F16>(o) * S64[2 * e]),
                            single(d * C64[2 * e + 1] - hi_of<F16>(o) * S64[2 * e + 1]));
            }
            y[e] = is_key && (INTERLEAVED ? e < turning : turning > 0) ? w : y[e];
          }
        }
        uint32_t exponent;
        const u32x2 z = quantise<F16>(y, &exponent);
        if (scale_to[u]) {
          *reinterpret_cast<u32x2*>(to[u]) = z;
          if (c == 0) *scale_to[u] = (uint8_t)exponent;
          continue;
        }
      }
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

struct ReadParams {
  const uint8_t *cache_k, *cache_v, *scales;
  long long kv_page, kv_head, s_page, s_head, k_tok, k_head, v_tok, v_head;
  const int32_t *table, *first, *starts;
  uint16_t *k, *v;
  int tokens, batch, per_seq, kv_heads, pages, table_pages, slices;
};

// Rows of an 8-bit cache as 16-bit ones.  Bound by memory: a wave takes one token, 16
// lanes a row (8 bytes in, 16 out), four rows an instruction and four of those at a
// time, as append_kernel.
template <bool F16>
__global__ __launch_bounds__(64 * kWaves) void read_kernel(ReadParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int t = (int)blockIdx.x * kWaves + wave;
  if (t >= p.tokens) return;
  int b, i;
  if (!place_of(p.starts, p.batch, p.per_seq, t, lane, &b, &i)) return;
  const long long row = cache_row(p.table, p.table_pages, p.pages, b, (long long)p.first[b] + i);
  const int c = lane & 15, sub = lane >> 4, rows = 2 * p.kv_heads;
  for (int r0 = blockIdx.y * kRowsPerWave; r0 < rows; r0 += kRowsPerWave * p.slices) {
    u32x2 x[4];
    uint32_t exponent[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = r0 + 4 * u + sub;
      x[u] = u32x2{};
      exponent[u] = 1;
      if (r < rows && row >= 0) {
        const bool is_v = r >= p.kv_heads;
        const int h = is_v ? r - p.kv_heads : r;
        x[u] = *reinterpret_cast<const u32x2*>((is_v ? p.cache_v : p.cache_k) + (row >> 6) * p.kv_page +
                                               (long long)h * p.kv_head + (row & 63) * kHeadDim + 8 * c);
        exponent[u] = p.scales[(row >> 6) * p.s_page + (long long)h * p.s_head + (is_v ? 64 : 0) + (row & 63)];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = r0 + 4 * u + sub;
      if (r >= rows) continue;
      const bool is_v = r >= p.kv_heads;
      const int h = is_v ? r - p.kv_heads : r;
      uint16_t* const to = is_v ? p.v + (long long)t * p.v_tok + (long long)h * p.v_head
                                : p.k + (long long)t * p.k_tok + (long long)h * p.k_head;
      __builtin_nontemporal_store(widen<F16>(x[u][0], x[u][1], __uint_as_float(exponent[u] << 23)),
                                  reinterpret_cast<u32x4*>(to + 8 * c));
    }
  }
}

// A grid holds less than 2^32 threads.
constexpr int kMostTokens = kWaves * (int)(((1ll << 32) - 1) / (64 * kWaves));

// The arguments of an append that do not depend on the cache's form.
bool append_fits(const AppendParams& p, int flags) {
  const bool interleaved = flags & 2;
  if (p.tokens < 0 || p.tokens > kMostTokens || p.batch <= 0 || p.heads < 0 || p.kv_heads <= 0 ||
      p.heads + 2ll * p.kv_heads > 65536 || p.pages <= 0 || p.table_pages <= 0 ||
      (!p.starts && p.tokens % p.batch) || (flags & ~3))
    return false;
  if (p.pairs < 0 || p.pairs > kHeadDim / 2 || (!interleaved && p.pairs % 8) || (p.pairs > 0 && !p.freqs) ||
      p.axes < 1 || p.axes > 3 || p.axis0 < 0 || p.axis1 < 0 || p.axis0 > p.pairs - p.axis1 ||
      (p.axes > 1 && !p.positions && p.pairs > 0))
    return false;
  // beyond, float64 does not hold every position
  if (p.first > 1ll << 53 || p.first < -(1ll << 53)) return false;
  // pairs behind the counts turn on the next axis, which positions must hold
  if (p.positions && p.pairs > 0 &&
      ((p.axes == 1 && p.axis0 != p.pairs) || (p.axes == 2 && p.axis0 + p.axis1 != p.pairs)))
    return false;
  if (!p.k || !p.v || !p.cache_k || !p.cache_v || !p.table || !p.held || (p.heads > 0 && (!p.q || !p.q_out)))
    return false;
  // 16-byte row pieces
  const long long strides = p.k_tok | p.k_head | p.v_tok | p.v_head |
                            (p.heads ? p.q_tok | p.q_head | p.o_tok | p.o_head : 0);
  const uintptr_t ptrs = (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.cache_k | (uintptr_t)p.cache_v |
                         (p.heads ? (uintptr_t)p.q | (uintptr_t)p.q_out : 0);
  return !(strides & 7) && strides >= 0 && !(ptrs & 15);
}

template <bool EIGHT>
int launch_append(AppendParams p, int flags, hipStream_t stream) {
  if (p.tokens == 0) return (int)hipSuccess;
  const bool interleaved = flags & 2;
  p.per_seq = p.starts ? 0 : p.tokens / p.batch;
  p.slices = wave_slices(p.tokens, p.heads + 2 * p.kv_heads);
  const dim3 grid((p.tokens - 1) / kWaves + 1, p.slices);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, stream, p); };
  if (flags & 1)
    interleaved ? launch(append_kernel<true, true, EIGHT>) : launch(append_kernel<true, false, EIGHT>);
  else
    interleaved ? launch(append_kernel<false, true, EIGHT>) : launch(append_kernel<false, false, EIGHT>);
  return (int)hipGetLastError();
}

AppendParams append_params(const void* q, long long q_token_stride, long long q_head_stride, void* q_out,
                           long long out_token_stride, long long out_head_stride, const void* k,
                           long long k_token_stride, long long k_head_stride, const void* v, long long v_token_stride,
                           long long v_head_stride, void* cache_k, void* cache_v, long long kv_stride,
                           long long kv_head_stride, const int32_t* table, const int32_t* held, const int32_t* starts,
                           const int32_t* positions, const double* freqs, long long first, int tokens, int batch,
                           int heads, int kv_heads, int pages, int table_pages, int pairs, int axis0, int axis1,
                           int axes) {
  AppendParams p{};
  p.q = (const uint16_t*)q;
  p.k = (const uint16_t*)k;
  p.v = (const uint16_t*)v;
  p.q_out = (uint16_t*)q_out;
  p.cache_k = cache_k;
  p.cache_v = cache_v;
  p.q_tok = q_token_stride;
  p.q_head = q_head_stride;
  p.o_tok = out_token_stride;
  p.o_head = out_head_stride;
  p.k_tok = k_token_stride;
  p.k_head = k_head_stride;
  p.v_tok = v_token_stride;
  p.v_head = v_head_stride;
  p.kv_tok = kv_stride;
  p.kv_head = kv_head_stride;
  p.table = table;
  p.held = held;
  p.starts = starts;
  p.positions = positions;
  p.freqs = freqs;
  p.first = first;
  p.tokens = tokens;
  p.batch = batch;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.pages = pages;
  p.table_pages = table_pages;
  p.pairs = pairs;
  p.axis0 = axis0;
  p.axis1 = axis1;
  p.axes = axes;
  return p;
}

// Strides of an 8-bit cache: 16-byte pieces of rows, 4-byte pieces of exponents.
bool cache8_fits(const void* cache_k, const void* cache_v, long long page, long long head, const void* scales,
                 long long s_page, long long s_head) {
  return cache_k && cache_v && scales && !(((uintptr_t)cache_k | (uintptr_t)cache_v) & 15) && !((uintptr_t)scales & 3) &&
         !((page | head) & 15) && (page | head) >= 0 && !((s_page | s_head) & 3) && (s_page | s_head) >= 0;
}

}  // namespace

extern "C" {

int ssa_paged_append(const void* q, long long q_token_stride, long long q_head_stride, void* q_out,
                     long long out_token_stride, long long out_head_stride, const void* k, long long k_token_stride,
                     long long k_head_stride, const void* v, long long v_token_stride, long long v_head_stride,
                     void* cache_k, void* cache_v, long long kv_token_stride, long long kv_head_stride,
                     const int32_t* table, const int32_t* held, const int32_t* starts, const int32_t* positions,
                     const double* freqs, long long first, int tokens, int batch, int heads, int kv_heads, int pages,
                     int table_pages, int pairs, int axis0, int axis1, int axes, int flags, hipStream_t stream) {
  const AppendParams p = append_params(
      q, q_token_stride, q_head_stride, q_out, out_token_stride, out_head_stride, k, k_token_stride, k_head_stride, v,
      v_token_stride, v_head_stride, cache_k, cache_v, kv_token_stride, kv_head_stride, table, held, starts, positions,
      freqs, first, tokens, batch, heads, kv_heads, pages, table_pages, pairs, axis0, axis1, axes);
  if (!append_fits(p, flags) || ((kv_token_stride | kv_head_stride) & 7) || (kv_token_stride | kv_head_stride) < 0 ||
      kv_token_stride < kHeadDim)
    return (int)hipErrorInvalidValue;
  return launch_append<false>(p, flags, stream);
}

int ssa_paged8_append(const void* q, long long q_token_stride, long long q_head_stride, void* q_out,
                      long long out_token_stride, long long out_head_stride, const void* k, long long k_token_stride,
                      long long k_head_stride, const void* v, long long v_token_stride, long long v_head_stride,
                      void* cache_k, void* cache_v, long long kv_page_stride, long long kv_head_stride, void* scales,
                      long long scales_page_stride, long long scales_head_stride, const int32_t* table,
                      const int32_t* held, const int32_t* starts, const int32_t* positions, const double* freqs,
                      long long first, int tokens, int batch, int heads, int kv_heads, int pages, int table_pages,
                      int pairs, int axis0, int axis1, int axes, int flags, hipStream_t stream) {
  AppendParams p = append_params(
      q, q_token_stride, q_head_stride, q_out, out_token_stride, out_head_stride, k, k_token_stride, k_head_stride, v,
      v_token_stride, v_head_stride, cache_k, cache_v, kv_page_stride, kv_head_stride, table, held, starts, positions,
      freqs, first, tokens, batch, heads, kv_heads, pages, table_pages, pairs, axis0, axis1, axes);
  p.scales = (uint8_t*)scales;
  p.s_page = scales_page_stride;
  p.s_head = scales_head_stride;
  if (!append_fits(p, flags) || !cache8_fits(cache_k, cache_v, kv_page_stride, kv_head_stride, scales,
                                             scales_page_stride, scales_head_stride))
    return (int)hipErrorInvalidValue;
  return launch_append<true>(p, flags, stream);
}

int ssa_paged8_read(const void* cache_k, const void* cache_v, long long kv_page_stride, long long kv_head_stride,
                    const void* scales, long long scales_page_stride, long long scales_head_stride,
                    const int32_t* table, const int32_t* first, const int32_t* starts, void* k,
                    long long k_token_stride, long long k_head_stride, void* v, long long v_token_stride,
                    long long v_head_stride, int tokens, int batch, int kv_heads, int pages, int table_pages, int flags,
                    hipStream_t stream) {
  const long long strides = k_token_stride | k_head_stride | v_token_stride | v_head_stride;
  if (tokens < 0 || tokens > kMostTokens || batch <= 0 || kv_heads <= 0 || kv_heads > 32768 || pages <= 0 ||
      table_pages <= 0 || (!starts && tokens % batch) || (flags & ~1) || !table || !first || !k || !v ||
      (((uintptr_t)k | (uintptr_t)v) & 15) || (strides & 7) || strides < 0 ||
      !cache8_fits(cache_k, cache_v, kv_page_stride, kv_head_stride, scales, scales_page_stride, scales_head_stride))
    return (int)hipErrorInvalidValue;
  if (tokens == 0) return (int)hipSuccess;
  ReadParams p{};
  p.cache_k = (const uint8_t*)cache_k;
  p.cache_v = (const uint8_t*)cache_v;
  p.scales = (const uint8_t*)scales;
  p.kv_page = kv_page_stride;
  p.kv_head = kv_head_stride;
  p.s_page = scales_page_stride;
  p.s_head = scales_head_stride;
  p.table = table;
  p.first = first;
  p.starts = starts;
  p.k = (uint16_t*)k;
  p.v = (uint16_t*)v;
  p.k_tok = k_token_stride;
  p.k_head = k_head_stride;
  p.v_tok = v_token_stride;
  p.v_head = v_head_stride;
  p.tokens = tokens;
  p.batch = batch;
  p.per_seq = starts ? 0 : tokens / batch;
  p.kv_heads = kv_heads;
  p.pages = pages;
  p.table_pages = table_pages;
  p.slices = wave_slices(tokens, 2 * kv_heads);
  const dim3 grid((tokens - 1) / kWaves + 1, p.slices);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, stream, p); };
  (flags & 1) ? launch(read_kernel<true>) : launch(read_kernel<false>);
  return (int)hipGetLastError();
}

}  // extern "C"
