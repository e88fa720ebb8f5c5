// Attention of a batch of sequences behind a prefix they share, over a paged
// K/V cache.
//
// Query rows of one K/V head are numbered rho = token * group + query head
// within the group (group = heads / kv_heads), over the packed tokens of all
// sequences; a tile is a run of rows.  Its keys are the prefix's rows, then
// those of its sequence; one running maximum m and sum l per row,
//   O = sum_j 2^(s_j - m) v_j,  l = sum_j 2^(s_j - m),  s_j = scale log2(e) q.k_j,
// out = O / l, lse = ln 2 (m + log2 l).  A list of keys may be cut into pieces,
// each leaving its (O, m, l), joined by
//   M = max m_i, out = sum O_i 2^(m_i - M) / sum l_i 2^(m_i - M).
//
// The prefix is the same for every row, so where sequences bring few rows each,
// the rows of ALL sequences walk it together in tiles of their own (each page is
// read once per tile instead of once per sequence), and a sequence's own pages
// are further pieces of its rows.  Where a sequence fills tiles by itself, its
// tiles walk prefix and own pages in one list.
#include "common.h"
#include "../../include/ssattn_paged.h"

#include <algorithm>

using namespace ssa;

namespace {

typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

constexpr int kPage = 64;

struct PagedParams {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  float* lse;
  long long q_tok, q_head, o_tok, o_head, kv_tok, kv_head;
  const int32_t *prefix, *table, *lengths, *starts;
  float* part;
  int tokens, batch, per_seq, heads, kv_heads, group, pages, prefix_tokens, table_pages, causal;
  float scale_log2;
  int row_tiles;      // 32-row tiles of a K/V head's rows: the states' layout
  // Work items of the launch, prefix items first: prefix_tiles tiles per K/V
  // head (of all sequences' rows), each in prefix_pieces pieces; then
  // own_tiles tiles per K/V head (of one sequence's rows) in own_pieces pieces,
  // which walk the prefix too where there are no prefix items.
  int prefix_tiles, prefix_pieces, own_tiles, own_pieces;
};

// A piece's state of 32 rows: O [dim / 4][row] of 4 floats (dim / 4 = 8 dt + 2 j
// + hh), m [32], l [32].  Piece c of K/V head h, rows 32 T .. at ((c * kv_heads +
// h) * row_tiles + T) * kState.
constexpr int kState = 32 * kHeadDim + 64;

template <bool F16>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return mfma32(a, b, c);
}

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (F16) {
    f16x2 r;
    r[0] = (_Float16)lo;
    r[1] = (_Float16)hi;
    return __builtin_bit_cast(uint32_t, r);
  }
  return pack_bf16(lo, hi);
}

// The two 16-bit parts of a pair of probabilities: hi the rounded pair, lo what
// the rounding left (the empty asm keeps the compiler from converting twice).
template <bool F16>
__device__ __forceinline__ u32x2 split2(float p0, float p1) {
  uint32_t hi = pack2<F16>(p0, p1);
  asm volatile("" : "+v"(hi));
  float h0, h1;
  if constexpr (F16) {
    const f16x2 h = __builtin_bit_cast(f16x2, hi);
    h0 = (float)h[0];
    h1 = (float)h[1];
  } else {
    h0 = bf16_lo(hi);
    h1 = bf16_hi(hi);
  }
  return u32x2{hi, pack2<F16>(p0 - h0, p1 - h1)};
}

// Probabilities are 2^(s - m + kLift).  The accumulator is rescaled only when a
// row's maximum has grown by more than kSlack, so they stay below 2^(kSlack +
// kLift): bf16 has fp32's range and needs no lift; fp16 probabilities are lifted
// to 2^7 .. 2^15, so that those down to 2^-21 of the largest keep all their bits
// and those down to 2^-31 some of them.
constexpr float kSlack = 8.0f;
template <bool F16>
constexpr float kLift = F16 ? 7.0f : 0.0f;

// 16-byte chunk c of a K row r lies at chunk c ^ (r & 15); of a V row at c ^
// vswz(r), which keeps the transposing reads of four rows on distinct banks.
__device__ __forceinline__ int vswz(int row) { return (0xEA40 >> (4 * (row & 3))) & 15; }   // 0, 4, 10, 14

__device__ __forceinline__ float max3f(float a, float b, float c) { return __builtin_fmaxf(__builtin_fmaxf(a, b), c); }

// Maximum of a lane's 16 scores and its other half's (lane ^ 32: the other keys
// of the same row).
__device__ __forceinline__ float row_max(const f32x16& S) {
  const float a = max3f(S[0], S[1], S[2]), b = max3f(S[3], S[4], S[5]), c = max3f(S[6], S[7], S[8]);
  const float d = max3f(S[9], S[10], S[11]), e = max3f(S[12], S[13], S[14]);
  const float mx = __builtin_fmaxf(max3f(a, b, c), max3f(d, e, S[15]));
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
  return __builtin_fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}

__device__ __forceinline__ float half_sum(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}

__device__ __forceinline__ u32x4 tr_pair(const lds_u8* a, const lds_u8* b) {
  const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)a));
  const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)b));
  return u32x4{x[0], x[1], y[0], y[1]};
}

// One tile of work, the same for all lanes.
struct Job {
  int h;              // K/V head
  int rho0, rho1;     // rows
  int piece, pieces, state;   // this piece of the list; the state index it is written to, -1: out
  int b, n, length, first_token;   // the rows' sequence: new tokens, rows in the cache, first packed token
  int prefix_pages, own_pages;     // pages of the list
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

// Sequence and tile of the idx-th tile of T rows, sequence by sequence (each
// sequence's last tile may be short); b = -1 behind the last.  One pass per 64
// sequences: every lane counts one sequence's tiles, a wave scan sums them.
struct SeqTile {
  int b, tile, start, n;
};
__device__ __forceinline__ SeqTile find_tile(const PagedParams& p, int idx, int T, int lane) {
  if (!p.starts) {
    const int each = (p.per_seq * p.group + T - 1) / T, b = idx / each;
    if (b >= p.batch) return SeqTile{-1, 0, 0, 0};
    return SeqTile{b, idx - b * each, b * p.per_seq, p.per_seq};
  }
  int base = 0;
  for (int c = 0; c < p.batch; c += 64) {
    const int b = min(c + lane, p.batch - 1);
    const int s0 = clampi(p.starts[b], 0, p.tokens), s1 = clampi(p.starts[b + 1], 0, p.tokens);
    const int n = c + lane < p.batch ? max(s1 - s0, 0) : 0;
    const int tiles = (int)(((long long)n * p.group + T - 1) / T);
    int sum = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int below = __shfl_up(sum, o);
      if (lane >= o) sum += below;
    }
    const unsigned long long past = __ballot(base + sum > idx);
    if (past) {
      const int l = __ffsll((long long)past) - 1;
      const int before = base + __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l);
      return SeqTile{c + l, idx - before, __builtin_amdgcn_readlane(s0, l), __builtin_amdgcn_readlane(n, l)};
    }
    base += __builtin_amdgcn_readlane(sum, 63);
  }
  return SeqTile{-1, 0, 0, 0};
}

// Packed tokens of all sequences.
__device__ __forceinline__ int packed_tokens(const PagedParams& p) {
  return p.starts ? clampi(p.starts[p.batch], 0, p.tokens) : p.tokens;
}

// The job of work item `item` for tiles of T rows; false: nothing to do.
template <int T>
__device__ __forceinline__ bool find_job(const PagedParams& p, int item, int lane, Job& j) {
  const int prefix_items = p.kv_heads * p.prefix_tiles * p.prefix_pieces;
  const int all_prefix = (p.prefix_tokens + kPage - 1) / kPage;
  j.b = -1;
  j.n = j.length = j.first_token = 0;
  if (item < prefix_items) {
    const int tp = item / p.prefix_pieces;
    j.piece = item - tp * p.prefix_pieces;
    j.h = tp / p.prefix_tiles;
    j.rho0 = (tp - j.h * p.prefix_tiles) * T;
    j.rho1 = min(j.rho0 + T, packed_tokens(p) * p.group);
    j.pieces = p.prefix_pieces;
    j.state = j.piece;
    j.prefix_pages = all_prefix;
    j.own_pages = 0;
    return j.rho0 < j.rho1;
  }
  const int tp = (item - prefix_items) / p.own_pieces;
  j.piece = item - prefix_items - tp * p.own_pieces;
  j.h = tp / p.own_tiles;
  const SeqTile s = find_tile(p, tp - j.h * p.own_tiles, T, lane);
  if (s.b < 0) return false;
  j.b = s.b;
  j.n = s.n;
  j.first_token = s.start;
  j.length = clampi(p.lengths[s.b], 0, kPage * p.table_pages);
  j.rho0 = s.start * p.group + s.tile * T;
  j.rho1 = min(j.rho0 + T, (s.start + s.n) * p.group);
  j.pieces = p.own_pieces;
  j.state = prefix_items || p.own_pieces > 1 ? p.prefix_pieces + j.piece : -1;
  j.prefix_pages = prefix_items ? 0 : all_prefix;
  // rows the tile's last query sees
  int seen = j.length;
  if (p.causal) seen = clampi(j.length - j.n + (j.rho1 - 1) / p.group - j.first_token + 1, 0, j.length);
  j.own_pages = (seen + kPage - 1) / kPage;
  return j.rho0 < j.rho1;
}

// The pages of a job's list, walked upwards: lane l holds page base + l of the
// list (-1: absent) and of the 64 pages after, so that no step waits for a table
// entry.
struct Unit {
  int page, rows;     // the cache page, and how many of its rows the list holds
};
struct PageList {
  int base, cur, next;
  __device__ __forceinline__ static int fetch(const PagedParams& p, const Job& j, int u) {
    int id = -1;
    if (u < j.prefix_pages)
      id = p.prefix[u];
    else if (u < j.prefix_pages + j.own_pages)
      id = p.table[(long long)j.b * p.table_pages + (u - j.prefix_pages)];
    return id >= 0 && id < p.pages ? id : -1;
  }
  __device__ __forceinline__ PageList(const PagedParams& p, const Job& j, int first, int lane)
      : base(first), cur(fetch(p, j, first + lane)), next(fetch(p, j, first + 64 + lane)) {}
  // page u of the list; u never decreases by more than the list's base
  __device__ __forceinline__ Unit at(const PagedParams& p, const Job& j, int u, int lane) {
    if (u - base >= 64) {
      base += 64;
      cur = next;
      next = fetch(p, j, base + 64 + lane);
    }
    Unit r;
    r.page = __builtin_amdgcn_readlane(cur, u - base);
    r.rows = min(u < j.prefix_pages ? p.prefix_tokens - kPage * u : j.length - kPage * (u - j.prefix_pages), kPage);
    if (r.page < 0) r.rows = 0;
    return r;
  }
};

// ---------------------------------------------------------------------------
// Narrow tiles: 32 rows.  Bound by the pages' way from memory, so the four waves
// of a workgroup walk the list by themselves, 32 keys at a time: wave w takes
// half pages w, w + 4, ..., its K and V rows going straight to two LDS slots of
// its own (32 KB a wave) while it computes on the other, with no barrier before
// the end, where the four states are joined.  The matrix pipe has time to spare:
// probabilities meet V in two parts (hi + lo), so that no rounding of theirs
// shows in the output.
constexpr int kNarrow = 32, kNarrowWaves = 4;
constexpr int kHalf = 32 * 256;      // 32 rows of K or V

template <bool F16>
__global__ __launch_bounds__(64 * kNarrowWaves) void narrow_kernel(PagedParams p) {
  __shared__ alignas(16) uint8_t ring[kNarrowWaves * 4 * kHalf];   // per wave: K, V of slot 0, K, V of slot 1
  __shared__ float xm[kNarrowWaves][32], xl[kNarrowWaves][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  Job j;
  if (!find_job<kNarrow>(p, xcd_remap(blockIdx.x, gridDim.x), lane, j)) return;
  const int r = lane & 31, hh = lane >> 5;
  const int rho = j.rho0 + r;
  const bool live = rho < j.rho1;
  const int token = min(rho, j.rho1 - 1) / p.group, hq = j.h * p.group + min(rho, j.rho1 - 1) % p.group;
  // rows of its sequence that this row sees
  const int limit = p.causal ? j.length - j.n + (token - j.first_token) + 1 : j.length;

  // half pages [begin, end) of the list, every fourth from begin + wave
  const int units = j.prefix_pages + j.own_pages;
  const int begin = 2 * (int)((long long)units * j.piece / j.pieces);
  const int end = 2 * (int)((long long)units * (j.piece + 1) / j.pieces);

  lds_u8* const base = (lds_u8*)ring + wave * (4 * kHalf);
  // per-lane byte offsets of 16 rows' loads (instruction form: load jj leaves
  // out the 1024 jj that its offset field adds)
  uint32_t koff[4], voff[4];
#pragma unroll
  for (int jj = 0; jj < 4; ++jj) {
    const int row = 4 * jj + (lane >> 4), c = lane & 15;
    const uint32_t at = (uint32_t)(row * p.kv_tok);
    koff[jj] = 2u * (at + 8u * (uint32_t)(c ^ row)) - 1024u * jj;
    voff[jj] = 2u * (at + 8u * (uint32_t)(c ^ vswz(row))) - 1024u * jj;
  }
  const long long rows16 = 32 * p.kv_tok;       // bytes of 16 rows
  const uint8_t* const kh = (const uint8_t*)(p.k + (long long)j.h * p.kv_head);
  const uint8_t* const vh = (const uint8_t*)(p.v + (long long)j.h * p.kv_head);
  auto issue = [&](const Unit& u, int hu, int slot) {
    // an absent page reads page 0: its rows are masked and its values cleared
    const long long at = (4ll * max(u.page, 0) + 2 * (hu & 1)) * rows16;
    const uint32_t l = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)base + slot * (2 * kHalf));
    dma_rows<4>(kh + at, koff, l);
    dma_rows<4>(kh + at + rows16, koff, l + 4096);
    dma_rows<4>(vh + at, voff, l + kHalf);
    dma_rows<4>(vh + at + rows16, voff, l + kHalf + 4096);
  };

  f32x16 O[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) O[dt] = f32x16{};
  float m = -INFINITY, ls = 0.0f;
  int hu = begin + wave;
  PageList list(p, j, hu >> 1, lane);
  Unit u0{-1, 0}, u1{-1, 0};
  if (hu < end) {
    u0 = list.at(p, j, hu >> 1, lane);
    issue(u0, hu, 0);
  }
  if (hu + kNarrowWaves < end) {
    u1 = list.at(p, j, (hu + kNarrowWaves) >> 1, lane);
    issue(u1, hu + kNarrowWaves, 1);
  }
  u32x4 qop[8];
  {
    const uint16_t* qp = p.q + (long long)token * p.q_tok + (long long)hq * p.q_head + 8 * hh;
#pragma unroll
    for (int st = 0; st < 8; ++st) qop[st] = ldg16(qp + 16 * st);
  }
  // everything so far, once and in a form the compiler counts: it does not
  // know of the loads above, and would wait for the query rows in every step
  wait_loads();
  for (int slot = 0; hu < end; hu += kNarrowWaves, slot ^= 1) {
    const bool more = hu + kNarrowWaves < end;
    const lds_u8* kb = base + slot * (2 * kHalf);
    lds_u8* vb = base + slot * (2 * kHalf) + kHalf;
    // K landed: at most this slot's V and the next slot's 16 loads are out
    if (more)
      asm volatile("s_waitcnt vmcnt(24)" ::: "memory");
    else
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    f32x16 S = {};
#pragma unroll
    for (int st = 0; st < 8; ++st) {
      const u32x4 a = *(lds_u32x4*)(kb + r * 256 + (((2 * st + hh) ^ (r & 15)) << 4));
      S = mma<F16>(a, qop[st], S);
    }
    // keys of this half page that the row sees; S[i] is key 8 (i / 4) + 4 hh + i % 4
    const int rows = u0.rows - 32 * (hu & 1);
    int see = rows;
    if ((hu >> 1) >= j.prefix_pages) see = min(see, limit - 32 * (hu - 2 * j.prefix_pages));
    if (!__all(see >= 32)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) S[i] = 8 * (i / 4) + 4 * hh + i % 4 < see ? S[i] : -INFINITY;
    }
    const float mx = row_max(S) * p.scale_log2;
    if (__any(mx > m + kSlack)) {
      const float to = __builtin_fmaxf(m, mx);
      const float a = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.0f : to));
      ls *= a;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) O[dt] *= a;
      m = to;
    }
    const float nb = kLift<F16> - (m == -INFINITY ? 0.0f : m);
    float P[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      P[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], p.scale_log2, nb));
      ls += P[i];
    }
    if (more)
      asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (rows < 32) {
      // rows behind the end hold anything: 0 * NaN must not reach the sums
#pragma unroll
      for (int jj = 0; jj < 8; ++jj)
        if (4 * jj + (lane >> 4) >= rows) *(lds_u32x4*)(vb + jj * 1024 + lane * 16) = u32x4{};
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      u32x4 hi, lo;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const u32x2 x = split2<F16>(P[8 * ks + 2 * w], P[8 * ks + 2 * w + 1]);
        hi[w] = x[0];
        lo[w] = x[1];
      }
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        // dims 32 dt + lane % 32 of keys 16 ks + 8 (e / 4) + 4 hh + e % 4
        const int g = lane >> 4, i = lane & 15;
        const int chunk = 4 * dt + 2 * (g & 1) + ((i & 3) >> 1), row = 16 * ks + 4 * (g >> 1) + (i >> 2);
        const lds_u8* a = vb + row * 256 + ((chunk ^ vswz(row)) << 4) + (i & 1) * 8;
        const u32x4 va = tr_pair(a, a + 2048);
        O[dt] = mma<F16>(va, hi, O[dt]);
        O[dt] = mma<F16>(va, lo, O[dt]);
      }
    }
    // this slot's reads are done before its next rows land
    u0 = u1;
    if (hu + 2 * kNarrowWaves < end) {
      u1 = list.at(p, j, (hu + 2 * kNarrowWaves) >> 1, lane);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      issue(u1, hu + 2 * kNarrowWaves, slot);
    }
  }

  // the four waves' states into one: the sums of a row's two half waves first
  const float l = half_sum(ls);
  const float mine = m == -INFINITY ? m : m - kLift<F16>;
  if (hh == 0) {
    xm[wave][r] = mine;
    xl[wave][r] = l;
  }
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kNarrowWaves; ++w) M = __builtin_fmaxf(M, xm[w][r]);
  const float Mu = M == -INFINITY ? 0.0f : M;
  float L = 0.0f;
#pragma unroll
  for (int w = 0; w < kNarrowWaves; ++w) L += xl[w][r] * __builtin_amdgcn_exp2f(xm[w][r] - Mu);
  const float a = __builtin_amdgcn_exp2f(mine - Mu);
  // every wave hands over its 32 x 128 sums, [dim tile][j][lane] of 4 floats,
  // and adds up one dim tile (the rings are free: all loads have landed)
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
  lds_u8* const x = (lds_u8*)ring;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *(lds_f32x4*)(x + wave * 16384 + (dt * 4 + i) * 1024 + lane * 16) =
          f32x4{O[dt][4 * i], O[dt][4 * i + 1], O[dt][4 * i + 2], O[dt][4 * i + 3]} * a;
  __syncthreads();
  f32x4 R[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    R[i] = f32x4{};
#pragma unroll
    for (int w = 0; w < kNarrowWaves; ++w) R[i] += *(lds_f32x4*)(x + w * 16384 + (wave * 4 + i) * 1024 + lane * 16);
  }
  if (!live) return;
  if (j.state >= 0) {
    float* st = p.part + (((long long)j.state * p.kv_heads + j.h) * p.row_tiles + (rho >> 5)) * kState;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<f32x4*>(st + ((8 * wave + 2 * i + hh) * 32 + (rho & 31)) * 4) = R[i];
    if (wave == 0 && hh == 0) {
      st[32 * kHeadDim + (rho & 31)] = M;
      st[32 * kHeadDim + 32 + (rho & 31)] = L;
    }
    return;
  }
  const bool none = __float_as_uint(L) == 0u;
  const float inv = none ? 0.0f : 1.0f / L;
  uint16_t* op = p.out + (long long)token * p.o_tok + (long long)hq * p.o_head + 32 * wave + 4 * hh;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    R[i] *= inv;
    *reinterpret_cast<u32x2*>(op + 8 * i) = u32x2{pack2<F16>(R[i][0], R[i][1]), pack2<F16>(R[i][2], R[i][3])};
  }
  if (p.lse && wave == 0 && hh == 0)
    p.lse[(long long)token * p.heads + hq] = none ? -INFINITY : (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f;
}

// Joins the pieces' states of 32 rows of a K/V head, dims 32 dt ..: block (h,
// tile, dt), wave w takes dims 8 w .. 8 w + 7.  Bound by the latency of its loads:
// those of 8 pieces are out together.
constexpr int kJoin = 8;

template <bool F16>
__global__ __launch_bounds__(256) void join_kernel(PagedParams p, int pieces) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int dt = blockIdx.x & 3, T = (blockIdx.x >> 2) % p.row_tiles, h = (blockIdx.x >> 2) / p.row_tiles;
  const int r = lane & 31, hh = lane >> 5;
  const int rho = 32 * T + r;
  const bool live = rho < packed_tokens(p) * p.group;
  const long long step = (long long)p.kv_heads * p.row_tiles * kState;
  const float* st = p.part + ((long long)h * p.row_tiles + T) * kState;
  float M = -INFINITY, L = 0.0f;
  f32x4 acc = {};
  for (int c = 0; c < pieces; c += kJoin, st += kJoin * step) {
    float m[kJoin], l[kJoin];
    f32x4 o[kJoin];
#pragma unroll
    for (int i = 0; i < kJoin; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
      o[i] = f32x4{};
      if (c + i < pieces && live) {
        m[i] = st[i * step + 32 * kHeadDim + r];
        l[i] = st[i * step + 32 * kHeadDim + 32 + r];
        o[i] = *reinterpret_cast<const f32x4*>(st + i * step + ((8 * dt + 2 * wave + hh) * 32 + r) * 4);
      }
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < kJoin; ++i) top = __builtin_fmaxf(top, m[i]);
    const float ref = top == -INFINITY ? 0.0f : top;
    const float a = __builtin_amdgcn_exp2f(M - ref);
    acc *= a;
    L *= a;
#pragma unroll
    for (int i = 0; i < kJoin; ++i) {
      const float w = __builtin_amdgcn_exp2f(m[i] - ref);
      L += l[i] * w;
      acc += o[i] * w;
    }
    M = top;
  }
  if (!live) return;
  const int token = rho / p.group, hq = h * p.group + rho % p.group;
  const bool none = __float_as_uint(L) == 0u;
  acc *= none ? 0.0f : 1.0f / L;
  *reinterpret_cast<u32x2*>(p.out + (long long)token * p.o_tok + (long long)hq * p.o_head + 32 * dt + 8 * wave + 4 * hh) =
      u32x2{pack2<F16>(acc[0], acc[1]), pack2<F16>(acc[2], acc[3])};
  if (p.lse && dt == 0 && wave == 0 && hh == 0)
    p.lse[(long long)token * p.heads + hq] = none ? -INFINITY : (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f;
}

// How a call is cut up, from sizes alone.
struct Plan {
  int row_tiles, prefix_tiles, prefix_pieces, own_tiles, own_pieces;
  bool split() const { return prefix_tiles > 0 || own_pieces > 1; }
  long long bytes(int kv_heads) const {
    return split() ? 4ll * kState * (prefix_pieces + own_pieces) * kv_heads * row_tiles : 0;
  }
};

bool sizes_fit(int tokens, int batch, int heads, int kv_heads, int prefix_tokens, int table_pages, bool ragged) {
  return tokens > 0 && batch > 0 && kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && prefix_tokens >= 0 &&
         table_pages > 0 && (ragged || tokens % batch == 0) && (long long)tokens * heads < (1ll << 31) &&
         (long long)table_pages * kPage < (1ll << 30) && prefix_tokens < (1 << 30) && batch <= (1 << 20);
}

int make_plan(int tokens, int batch, int heads, int kv_heads, int prefix_tokens, int table_pages, bool ragged,
              Plan* plan) {
  int cus = 0;
  const int e = device_cus(&cus);
  if (e != (int)hipSuccess) return e;
  const int group = heads / kv_heads;
  const long long rows = (long long)tokens * group;
  const int prefix_pages = (prefix_tokens + kPage - 1) / kPage;
  plan->row_tiles = (int)((rows + 31) / 32);
  const long long own_tiles =
      ragged ? rows / kNarrow + batch : (long long)batch * ((rows / batch + kNarrow - 1) / kNarrow);
  plan->own_tiles = (int)own_tiles;
  const bool together = batch > 1 && prefix_pages > 0 && rows < 32ll * batch;
  auto pieces = [&](long long tiles, int units) {
    const long long fill = std::max(1ll, cus / std::max(1ll, tiles));
    return (int)std::min(fill, (long long)std::max(1, units / 4));
  };
  plan->prefix_tiles = together ? plan->row_tiles : 0;
  plan->prefix_pieces = together ? pieces((long long)kv_heads * plan->prefix_tiles, prefix_pages) : 0;
  plan->own_pieces = pieces(kv_heads * own_tiles, table_pages + (together ? 0 : prefix_pages));
  return (int)hipSuccess;
}

}  // namespace

extern "C" {

long long ssa_paged_attention_workspace_bytes(int tokens, int batch, int heads, int kv_heads, int prefix_tokens,
                                              int table_pages, int ragged) {
  Plan plan;
  if (!sizes_fit(tokens, batch, heads, kv_heads, prefix_tokens, table_pages, ragged != 0) ||
      make_plan(tokens, batch, heads, kv_heads, prefix_tokens, table_pages, ragged != 0, &plan) != (int)hipSuccess)
    return -1;
  return plan.bytes(kv_heads);
}

int ssa_paged_attention(const void* q, long long q_token_stride, long long q_head_stride, const void* cache_k,
                        const void* cache_v, long long kv_token_stride, long long kv_head_stride,
                        const int32_t* prefix, int prefix_tokens, const int32_t* table, const int32_t* lengths,
                        const int32_t* starts, void* out, long long out_token_stride, long long out_head_stride,
                        float* lse, int tokens, int batch, int heads, int kv_heads, int pages, int table_pages,
                        float scale, int flags, void* workspace, long long workspace_bytes, hipStream_t stream) {
  if (!sizes_fit(tokens, batch, heads, kv_heads, prefix_tokens, table_pages, starts != nullptr) || pages <= 0 ||
      (flags & ~3) || !(scale > 0.0f))
    return (int)hipErrorInvalidValue;
  if (!q || !cache_k || !cache_v || !table || !lengths || !out || (prefix_tokens > 0 && !prefix))
    return (int)hipErrorInvalidValue;
  // 16-byte row pieces; a page's byte offsets fit 32 bits
  const long long strides = q_token_stride | q_head_stride | kv_token_stride | kv_head_stride | out_token_stride |
                            out_head_stride;
  if ((strides & 7) || strides < 0 || kv_token_stride < kHeadDim || kv_token_stride >= (1ll << 24) ||
      (((uintptr_t)q | (uintptr_t)cache_k | (uintptr_t)cache_v | (uintptr_t)out) & 15) || ((uintptr_t)lse & 3))
    return (int)hipErrorInvalidValue;
  Plan plan;
  const int e = make_plan(tokens, batch, heads, kv_heads, prefix_tokens, table_pages, starts != nullptr, &plan);
  if (e != (int)hipSuccess) return e;
  const long long need = plan.bytes(kv_heads);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
    return (int)hipErrorInvalidValue;
  PagedParams p;
  p.q = (const uint16_t*)q;
  p.k = (const uint16_t*)cache_k;
  p.v = (const uint16_t*)cache_v;
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
  p.part = (float*)workspace;
  p.tokens = tokens;
  p.batch = batch;
  p.per_seq = starts ? 0 : tokens / batch;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.pages = pages;
  p.prefix_tokens = prefix_tokens;
  p.table_pages = table_pages;
  p.causal = (flags & 2) != 0;
  p.scale_log2 = scale * kLog2e;
  p.row_tiles = plan.row_tiles;
  p.prefix_tiles = plan.prefix_tiles;
  p.prefix_pieces = plan.prefix_pieces;
  p.own_tiles = plan.own_tiles;
  p.own_pieces = plan.own_pieces;
  const long long items = (long long)kv_heads * (1ll * plan.prefix_tiles * plan.prefix_pieces +
                                                 1ll * plan.own_tiles * plan.own_pieces);
  if (items > 0x7fffffffll || 4ll * kv_heads * plan.row_tiles > 0x7fffffffll) return (int)hipErrorInvalidValue;
  const bool f16 = flags & 1;
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)items), dim3(64 * kNarrowWaves), 0, stream, p);
  };
  f16 ? launch(narrow_kernel<true>) : launch(narrow_kernel<false>);
  if (plan.split()) {
    const dim3 grid(4 * kv_heads * plan.row_tiles);
    const int pieces = plan.prefix_pieces + plan.own_pieces;
    if (f16)
      hipLaunchKernelGGL(join_kernel<true>, grid, dim3(256), 0, stream, p, pieces);
    else
      hipLaunchKernelGGL(join_kernel<false>, grid, dim3(256), 0, stream, p, pieces);
  }
  return (int)hipGetLastError();
}

}  // extern "C"
