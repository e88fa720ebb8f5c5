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
#pragma once
#include "common.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

using namespace ssa;

namespace {

typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

constexpr int kPage = 64;
constexpr int kMostRows = (1 << 30) - 1;       // of a sequence, and of a window

// What a kernel is made for: fp16 rows (else bf16), a cache of 8-bit rows (else of
// 16-bit ones in the queries' type), shaped scores (else plain ones), two parts of a
// probability as such (else one of fp16 may stand for two of bf16 over 8-bit rows).
template <bool F16_, bool Q8_, bool SHAPED_, bool BOTH_ = false>
struct Mode {
  static constexpr bool F16 = F16_, Q8 = Q8_, SHAPED = SHAPED_, BOTH = BOTH_;
};

struct PagedParams {
  const uint16_t *q;
  // 16-bit rows at row * kv_tok + head * kv_head elements; of an 8-bit cache the 64 rows
  // of 128 bytes of a page and head at page * kv_tok + head * kv_head bytes
  const void *k, *v;
  uint16_t* out;
  float* lse;
  long long q_tok, q_head, o_tok, o_head, kv_tok, kv_head;
  const int32_t *prefix, *table, *lengths, *starts;
  float* part;
  int tokens, batch, per_seq, heads, kv_heads, group, pages, prefix_tokens, table_pages, causal;
  float scale_log2;
  // Work items of the launch: prefix_items of the prefix by itself
  // (prefix_tiles tiles per K/V head, of all sequences' rows, each in
  // prefix_pieces pieces of prefix_cut pages), then those of the sequences:
  // own_tiles tiles per K/V head, the first own_whole of all heads' whole, the
  // others in up to own_pieces pieces of own_cut pages.  They walk the prefix
  // too unless it is `apart`.  longest_first (own_whole 0, or all): the tiles with
  // the longest lists, a causal sequence's last, come first.
  int prefix_items, prefix_tiles, prefix_pieces, prefix_cut, own_tiles, own_whole, own_pieces, own_cut, apart,
      longest_first;
  int log_rows;       // of an own tile's rows (beside prefix tiles they have 32)
  int row_tiles;      // 32-row tiles of a K/V head's rows, where the prefix is apart
  int own_waves;      // and the waves of a workgroup that take own items then
  // 8-bit caches: the biased exponents of a page and head, 64 of K and 64 of V, at page *
  // s_page + head * s_head
  const uint8_t* scales;
  long long s_page, s_head;
  // Shaped scores: cap * log2(e), 0: none, and what a product is multiplied by in the
  // exponent of the tanh; slopes [heads] or null; rows up to itself that a query sees
  // of its sequence, 0: all
  float cap_log2, cap_scale;
  const float* slopes;
  int window;
};

// A piece's state of 32 rows: O [dim / 4][row] of 4 floats, m [32], l [32].  Where
// the prefix is apart, rows keep their places: piece c of K/V head h, rows 32 T ..
// at ((c * kv_heads + h) * row_tiles + T) * kState, the prefix's pieces first.
// Otherwise the tiles behind own_whole have theirs, piece by piece.
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

// Maximum of a lane's 16 scores, and of both lanes that hold a row (l, l ^ 32).
template <typename V>
__device__ __forceinline__ float lane_max(const V& S) {
  const float a = max3f(S[0], S[1], S[2]), b = max3f(S[3], S[4], S[5]), c = max3f(S[6], S[7], S[8]);
  const float d = max3f(S[9], S[10], S[11]), e = max3f(S[12], S[13], S[14]);
  return __builtin_fmaxf(max3f(a, b, c), max3f(d, e, S[15]));
}
__device__ __forceinline__ float half_max(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}

__device__ __forceinline__ float half_sum(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}

__device__ __forceinline__ float lse_of(float M, float l) {
  return __float_as_uint(l) == 0u ? -INFINITY : (M + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

__device__ __forceinline__ u32x4 tr_pair(const lds_u8* a, const lds_u8* b) {
  const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)a));
  const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)b));
  return u32x4{x[0], x[1], y[0], y[1]};
}

// Eight rows of 8-bit values, 16 lanes' addresses two to a row: lane i gets column i.
__device__ __forceinline__ u32x2 tr8(const lds_u8* a) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)a));
}

// One tile of work, the same for all lanes.
struct Job {
  int h;              // K/V head
  int rho0, rho1;     // rows
  int state;          // where its states go, -1: it writes out
  int b, n, length, first_token;   // the rows' sequence: new tokens, rows with them, first packed token
  int prefix_pages, own_pages;     // pages of the list
  int skip;           // pages of the sequence before them, that no row of the tile sees
  int low;            // rows of the sequence before it are seen by none of its queries
  int begin, end;                  // this piece of it
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

// Sequence and tile of the idx-th tile of T = 2^log_rows rows, sequence by sequence (each
// sequence's last tile may be short); b = -1 behind the last.  One pass per 256
// sequences: every lane counts four sequences' tiles, a wave scan sums them.
// `last_first`: the last tile of each sequence first, and where the sequences
// have equal counts the last tiles of all before the others.
struct SeqTile {
  int b, tile, start, n;
};
__device__ __forceinline__ SeqTile find_tile(const PagedParams& p, int idx, int log_rows, bool last_first, int lane) {
  const int T = 1 << log_rows;
  if (!p.starts) {
    const int each = (p.per_seq * p.group + T - 1) >> log_rows;
    if (last_first) {
      const int level = idx / p.batch, b = idx - level * p.batch;
      return SeqTile{level < each ? b : -1, each - 1 - level, b * p.per_seq, p.per_seq};
    }
    const int b = idx / each;
    return SeqTile{b < p.batch ? b : -1, idx - b * each, b * p.per_seq, p.per_seq};
  }
  int base = 0;
  for (int c = 0; c < p.batch; c += 256) {
    int s[5], tiles[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 5; ++i) s[i] = clampi(p.starts[min(c + 4 * lane + i, p.batch)], 0, p.tokens);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      tiles[i] = (max(s[i + 1] - s[i], 0) * p.group + T - 1) >> log_rows;
      sum += tiles[i];
    }
    const int mine = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int below = __shfl_up(sum, o);
      if (lane >= o) sum += below;
    }
    const unsigned long long past = __ballot(base + sum > idx);
    if (past) {
      const int l = __ffsll((long long)past) - 1;
      int tile = idx - (base + __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(mine, l));
      int b = c + 4 * l, count = 0, at = 0, n = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        count = __builtin_amdgcn_readlane(tiles[i], l);
        at = __builtin_amdgcn_readlane(s[i], l);
        n = __builtin_amdgcn_readlane(s[i + 1], l) - at;
        if (tile < count) break;
        tile -= count;
        ++b;
      }
      return SeqTile{b, last_first ? count - 1 - tile : tile, at, n};
    }
    base += __builtin_amdgcn_readlane(sum, 63);
  }
  return SeqTile{-1, 0, 0, 0};
}

// Packed tokens of all sequences.
__device__ __forceinline__ int packed_tokens(const PagedParams& p) {
  return p.starts ? clampi(p.starts[p.batch], 0, p.tokens) : p.tokens;
}

// Prefix item `item` of tiles of T rows; false: no rows.
__device__ __forceinline__ bool prefix_job(const PagedParams& p, int item, int T, Job& j) {
  const int tp = item / p.prefix_pieces;
  j.state = item - tp * p.prefix_pieces;
  j.h = tp / p.prefix_tiles;
  j.rho0 = (tp - j.h * p.prefix_tiles) * T;
  j.rho1 = min(j.rho0 + T, packed_tokens(p) * p.group);
  j.b = 0;
  j.n = j.length = j.first_token = 0;
  j.prefix_pages = (p.prefix_tokens + kPage - 1) / kPage;
  j.own_pages = j.skip = j.low = 0;
  j.begin = j.state * p.prefix_cut;
  j.end = min(j.begin + p.prefix_cut, j.prefix_pages);
  return j.rho0 < j.rho1;
}

// Own item `item` (behind the prefix items) of tiles of 2^log_rows rows; false: nothing
// to do.
template <bool SHAPED>
__device__ __forceinline__ bool own_job(const PagedParams& p, int item, int log_rows, int lane, Job& j) {
  // the tile over all heads, and its piece
  int idx = item, piece = 0, t;
  if (p.longest_first) {
    // the first pieces of all tiles, then the second ones, ...; the heads of a
    // tile next to each other, so that with 8 heads an XCD keeps to one
    const int all = p.kv_heads * p.own_tiles;
    piece = item / all;
    idx = item - piece * all;
    t = idx / p.kv_heads;
    j.h = idx - t * p.kv_heads;
  } else {
    if (item >= p.own_whole) {
      const int u = (item - p.own_whole) / p.own_pieces;
      piece = item - p.own_whole - u * p.own_pieces;
      idx = p.own_whole + u;
    }
    j.h = idx / p.own_tiles;
    t = idx - j.h * p.own_tiles;
  }
  const SeqTile s = find_tile(p, t, log_rows, p.longest_first, lane);
  if (s.b < 0 || s.tile < 0) return false;
  j.b = s.b;
  j.n = s.n;
  j.first_token = s.start;
  j.rho0 = s.start * p.group + (s.tile << log_rows);
  j.rho1 = min(j.rho0 + (1 << log_rows), (s.start + s.n) * p.group);
  if (j.rho0 >= j.rho1) return false;
  // A length may pass the table (tokens whose rows it does not hold): the causal
  // limit goes by the length, which beyond `held + n` changes nothing more, the pages
  // by the rows that the table holds.
  const int held = kPage * p.table_pages;
  // Shaped scores go by the queries' places themselves.
  j.length = clampi(p.lengths[j.b], 0, SHAPED ? kMostRows : held + j.n);
  j.prefix_pages = p.apart ? 0 : (p.prefix_tokens + kPage - 1) / kPage;
  // rows the tile's last query sees
  int seen = j.length;
  if (p.causal) seen = j.length - j.n + (j.rho1 - 1) / p.group - j.first_token + 1;
  seen = clampi(seen, 0, min(j.length, held));
  j.own_pages = (seen + kPage - 1) / kPage;
  j.skip = j.low = 0;
  if constexpr (SHAPED) {
    if (p.window > 0) {
      j.low = j.length - j.n - p.window + 1;
      // the rows before the window of the tile's first query
      const int first = j.length - j.n + j.rho0 / p.group - j.first_token - p.window + 1;
      j.skip = __builtin_amdgcn_readfirstlane(min(max(first, 0) / kPage, j.own_pages));
      j.own_pages -= j.skip;
    }
  }
  const int units = j.prefix_pages + j.own_pages;
  const int cut = item < p.own_whole || p.own_pieces == 1 ? max(units, 1) : p.own_cut;
  j.begin = min(piece * cut, units);
  j.end = min(j.begin + cut, units);
  if (p.apart) {
    j.state = p.prefix_pieces + piece;       // a piece without pages leaves an empty state
    return true;
  }
  // a list that fits one piece is written out by it
  j.state = units > cut ? (idx - p.own_whole) * p.own_pieces + piece : -1;
  return piece == 0 || j.begin < units;
}

// The state that holds row rho (32-row block `blk` of its tile) of a job, and its
// place in it.
__device__ __forceinline__ float* state_of(const PagedParams& p, const Job& j, int rho, int blk, int* col) {
  if (p.apart) {
    *col = rho & 31;
    return p.part + (((long long)j.state * p.kv_heads + j.h) * p.row_tiles + (rho >> 5)) * kState;
  }
  *col = (rho - j.rho0) & 31;
  return p.part + ((long long)j.state * (1 << (p.log_rows - 5)) + blk) * kState;
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
    else if (u - j.prefix_pages + j.skip < p.table_pages)
      id = p.table[(long long)j.b * p.table_pages + (u - j.prefix_pages + j.skip)];
    return id >= 0 && id < p.pages ? id : -1;
  }
  // A list that fits both windows is held from its start, so that its entries
  // are requested without waiting for the sequence's length.
  __device__ __forceinline__ PageList(const PagedParams& p, const Job& j, int first, int lane)
      : base(j.prefix_pages + p.table_pages <= 128 ? 0 : first), cur(fetch(p, j, base + lane)),
        next(fetch(p, j, base + 64 + lane)) {}
  // page u of the list; u never decreases
  __device__ __forceinline__ Unit at(const PagedParams& p, const Job& j, int u, int lane) {
    if (u - base >= 64) {
      base += 64;
      cur = next;
      next = fetch(p, j, base + 64 + lane);
    }
    Unit r;
    r.page = __builtin_amdgcn_readlane(cur, u - base);
    r.rows = min(u < j.prefix_pages ? p.prefix_tokens - kPage * u : j.length - kPage * (u - j.prefix_pages + j.skip),
                 kPage);
    if (r.page < 0) r.rows = 0;
    return r;
  }
};

// What a lane's query row sees: rows `from` <= j < limit of its sequence (`from` 0
// but for windows).  all_see, all_from: what every row of the wave sees, the rows
// being those of one sequence in order.
struct Sight {
  int limit, all_see, from, all_from;
  int at;             // the query's place, the prefix counted
  float slope;        // what a row of distance costs, in log2 units

  // Whether some row of the wave does not see all of `count` keys from row `at` on of the
  // sequence (own) or the prefix, of which `rows` are there.
  template <bool SHAPED>
  __device__ __forceinline__ bool cuts(bool own, int at, int count, int rows) const {
    return min(rows, own ? all_see - at : count) < count || (SHAPED && own && all_from > at);
  }
  // Drops the scores of the keys that the row does not see; key(i): which one, from `at` on, S[i] is.
  template <bool SHAPED, class Key>
  __device__ __forceinline__ void mask(f32x16& S, bool own, int at, int rows, Key key) const {
    const int see = own ? min(rows, limit - at) : rows, low = SHAPED && own ? from - at : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) S[i] = key(i) < see && (!SHAPED || key(i) >= low) ? S[i] : -INFINITY;
  }
};

// The row of its sequence that packed token `token` is.
__device__ __forceinline__ int own_row(const PagedParams& p, int token) {
  int b, first, n;
  if (p.starts) {
    int above = p.batch;       // the last sequence that starts at or before the token
    for (b = 0; above - b > 1;) {
      const int mid = (b + above) >> 1;
      (p.starts[mid] <= token ? b : above) = mid;
    }
    first = p.starts[b];
    n = p.starts[b + 1] - first;
  } else {
    b = token / p.per_seq;
    n = p.per_seq;
    first = b * n;
  }
  return clampi(p.lengths[b], 0, kMostRows) - n + token - first;
}

template <bool SHAPED>
__device__ __forceinline__ Sight sight_of(const PagedParams& p, const Job& j, int token, int hq) {
  Sight x;
  const int row = j.length - j.n + (token - j.first_token);
  x.limit = p.causal ? row + 1 : j.length;
  x.all_see = __builtin_amdgcn_readfirstlane(x.limit);
  x.from = x.all_from = x.at = 0;
  x.slope = 0.0f;
  if constexpr (SHAPED) {
    if (p.window > 0) {
      x.from = max(row - p.window + 1, 0);
      x.all_from = __builtin_amdgcn_readlane(x.from, 31);
    }
    if (p.slopes) {
      // the rows of a prefix tile are those of many sequences
      x.at = p.prefix_tokens + (j.n > 0 ? row : own_row(p, token));
      x.slope = p.slopes[hq] * kLog2e;
    }
  }
  return x;
}

// Products q.k into scores in log2 units: cap tanh(s / cap), s = scale q.k, as cap - 2
// cap / (1 + e^(2 s / cap)) (its error is at most 2^-22 of the cap), less slope *
// |distance| (2^-22 of that product).  `place`: that of key 0, the prefix counted.
template <class Key>
__device__ __forceinline__ void shape(const PagedParams& p, f32x16& S, const Sight& x, int place, Key key) {
  if (p.cap_log2 > 0.0f) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      S[i] = __builtin_fmaf(__builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(S[i] * p.cap_scale)), -2.0f * p.cap_log2,
                            p.cap_log2);
  } else {
    S *= p.scale_log2;
  }
  if (p.slopes) {
    const float away = (float)(x.at - place);
#pragma unroll
    for (int i = 0; i < 16; ++i) S[i] = __builtin_fmaf(-x.slope, __builtin_fabsf(away - (float)key(i)), S[i]);
  }
}

// ---------------------------------------------------------------------------
// Narrow tiles: 32 rows.  Bound by the pages' way from memory, so waves walk the
// list by themselves, 32 keys at a time: of the NW waves that share a tile, wave
// w takes half pages w, w + NW, ..., its K and V rows going straight to 16 KB of
// LDS of its own, with no barrier before the end, where the states are joined.
// K of the wave's next half page is requested as soon as the scores are formed,
// its V as soon as V is read, and eight waves of a CU wait at different times, so
// that something is always on its way.  The matrix pipe has time to spare:
// probabilities meet V in two parts (hi + lo), so that no rounding of theirs
// shows in the output.  One token of 32 heads on 8 K/V heads behind 60000 rows:
// 52.8 us, 4.7 TB/s (a large copy 5.1).
constexpr int kNarrow = 32, kLogNarrow = 5, kNarrowWaves = 4;
constexpr int kHalf = 32 * 256;      // 32 rows of K or V

template <int N>
__device__ __forceinline__ void loads_left() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// 16 bytes from each lane's own address into lds + 16 * lane; not counted by the
// compiler, as dma_rows.
__device__ __forceinline__ void dma_at(const void* from, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "{m0}"(lds) : "memory");
}

// Lane `from`'s pointer.
template <typename T>
__device__ __forceinline__ T* of_lane(T* p, int from) {
  const uint64_t a = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_ds_bpermute(from << 2, (int)(uint32_t)a);
  const uint32_t hi = __builtin_amdgcn_ds_bpermute(from << 2, (int)(uint32_t)(a >> 32));
  return (T*)((uint64_t)hi << 32 | lo);
}

// All waves of a workgroup, their LDS reads and writes done.
__device__ __forceinline__ void meet() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");      // nothing behind it is read ahead of it
}

// Writes what a lane holds of a row to the row's state: 16 groups of 4 dims (8 c +
// 4 hh of row rho = j.rho0 + 32 blk + lane % 32), the maximum M and the sum l.  Those of
// wide tiles go past the L2, which would hand 17 MB of them on at the kernel's end (64 x 1
// behind 16384, 8 bits, 42.2 -> 41.5 us; the small ones of narrow tiles do not: 4 x 1, 12
// heads, behind 2000 11.8 and 12.2).
template <bool PAST_L2>
__device__ __forceinline__ void write_state(const PagedParams& p, const Job& j, const f32x16 (&O)[4], float M, float l,
                                            int blk, int lane) {
  const int rho = j.rho0 + 32 * blk + (lane & 31), hh = lane >> 5;
  if (rho >= j.rho1) return;
  int col;
  float* st = state_of(p, j, rho, blk, &col);
  // the sums of an empty state are not read
#pragma unroll
  for (int c = 0; c < 16 && j.begin < j.end; ++c) {
    const f32x16& o = O[c >> 2];
    const int i = 4 * (c & 3);
    const f32x4 x{o[i], o[i + 1], o[i + 2], o[i + 3]};
    f32x4* const to = reinterpret_cast<f32x4*>(st + ((2 * c + hh) * 32 + col) * 4);
    if constexpr (PAST_L2)
      __builtin_nontemporal_store(x, to);
    else
      *to = x;
  }
  if (hh == 0) {
    st[32 * kHeadDim + col] = M;
    st[32 * kHeadDim + 32 + col] = l;
  }
}

// A wave's walk over a tile's 16-bit pages: half pages w, w + NW, ... of the list.
template <class How, int NW>
__device__ __forceinline__ void walk(const PagedParams& p, const Job& j, lds_u8* ring, int lane, int wave,
                                     f32x16 (&O)[4], float& m, float& ls) {
  constexpr bool F16 = How::F16, SHAPED = How::SHAPED;
  const int r = lane & 31, hh = lane >> 5;
  u32x4 qop[8];
  Sight x;
  {
    const int rho = min(j.rho0 + r, j.rho1 - 1);
    const int token = rho / p.group, hq = j.h * p.group + rho % p.group;
    x = sight_of<SHAPED>(p, j, token, hq);
    const uint16_t* qp = p.q + (long long)token * p.q_tok + (long long)hq * p.q_head + 8 * hh;
#pragma unroll
    for (int st = 0; st < 8; ++st) qop[st] = ldg16(qp + 16 * st);
  }
  const float per_score = SHAPED ? 1.0f : p.scale_log2;

  const int begin = 2 * j.begin, end = 2 * j.end;      // half pages

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
  const uint8_t* const kh = (const uint8_t*)((const uint16_t*)p.k + (long long)j.h * p.kv_head);
  const uint8_t* const vh = (const uint8_t*)((const uint16_t*)p.v + (long long)j.h * p.kv_head);
  lds_u8* const kb = ring + wave * (2 * kHalf);
  lds_u8* const vb = kb + kHalf;
  auto issue = [&](const uint8_t* from, const uint32_t (&off)[4], const Unit& u, int hu, lds_u8* to) {
    // an absent page reads page 0: its rows are masked and its values cleared
    const long long at = (4ll * max(u.page, 0) + 2 * (hu & 1)) * rows16;
    const uint32_t l = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)to);
    dma_rows<4>(from + at, off, l);
    dma_rows<4>(from + at + rows16, off, l + 4096);
  };

  int hu = begin + (NW == 1 ? 0 : wave);
  PageList list(p, j, hu >> 1, lane);
  // the query rows and the list, in a form the compiler counts: it does not
  // know of the row loads to come, and would wait for the query rows in every
  // step
  wait_loads();
  Unit u{-1, 0};
  if (hu < end) {
    u = list.at(p, j, hu >> 1, lane);
    issue(kh, koff, u, hu, kb);
    issue(vh, voff, u, hu, vb);
  }
  for (; hu < end; hu += NW) {
    const bool more = hu + NW < end;
    loads_left<8>();                                        // K landed, V behind it
    f32x16 S = {};
#pragma unroll
    for (int st = 0; st < 8; ++st)
      S = mma<F16>(*(lds_u32x4*)(kb + r * 256 + (((2 * st + hh) ^ (r & 15)) << 4)), qop[st], S);
    Unit after{-1, 0};
    if (more) {
      after = list.at(p, j, (hu + NW) >> 1, lane);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // K is read
      issue(kh, koff, after, hu + NW, kb);
    }
    // keys of this half page that a row sees; S[i] is key 8 (i / 4) + 4 hh + i % 4
    const int rows = u.rows - 32 * (hu & 1);
    const bool own = hu >= 2 * j.prefix_pages;
    const int at = 32 * (hu - (own ? 2 * (j.prefix_pages - j.skip) : 0));     // its first row in the prefix, or of its own
    auto key = [](int i) { return 8 * (i / 4) + i % 4; };
    if constexpr (SHAPED) shape(p, S, x, (own ? p.prefix_tokens : 0) + at + 4 * hh, key);
    if (x.cuts<SHAPED>(own, at, 32, rows)) x.mask<SHAPED>(S, own, at + 4 * hh, rows - 4 * hh, key);
    const float mx = half_max(lane_max(S)) * per_score;
    if (__any(mx > m + kSlack)) {
      const float to = __builtin_fmaxf(m, mx);
      const float a = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.0f : to));
      ls *= a;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) O[dt] *= a;
      m = to;
    }
    const float nb = kLift<F16> - (m == -INFINITY ? 0.0f : m);
    u32x4 hi[2], lo[2];
    {
      float P[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        P[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], per_score, nb));
        ls += P[i];
      }
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const u32x2 x = split2<F16>(P[2 * w], P[2 * w + 1]);
        hi[w >> 2][w & 3] = x[0];
        lo[w >> 2][w & 3] = x[1];
      }
    }
    if (more)
      loads_left<8>();                                      // V landed, the K just requested behind it
    else
      loads_left<0>();
    const int low = SHAPED && own ? j.low - at : 0;
    if (rows < 32 || low > 0) {
      // rows behind the end, or before every window, hold anything: 0 * NaN must not
      // reach the sums
#pragma unroll
      for (int jj = 0; jj < 8; ++jj)
        if (4 * jj + (lane >> 4) >= rows || 4 * jj + (lane >> 4) < low) *(lds_u32x4*)(vb + jj * 1024 + lane * 16) = u32x4{};
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        // dims 32 dt + lane % 32 of keys 16 ks + 8 (e / 4) + 4 hh + e % 4
        const int g = lane >> 4, i = lane & 15;
        const int chunk = 4 * dt + 2 * (g & 1) + ((i & 3) >> 1), row = 16 * ks + 4 * (g >> 1) + (i >> 2);
        const lds_u8* a = vb + row * 256 + ((chunk ^ vswz(row)) << 4) + (i & 1) * 8;
        const u32x4 va = tr_pair(a, a + 2048);
        O[dt] = mma<F16>(va, hi[ks], O[dt]);
        O[dt] = mma<F16>(va, lo[ks], O[dt]);
      }
    }
    if (more) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // V is read
      issue(vh, voff, after, hu + NW, vb);
    }
    u = after;
  }
}

// A pointer that is the same for all lanes in scalar registers, which the loads below
// take it in after five wait states (under pressure the compiler holds it in
// vector registers).
__device__ __forceinline__ const uint8_t* scalar(const uint8_t* p) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)(uint64_t)p);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)p >> 32));
  return (const uint8_t*)((uint64_t)hi << 32 | lo);
}

// 4 bytes of each lane l, from base + off, into lds + 4 * l; not counted by the
// compiler.
__device__ __forceinline__ void dma4(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
}

// V's 8-bit values against bf16 queries where a probability has two parts (RELATIVE).  Two
// bf16 parts are half as many products again as one; one fp16 part has 11 bits, beside
// which an output's 8 are all that counts (against 64 bits both 0.00166), and 8-bit
// values are exact in fp16, but not their powers of two.  So V counts in units of 2^E,
// one E for all pages so far (when it rises the sums follow), in which values of the
// exponents E - 15 .. E are exact in fp16, and so are zeros: rows of the least exponent
// count as such (what they may hold is below 2^-117).  Values take their powers
// themselves: in the probabilities, whose smallest fp16 then holds no longer, 4096 keys
// of 2^-17 of the largest beside values of E - 15 went missing, 3% of an output.  From
// the first page on that has other exponents pages meet two bf16 parts in units of 1, in
// a loop of its own (as a branch in a wide tile's first one it took its registers: 64 x 1
// token behind 16384 127 us).  64 x 1 behind 16384 41.4 us, by two bf16 parts (BOTH)
// 45.7, and 50.1 where every list's first page has such exponents; 16 x 1 behind 131001
// 77, 85 and 85; 64 x 1 behind 64, up to 2000 own rows, 33.6, 36.1 and 36.5.  Waves by
// themselves, which wait for their pages, keep the two parts: a second loop beside the
// prefix tiles' costs more than it saves (4 x 1, 12 heads, behind 2000 12.7 and 11.9).
constexpr int kUnitLow = 127 - 40, kUnitHigh = 127 + 40, kUnitSpan = 15;      // as floats' exponents

// A wave's walk over a tile's 8-bit pages: pages w, w + NW, ... of the list, 8 KB of K
// and as much of V at a time.  16-byte chunk c of row r lies at c ^ swz8(r), with which
// neither the rows that 16 lanes read nor the transposing reads meet on a bank.
//
// K's powers of two go into its values on their way to 16 bits.  V's operand holds
// eight rows of one dim, so its powers go into the probabilities, p v = (p 2^e) (v /
// 2^e), which meet V in bf16 whatever the queries' type: its range holds every power of
// two and two parts carry more bits than an fp16 output.  On RELATIVE pages they go into
// V all the same, by a product a pair of rows, which costs 1 to 2% (16 x 1 behind 131001
// 71.4 and 73.0 us).  Score S[i] is key 16 (i / 8) + 8 hh + i % 8 of its half page (the K
// operand's rows are taken in that order), so that a lane's probabilities belong to the
// eight rows of an operand.
constexpr int kWave8 = 2 * kPage * kHeadDim + 512;     // K, V, the exponents as they come, V's as floats
__device__ __forceinline__ int swz8(int row) { return (row & 6) | ((row >> 3) & 1); }

template <class How, int NW>
__device__ __forceinline__ void walk8(const PagedParams& p, const Job& j, lds_u8* ring, int lane, int wave,
                                      f32x16 (&O)[4], float& m, float& ls) {
  constexpr bool F16 = How::F16, SHAPED = How::SHAPED, RELATIVE = !F16 && !How::BOTH && NW > 1;
  typedef __attribute__((address_space(3))) float lds_f32;
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
  typedef __attribute__((address_space(3))) _Float16 lds_f16;
  const int r = lane & 31, hh = lane >> 5;
  u32x4 qop[8];
  Sight x;
  {
    const int rho = min(j.rho0 + r, j.rho1 - 1);
    const int token = rho / p.group, hq = j.h * p.group + rho % p.group;
    x = sight_of<SHAPED>(p, j, token, hq);
    // a lane's 16 bytes of K are two operands' dims
    const uint16_t* qp = p.q + (long long)token * p.q_tok + (long long)hq * p.q_head + 16 * hh;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      qop[2 * t] = ldg16(qp + 32 * t);
      qop[2 * t + 1] = ldg16(qp + 32 * t + 8);
    }
  }
  const float per_score = SHAPED ? 1.0f : p.scale_log2;

  // load jj takes rows 8 jj .. 8 jj + 7
  uint32_t off[4];
#pragma unroll
  for (int jj = 0; jj < 4; ++jj) off[jj] = (lane >> 3) * 128 + (((lane & 7) ^ swz8(8 * (jj & 1) + (lane >> 3))) << 4);
  const uint8_t* const kh = (const uint8_t*)p.k + (long long)j.h * p.kv_head;
  const uint8_t* const vh = (const uint8_t*)p.v + (long long)j.h * p.kv_head;
  const uint8_t* const sh = p.scales + (long long)j.h * p.s_head;
  lds_u8* const kb = ring + wave * kWave8;
  lds_u8* const vb = kb + kPage * kHeadDim;
  lds_u8* const raw = vb + kPage * kHeadDim;
  lds_f32* const vscale = (lds_f32*)(raw + 256);
  lds_f16* const vfactor = (lds_f16*)vscale;
  auto issue = [&](const uint8_t* from, const Unit& u, lds_u8* to) {
    // an absent page reads page 0: its rows are masked and its values cleared
    const uint8_t* const at = scalar(from + max(u.page, 0) * p.kv_tok);
    const uint32_t l = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)to);
    dma_rows<4, 4>(at, off, l);
    dma_rows<4, 4>(at + 4096, off, l + 4096);
  };
  auto issue_keys = [&](const Unit& u) {
    issue(kh, u, kb);
    dma4(scalar(sh + max(u.page, 0) * p.s_page), 4 * (lane & 31), __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)raw));
  };
  auto exponent = [](uint32_t byte) { return __uint_as_float(byte << 23); };

  // the K row of the lane's operand: bits 2 and 3 change places
  const int kr = (r & 19) | (r & 4) << 1 | (r & 8) >> 1;
  int pu = j.begin + (NW == 1 ? 0 : wave);
  PageList list(p, j, pu, lane);
  wait_loads();       // as in walk
  Unit u{-1, 0};
  if (pu < j.end) {
    u = list.at(p, j, pu, lane);
    issue_keys(u);
    issue(vh, u, vb);
  }
  int unit = 0;               // E of the sums, once there are any
  // Page pu; with `fine` false, nothing done, where its powers of two are too far apart.
  auto step = [&](auto fine_c) {
    constexpr bool fine = RELATIVE && decltype(fine_c)::value;
    const bool more = pu + NW < j.end;
    const bool own = pu >= j.prefix_pages;
    const int at = kPage * (pu - (own ? j.prefix_pages - j.skip : 0));       // its first row in the prefix, or of its own
    const int low = SHAPED && own ? j.low - at : 0;
    loads_left<8>();                                        // K and the exponents landed, V behind them
    f32x16 S[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      S[h] = f32x16{};
      const float scale = exponent(raw[32 * h + kr]);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const u32x4 w = *(lds_u32x4*)(kb + (32 * h + kr) * 128 + (((2 * t + hh) ^ swz8(kr)) << 4));
        S[h] = mma<F16>(widen<F16>(w[0], w[1], scale), qop[2 * t], S[h]);
        S[h] = mma<F16>(widen<F16>(w[2], w[3], scale), qop[2 * t + 1], S[h]);
      }
    }
    // (while the products run) rows behind the end, or before every window, hold
    // anything, their exponents too
    const bool seen = lane < u.rows && lane >= low;
    if constexpr (RELATIVE) {
      const int e = raw[kPage + lane];
      int to = fine ? max(unit, kUnitLow) : 127;
      if constexpr (fine) {
        for (uint64_t up; to < kUnitHigh && (up = __ballot(seen && e > to));)
          to = min(__builtin_amdgcn_readlane(e, __builtin_ctzll(up)), kUnitHigh);
        if (__builtin_expect(__ballot(seen && (e > to || (e < to - kUnitSpan && e > 1))) != 0, 0)) return false;
      }
      if (to != unit && unit > 0) {
        const float a = __uint_as_float((uint32_t)(127 + unit - to) << 23);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) O[dt] *= a;
      }
      unit = to;
      const float f = seen && !(fine && e == 1) ? exponent(e + 127 - to) : 0.0f;
      if constexpr (fine)
        vfactor[lane] = (_Float16)f;
      else
        vscale[lane] = f;
    } else {
      vscale[lane] = seen ? exponent(raw[kPage + lane]) : 0.0f;
    }
    Unit after{-1, 0};
    if (more) {
      after = list.at(p, j, pu + NW, lane);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // K and the exponents are read
      issue_keys(after);
    }
    auto key = [](int i) { return 16 * (i / 8) + i % 8; };
    if constexpr (SHAPED) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        shape(p, S[h], x, (own ? p.prefix_tokens : 0) + at + 32 * h + 8 * hh, key);
    }
    if (x.cuts<SHAPED>(own, at, kPage, u.rows)) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        x.mask<SHAPED>(S[h], own, at + 32 * h + 8 * hh, u.rows - 32 * h - 8 * hh, key);
    }
    const float mx = half_max(__builtin_fmaxf(lane_max(S[0]), lane_max(S[1]))) * per_score;
    if (__any(mx > m + kSlack)) {
      const float to = __builtin_fmaxf(m, mx);
      const float a = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.0f : to));
      ls *= a;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) O[dt] *= a;
      m = to;
    }
    const float nb = kLift<RELATIVE> - (m == -INFINITY ? 0.0f : m);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        S[h][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[h][i], per_score, nb));
        ls += S[h][i];
      }
    if (more)
      loads_left<9>();                                      // V landed, the K just requested behind it
    else
      loads_left<0>();
    if (u.rows < kPage || low > 0) {
#pragma unroll
      for (int jj = 0; jj < 8; ++jj) {
        const int row = 8 * jj + (lane >> 3);
        if (row >= u.rows || row < low) *(lds_u32x4*)(vb + jj * 1024 + lane * 16) = u32x4{};
      }
    }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      // the probabilities of keys 16 ks + 8 hh .. + 7, in two parts, or in one beside values
      // times their rows' powers
      u32x4 hi, lo, factor;
      if constexpr (fine) factor = *(lds_u32x4*)(vfactor + 16 * ks + 8 * hh);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const f32x16& P = S[ks >> 1];
        const int i = 8 * (ks & 1) + 4 * half;
        if constexpr (fine) {
          hi[2 * half] = pack2<true>(P[i], P[i + 1]);
          hi[2 * half + 1] = pack2<true>(P[i + 2], P[i + 3]);
        } else {
          const f32x4 f = *(lds_f32x4*)(vscale + 16 * ks + 8 * hh + 4 * half);
          const u32x2 a = split2<false>(P[i] * f[0], P[i + 1] * f[1]), b = split2<false>(P[i + 2] * f[2], P[i + 3] * f[3]);
          hi[2 * half] = a[0];
          hi[2 * half + 1] = b[0];
          lo[2 * half] = a[1];
          lo[2 * half + 1] = b[1];
        }
      }
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        // dim 32 dt + lane % 32 of the same keys
        const int g = lane >> 4, i = lane & 15, row = 16 * ks + 8 * (g >> 1) + (i >> 1);
        const u32x2 w = tr8(vb + row * 128 + (((2 * dt + (g & 1)) ^ swz8(row)) << 4) + (i & 1) * 8);
        u32x4 va = widen<fine>(w[0], w[1], 1.0f);
        if constexpr (fine)
          va = __builtin_bit_cast(u32x4, __builtin_bit_cast(f16x8, va) * __builtin_bit_cast(f16x8, factor));
        O[dt] = mma<fine>(va, hi, O[dt]);
        if constexpr (!fine) O[dt] = mma<false>(va, lo, O[dt]);
      }
    }
    if (more) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // V is read
      issue(vh, after, vb);
    }
    u = after;
    pu += NW;
    return true;
  };
  if constexpr (RELATIVE) {
    while (pu < j.end && step(std::true_type{})) {
    }
  }
  while (RELATIVE ? __builtin_expect(pu < j.end, 0) : pu < j.end) step(std::false_type{});
  if constexpr (RELATIVE) {
    const float a = __uint_as_float((uint32_t)unit << 23);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) O[dt] *= a;
  }
}

template <class How>
constexpr int kWaveBytes = How::Q8 ? kWave8 : 2 * kHalf;      // a narrow wave's LDS

// NW waves share a tile; NW = 1: a wave by itself.
template <class How, int NW>
__device__ __forceinline__ void narrow_tile(const PagedParams& p, const Job& j, lds_u8* ring, int lane, int wave) {
  constexpr bool F16 = How::F16;
  constexpr float lift = kLift<How::Q8 ? !F16 && !How::BOTH && NW != 1 : F16>;
  f32x16 O[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) O[dt] = f32x16{};
  float m = -INFINITY, ls = 0.0f;
  if constexpr (How::Q8)
    walk8<How, NW>(p, j, ring, lane, wave, O, m, ls);
  else
    walk<How, NW>(p, j, ring, lane, wave, O, m, ls);

  // the lane's row, formed anew so that no register holds it across the loop
  int e = lane;
  asm volatile("" : "+v"(e));
  const float l = half_sum(ls);
  const float mine = m == -INFINITY ? m : m - lift;
  if constexpr (NW == 1) {
    write_state<false>(p, j, O, mine, l, 0, e);      // beside prefix tiles, so never the last word
  } else {
    // the waves' states into one: every wave hands over m, l and its 32 x 128
    // sums, [dim tile][j][lane] of 4 floats, two dim tiles at a time (8 KB a wave;
    // all row loads have landed), and adds up its share
    const int re = e & 31, he = e >> 5;
    typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
    typedef __attribute__((address_space(3))) float lds_f32;
    constexpr int kItems = 16 / NW;
    lds_f32* const xm = (lds_f32*)(ring + NW * 8192);
    __syncthreads();
    if (he == 0) {
      xm[wave * 64 + re] = mine;
      xm[wave * 64 + 32 + re] = l;
    }
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = __builtin_fmaxf(M, xm[w * 64 + re]);
    const float Mu = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int w = 0; w < NW; ++w) L += xm[w * 64 + 32 + re] * __builtin_amdgcn_exp2f(xm[w * 64 + re] - Mu);
    const float a = __builtin_amdgcn_exp2f(mine - Mu);
    f32x4 R[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) R[i] = f32x4{};
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      if (part) __syncthreads();
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const f32x16& o = O[2 * part + (c >> 2)];
        const int i = 4 * (c & 3);
        *(lds_f32x4*)(ring + wave * 8192 + c * 1024 + e * 16) = f32x4{o[i], o[i + 1], o[i + 2], o[i + 3]} * a;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int c = wave * kItems + i - 8 * part;
        if (c >= 0 && c < 8) {
#pragma unroll
          for (int w = 0; w < NW; ++w) R[i] += *(lds_f32x4*)(ring + w * 8192 + c * 1024 + e * 16);
        }
      }
    }
    const int rho = j.rho0 + re;
    if (rho >= j.rho1) return;
    if (j.state >= 0) {
      int col;
      float* st = state_of(p, j, rho, 0, &col);
#pragma unroll
      for (int i = 0; i < kItems; ++i)
        *reinterpret_cast<f32x4*>(st + ((2 * (wave * kItems + i) + he) * 32 + col) * 4) = R[i];
      if (wave == 0 && he == 0) {
        st[32 * kHeadDim + col] = M;
        st[32 * kHeadDim + 32 + col] = L;
      }
      return;
    }
    const int token = rho / p.group, hq = j.h * p.group + rho % p.group;
    const bool none = __float_as_uint(L) == 0u;
    const float inv = none ? 0.0f : 1.0f / L;
    uint16_t* op = p.out + (long long)token * p.o_tok + (long long)hq * p.o_head + 4 * he;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      R[i] *= inv;
      *reinterpret_cast<u32x2*>(op + 8 * (wave * kItems + i)) =
          u32x2{pack2<F16>(R[i][0], R[i][1]), pack2<F16>(R[i][2], R[i][3])};
    }
    if (p.lse && wave == 0 && he == 0) p.lse[(long long)token * p.heads + hq] = lse_of(M, L);
  }
}

// Where the prefix is apart: the own items of workgroup `group` of `groups`, a wave
// each, one after the other.  Waves that begin and end at different times keep the
// CU's loads on their way, where a workgroup for every eight items leaves it idle
// between them.
template <class How>
__device__ __forceinline__ void own_items(const PagedParams& p, int group, int groups, lds_u8* ring, int lane,
                                          int wave) {
  if (wave >= p.own_waves) return;
  const int all = p.kv_heads * p.own_tiles * p.own_pieces;
  Job j;
  for (long long own = group * p.own_waves + wave; own < all; own += (long long)groups * p.own_waves) {
    // what an item forms from the lane is not kept for the next: it has no registers to spare
    int e = lane;
    if constexpr (How::Q8) asm volatile("" : "+v"(e));
    if (own_job<How::SHAPED>(p, (int)own, kLogNarrow, lane, j)) narrow_tile<How, 1>(p, j, ring, e, wave);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // its rows are read before the next ones come
  }
}

// APART: prefix tiles, then own tiles, a wave each.
template <class How, bool APART>
__global__ __launch_bounds__(64 * kNarrowWaves, 2) void narrow_kernel(PagedParams p) {
  __shared__ alignas(16) uint8_t ring[kNarrowWaves * kWaveBytes<How>];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int b = blockIdx.x, first = APART ? p.prefix_items : 0;
  const int item = b < first ? xcd_remap(b, first) : xcd_remap(b - first, gridDim.x - first);
  Job j;
  if constexpr (APART) {
    if (b < first) {
      if (prefix_job(p, item, kNarrow, j)) narrow_tile<How, kNarrowWaves>(p, j, (lds_u8*)ring, lane, wave);
    } else {
      own_items<How>(p, item, gridDim.x - first, (lds_u8*)ring, lane, wave);
    }
  } else {
    if (own_job<How::SHAPED>(p, item, kLogNarrow, lane, j)) narrow_tile<How, kNarrowWaves>(p, j, (lds_u8*)ring, lane, wave);
  }
}

// ---------------------------------------------------------------------------
// Wide tiles: 256 rows, or 128.  Bound by the matrix pipe and the vector work of the
// softmax together: eight waves, two on a SIMD, so that one's products run under
// the other's exponentials; each holds 32 rows with their sums in registers and
// walks every key, and all share the pages.  S^T = K Q^T and O^T += V^T P^T on
// 32 x 32 x 16 products: a lane holds one query, its softmax needs no other lane
// but l ^ 32.
// A probability meets V in one 16-bit part or in two (TWO).  One: it is rounded,
// and the outputs' error is 1.4 times that of their own rounding (of bf16 outputs
// 0.00235 relative, with two parts 0.00166; fp16 0.000286 and 0.000207).  The second
// part is half as many products again: 4 x 4608 tokens behind 23040 rows 2686 and
// 3722 us, 8 x 1536 behind 4608 422 and 573, six prompts of up to 901 behind 8192
// 464 and 635.  So it is the caller's to ask for, but for sequences of up to 32 rows
// a K/V head (their mean), which alone would take narrow tiles: where they meet in
// the tiles of a prefix apart they have two parts as well, so that a step's precision
// does not change with the batch (64 x 1 behind 16384 48 and 51 us, 16 x 1 behind
// 131001 118 and 121).
// 4 sequences of 4608 tokens, 12 heads, behind 23040 rows: 2649 us, 1.18 PFLOP/s
// (an 8192^3 library product 1.40), the matrix pipe busy 64% of the time and the
// vector pipe 56 at the 1.65 GHz that the chip holds under this load.  Waves of 64
// rows, one on a SIMD, read half as much LDS and took 2948 us where these took 2711;
// from there the slots at fixed offsets, the raised priority and the loads between
// the half pages.  The sums as dot products of the rounded pairs, half as many
// instructions: 2703 us.
constexpr int kWide = 256, kHalfWide = 128, kWideWaves = 8;
constexpr int kTile = 64 * 256;      // a page's K or V rows

// Pages of the ring, K of all and then V.  One step, from barrier to barrier, is one
// page, or with PAIRS two: half as many barriers, from which the waves of a SIMD
// set out in step (4608 tokens as above 2690 -> 2642 us, 8 x 1536 behind 4608 422 ->
// 416), but pages come in twos, which a list from memory waits for (16 sequences
// behind 131001 rows 118 and 123; 20 x 64 tokens, 12 heads, 43 and 47; one of 160, 8
// heads, behind 30000 42.5 and 44.6; 12 x 200 behind 1500 38.2 and 37.7): so tiles of
// the prefix by itself, and sequences of up to 192 rows a head, go page by page.
template <bool PAIRS>
constexpr int kRing = PAIRS ? 5 : 4;

// What a lane has taken of an 8-bit page on its way to LDS: 16 values of K and of V,
// their rows' exponents, and that of V's row `lane`.
struct Staged {
  u32x4 k, v;
  uint32_t ks, vs, all;
};

template <class How, bool PAIRS, bool TWO>
__device__ __forceinline__ void wide_tile(const PagedParams& p, const Job& j, lds_u8* ring, int lane, int wave) {
  constexpr bool F16 = How::F16, Q8 = How::Q8, SHAPED = How::SHAPED, RELATIVE = Q8 && !F16 && !How::BOTH && TWO,
                 V16 = F16 || RELATIVE;
  constexpr int kSlots = kRing<PAIRS>;
  const int r = lane & 31, hh = lane >> 5;
  Sight x;
  const uint16_t* qp;
  {
    const int rho = min(j.rho0 + 32 * wave + r, j.rho1 - 1);
    const int token = rho / p.group, hq = j.h * p.group + rho % p.group;
    x = sight_of<SHAPED>(p, j, token, hq);
    qp = p.q + (long long)token * p.q_tok + (long long)hq * p.q_head;
  }
  const float per_score = SHAPED ? 1.0f : p.scale_log2;
  // a wave without rows only loads
  const bool alive = j.rho0 + 32 * wave < j.rho1;
  const int begin = j.begin, end = j.end;

  lds_u8* const kring = ring;
  lds_u8* const vring = kring + kSlots * kTile;
  // this wave loads rows 8 wave .. 8 wave + 7 of every page
  uint32_t koff[4] = {}, voff[4] = {};
#pragma unroll
  for (int jj = 0; jj < 2 && !Q8; ++jj) {
    const int row = 8 * wave + 4 * jj + (lane >> 4), c = lane & 15;
    const uint32_t at = (uint32_t)(row * p.kv_tok);
    koff[jj] = 2u * (at + 8u * (uint32_t)(c ^ (row & 15))) - 1024u * jj;
    voff[jj] = 2u * (at + 8u * (uint32_t)(c ^ vswz(row))) - 1024u * jj;
  }
  const long long page_bytes = 128 * p.kv_tok;
  const uint8_t* const kh = (const uint8_t*)p.k + (long long)j.h * p.kv_head * (Q8 ? 1 : 2);
  const uint8_t* const vh = (const uint8_t*)p.v + (long long)j.h * p.kv_head * (Q8 ? 1 : 2);
  PageList list(p, j, begin, lane);
  wait_loads();       // as in walk
  // The query rows, and in the end the output's, go by way of the parts of slots 2
  // and 3 that this wave itself loads (8 rows of each of the four 16 KB), so that
  // memory sees whole rows and no wave waits for another.  Operands' own form, 32
  // bytes of 32 rows an instruction, took 3.0 us of a tile's start and 3.8 of its
  // end where all CUs begin and end together.  Chunk c of row x lies at c ^ (x &
  // 15).
  auto row_place = [&](int x) {
    return ring + (2 + (x >> 4)) * kTile + ((x >> 3) & 1) * (kSlots * kTile) + wave * 2048 + (x & 7) * 256;
  };
  auto chunk_of = [](int x, int c) { return (c ^ (x & 15)) << 4; };
#pragma unroll
  for (int jj = 0; jj < 8; ++jj) {
    const int x = 4 * jj + (lane >> 4);
    dma_at((const uint8_t*)of_lane(qp, x) + chunk_of(x, lane & 15),
           __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)row_place(4 * jj)));
  }
  int rows_ahead[5] = {};      // rows of units u .. u + 4
  // rows of unit u's sequence before `low_of` are seen by no query of it
  auto low_of = [&](int u) {
    return SHAPED && u >= j.prefix_pages ? j.low - kPage * (u - j.prefix_pages + j.skip) : 0;
  };
  // 8-bit rows come into registers and go to LDS as 16-bit ones, their powers of two
  // in them: a lane takes 16 dims of row 8 wave + lane / 8, two pages before they are
  // read.  (Its two 16-byte stores meet others' on the banks, 256 cycles a page; 8-byte
  // loads in an order that avoids it: 64 x 1 behind 16384 42.0 -> 42.6 us, 4 x 4608
  // behind 23040 2660 -> 2690.)
  Staged staged[2];
  const uint8_t* const sh = Q8 ? p.scales + (long long)j.h * p.s_head + 8 * wave + (lane >> 3) : nullptr;
  const uint8_t* const every = RELATIVE ? p.scales + (long long)j.h * p.s_head + kPage + lane : nullptr;
  int unit = kUnitLow;                  // E of the pages in LDS, as a float's exponent
  int units[3] = {kUnitLow, kUnitLow, kUnitLow};       // of units u .. u + 2
  int fine_end = end;                   // units that are landed as fp16
  auto fetch = [&](int u, Staged& to) {
    if (u >= end) return 0;
    const Unit x = list.at(p, j, u, lane);
    const long long page = max(x.page, 0);
    const uint32_t at = 1024 * wave + 16 * lane;
    to.k = *reinterpret_cast<const u32x4*>(kh + page * p.kv_tok + at);
    to.v = *reinterpret_cast<const u32x4*>(vh + page * p.kv_tok + at);
    to.ks = sh[page * p.s_page];
    to.vs = sh[page * p.s_page + kPage];
    if constexpr (RELATIVE) to.all = every[page * p.s_page];
    return x.rows;
  };
  auto land = [&](int u, int slot, const Staged& from, int rows) {
    if (u >= end) return unit;
    const int row = 8 * wave + (lane >> 3), c = 2 * (lane & 7), low = low_of(u);
    if constexpr (RELATIVE) {
      // the same in every wave
      const bool seen = lane < rows && lane >= low;
      const int e = (int)from.all;
      if (u < fine_end) {
        for (uint64_t more; unit < kUnitHigh && (more = __ballot(seen && e > unit));)
          unit = min(__builtin_amdgcn_readlane(e, __builtin_ctzll(more)), kUnitHigh);
        if (__ballot(seen && (e > unit || (e < unit - kUnitSpan && e > 1)))) fine_end = u;
      }
      if (u >= fine_end) unit = 127;
    }
    lds_u8* const kt = kring + slot * kTile + row * 256;
    lds_u8* const vt = vring + slot * kTile + row * 256;
    const float ks = __uint_as_float(from.ks << 23);
    const float vs = __uint_as_float((RELATIVE ? (uint32_t)max((int)from.vs + 127 - unit, 1) : from.vs) << 23);
    *(lds_u32x4*)(kt + ((c ^ (row & 15)) << 4)) = widen<F16>(from.k[0], from.k[1], ks);
    *(lds_u32x4*)(kt + (((c + 1) ^ (row & 15)) << 4)) = widen<F16>(from.k[2], from.k[3], ks);
    u32x4 a, b;
    if (RELATIVE && u >= fine_end) {
      a = widen<false>(from.v[0], from.v[1], vs);
      b = widen<false>(from.v[2], from.v[3], vs);
    } else {
      a = widen<V16>(from.v[0], from.v[1], vs);
      b = widen<V16>(from.v[2], from.v[3], vs);
    }
    if (rows < kPage || low > 0) {
      // as clear_rows
      const bool there = row < rows && row >= low;
      a = there ? a : u32x4{};
      b = there ? b : u32x4{};
    }
    *(lds_u32x4*)(vt + ((c ^ vswz(row)) << 4)) = a;
    *(lds_u32x4*)(vt + (((c + 1) ^ vswz(row)) << 4)) = b;
    return unit;
  };
  auto issue = [&](int u) {
    if (u >= end) return 0;
    const Unit x = list.at(p, j, u, lane);
    const long long at = max(x.page, 0) * page_bytes;
    const uint32_t l =
        __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)kring + ((u - begin) % kSlots) * kTile + wave * 2048);
    dma_rows<2>(kh + at, koff, l);
    dma_rows<2>(vh + at, voff, l + kSlots * kTile);
    return x.rows;
  };
  if constexpr (Q8) {
    Staged first[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) rows_ahead[i] = fetch(begin + i, first[i]);
#pragma unroll
    for (int i = 0; i < 2; ++i) rows_ahead[2 + i] = fetch(begin + 2 + i, staged[i]);
#pragma unroll
    for (int i = 0; i < 2; ++i) units[i] = land(begin + i, i, first[i], rows_ahead[i]);
    if (begin >= end) loads_left<0>();          // the query rows came before the first page's
  } else {
    rows_ahead[0] = issue(begin);
    rows_ahead[1] = issue(begin + 1);
    if (begin + 2 <= end)
      loads_left<8>();          // the query rows landed, two units behind them
    else
      loads_left<0>();
  }
  u32x4 qop[8];
#pragma unroll
  for (int st = 0; st < 8; ++st) qop[st] = *(lds_u32x4*)(row_place(r) + chunk_of(r, 2 * st + hh));
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if constexpr (!Q8) rows_ahead[2] = issue(begin + 2);

  f32x16 O[4], S;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) O[dt] = f32x16{};
  // the running maximum in log2 units; the exponents' offset and the raw score
  // that the accumulators are rescaled beyond, which change with it alone
  float m = -INFINITY, nb = kLift<V16>, beyond = -INFINITY, ls = 0.0f, mx;
  const float slack = kSlack / per_score;
  const uint32_t klane = (uint32_t)(r * 256 + ((hh ^ (r & 15)) << 4));
  uint32_t vlane;
  {
    const int g = lane >> 4, i = lane & 15, row = 4 * (g >> 1) + (i >> 2);
    vlane = (uint32_t)(row * 256 + (((2 * (g & 1) + ((i & 3) >> 1)) ^ vswz(row)) << 4) + (i & 1) * 8);
  }
  // addresses of the K and V operands in slot 0: the slots lie at instruction
  // offsets, so that a step forms none (12 fewer vector instructions per half page)
  const lds_u8 *kat[8], *vat[4];
#pragma unroll
  for (int x = 0; x < 8; ++x) kat[x] = kring + (klane ^ (uint32_t)(x << 5));
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) vat[dt] = vring + (vlane ^ (uint32_t)(dt << 6));
  // rows of a page behind its end, or before every window, hold anything: 0 * NaN must
  // not reach the sums, so each wave clears those of its V rows once they have landed
  auto clear_rows = [&](int u, int rows) {
    const int low = low_of(u);
    if (rows < kPage || low > 0) {
#pragma unroll
      for (int jj = 0; jj < 2; ++jj)
        if (8 * wave + 4 * jj + (lane >> 4) >= rows || 8 * wave + 4 * jj + (lane >> 4) < low)
          *(lds_u32x4*)(vring + ((u - begin) % kSlots) * kTile + wave * 2048 + jj * 1024 + lane * 16) = u32x4{};
    }
  };
  // the products of half page `half` of unit u, which holds `rows` rows, into scores,
  // those dropped that a row does not see, and their maximum
  auto key = [](int i) { return 8 * (i / 4) + i % 4; };
  auto settle = [&](f32x16& X, int u, int half, int rows) {
    const bool own = u >= j.prefix_pages;
    const int at = kPage * (u - (own ? j.prefix_pages - j.skip : 0)) + 32 * half;
    if constexpr (SHAPED) shape(p, X, x, (own ? p.prefix_tokens : 0) + at + 4 * hh, key);
    mx = half_max(lane_max(X));
    if (x.cuts<SHAPED>(own, at, 32, rows - 32 * half)) {
      x.mask<SHAPED>(X, own, at + 4 * hh, rows - 32 * half - 4 * hh, key);
      mx = half_max(lane_max(X));
    }
  };
  auto rescale = [&]() {
    if (__any(mx > beyond)) {
      const float to = __builtin_fmaxf(m, mx * per_score), at = to == -INFINITY ? 0.0f : to;
      const float a = __builtin_amdgcn_exp2f(m - at);
      ls *= a;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) O[dt] *= a;
      m = to;
      nb = kLift<V16> - at;
      beyond = __builtin_fmaxf(beyond - slack, mx) + slack;
    }
  };
  // Half a page: the probabilities of Sc meet V (rows 32 half .. of slot `slot`),
  // with the scores Sn of the next half page and their maximum.  ka holds the
  // first four K operands on entry, and on return those of the half page after.
  // The scores' products run at raised priority: a wave in them keeps the pipe
  // from the other one's sums, and the two fall out of step.
  u32x4 ka[8];
  auto kread = [&](int slot, int half, int x) {
    return *(lds_u32x4*)(kat[x] + slot * kTile + half * (kTile / 2));
  };
  auto half_step = [&](auto slot, auto half_c, auto coarse_c, const f32x16& Sc, f32x16& Sn, int next, int next_rows) {
    constexpr int half = decltype(half_c)::value;
    constexpr bool coarse = decltype(coarse_c)::value, two = TWO && !RELATIVE || coarse, V = V16 && !coarse;
    constexpr int nhalf = half ^ 1, ahalf = half;
    const int nslot = (slot + half) % kSlots;            // the next half page
    const int aslot = (slot + 1) % kSlots;                   // and the one after
    u32x4 va[2][4], pb[2], pl[2];       // pl: the second parts
    float P[16];
    auto vread = [&](int ks, int dt) {
      const lds_u8* a = vat[dt] + slot * kTile + half * (kTile / 2) + 4096 * ks;
      return tr_pair(a, a + 2048);
    };
    auto expo = [&](int i) {
      P[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(Sc[i], per_score, nb));
      ls += P[i];
      if (!(i & 1)) return;
      if constexpr (two) {
        const u32x2 x = split2<V>(P[i - 1], P[i]);
        pb[i >> 3][(i & 7) >> 1] = x[0];
        pl[i >> 3][(i & 7) >> 1] = x[1];
      } else {
        pb[i >> 3][(i & 7) >> 1] = pack2<V>(P[i - 1], P[i]);
      }
    };
    Sn = f32x16{};
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int st = 0; st < 8; ++st) {
      Sn = mma<F16>(ka[st], qop[st], Sn);
      if (st < 4)
        ka[st + 4] = kread(nslot, nhalf, st + 4);
      else
        va[0][st - 4] = vread(0, st - 4);
      expo(st);
    }
    __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      O[dt] = mma<V>(va[0][dt], pb[0], O[dt]);
      if constexpr (two) O[dt] = mma<V>(va[0][dt], pl[0], O[dt]);
      va[1][dt] = vread(1, dt);
      expo(8 + 2 * dt);
      expo(9 + 2 * dt);
    }
    asm volatile("" : "+v"(ls));   // the sums here, not behind the branches below
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      O[dt] = mma<V>(va[1][dt], pb[1], O[dt]);
      if constexpr (two) O[dt] = mma<V>(va[1][dt], pl[1], O[dt]);
      ka[dt] = kread(aslot, ahalf, dt);
    }
    settle(Sn, next, nhalf, next_rows);
    rescale();
  };

  int held = kUnitLow;       // E of the sums
  if (begin < end) {
    // The first steps' pages: K and V of one (two), and K of the next; each unit is 2
    // loads of K, then 2 of V.
    constexpr int kStep = PAIRS ? 2 : 1, kLater = PAIRS ? 2 : 6;
    if constexpr (!Q8) {
      if (begin + 3 <= end)
        loads_left<kLater>();
      else
        loads_left<0>();
      clear_rows(begin, rows_ahead[0]);
      if (PAIRS && begin + 1 < end) clear_rows(begin + 1, rows_ahead[1]);
    }
    meet();
    S = f32x16{};
    if (alive) {
#pragma unroll
      for (int st = 0; st < 8; ++st) S = mma<F16>(kread(0, 0, st), qop[st], S);
    }
    settle(S, begin, 0, rows_ahead[0]);
    rescale();
#pragma unroll
    for (int st = 0; st < 4; ++st) ka[st] = kread(0, 1, st);
    int u = begin;
    held = units[0];
    auto step = [&](auto slot, auto coarse) {
      constexpr std::integral_constant<int, 0> low;
      constexpr std::integral_constant<int, 1> high;
      f32x16 S1;
      if constexpr (RELATIVE) {
        if (units[0] != held) {
          const float a = __uint_as_float((uint32_t)(127 + held - units[0]) << 23);
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) O[dt] *= a;
          held = units[0];
        }
      }
      if (alive) half_step(slot, low, coarse, S, S1, u, rows_ahead[0]);
      if constexpr (Q8) {
        // the coarse loop's slots are not known here: its next page is staged[0] always
        const int i = coarse ? 0 : slot & 1;
        units[2] = land(u + 2, (slot + 2) % kSlots, staged[i], rows_ahead[2]);
        if constexpr (coarse) staged[0] = staged[1];
        rows_ahead[4] = fetch(u + 4, staged[coarse ? 1 : i]);
      } else {
        rows_ahead[3] = issue(u + 3);
      }
      if (alive) half_step(slot, high, coarse, S1, S, u + 1, rows_ahead[1]);
      if constexpr (PAIRS) {
        constexpr std::integral_constant<int, (slot + 1) % kSlots> slot_d;
        rows_ahead[4] = issue(u + 4);
        if (alive && u + 1 < end) {
          half_step(slot_d, low, coarse, S, S1, u + 1, rows_ahead[1]);
          half_step(slot_d, high, coarse, S1, S, u + 2, rows_ahead[2]);
        }
      }
      if constexpr (!Q8) {
        if (u + kStep + 2 < end)
          loads_left<kLater>();
        else
          loads_left<0>();
      }
      u += kStep;
#pragma unroll
      for (int i = 0; i < (Q8 ? 4 : 3); ++i) rows_ahead[i] = rows_ahead[i + kStep];
      units[0] = units[1];
      units[1] = units[2];
      if constexpr (!Q8) {
        if (u < end) clear_rows(u, rows_ahead[0]);
        if (PAIRS && u + 1 < end) clear_rows(u + 1, rows_ahead[1]);
      }
      meet();
      return u < (coarse || !RELATIVE ? end : fine_end);
    };
    auto slot = [](auto k) { return std::integral_constant<int, decltype(k)::value * kStep % kSlots>{}; };
    constexpr std::false_type fine;
    bool more = !RELATIVE || begin < fine_end;
    while (more) {
      more = step(slot(std::integral_constant<int, 0>{}), fine) && step(slot(std::integral_constant<int, 1>{}), fine) &&
             step(slot(std::integral_constant<int, 2>{}), fine) && step(slot(std::integral_constant<int, 3>{}), fine);
      if constexpr (PAIRS) more = more && step(slot(std::integral_constant<int, 4>{}), fine);
    }
    if constexpr (RELATIVE) {
      if (u < end && (u - begin) & 1) {
        const Staged x = staged[0];
        staged[0] = staged[1];
        staged[1] = x;
      }
      while (u < end) step((u - begin) % kSlots, std::true_type{});
    }
  }

  // the lane's row, formed anew so that no register holds it across the loop
  int e = lane;
  asm volatile("" : "+v"(e));
  const float M = m == -INFINITY ? m : m - kLift<V16>, l = half_sum(ls);
  if constexpr (RELATIVE) {
    const float a = __uint_as_float((uint32_t)held << 23);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) O[dt] *= a;
  }
  if (j.state >= 0) {
    write_state<true>(p, j, O, M, l, wave, e);
    return;
  }
  const int y = e & 31, he = e >> 5, rho = j.rho0 + 32 * wave + y;
  const int token = rho / p.group, hq = j.h * p.group + rho % p.group;
  uint16_t* const to = p.out + (long long)token * p.o_tok + (long long)hq * p.o_head;
  const float inv = __float_as_uint(l) == 0u ? 0.0f : 1.0f / l;
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const f32x16 o = O[c >> 2] * inv;
    const int i = 4 * (c & 3);
    *(lds_u32x2*)(row_place(y) + chunk_of(y, c) + 8 * he) =
        u32x2{pack2<F16>(o[i], o[i + 1]), pack2<F16>(o[i + 2], o[i + 3])};
  }
#pragma unroll
  for (int jj = 0; jj < 8; ++jj) {
    const int z = 4 * jj + (e >> 4);
    uint16_t* const at = of_lane(to, z);
    const u32x4 w = *(lds_u32x4*)(row_place(z) + chunk_of(z, e & 15));
    if (j.rho0 + 32 * wave + z < j.rho1) *reinterpret_cast<u32x4*>(at + 8 * (e & 15)) = w;
  }
  if (p.lse && he == 0 && rho < j.rho1) p.lse[(long long)token * p.heads + hq] = lse_of(M, l);
}

// APART: prefix tiles, then own tiles of 32 rows, a wave each.  TWO: a probability
// meets V in two parts.
template <class How, bool APART, bool PAIRS, bool TWO>
__global__ __launch_bounds__(64 * kWideWaves, 1) void wide_kernel(PagedParams p) {
  constexpr int kPages = 2 * kRing<PAIRS> * kTile, kOwn = APART ? kWideWaves * kWaveBytes<How> : 0;
  static_assert(!(How::Q8 && PAIRS), "8-bit pages come one by one");
  __shared__ alignas(16) uint8_t ring[kPages > kOwn ? kPages : kOwn];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int b = blockIdx.x, first = APART ? p.prefix_items : p.own_whole;
  // the longer items first; either kind by itself over the XCDs, but for tiles in
  // the order of their lists
  int item = b < first ? b : b - first;
  if (APART || !p.longest_first) item = xcd_remap(item, b < first ? first : gridDim.x - first);
  Job j;
  if constexpr (APART) {
    if (b < first) {
      if (prefix_job(p, item, kWide, j)) wide_tile<How, PAIRS, TWO>(p, j, (lds_u8*)ring, lane, wave);
    } else {
      own_items<How>(p, item, gridDim.x - first, (lds_u8*)ring, lane, wave);
    }
  } else {
    if (own_job<How::SHAPED>(p, b < first ? item : first + item, p.log_rows, lane, j))
      wide_tile<How, PAIRS, TWO>(p, j, (lds_u8*)ring, lane, wave);
  }
}

// What a lane gathers of the pieces c, c + stride, ... of a row: M, L and N groups
// of 4 dims, `at` floats into a state; kJoin pieces' loads are out together.
constexpr int kJoin = 8, kJoinWaves = 4;

template <int N>
struct Gathered {
  float M = -INFINITY, L = 0.0f;
  f32x4 o[N];
};

template <int N, int STEP>
__device__ __forceinline__ Gathered<N> gather(const float* st, long long step, int first, int pieces, int stride, int r,
                                              int at, bool live) {
  Gathered<N> got;
#pragma unroll
  for (int x = 0; x < N; ++x) got.o[x] = f32x4{};
  for (int c = first; c < pieces; c += kJoin * stride) {
    float m[kJoin], l[kJoin];
    f32x4 o[kJoin][N];
#pragma unroll
    for (int i = 0; i < kJoin; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
#pragma unroll
      for (int x = 0; x < N; ++x) o[i][x] = f32x4{};
      if (c + i * stride < pieces && live) {
        const float* s = st + (c + i * stride) * step;
        m[i] = s[32 * kHeadDim + r];
        l[i] = s[32 * kHeadDim + 32 + r];
#pragma unroll
        for (int x = 0; x < N; ++x) o[i][x] = *reinterpret_cast<const f32x4*>(s + at + x * STEP);
      }
    }
    float top = got.M;
#pragma unroll
    for (int i = 0; i < kJoin; ++i) top = __builtin_fmaxf(top, m[i]);
    const float ref = top == -INFINITY ? 0.0f : top;
    const float a = __builtin_amdgcn_exp2f(got.M - ref);
    got.L *= a;
#pragma unroll
    for (int x = 0; x < N; ++x) got.o[x] *= a;
#pragma unroll
    for (int i = 0; i < kJoin; ++i) {
      const float w = __builtin_amdgcn_exp2f(m[i] - ref);
      got.L += l[i] * w;
      // an empty state's sums are not there
#pragma unroll
      for (int x = 0; x < N; ++x)
#pragma unroll
        for (int k = 0; k < 4; ++k) got.o[x][k] += m[i] == -INFINITY ? 0.0f : o[i][x][k] * w;
    }
    got.M = top;
  }
  return got;
}

// Joins the pieces' states of 32 rows of a K/V head, 528 bytes a row and piece:
// block (h, rows 32 T .., group) where the prefix is apart, else (split tile,
// block of 32, group).  Bound by the latency of its loads.  Few pieces: a group is
// 32 dims, a wave gathers 8 of them over all pieces.  MANY: a group is 16 dims,
// which the four waves gather over a quarter of the pieces each; their sums meet
// in LDS (32 pieces, 8 rows: 3.7 us).
template <class How, bool APART, bool MANY>
__global__ __launch_bounds__(64 * kJoinWaves) void join_kernel(PagedParams p) {
  constexpr bool F16 = How::F16;
  constexpr int kGroups = MANY ? 8 : 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = blockIdx.x % kGroups, block = blockIdx.x / kGroups, r = lane & 31, hh = lane >> 5;
  int h, rho, end, pieces;
  long long step;                 // floats from a piece to the next
  const float* st;
  if constexpr (APART) {
    h = block / p.row_tiles;
    rho = 32 * (block - h * p.row_tiles) + r;
    end = packed_tokens(p) * p.group;
    pieces = p.prefix_pieces + p.own_pieces;
    step = (long long)p.kv_heads * p.row_tiles * kState;
    st = p.part + (long long)block * kState;
  } else {
    const int log_blocks = p.log_rows - 5, t = block >> log_blocks, blk = block - (t << log_blocks);
    Job j;
    // the tile's first piece
    if (!own_job<How::SHAPED>(p, p.longest_first ? t : p.own_whole + t * p.own_pieces, p.log_rows, lane, j) || j.state < 0) return;
    h = j.h;
    rho = j.rho0 + 32 * blk + r;
    end = j.rho1;
    pieces = (j.prefix_pages + j.own_pages + p.own_cut - 1) / p.own_cut;
    step = (long long)kState << log_blocks;
    st = p.part + (((long long)t * p.own_pieces << log_blocks) + blk) * kState;
  }
  const bool live = rho < end;
  float M, L;
  f32x4 o;
  int dims;
  if constexpr (MANY) {
    __shared__ f32x4 xo[kJoinWaves][2][64];
    __shared__ float xm[kJoinWaves][32], xl[kJoinWaves][32];
    const Gathered<2> got =
        gather<2, 256>(st, step, wave, pieces, kJoinWaves, r, ((4 * g + hh) * 32 + r) * 4, live);
    if (hh == 0) {
      xm[wave][r] = got.M;
      xl[wave][r] = got.L;
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) xo[wave][x][lane] = got.o[x];
    __syncthreads();
    if (wave >= 2) return;              // waves 0 and 1 finish 8 dims each
    M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) M = __builtin_fmaxf(M, xm[w][r]);
    const float ref = M == -INFINITY ? 0.0f : M;
    L = 0.0f;
    o = f32x4{};
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
      const float a = __builtin_amdgcn_exp2f(xm[w][r] - ref);
      L += xl[w][r] * a;
      o += xo[w][wave][lane] * a;
    }
    dims = 16 * g + 8 * wave + 4 * hh;
  } else {
    const Gathered<1> got = gather<1, 0>(st, step, 0, pieces, 1, r, ((8 * g + 2 * wave + hh) * 32 + r) * 4, live);
    M = got.M;
    L = got.L;
    o = got.o[0];
    dims = 32 * g + 8 * wave + 4 * hh;
  }
  if (!live) return;
  const int token = rho / p.group, hq = h * p.group + rho % p.group;
  const bool none = __float_as_uint(L) == 0u;
  o *= none ? 0.0f : 1.0f / L;
  *reinterpret_cast<u32x2*>(p.out + (long long)token * p.o_tok + (long long)hq * p.o_head + dims) =
      u32x2{pack2<F16>(o[0], o[1]), pack2<F16>(o[2], o[3])};
  if (p.lse && dims == 0) p.lse[(long long)token * p.heads + hq] = lse_of(M, L);
}

// How a call is cut up, from sizes alone.  Tiles are of 32 rows (narrow), or of 256
// or, in one list, 128 (wide); own tiles beside prefix tiles are narrow.
struct Plan {
  int rows, row_tiles, prefix_tiles, prefix_pieces, prefix_cut, own_tiles, own_whole, own_pieces, own_cut;
  int own_groups, own_waves;     // apart: workgroups of own items, and their waves that take some
  bool longest_first, pairs;     // pairs: wide tiles take two pages between barriers
  bool apart() const { return prefix_tiles > 0; }
  long long split_tiles(int kv_heads) const { return (long long)kv_heads * own_tiles - own_whole; }
  long long states(int kv_heads) const {
    if (apart()) return (long long)(prefix_pieces + own_pieces) * kv_heads * row_tiles;
    return own_pieces > 1 ? split_tiles(kv_heads) * own_pieces * (rows / 32) : 0;
  }
  long long bytes(int kv_heads) const { return 4ll * kState * states(kv_heads); }
  // workgroups of the launches, and whether a grid holds them (2^32 threads)
  bool wide() const { return rows > kNarrow; }
  int waves() const { return wide() ? kWideWaves : kNarrowWaves; }
  long long prefix_items(int kv_heads) const { return 1ll * kv_heads * prefix_tiles * prefix_pieces; }
  long long own_items(int kv_heads) const { return own_whole + split_tiles(kv_heads) * own_pieces; }
  long long items(int kv_heads) const {
    return prefix_items(kv_heads) + (apart() ? own_groups : own_items(kv_heads));
  }
  bool many() const { return prefix_pieces + own_pieces > kJoin; }
  long long joins(int kv_heads) const {
    const long long blocks =
        apart() ? 1ll * kv_heads * row_tiles : own_pieces > 1 ? split_tiles(kv_heads) * (rows / 32) : 0;
    return (many() ? 8 : 4) * blocks;
  }
  bool fits(int kv_heads) const {
    return own_items(kv_heads) <= 0x7fffffffll && items(kv_heads) * 64 * waves() < (1ll << 32) &&
           joins(kv_heads) * 64 * kJoinWaves < (1ll << 32);
  }
};

// The sizes that a plan goes by.
struct Sizes {
  int cus, tokens, batch, heads, kv_heads, prefix_tokens, table_pages, ragged, causal;
  int eight = 0, shaped = 0, window = 0;       // 8-bit rows; shaped scores, and their window
  bool operator==(const Sizes& o) const {
    return cus == o.cus && tokens == o.tokens && batch == o.batch && heads == o.heads && kv_heads == o.kv_heads &&
           prefix_tokens == o.prefix_tokens && table_pages == o.table_pages && ragged == o.ragged &&
           causal == o.causal && eight == o.eight && shaped == o.shaped && window == o.window;
  }
  // Pages of its sequence that a tile of T rows walks, at most: with a window those of
  // its queries' windows (without `causal` up to the sequence's end).
  int own_pages(int T) const {
    if (window == 0) return table_pages;
    const long long group = heads / kv_heads, most = ragged ? tokens : tokens / batch;
    const long long behind = causal ? std::min(most, (T + group - 2) / group + 1) : most;
    return (int)std::min<long long>(table_pages, (window - 1ll + behind + kPage - 2) / kPage + 1);
  }
  // pages that the first tile of a sequence sees fewer of than the last
  double spread(int T) const {
    return causal && own_pages(T) == table_pages ? (double)(tokens / batch) / kPage : 0.0;
  }
  int prefix_pages() const { return (prefix_tokens + kPage - 1) / kPage; }
  long long rows() const { return (long long)tokens * (heads / kv_heads); }     // of a K/V head
  bool few() const { return rows() <= (long long)kNarrow * batch; }    // a sequence fills no wide tile
  // tiles of T rows of a K/V head, of sequences by themselves, at most
  int seq_tiles(int T) const {
    return (int)(ragged ? rows() / T + batch : batch * ((rows() / batch + T - 1) / T));
  }
};

// Estimates, in us, that the pieces are chosen by, from captured calls (224, 96
// and 32 workgroups, 17 and 65 pages each): a workgroup's start and end and a page
// of its tile, a state written and read again, pages from memory.  A wide tile's
// page takes 0.93 to 0.98 us with up to 128 rows (a wave on each SIMD), 1.35 with
// 192, with 256 1.62 where all CUs work and 1.32 where few do (the clock falls
// under the matrix pipe's load), 7% less with two pages between barriers; in two
// parts (steps behind a prefix apart) 1.15 to 2.0 (64 x 1 token behind 16384 cut by
// the figures of one part 55.9 us, by these 51.4; 128 x 1 behind 4096 69.3 and 58.4);
// a narrow tile's 0.47, 0.72 with two workgroups on a CU.  A page that no other tile
// reads takes 1.1 and 1.2 at least, which is what one workgroup draws from memory.
// Waves by themselves: a CU draws a page in 0.85 us (8 of them one each in 6.8), a
// wave one in 3.5, and an item begins and ends in 5.  The lengths being known to the
// device alone, tables are taken to be 0.6 to 0.7 full and sequences to be of mean
// size.  In a table much wider than its sequences the own pages seem to cover for a
// longer walk of the prefix, which is then cut too little (64 x 1 token behind 16384,
// up to 600 rows of their own: 51 us with a table of 10 pages, 69 with 32, 123 with 64,
// 460 with 256; 16 x 1 behind 131001 128 us with 33 pages, 211 with 256).
// Pages of 8 bits: a narrow tile's take 0.42 us, 0.92 with two workgroups on a CU, and
// no less where a page comes from memory; a wave by itself draws one in 1.8 and a CU
// in 0.5; an item begins and ends in 2.5 (4 x 1 token, 12 heads, behind 2000: the
// prefix apart 12.1, joint 15.5 by the 16-bit figures); a tile over prefix and own
// pages starts in 9.  A joint plan's lists are taken to be 0.65 full also where
// memory bounds them (64 x 1 behind 64, up to 2000 own rows: whole lists in narrow
// tiles 39, apart in wide ones 47).
constexpr double kJoinStart = 3.0, kSoloPage[] = {0.85, 0.5}, kSoloLatency[] = {3.5, 1.8}, kSoloStart = 3.0,
                 kSoloItem[] = {5.0, 2.5};
double start_time(int T, double rows, bool singly) {
  return T == kNarrow ? 7.0 : singly ? 6.0 + 5.0 * rows / kWide : 5.0 + 3.0 * rows / kWide;
}
double tile_page(int T, double rows, double active, double cus, double unshared, bool singly, const Sizes& z,
                 bool two = false) {
  const double busy = active / cus;
  double page;
  if (T == kNarrow && z.eight) {
    page = 0.42 + 0.5 * std::min(1.0, std::max(0.0, busy - 1.0));
  } else if (T == kNarrow) {
    page = 0.47 + 0.25 * std::min(1.0, std::max(0.0, busy - 1.0));
  } else {
    const double second = std::max(0.0, std::ceil(rows / 32) - 4) / 4;     // SIMDs with two waves
    const double few = two ? 1.7 : singly ? 1.3 : 1.2, more = singly ? 0.3 : 0.25;
    page = second > 0 ? few + more * std::min(1.0, busy) * second * second : two ? 1.15 : 0.95;
  }
  return page + unshared * std::max(0.0, (z.eight ? 0.42 : T == kNarrow ? 1.2 : 1.1) - page);
}
double state_time(double rows) { return rows * 2 * (4.0 * kState / 32) / 4.5e6; }
// Two workgroups on a CU draw less together (8 heads behind 30000 rows: 32 pieces
// each 31.9 us, 64 38.9).
double page_time(double pages, bool eight, double busy = 1.0) {
  return pages * (eight ? 16512 / 6.0e6 : 32768 / 5.2e6) * (1.0 + 0.2 * std::max(0.0, busy - 1.0));
}

constexpr int kCuts[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 56, 64, 96, 128, 192, 256};

bool sizes_fit(int tokens, int batch, int heads, int kv_heads, int prefix_tokens, int table_pages, bool ragged) {
  return tokens > 0 && batch > 0 && kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && prefix_tokens >= 0 &&
         table_pages > 0 && (ragged || tokens % batch == 0) && (long long)tokens * heads < (1ll << 30) &&
         (long long)table_pages * kPage < (1ll << 30) && prefix_tokens < (1 << 30) && batch <= (1 << 20);
}

// `units` pages in about c pieces of *cut; returns how many.
int cut_in(int units, int c, int* cut) {
  *cut = (units + c - 1) / c;
  return (units + *cut - 1) / *cut;
}

// The prefix apart: all rows together over the prefix, each sequence over its own
// pages.  Returns the estimated time.  Against one list, us: 64 x 1 token, 32 heads on
// 8, behind 16384: 51 and 228; 16 x 1 behind 131001: 121 and 1089; 24 x 5, 28 on 4,
// behind 5003: 27 and 54; where sequences fill tiles, 8 x 1536 behind 4608, 579 and
// 422.  The own lists' first pieces come first, then the second ones, on the CUs the
// prefix leaves (64 x 1 behind 2048, up to 2000 own rows: 75, list by list 85), as
// many workgroups as there are places, each wave several items (128 x 1 behind 4096,
// up to 1000: 80, with a workgroup for every eight items 87).  In 8 bits up to 64 rows
// may go in two narrow tiles, which both read the prefix, the second time from L2; a
// wide tile of so few rows waits for its own barriers (16 x 1 behind 131001: 87 and
// 113; 40 x 1, 12 heads, behind 9000: 22 and 27).  Two such tiles may share a CU (16 x 1
// behind 20000: 24 and 28).
double plan_apart(const Sizes& z, int T, Plan* plan) {
  const long long rows = z.rows();
  const int prefix_pages = z.prefix_pages(), table = z.own_pages(kNarrow);
  const int slots = T == kNarrow && rows > T ? 2 * z.cus : z.cus;
  plan->rows = T;
  plan->row_tiles = (int)((rows + 31) / 32);
  plan->prefix_tiles = (int)((rows + T - 1) / T);
  plan->own_tiles = z.seq_tiles(kNarrow);
  plan->own_whole = 0;
  plan->longest_first = true;
  plan->pairs = false;
  const double tiles = (double)z.kv_heads * plan->prefix_tiles, own_tiles = (double)z.kv_heads * plan->own_tiles;
  const double live = (double)rows / plan->prefix_tiles;
  const double floor_time = page_time(z.kv_heads * (prefix_pages + 0.6 * z.batch * table), z.eight);
  // pages of a sequence's mean list
  const double mean = std::max(1.0, table - 0.5 * z.spread(kNarrow));
  // n own items over at most *g workgroups, of which *w waves take some: as many as
  // give every item a wave, or a power of two, with which the rows of the heads, that
  // lie side by side, are read together
  auto own_time = [&](double n, int cut, double* g, int* w) {
    const double places = *g;
    const int exact = (int)std::min<double>(plan->waves(), std::ceil(n / places));
    double least = 1e30;
    for (int x = 1; x <= plan->waves(); ++x) {
      const bool even = !(x & (x - 1));
      if (!even && x != exact) continue;
      const double groups = std::min(places, std::ceil(n / x));
      const double page = std::max({kSoloLatency[z.eight], kSoloPage[z.eight] * x * (even ? 1.0 : 1.15),
                                     page_time(0.7 * groups * x, z.eight)});
      const double time =
          kSoloStart + std::ceil(n / (groups * x)) * (kSoloItem[z.eight] + page * std::min<double>(cut, mean));
      if (time < least) {
        least = time;
        *g = groups;
        *w = x;
      }
    }
    return least;
  };
  double least = 1e30;
  for (int c : kCuts) {
    if (c > 1 && 2 * c > prefix_pages) break;
    int cut;
    const int pieces = cut_in(prefix_pages, c, &cut);
    const double t = start_time(T, live, true) + cut * tile_page(T, std::min<double>(rows, T),
                                                           std::min(tiles * pieces, (double)slots), z.cus,
                                                           plan->prefix_tiles == 1 ? 1.0 : 0.0, true, z, z.few());
    const double rounds = std::ceil(tiles * pieces / slots), left = rounds * slots - tiles * pieces;
    for (int d : kCuts) {
      if (d > 16 || (d > 1 && 2 * d > table)) break;
      int own_cut;
      const int own = cut_in(table, d, &own_cut);
      const double n = own_tiles * own;
      // on the places that the last round of the prefix leaves, or behind it too
      double g = slots;
      int w;
      double time = rounds * t + own_time(n, own_cut, &g, &w);
      if (left > 0) {
        double beside = left;
        int v;
        const double u = std::max(rounds * t, (rounds - 1) * t + own_time(n, own_cut, &beside, &v));
        if (u < time) {
          g = beside;
          w = v;
          time = u;
        }
      }
      const double cost =
          std::max(floor_time, time) + state_time((double)z.kv_heads * rows * (pieces + own)) + kJoinStart;
      if (cost < least) {
        least = cost;
        plan->prefix_pieces = pieces;
        plan->prefix_cut = cut;
        plan->own_pieces = own;
        plan->own_cut = own_cut;
        plan->own_groups = (int)g;
        plan->own_waves = w;
      }
    }
  }
  return least;
}

// Every tile over prefix and own pages.  Where their lists are alike and there
// are more wide tiles than CUs, only those behind the last full round are cut
// (8 x 1536 tokens, 12 heads, behind 4608, 422 us and 494 uncut, page by page); where a causal
// sequence's first tiles have much shorter lists than its last, every list is cut
// at the same length and the longest come first (2717 tokens, 12 heads: 58 us, 76
// uncut, 76 in their order; 9 x 2786, 4 heads: 96, 127 in their order).  Sequences
// of up to 32 rows a K/V head take narrow tiles (40 x 3 tokens: 16.3 us, 22.7 with
// wide ones); others tiles of 256 rows or, where those leave CUs idle, of 128, whose
// waves have a SIMD each (12 x 200 tokens, 8 heads, behind 1500: 33.6 us, 38.4 with
// 256; 3 x 601 behind 126: 18.4 and 23.0; 5 x 531 behind 4389 86.4 and 82.7).
double plan_joint(const Sizes& z, int T, Plan* plan) {
  const double per_seq = (double)z.rows() / z.batch;
  const int table = z.own_pages(T), units = table + z.prefix_pages();
  const bool wide = T > kNarrow, singly = z.eight || per_seq <= 192;       // pages one by one
  const int slots = wide ? z.cus : 2 * z.cus;
  plan->rows = T;
  plan->pairs = wide && !singly;
  plan->row_tiles = plan->prefix_tiles = plan->prefix_pieces = plan->prefix_cut = 0;
  plan->own_groups = plan->own_waves = 0;
  plan->own_tiles = z.seq_tiles(T);
  const double spread = z.spread(T);
  plan->longest_first = wide && spread > 0.2 * units;
  const long long own_tiles = (long long)z.kv_heads * plan->own_tiles;
  const long long whole = wide && !plan->longest_first ? own_tiles / z.cus * z.cus : 0;
  const double tiles = (double)(own_tiles - whole);
  const double full = std::min<double>(per_seq, T);         // rows of the fullest tile
  const double live = per_seq / std::ceil(per_seq / T);     // and of the mean one
  const double start = start_time(T, live, singly) + (z.eight && !wide ? 2.0 : 0.0);
  // the part of all lists' pages that come from memory, and of a list that no other
  // tile reads
  const double read = std::min(1.0, z.kv_heads * (z.prefix_pages() + (double)z.batch * table) /
                                        ((double)own_tiles * units));
  const double unshared = per_seq > T ? 0.0 : z.batch == 1 ? 1.0 : (double)table / units;
  double least = tiles > 0 ? 1e30 : 0.0;
  plan->own_pieces = 1;
  plan->own_cut = units;
  for (int c : kCuts) {
    if (tiles == 0 || (c > 1 && 2 * c > units)) break;
    int cut;
    const int pieces = cut_in(units, c, &cut);
    double time, states = 0.0;
    if (plan->longest_first) {
      const double mean = units - 0.5 * spread, each = std::max(1.0, mean / cut + (c > 1 ? 0.5 : 0.0));
      const double page = tile_page(T, full, std::min(tiles * each, (double)slots), z.cus, unshared, singly, z);
      const double longest = start + cut * page;
      time = tiles * each <= slots ? longest
                                   : std::max(longest, tiles * (each * start + mean * page) / slots + 0.5 * longest);
      states = c > 1 ? tiles * each : 0.0;
    } else {
      const double active = std::min(tiles * pieces, (double)slots);
      time = std::ceil(tiles * pieces / slots) *
             (start + std::max(cut * tile_page(T, full, active, z.cus, unshared, singly, z),
                               page_time(read * active * cut * (z.eight ? 0.65 : 1.0), z.eight, active / z.cus)));
      states = pieces > 1 ? tiles * pieces : 0.0;
    }
    const double cost = time + (states > 0 ? state_time(states * live) + kJoinStart : 0.0);
    if (cost < least) {
      least = cost;
      plan->own_pieces = pieces;
      plan->own_cut = cut;
    }
  }
  plan->own_whole = (int)(plan->own_pieces == 1 ? own_tiles : whole);
  return least + (double)(whole / z.cus) * (start + units * tile_page(T, full, slots, z.cus, unshared, singly, z));
}

// The plan of a call's sizes (z.cus is filled in).  A thread keeps its last one:
// the estimates of all cuts take longer than a launch.
int make_plan(Sizes z, Plan* plan) {
  const int e = device_cus(&z.cus);
  if (e != (int)hipSuccess) return e;
  static thread_local Sizes last_sizes{};
  static thread_local Plan last_plan;
  if (!(z == last_sizes)) {
    Plan joint, other;
    double t = plan_joint(z, z.few() ? kNarrow : kWide, &joint);
    auto consider = [&](double time) {
      if (time < t) {
        joint = other;
        t = time;
      }
    };
    if (!z.few()) consider(plan_joint(z, kHalfWide, &other));
    if (z.batch > 1 && z.prefix_tokens > 0) {
      const bool narrow = z.rows() <= kNarrow;
      consider(plan_apart(z, narrow ? kNarrow : kWide, &other));
      if (z.eight && !narrow && z.rows() <= 2 * kNarrow) consider(plan_apart(z, kNarrow, &other));
    }
    last_plan = joint;
    last_sizes = z;
  }
  *plan = last_plan;
  return (int)hipSuccess;
}

// The arguments of an attention call that do not depend on the cache's form.
bool call_fits(const PagedParams& p, const Sizes& z, float scale, int flags) {
  if (!sizes_fit(z.tokens, z.batch, z.heads, z.kv_heads, z.prefix_tokens, z.table_pages, z.ragged) || p.pages <= 0 ||
      (flags & ~(3 | 3 << 3)) || flags >> 3 == 3 || !(scale > 0.0f && scale < INFINITY))
    return false;
  if (!p.q || !p.k || !p.v || !p.table || !p.lengths || !p.out || (z.prefix_tokens > 0 && !p.prefix)) return false;
  // 16-byte row pieces
  const long long strides = p.q_tok | p.q_head | p.o_tok | p.o_head;
  return !(strides & 7) && strides >= 0 &&
         !(((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.out) & 15) && !((uintptr_t)p.lse & 3);
}

// Plans and launches a call whose arguments are checked; p holds them but for the
// sizes' and the plan's.
template <bool Q8, bool SHAPED>
int run(PagedParams p, Sizes z, float scale, int flags, void* workspace, long long workspace_bytes,
        hipStream_t stream) {
  z.eight = Q8;
  z.shaped = SHAPED;
  z.window = p.window;
  Plan plan;
  const int e = make_plan(z, &plan);
  if (e != (int)hipSuccess) return e;
  if (!plan.fits(z.kv_heads)) return (int)hipErrorInvalidValue;
  const long long need = plan.bytes(z.kv_heads);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
    return (int)hipErrorInvalidValue;
  p.part = (float*)workspace;
  p.tokens = z.tokens;
  p.batch = z.batch;
  p.per_seq = z.ragged ? 0 : z.tokens / z.batch;
  p.heads = z.heads;
  p.kv_heads = z.kv_heads;
  p.group = z.heads / z.kv_heads;
  p.prefix_tokens = z.prefix_tokens;
  p.table_pages = z.table_pages;
  p.causal = z.causal;
  p.scale_log2 = scale * kLog2e;
  p.log_rows = plan.rows == kNarrow ? 5 : plan.rows == kHalfWide ? 7 : 8;
  p.row_tiles = plan.row_tiles;
  p.own_waves = plan.own_waves;
  p.prefix_tiles = plan.prefix_tiles;
  p.prefix_pieces = plan.prefix_pieces;
  p.prefix_cut = plan.prefix_cut;
  p.own_tiles = plan.own_tiles;
  p.own_whole = plan.own_whole;
  p.own_pieces = plan.own_pieces;
  p.own_cut = plan.own_cut;
  p.longest_first = plan.longest_first;
  p.apart = plan.apart();
  p.prefix_items = (int)plan.prefix_items(z.kv_heads);
  const long long items = plan.items(z.kv_heads), joins = plan.joins(z.kv_heads);
  const int waves = plan.waves();
  // parts of a probability in wide tiles: as asked, else two for sequences of few rows
  const int parts = flags >> 3;
  const bool two = parts ? parts == 2 : z.few();
  auto launch = [&](auto kernel, long long blocks, int threads) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, stream, p);
  };
  auto with = [&](auto how) {
    typedef decltype(how) How;
    auto start = [&](auto kernel) { launch(kernel, items, 64 * waves); };
    auto join = [&](auto kernel) { launch(kernel, joins, 64 * kJoinWaves); };
    if (!plan.wide())
      plan.apart() ? start(narrow_kernel<How, true>) : start(narrow_kernel<How, false>);
    else if constexpr (How::BOTH)
      plan.apart() ? start(wide_kernel<How, true, false, true>) : start(wide_kernel<How, false, false, true>);
    else if (plan.apart())
      two ? start(wide_kernel<How, true, false, true>) : start(wide_kernel<How, true, false, false>);
    else if (plan.pairs) {
      if constexpr (!Q8) two ? start(wide_kernel<How, false, true, true>) : start(wide_kernel<How, false, true, false>);
    } else
      two ? start(wide_kernel<How, false, false, true>) : start(wide_kernel<How, false, false, false>);
    if (joins == 0) return;
    if (plan.apart())
      plan.many() ? join(join_kernel<How, true, true>) : join(join_kernel<How, true, false>);
    else
      plan.many() ? join(join_kernel<How, false, true>) : join(join_kernel<How, false, false>);
  };
  if (flags & 1)
    with(Mode<true, Q8, SHAPED>{});
  else if (Q8 && parts == 2)
    with(Mode<false, Q8, SHAPED, Q8>{});
  else
    with(Mode<false, Q8, SHAPED>{});
  return (int)hipGetLastError();
}

// Bytes of the workspace of a call of these sizes; -1 for sizes that are rejected.
long long workspace_of(const Sizes& z) {
  Plan plan;
  if (!sizes_fit(z.tokens, z.batch, z.heads, z.kv_heads, z.prefix_tokens, z.table_pages, z.ragged) || z.window < 0 ||
      make_plan(z, &plan) != (int)hipSuccess || !plan.fits(z.kv_heads))
    return -1;
  return plan.bytes(z.kv_heads);
}

}  // namespace
