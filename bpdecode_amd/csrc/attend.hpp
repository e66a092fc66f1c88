// The attention kernels over the 4-bit paged cache (kv4.hpp) and the cut of a
// call's work: for requests by themselves (attend.hip) and, with Prefix, for
// what follows a prefix that a batch shares (shared.hip).
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "kv4.hpp"
#include "wave.hpp"

namespace bpd {
namespace {

struct AttendArgs {
  const uint8_t* pages;
  KvPage page;
  KvTable table;
  int32_t kv_heads, heads;
  const uint16_t* q;
  int64_t q_row, q_token, q_head;  // strides in elements
  uint16_t* out;                   // [rows, tokens, heads, dim]
  int64_t rows;
  int32_t tokens;
  const int32_t *lengths, *query_lens;
  float scale;
  int32_t* err;
};

// Tokens that query i of request b sees: none past the request's block table,
// whatever its length says (*past is set where it says more).  The host's.
inline int64_t seen_tokens(const AttendArgs& a, int64_t b, int32_t i, bool* past) {
  *past = false;
  int32_t n = a.tokens;
  if (a.query_lens) n = a.query_lens[b] < n ? a.query_lens[b] : n;
  if (i >= n) return 0;
  const int64_t s = int64_t(a.lengths[b]) - n + 1 + i, room = int64_t(a.table.blocks) * a.page.page_size;
  *past = s > room;
  return s < 0 ? 0 : s < room ? s : room;
}

constexpr int kWave = 64;
constexpr int kTile = 64;   // cache tokens that a wave takes at a time
constexpr int kWaves = 4;   // waves of a block, but for blocks that have a CU to themselves
constexpr int kManyWaves = 16, kManyPieces = 16;  // of a join of that many pieces a unit
constexpr int kNever = 0x7FFFFFFF;

// The power of two at which a row's largest weight stands when its maximum is
// taken up: with the 2^8 that it may grow by, the largest that float16 holds.
template <int DT>
constexpr float kLift = DT == BPD_DTYPE_F16 ? 7.0f : 0.0f;

// How a call's work is cut.  A unit is one request, one key head and one group
// of query columns (tokens x heads that share the key head); all units' tiles
// stand in one row, request by request, and every block takes an equal run of
// them.  A run may end one unit and begin others: a unit that lies in one run
// is finished by its block, the pieces of the others are joined afterwards.
// The lengths are on the device, so every wave works the cut out for itself.
struct AttendPlan {
  int32_t groups;   // column groups
  int32_t cols;     // columns of a group, at most 16 * NT
  int32_t blocks;   // runs that fill the device, 0: one block takes one unit
  float* partials;  // two pieces per run: of its first unit, of its last
};

__device__ __forceinline__ int32_t queries_of(const AttendArgs& a, int64_t b) {
  if (!a.query_lens) return a.tokens;
  const int32_t n = a.query_lens[b];
  return n < 0 ? 0 : n < a.tokens ? n : a.tokens;
}
// Tokens of request b that its last query sees.
__device__ __forceinline__ int64_t length_of(const AttendArgs& a, int64_t b) {
  const int64_t s = a.lengths[b], room = int64_t(a.table.blocks) * a.page.page_size;
  return s < 0 ? 0 : s < room ? s : room;
}
// A value that all lanes share, in scalar registers.
__device__ __forceinline__ int32_t scalar(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t scalar(int64_t x) { return of_lane(x, 0); }

__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {  // of numbers that are not negative
  if (((x | y) >> 32) == 0) return scalar(int32_t(uint32_t(x) / uint32_t(y)));
  return scalar(x / y);
}

// Tokens that a batch shares.
struct Spans {
  int32_t paged;  // of whole pages: in the prefix's table, not in a request's
  int32_t whole;  // of whole tiles of these: attended for all requests at once
};
// A call's prefix, and what its attention left for each column of each key
// head (request, query, head that shares the key head): of every chunk of the
// prefix the exponent that counts as 0 and the sum of weights, and the weighted
// values, channels in the order in which a lane of a join takes them.
struct Prefix {
  const int32_t* table;
  int32_t blocks;
  const int32_t* shared;  // tokens, or shared_all
  int32_t shared_all;
  int32_t chunks;
  int64_t columns;  // of one key head
  float2* stats;    // [chunks, kv_heads, columns]
  float* values;    // [chunks, kv_heads, columns, dim]
  __host__ __device__ __forceinline__ Spans spans(int32_t page_size, bool* past = nullptr) const {
    int64_t n = shared ? *shared : shared_all, room = int64_t(blocks) * page_size;
    if (past) *past = n > room;
    n = n < 0 ? 0 : n < room ? n : room;
    const int32_t paged = int32_t(n) & ~(page_size - 1);
    return Spans{paged, paged & ~(kTile - 1)};
  }
};
struct NoPrefix {
  __device__ __forceinline__ Spans spans(int32_t) const { return Spans{0, 0}; }
};

// The token at which a request's own part begins: past the prefix where all
// its queries see that, else 0.
__device__ __forceinline__ int32_t begin_of(const AttendArgs& a, const Spans& sp, int64_t b) {
  if (sp.whole == 0) return 0;
  const int64_t first = int64_t(a.lengths[b]) - queries_of(a, b) + 1, end = length_of(a, b);
  return (first < end ? first : end) >= sp.whole ? sp.whole : 0;
}

// Tiles of one of its units, one at least: someone has to write the zeros.
__device__ __forceinline__ int32_t tiles_of(const AttendArgs& a, const Spans& sp, int64_t b) {
  const int32_t n = queries_of(a, b) > 0 ? int32_t((length_of(a, b) - begin_of(a, sp, b) + kTile - 1) / kTile) : 0;
  return n < 1 ? 1 : n;
}

// A request's place in the row of tiles.
struct Place {
  int64_t first;  // its first tile
  int64_t whole;  // tiles of the call
  int64_t row;
  int32_t tiles;  // of each of its units
};

// The request that holds tile `at` (row < 0) or request `row`; `run` becomes
// the tiles of a run, `at` = run number * run.  False past the last tile.
__device__ __forceinline__ bool find_place(const AttendArgs& a, const AttendPlan& p, const Spans& sp, int64_t number,
                                           int64_t row, int lane, int64_t* run, Place* place) {
  const int32_t units = a.kv_heads * p.groups;
  const int32_t mine = lane < a.rows ? tiles_of(a, sp, lane) : 0;
  int64_t whole = mine;
  for (int64_t b = lane + kWave; b < a.rows; b += kWave) whole += tiles_of(a, sp, b);
  whole = wave_sum(whole);
  const int64_t per = quotient(whole * units + p.blocks - 1, p.blocks);
  *run = per < kWaves ? kWaves : per;
  place->whole = whole * units;
  const int64_t at = number * *run;
  if (row < 0 && at >= place->whole) return false;
  int64_t before = 0;
  for (int64_t b0 = 0;; b0 += kWave) {
    const int32_t here = b0 == 0 ? mine : b0 + lane < a.rows ? tiles_of(a, sp, b0 + lane) : 0;
    const int64_t upto = wave_scan_sum(int64_t(here));
    const uint64_t m = __ballot(row < 0 ? (before + upto) * units > at : b0 + lane == row);
    if (m) {
      const int hit = __builtin_ctzll(m);
      place->row = b0 + hit;
      place->tiles = __builtin_amdgcn_readlane(here, hit);
      place->first = (before + of_lane(upto, hit) - place->tiles) * units;
      return true;
    }
    before += of_lane(upto, kWave - 1);
  }
}

// A head's channels as one or two parts of 128, 64 or 32: what 16 lanes take
// in one load of 4, 2 or 1 bytes of values each, and 4 lanes in one load of
// 16, 8 or 4 bytes of keys.
template <int D>
struct Parts {
  static constexpr int first = D >= 128 ? 128 : 64;
  static constexpr int second = D - first;
  static constexpr int count = second ? 2 : 1;
  static constexpr int width(int p) { return p ? second : first; }
  static constexpr int begin(int p) { return p ? first : 0; }
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
union Frag {  // 8 channels (or tokens) of one row of a matrix operand
  uint32_t u[4];
  bf16x8 b;
  f16x8 h;
};

template <int DT>
__device__ __forceinline__ f32x4 mfma(const Frag& x, const Frag& y, f32x4 c) {
  if constexpr (DT == BPD_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.b, y.b, c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x.h, y.h, c, 0, 0, 0);
}

// Byte `at` + `lane_at` of an array of words as a power of two (the float
// whose exponent it is); lane_at < 4 differs between lanes.
__device__ __forceinline__ float scale_at(const uint32_t* w, int at, int words, uint32_t sel) {
  const int i = at / 4, o = at % 4;
  const uint32_t hi = i + 1 < words ? w[i + 1] : 0;
  return bits_float(__builtin_amdgcn_perm(hi, w[i], sel + (uint32_t(o) << 24)) >> 1);
}

// N neighbouring value tiles from v on of one column, times `inv`, to its head:
// rows 4 g .. 4 g + 3 of each are channels (width / 16) row + tile of a part.
template <int DT, int D, int N>
__device__ __forceinline__ void store_columns(uint16_t* out, int v, int g, const f32x4* x, float inv) {
  using Pt = Parts<D>;
  const int p = 16 * v < Pt::first ? 0 : 1, per = p ? Pt::second / 16 : Pt::first / 16;
  uint16_t* to = out + (p ? Pt::first : 0) + 4 * g * per + (v - (p ? Pt::first / 16 : 0));
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      if (N == 1)
        to[r * per] = uint16_t(two_rounded<DT>(x[0][r] * inv, 0.0f));
      else
        *reinterpret_cast<uint32_t*>(to + r * per + k) = two_rounded<DT>(x[k][r] * inv, x[k + (N > 1)][r] * inv);
    }
}

// A chunk of the prefix's sums for a lane's column (at `at`; in: there is one)
// into what the lane has accumulated: its value tiles as a product leaves them,
// the sum of weights on the first of the column's four lanes.
template <int D>
__device__ __forceinline__ void take_chunk(const Prefix& px, int64_t at, bool in, int g, float* top, float* sum, f32x4* acc) {
  constexpr int VT = D / 16;
  float2 st = {-3e38f, 0.0f};
  f32x4 y[VT];
  if (in) {
    st = px.stats[at];
    const f32x4* from = reinterpret_cast<const f32x4*>(px.values + at * D) + g * VT;
#pragma unroll
    for (int v = 0; v < VT; ++v) y[v] = from[v];
  }
  const bool some = in && st.y != 0.0f;  // else nothing was written
  const float now = some ? fmaxf(*top, st.x) : *top;
  const float keep = __builtin_amdgcn_exp2f(*top - now), f = some ? __builtin_amdgcn_exp2f(st.x - now) : 0.0f;
  *top = now;
  *sum = *sum * keep + (some && g == 0 ? st.y * f : 0.0f);
#pragma unroll
  for (int v = 0; v < VT; ++v)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[v][i] = acc[v][i] * keep + (some ? y[v][i] * f : 0.0f);
}

// Blocks that a CU is to hold, by registers (a block puts one wave on each SIMD).
constexpr int attend_blocks(int dim, int nt) {
  if (nt == 1) return dim == 64 ? 4 : dim == 128 ? 3 : 2;
  return dim == 64 ? 3 : dim <= 128 ? 2 : 1;
}

// A value that the compiler forms anew here instead of keeping it (or what
// follows from it) in registers across a loop.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// One block per run, the tiles of each unit in it dealt to the waves in turn.
//
// Scores: with keys as the left operand and queries as the right, a lane holds
// column n = lane % 16 (a query) and, of each 16 tokens, rows 4 g .. 4 g + 3
// (g = lane / 16).  The 64 tokens are handed to the four products so that row
// m of product j is token 4 m + j: the lane's 16 scores are then the 16
// consecutive tokens from 16 g, in the order in which the second product's
// right operand wants them, and the weights never leave their lane.  That
// product takes values with channels as rows: lane (m, g) loads the channels
// of row m, next to each other, of the tokens from 16 g, converts two codes
// of a token at a time and swaps halves with the next token's.
// The running maximum is followed loosely: weights may grow by 2^8 before the
// sums are scaled down, so most tiles cost no exchange between lanes.  Scores,
// maximum, sums and the accumulated values are floats; the weights are rounded
// to the cache's type, because the second product takes its operands in 16
// bits (the values themselves are exact in them).  A weight is off by half a
// step, which the sum that divides does not follow here, where it is of weights
// as they were before (a prefix's own sum, shared.hip, is of rounded ones): with
// bfloat16 an output of 1,000 tokens is off by 0.0020 of itself, the roundings
// of inputs and output alone make that 0.0016.  (Weights as two terms of 16 bits, for
// twice the second product: 16 columns of 128 channels 174 -> 200 us, 20 of
// them 57 -> 66, one short request 10.6 -> 11.9.)  In float16 a row's
// largest weight lies between kLift and kLift + 8 powers of two, so that
// weights down to 2^-21 of it keep all their bits, and those below are off by
// 2^-32 of it at most (with the largest at 1, those 2^-24 below, 17 nats,
// would lose half of themselves or all).
//
// (The product that takes codes and scales as they are, fp4 by fp8, was left:
// of 8 neighbouring products it keeps bits down to 2^-13 of the largest, and
// queries would need two or three fp8 terms each.)
//
// What bounds it: the cache's bytes for long contexts (32 requests of up to
// 32,768 tokens, 64/8 heads of 128, two tokens: 866 MB in 173 us, 5.0 TB/s of
// the 5.8 that a plain read reaches), and before that the conversions: a tile
// of 64 tokens takes about 360 vector instructions, 430 with two column tiles,
// which two or three waves on a SIMD issue one in five cycles (64 blocks of 5
// drafts over up to 4,096 tokens: 220 MB in 57 us).  A block that finds
// nothing to do takes 5 us, each of its first tiles 1.4.
template <int DT, int D, int NT, int W, class Px>
__global__ __launch_bounds__(W* kWave, W == kWaves ? attend_blocks(D, NT) : 1) void kv_attend_kernel(AttendArgs a,
                                                                                                 AttendPlan plan, Px px) {
  using Pt = Parts<D>;
  constexpr bool kShared = std::is_same<Px, Prefix>::value;
  constexpr int G = D / kKvGroup, KW = D / 32, VT = D / 16;  // scales, key words of a lane, value tiles
  constexpr int kScaleWords = 4 * G;                          // of 16 tokens
  constexpr int kJoin = VT <= W ? VT : W == kWaves ? 2 * W : W;  // value tiles joined at a time
  __shared__ f32x4 joined[W][kJoin][kWave];
  __shared__ float tops[W][kWave], sums[W][kWave];
  __shared__ Frag queries[NT][KW][kWave];  // as the lanes of every wave take them

  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int m = lane & 15, g = lane >> 4;
  const int32_t share = a.heads / a.kv_heads, units = a.kv_heads * plan.groups;
  const Spans sp = px.spans(a.page.page_size);
  int64_t b, pos = 0, stop, begin = 0;
  int32_t tiles, unit, tile0 = 0;
  if (plan.blocks == 0) {
    b = scalar(int32_t(blockIdx.x / uint32_t(units)));
    unit = int32_t(blockIdx.x) - int32_t(b) * units;
    stop = tiles = tiles_of(a, sp, b);
  } else {
    int64_t run;
    Place place;
    if (!find_place(a, plan, sp, blockIdx.x, -1, lane, &run, &place)) return;
    begin = pos = run * blockIdx.x;
    stop = pos + run < place.whole ? pos + run : place.whole;
    b = place.row;
    tiles = place.tiles;
    // (a request's tiles are fewer than 2^31, which the host checks)
    unit = scalar(int32_t(uint32_t(pos - place.first) / uint32_t(tiles)));
    tile0 = int32_t(pos - place.first) - unit * tiles;
  }

  // which of 4 neighbouring scales a lane takes: as a key lane, as a value lane
  uint32_t ksel[Pt::count], vsel[Pt::count];
#pragma unroll
  for (int p = 0; p < Pt::count; ++p) {
    ksel[p] = uint32_t(g * Pt::width(p) / 128) << 24 | 0x0C0C0C;
    vsel[p] = uint32_t(m * Pt::width(p) / 512) << 24 | 0x0C0C0C;
  }
  // scores times this are exponents of two; a negative scale turns the queries
  // around and a scale of zero clears them, so that a larger score stays larger
  const float to_log2 = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.44269504088896340736f;
  const int32_t P = a.page.page_size;
  const int shift = __builtin_ctz(P);

  for (;;) {
    const int32_t n_here = int32_t(stop - pos < tiles - tile0 ? stop - pos : tiles - tile0);
    const int32_t kvh = scalar(unit / plan.groups), group = unit - kvh * plan.groups;
    const int32_t n_q = queries_of(a, b);
    const int64_t end = n_q > 0 ? length_of(a, b) : 0;
    const int32_t base = kShared ? scalar(begin_of(a, sp, b)) : 0;  // a multiple of kTile
    const int32_t tile1 = end > base ? tile0 + n_here : tile0;
    if (a.err && n_q > 0 && a.lengths[b] > end && threadIdx.x == 0) atomicOr(a.err, BPD_FLAG_PAGE_RANGE);

    const int32_t* table = a.table.block_table + b * a.table.ld;
    // page of the chunk of 16 tokens that starts at t, -1: none
    const auto page_at = [&](int64_t t) -> int32_t {
      if constexpr (kShared) {
        if (t < sp.paged) return t < end ? px.table[t >> shift] : -1;
      }
      return t < end ? table[t >> shift] : -1;
    };
    const auto block_at = [&](int32_t page) -> const uint8_t* {
      // a page outside the pool is masked below
      const int64_t ok = page >= 0 && page < a.table.num_pages ? page : 0;
      return a.pages + (ok * a.kv_heads + kvh) * int64_t(a.page.bytes());
    };

    uint32_t kc[4][KW], ks[G], vc[16][Pt::count], vs[kScaleWords];
    const auto load_keys = [&](const uint8_t* block, int32_t slot) {  // tokens 4 m + j of a tile
      const uint8_t* codes = block + slot * (D / 2);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int p = 0; p < Pt::count; ++p) {
          const uint32_t* from =
              reinterpret_cast<const uint32_t*>(codes + j * (D / 2) + Pt::begin(p) / 2 + g * (Pt::width(p) / 8));
#pragma unroll
          for (int k = 0; k < Pt::width(p) / 32; ++k) kc[j][Pt::begin(p) / 32 + k] = from[k];
        }
      const uint32_t* scales = reinterpret_cast<const uint32_t*>(block + a.page.k_scales() + slot * G);
#pragma unroll
      for (int k = 0; k < G; ++k) ks[k] = scales[k];
    };
    const auto load_values = [&](const uint8_t* block, int32_t slot) {  // tokens 16 g + u of a tile
      const uint8_t* codes = block + a.page.v_codes() + slot * (D / 2);
#pragma unroll
      for (int u = 0; u < 16; ++u)
#pragma unroll
        for (int p = 0; p < Pt::count; ++p) {
          const uint8_t* from = codes + u * (D / 2) + Pt::begin(p) / 2 + m * (Pt::width(p) / 32);
          if (Pt::width(p) == 128) vc[u][p] = *reinterpret_cast<const uint32_t*>(from);
          if (Pt::width(p) == 64) vc[u][p] = *reinterpret_cast<const uint16_t*>(from);
          if (Pt::width(p) == 32) vc[u][p] = *from;
        }
      const uint4* scales = reinterpret_cast<const uint4*>(block + a.page.v_scales() + slot * G);
#pragma unroll
      for (int k = 0; k < kScaleWords / 4; ++k) {
        const uint4 w = scales[k];
        vs[4 * k] = w.x, vs[4 * k + 1] = w.y, vs[4 * k + 2] = w.z, vs[4 * k + 3] = w.w;
      }
    };
    int32_t tile = tile0 + wave;
    int32_t kpage = -1, vpage = -1, knext = -1, vnext = -1;
    if (tile < tile1) {
      kpage = page_at(base + int64_t(tile) * kTile + (m >> 2) * 16);
      vpage = page_at(base + int64_t(tile) * kTile + g * 16);
    }
    // this lane's columns: the queries, and how many tokens each sees
    const int ql = here(lane), qm = ql & 15;
    Frag q[NT][KW];  // every fourth of them
    int32_t sees[NT];
    int32_t least = int32_t(end);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int32_t c = group * plan.cols + t * 16 + qm;
      const int32_t i = c / share, h = kvh * share + c % share;
      const bool in = t * 16 + qm < plan.cols && i < n_q;
      const int64_t s = in ? int64_t(a.lengths[b]) - n_q + 1 + i : 0;
      sees[t] = int32_t(s < 0 ? 0 : s < end ? s : end);
      if (in) least = min(least, sees[t]);
      const uint16_t* row = a.q + b * a.q_row + (in ? i : 0) * a.q_token + (in ? h : 0) * a.q_head;
#pragma unroll
      for (int p = 0; p < Pt::count; ++p)
#pragma unroll
        for (int k = 0; k < Pt::width(p) / 32; ++k) {
          const uint16_t* from = row + Pt::begin(p) + (ql >> 4) * (Pt::width(p) / 4) + 8 * k;
          Frag f = {{0u, 0u, 0u, 0u}};
          const bool own = (t * KW + Pt::begin(p) / 32 + k) % W == wave;
          if (own && in && a.scale != 0.0f) __builtin_memcpy(&f, from, 16);  // at any element
          if (a.scale < 0.0f)
#pragma unroll
            for (int j = 0; j < 4; ++j) f.u[j] ^= 0x80008000u;
          q[t][Pt::begin(p) / 32 + k] = f;
        }
    }
    if (tile < tile1) {
      const int64_t t0 = base + int64_t(tile) * kTile;
      load_keys(block_at(kpage), int32_t((t0 + 4 * m) & (P - 1)));
      load_values(block_at(vpage), int32_t((t0 + 16 * g) & (P - 1)));
      const int64_t t1 = t0 + W * kTile;
      if (tile + W < tile1) knext = page_at(t1 + (m >> 2) * 16), vnext = page_at(t1 + g * 16);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < KW; ++k)
        if ((t * KW + k) % W == wave) queries[t][k][ql] = q[t][k];
    __syncthreads();
    least = wave_min(least);

    f32x4 acc[NT][VT];
    float top[NT], sum[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      top[t] = -3e38f, sum[t] = 0.0f;
#pragma unroll
      for (int v = 0; v < VT; ++v) acc[t][v] = f32x4{0, 0, 0, 0};
    }
    // the prefix's chunks, dealt to the waves of the block that begins the unit
    if constexpr (kShared) {
      if (base > 0 && tile0 == 0) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int32_t c = group * plan.cols + t * 16 + qm;
          const bool in = t * 16 + qm < plan.cols && c / share < n_q;
          const int64_t step = int64_t(a.kv_heads) * px.columns;
          const int64_t at = int64_t(kvh) * px.columns + b * (a.tokens * share) + c;
#pragma unroll 1
          for (int32_t k = wave; k < px.chunks; k += W) take_chunk<D>(px, k * step + at, in, g, &top[t], &sum[t], acc[t]);
        }
      }
    }
    int32_t nan_at[Pt::count];  // first token of the tail whose value group is bad, as a value lane
#pragma unroll
    for (int p = 0; p < Pt::count; ++p) nan_at[p] = kNever;
    for (; tile < tile1; tile += W) {
      const int64_t t0 = base + int64_t(tile) * kTile, t1 = t0 + W * kTile;
      const bool more = tile + W < tile1;
      // read anew for every tile: the registers hold loads in flight instead
      const int q_lane = here(lane);
      f32x4 s[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[t][j] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int p = 0; p < Pt::count; ++p) {
        float sc[4];  // of the lane's group of channels, by token
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[j] = scale_at(ks, G * j + Pt::begin(p) / kKvGroup, G, ksel[p]);
#pragma unroll
        for (int k = 0; k < Pt::width(p) / 32; ++k) {
          Frag q[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) q[t] = queries[t][Pt::begin(p) / 32 + k][q_lane];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t w = kc[j][Pt::begin(p) / 32 + k];
            Frag f;
            f.u[0] = two_values<DT, 0>(w, sc[j]);
            f.u[1] = two_values<DT, 1>(w, sc[j]);
            f.u[2] = two_values<DT, 2>(w, sc[j]);
            f.u[3] = two_values<DT, 3>(w, sc[j]);
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t][j] = mfma<DT>(f, q[t], s[t][j]);
          }
        }
      }
      if (more) load_keys(block_at(knext), int32_t((t1 + 4 * m) & (P - 1)));

      // token 16 g + 4 i + j of the tile is s[t][j][i]
      const int32_t mine = int32_t(t0) + 16 * g;
      const bool there = vpage >= 0 && vpage < a.table.num_pages;
      const bool tail = t0 + kTile > least;
      const bool masked = __any(!there || tail);
      if (masked) {
        const int32_t present = there ? int32_t(end) - mine : 0;
        if (!there && mine < int32_t(end) && a.err) atomicOr(a.err, BPD_FLAG_PAGE_RANGE);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (4 * i + j >= (there ? sees[t] - mine : 0)) s[t][j][i] = -INFINITY;
        // values that no query or not every query sees: nothing where there is
        // no token, and bad groups are noted, so that a weight of 0 meets no NaN
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const bool gone = u >= present;
#pragma unroll
          for (int p = 0; p < Pt::count; ++p) {
            const int byte = G * u + Pt::begin(p) / kKvGroup;
            const uint32_t e = float_bits(scale_at(vs, byte, kScaleWords, vsel[p])) >> 23;
            if (e == kKvBadScale && !gone && tail) {
              nan_at[p] = min(nan_at[p], mine + u);
            }
            if (gone || (e == kKvBadScale && tail)) {  // zeros, at a scale of one
              vc[u][p] = 0;
              const uint32_t at_byte = byte % 4 + (vsel[p] >> 24), put = 0xFFu << (8 * (at_byte & 3));
              if (at_byte < 4) vs[byte / 4] = (vs[byte / 4] & ~put) | (put & 0x7F7F7F7Fu);
              if (at_byte >= 4 && byte / 4 + 1 < kScaleWords)
                vs[byte / 4 + 1] = (vs[byte / 4 + 1] & ~put) | (put & 0x7F7F7F7Fu);
            }
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float most_here = s[t][0][0];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) most_here = fmaxf(most_here, s[t][j][i]);
        most_here *= to_log2;
        // (top[t] is the exponent that counts as 0, kLift below a maximum)
        if (__any(most_here > top[t] + (kLift<DT> + 8.0f))) {
          float now = fmaxf(top[t], most_here - kLift<DT>);
          now = fmaxf(now, __shfl_xor(now, 16));
          now = fmaxf(now, __shfl_xor(now, 32));
          const float keep = __builtin_amdgcn_exp2f(top[t] - now);
          top[t] = now;
          sum[t] *= keep;
#pragma unroll
          for (int v = 0; v < VT; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][v][i] *= keep;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[t][j][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][j][i], to_log2, -top[t]));
            sum[t] += s[t][j][i];
          }
      }
      // the weights, rounded to the type: tokens 8 h .. 8 h + 7 of the lane's 16
      Frag w[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[t][h].u[k] = two_rounded<DT>(s[t][2 * (k & 1)][2 * h + (k >> 1)], s[t][2 * (k & 1) + 1][2 * h + (k >> 1)]);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int p = 0; p < Pt::count; ++p) {
          constexpr int kMost = 8;
          Frag f[kMost];  // one value tile each: channels Pt::begin + row * (width / 16) + tile
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int u = 8 * h + 2 * k;
            float sc[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
              sc[e] = scale_at(vs, G * (u + e) + Pt::begin(p) / kKvGroup, kScaleWords, vsel[p]);
            const auto pair = [&](auto byte) {
              constexpr int B = decltype(byte)::value;
              if constexpr (2 * B < kMost) {
                const uint32_t x0 = two_values<DT, B>(vc[u][p], sc[0]), x1 = two_values<DT, B>(vc[u + 1][p], sc[1]);
                f[2 * B].u[k] = __builtin_amdgcn_perm(x1, x0, 0x05040100);
                f[2 * B + 1].u[k] = __builtin_amdgcn_perm(x1, x0, 0x07060302);
              }
            };
            pair(std::integral_constant<int, 0>());
            if (Pt::width(p) >= 64) pair(std::integral_constant<int, 1>());
            if (Pt::width(p) >= 128) pair(std::integral_constant<int, 2>()), pair(std::integral_constant<int, 3>());
          }
#pragma unroll
          for (int v = 0; v < Pt::width(p) / 16; ++v)
#pragma unroll
            for (int t = 0; t < NT; ++t)
              acc[t][Pt::begin(p) / 16 + v] = mfma<DT>(f[v], w[t][h], acc[t][Pt::begin(p) / 16 + v]);
        }
      vpage = vnext;
      if (more) load_values(block_at(vpage), int32_t((t1 + 16 * g) & (P - 1)));
      const int64_t t2 = t1 + W * kTile;
      if (tile + 2 * W < tile1) knext = page_at(t2 + (m >> 2) * 16), vnext = page_at(t2 + g * 16);
    }

    // bad value groups among the tokens that not every query sees
#pragma unroll
    for (int p = 0; p < Pt::count; ++p) {
      if (!__any(nan_at[p] != kNever)) continue;
      int32_t t = nan_at[p];
      t = min(t, __shfl_xor(t, 16));
      t = min(t, __shfl_xor(t, 32));
      // rows 4 g .. 4 g + 3 of a value tile lie in one group: that of value lane 4 g
      t = __shfl(t, 4 * g);
#pragma unroll
      for (int c = 0; c < NT; ++c)
        if (t < sees[c])
#pragma unroll
          for (int v = 0; v < Pt::width(p) / 16; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[c][Pt::begin(p) / 16 + v][i] = bits_float(0x7FC00000u);
    }

    // join the waves: each takes its share of the value tiles
    const int el = here(lane);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      sum[t] += __shfl_xor(sum[t], 16);
      sum[t] += __shfl_xor(sum[t], 32);
#pragma unroll
      for (int v0 = 0; v0 < VT; v0 += kJoin) {
        constexpr int kMine = kJoin > W ? kJoin / W : 1;
        __syncthreads();
        if (v0 == 0) tops[wave][el] = top[t], sums[wave][el] = sum[t];
#pragma unroll
        for (int v = 0; v < kJoin; ++v) {
          if (v0 + v < VT) joined[wave][v][el] = acc[t][v0 + v];
        }
        __syncthreads();
        const int v = v0 + wave * kMine;  // the first of the wave's value tiles
        if (wave * kMine >= kJoin || v >= VT) continue;
        float now = tops[0][el], whole = 0.0f, f[W];
#pragma unroll
        for (int w = 1; w < W; ++w) now = fmaxf(now, tops[w][el]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          f[w] = __builtin_amdgcn_exp2f(tops[w][el] - now);
          whole += sums[w][el] * f[w];
        }
        f32x4 mine[kMine];
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
          mine[k] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const f32x4 y = joined[w][wave * kMine + k][el];
#pragma unroll
            for (int i = 0; i < 4; ++i) mine[k][i] += y[i] * f[w];
          }
        }
        const int32_t column = t * 16 + (el & 15);
        if (n_here == tiles) {
          const int32_t c = group * plan.cols + column;
          const int32_t i = c / share, h = kvh * share + c % share;
          if (column >= plan.cols || i >= a.tokens) continue;
          // a row past the request's queries has summed what no mask kept out
          if (i >= n_q)
#pragma unroll
            for (int k = 0; k < kMine; ++k) mine[k] = f32x4{0, 0, 0, 0};
          store_columns<DT, D, kMine>(a.out + ((b * a.tokens + i) * a.heads + h) * D, v, el >> 4, mine,
                                      whole == 0.0f || i >= n_q ? 0.0f : 1.0f / whole);
        } else {
          const int64_t piece = 2 * int64_t(blockIdx.x) + (pos == begin ? 0 : 1);
          float* to = plan.partials + (piece * NT + t) * ((2 + 4 * VT) * kWave);
          if (v == 0) to[el] = now, to[kWave + el] = whole;
#pragma unroll
          for (int k = 0; k < kMine; ++k)
            if (v + k < VT) *reinterpret_cast<f32x4*>(to + 2 * kWave + ((v + k) * kWave + el) * 4) = mine[k];
        }
      }
    }
    pos += n_here;
    if (pos >= stop) break;
    tile0 = 0;
    if (++unit == units) unit = 0, tiles = tiles_of(a, sp, ++b);
    __syncthreads();
  }
}

// Joins the pieces of a unit that lies in several runs: one block per unit,
// column tile and pair of value tiles, its waves over the pieces.
template <int DT, int D, int NT, int W, class Px>
__global__ __launch_bounds__(W* kWave) void kv_attend_join_kernel(AttendArgs a, AttendPlan plan, Px px) {
  constexpr int VT = D / 16, kPiece = (2 + 4 * VT) * kWave, kAtOnce = 4;
  __shared__ f32x4 joined[W][2][kWave];
  __shared__ float tops[W][kWave], sums[W][kWave];
  const int lane = threadIdx.x % kWave, wave = scalar(int32_t(threadIdx.x / kWave));
  uint32_t x = blockIdx.x;
  const int v0 = int(x % (VT / 2)) * 2;
  x /= VT / 2;
  const int t = int(x % NT);
  x /= NT;
  const int32_t units = a.kv_heads * plan.groups;
  const int32_t unit = scalar(int32_t(x % uint32_t(units)));
  const int64_t b = scalar(int32_t(x / uint32_t(units)));
  const Spans sp = px.spans(a.page.page_size);
  int64_t run;
  Place place;
  find_place(a, plan, sp, 0, b, lane, &run, &place);
  const int64_t begin = place.first + int64_t(unit) * place.tiles;
  const int64_t run0 = quotient(begin, run), run1 = quotient(begin + place.tiles - 1, run);
  if (run0 == run1) return;
  float top = -3e38f, sum = 0.0f;
  f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  for (int64_t i0 = run0 + wave; i0 <= run1; i0 += W * kAtOnce) {
    float m[kAtOnce], l[kAtOnce];
    f32x4 y[kAtOnce][2];
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const int64_t i = i0 + n * W;
      m[n] = -3e38f, l[n] = 0.0f, y[n][0] = y[n][1] = f32x4{0, 0, 0, 0};
      if (i > run1) continue;
      const float* p = plan.partials + ((2 * i + (i == run0 && begin != run0 * run ? 1 : 0)) * NT + t) * kPiece;
      m[n] = p[lane], l[n] = p[kWave + lane];
#pragma unroll
      for (int v = 0; v < 2; ++v) y[n][v] = *reinterpret_cast<const f32x4*>(p + 2 * kWave + ((v0 + v) * kWave + lane) * 4);
    }
    float now = top;
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) now = fmaxf(now, m[n]);
    const float keep = __builtin_amdgcn_exp2f(top - now);
    top = now;
    sum *= keep;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[v][k] *= keep;
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const float f = __builtin_amdgcn_exp2f(m[n] - now);
      sum += l[n] * f;
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[v][k] += y[n][v][k] * f;
    }
  }
  tops[wave][lane] = top, sums[wave][lane] = sum, joined[wave][0][lane] = acc[0], joined[wave][1][lane] = acc[1];
  __syncthreads();
  if (wave) return;
  float now = top;
#pragma unroll
  for (int w = 1; w < W; ++w) now = fmaxf(now, tops[w][lane]);
  const float keep = __builtin_amdgcn_exp2f(top - now);
  sum *= keep;
#pragma unroll
  for (int v = 0; v < 2; ++v)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[v][k] *= keep;
#pragma unroll
  for (int w = 1; w < W; ++w) {
    const float f = __builtin_amdgcn_exp2f(tops[w][lane] - now);
    sum += sums[w][lane] * f;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const f32x4 y = joined[w][v][lane];
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[v][k] += y[k] * f;
    }
  }
  const int32_t share = a.heads / a.kv_heads, column = t * 16 + (lane & 15);
  const int32_t c = unit % plan.groups * plan.cols + column;
  const int32_t i = c / share, h = unit / plan.groups * share + c % share;
  if (column >= plan.cols || i >= a.tokens) return;
  const bool none = i >= queries_of(a, b);
  if (none) acc[0] = acc[1] = f32x4{0, 0, 0, 0};
  store_columns<DT, D, 2>(a.out + ((b * a.tokens + i) * a.heads + h) * D, v0, lane >> 4, acc,
                          none || sum == 0.0f ? 0.0f : 1.0f / sum);
}

struct AttendSizes {
  AttendPlan plan;
  int32_t nt, waves;
  int64_t tiles;  // at most, over all units
  int32_t blocks;  // that the device holds at a time
  size_t piece;   // floats of a unit's piece
};

constexpr int kCus = 256;
// Tiles of a unit up to which it is short, or of a middling length, by the width
// of the block table: the lengths are on the device.  Eight units of 1,000
// tokens: 10.6 us, cut in runs (as in a table for 4,096 tokens or more) 12.8;
// 128 units 11.4 and 13.7; eight of 2,000: 15.9 and 14.6.
// 512 units of 4,000 tokens: 50 and 59, of 8,000: 92 and 99; 128 units of
// 4,000 (a sixth of the device): 30 and 26.
constexpr int kShort = 16, kMiddling = 128;
// Waves of a block that has a CU to itself: units no more than CUs, and no more
// than a fourth as many tiles as there are units, for which runs with their
// join take longer.  One token, 32 heads of 128, lengths down to a half, runs and
// this: 9 requests of 1,100 tokens 16.0 and 11.6 us, 16 of 2,000 21.9 and 16.4, 32 of
// 4,000 32.4 and 26.2 (one of them 4,000 and the others 500: 17.1 and 24.0), 4 of
// 4,000 (not taken) 18.7 and 23.2; five tokens: 28.7 and 21.3, 39.1 and 34.2 for
// 16 and 32; heads of 64: 17.9 and 12.9, 25.3 and 20.0.  Up to kShort tiles four waves
// do as well (16 of 1,000: 12.2 and 11.6, five tokens 15.3 and 16.0).
constexpr int kUnitWaves = 8;

// `longest`: tokens of a request at most; `most` of them, if not all, are what
// is to be expected (behind a prefix).
AttendSizes attend_sizes(int64_t rows, int32_t tokens, int32_t heads, int32_t kv_heads, int32_t dim, int64_t longest,
                         int64_t most) {
  AttendSizes z{};
  const int64_t cols = int64_t(tokens) * (heads / kv_heads);
  // Two column tiles to a wave share the conversions of keys and values; four
  // leave one wave to a SIMD, and groups of two are read again from L2 instead
  // (72 columns of 128 channels, 64 requests of 4,000 tokens: one tile 91 us,
  // two 83, four 114; 40 columns of 64 channels: 40, 37 and 46).
  const int64_t col_tiles = (cols + 15) / 16;
  z.nt = col_tiles <= 1 ? 1 : 2;
  z.plan.groups = int32_t((col_tiles + z.nt - 1) / z.nt);
  z.plan.cols = int32_t((cols + z.plan.groups - 1) / z.plan.groups);
  const auto tiles = [](int64_t n) { return std::max<int64_t>(1, (std::min<int64_t>(n, 0x7FFFFFFF) + kTile - 1) / kTile); };
  const int64_t per_unit = tiles(most);
  z.tiles = tiles(longest) * kv_heads * z.plan.groups;
  z.blocks = kCus * attend_blocks(dim, z.nt);
  // one block per unit where that fills half the device with units of a
  // middling length, or where units are short: nothing is searched or joined
  const int64_t units = rows * kv_heads * z.plan.groups;
  const bool alone =
      units <= kCus && per_unit > kShort && 4 * per_unit <= units && attend_blocks(dim, z.nt) >= kUnitWaves / kWaves;
  z.waves = alone ? kUnitWaves : kWaves;
  z.plan.blocks = alone || per_unit <= kShort || (per_unit <= kMiddling && 2 * units >= z.blocks) ? 0 : z.blocks;
  z.piece = size_t(z.nt) * (2 + dim / 4) * kWave;
  return z;
}

// Runs that a call can have: each of kWaves tiles at least.
int64_t attend_runs(const AttendSizes& z, int64_t rows) {
  const int64_t runs = (z.tiles + kWaves - 1) / kWaves * rows;
  return runs < z.plan.blocks ? runs : z.plan.blocks;
}

template <int DT, int D, int NT, class Px>
int launch_attend(const AttendArgs& a, const AttendSizes& z, const Px& px, hipStream_t s) {
  const int64_t joins = a.rows * a.kv_heads * z.plan.groups * NT * (D / 32);
  BPD_REQUIRE(z.tiles < (int64_t(1) << 31) && joins < (int64_t(1) << 31), "too many queries or tokens in one call");
  const int64_t blocks = z.plan.blocks ? attend_runs(z, a.rows) : a.rows * a.kv_heads * z.plan.groups;
  if constexpr (attend_blocks(D, NT) >= kUnitWaves / kWaves) {
    if (z.waves == kUnitWaves)
      kv_attend_kernel<DT, D, NT, kUnitWaves, Px><<<uint32_t(blocks), kUnitWaves * kWave, 0, s>>>(a, z.plan, px);
  }
  if (z.waves == kWaves) kv_attend_kernel<DT, D, NT, kWaves, Px><<<uint32_t(blocks), kWaves * kWave, 0, s>>>(a, z.plan, px);
  // few units have many pieces each: more waves to a unit's join
  if (z.plan.blocks >= kManyPieces * a.rows * a.kv_heads * z.plan.groups)
    kv_attend_join_kernel<DT, D, NT, kManyWaves, Px><<<uint32_t(joins), kManyWaves * kWave, 0, s>>>(a, z.plan, px);
  else if (z.plan.blocks)
    kv_attend_join_kernel<DT, D, NT, kWaves, Px><<<uint32_t(joins), kWaves * kWave, 0, s>>>(a, z.plan, px);
  BPD_LAUNCHED();
  return BPD_OK;
}

// f(head size, column tiles of a wave) of a call.
template <class F>
int with_attend(int32_t dim, int32_t nt, F f) {
  const auto with_tiles = [&](auto d) -> int {
    return nt == 1 ? f(d, std::integral_constant<int, 1>()) : f(d, std::integral_constant<int, 2>());
  };
  switch (dim) {
    case 64: return with_tiles(std::integral_constant<int, 64>());
    case 96: return with_tiles(std::integral_constant<int, 96>());
    case 128: return with_tiles(std::integral_constant<int, 128>());
    case 192: return with_tiles(std::integral_constant<int, 192>());
    default: return with_tiles(std::integral_constant<int, 256>());
  }
}

// Tokens before `paged` lie in the pages of `prefix`.
template <int DT>
void host_attend(const AttendArgs& a, const int32_t* prefix = nullptr, int64_t paged = 0) {
  const int32_t D = a.page.dim;
  const auto page_of = [&](int64_t b, int64_t t) -> int64_t {
    if (t >= paged) return a.table.page_of(b, t, a.page.page_size);
    const int32_t page = prefix[t / a.page.page_size];
    return page >= 0 && page < a.table.num_pages ? page : -1;
  };
  std::vector<double> w, acc(D);
  for (int64_t b = 0; b < a.rows; ++b)
    for (int32_t i = 0; i < a.tokens; ++i) {
      bool past;
      const int64_t n = seen_tokens(a, b, i, &past);
      if (past && a.err) *a.err |= BPD_FLAG_PAGE_RANGE;
      for (int32_t h = 0; h < a.heads; ++h) {
        const uint16_t* q = a.q + b * a.q_row + i * a.q_token + h * a.q_head;
        const int32_t kvh = h / (a.heads / a.kv_heads);
        double m = -INFINITY, l = 0.0;
        w.assign(size_t(n), -INFINITY);
        for (int64_t t = 0; t < n; ++t) {
          const int64_t page = page_of(b, t);
          if (page < 0) {
            if (a.err) *a.err |= BPD_FLAG_PAGE_RANGE;
            continue;
          }
          const uint8_t* block = a.pages + (page * a.kv_heads + kvh) * int64_t(a.page.bytes());
          const int32_t slot = int32_t(t % a.page.page_size);
          const uint8_t* codes = block + slot * a.page.codes();
          const uint8_t* scales = block + a.page.k_scales() + slot * a.page.groups();
          double s = 0.0;
          for (int32_t d = 0; d < D; ++d)
            s += double(elem16_float<DT>(q[d])) * kv_value(uint32_t(codes[d / 2]) >> (4 * (d & 1)) & 15u, scales[d / kKvGroup]);
          w[t] = s * a.scale;
          if (w[t] > m || w[t] != w[t]) m = w[t];
          if (m != m) break;
        }
        std::fill(acc.begin(), acc.end(), m != m ? m : 0.0);
        l = m != m ? 1.0 : 0.0;
        for (int64_t t = 0; t < n && m == m; ++t) {
          if (w[t] == -INFINITY) continue;
          const double p = std::exp(w[t] - m);
          const int64_t page = page_of(b, t);
          const uint8_t* block = a.pages + (page * a.kv_heads + kvh) * int64_t(a.page.bytes());
          const int32_t slot = int32_t(t % a.page.page_size);
          const uint8_t* codes = block + a.page.v_codes() + slot * a.page.codes();
          const uint8_t* scales = block + a.page.v_scales() + slot * a.page.groups();
          l += p;
          for (int32_t d = 0; d < D; ++d)
            acc[d] += p * kv_value(uint32_t(codes[d / 2]) >> (4 * (d & 1)) & 15u, scales[d / kKvGroup]);
        }
        uint16_t* out = a.out + ((b * a.tokens + i) * a.heads + h) * D;
        for (int32_t d = 0; d < D; ++d) out[d] = float_elem16<DT>(l == 0.0 ? 0.0f : float(acc[d] / l));
      }
    }
}

int check_attend(const AttendArgs& a, int dtype) {
  if (int rc = check_kv_cache(a.pages, a.page, a.table, a.kv_heads, dtype)) return rc;
  BPD_REQUIRE(a.rows >= 0 && a.tokens >= 0, "negative sizes");
  BPD_REQUIRE(a.heads >= 1 && a.heads % a.kv_heads == 0, "query heads (%d) must be a multiple of key heads (%d)",
              a.heads, a.kv_heads);
  BPD_REQUIRE(std::isfinite(a.scale), "the scale must be finite");
  BPD_REQUIRE(a.rows * int64_t(a.tokens) == 0 || (a.q && a.out && a.lengths), "null pointer argument");
  BPD_REQUIRE(a.table.block_table || a.table.blocks == 0 || a.rows == 0, "null block table");
  BPD_REQUIRE((reinterpret_cast<uintptr_t>(a.out) & 3u) == 0, "the output must lie at a multiple of 4 bytes");
  BPD_REQUIRE(a.rows * int64_t(a.tokens) * a.heads < (int64_t(1) << 31), "too many queries in one call");
  return BPD_OK;
}

}  // namespace
}  // namespace bpd
