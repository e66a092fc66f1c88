// Attention of a block of query tokens over the 4-bit paged cache (kv4.hpp),
// and its host form.
//
// Query token i of a block of n sees the request's first length - n + 1 + i
// tokens (the block's own keys are already in the cache), so a single token
// sees all of them; out = softmax(scale q k^T) v over those, zeros where
// there are none.  Query heads share key heads in order: head h reads key
// head h / (heads / kv_heads).
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "kv4.hpp"

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
// whatever its length says (*past is set where it says more).
__host__ __device__ __forceinline__ int64_t seen_tokens(const AttendArgs& a, int64_t b, int32_t i, bool* past) {
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
constexpr int kWaves = 4;   // waves of a block
constexpr int kNever = 0x7FFFFFFF;

// How a call's work is cut.  A unit is one request, one key head and one group
// of query columns (tokens x heads that share the key head); its tiles are
// cut into equal splits of at least kWaves tiles, so that all splits of a call
// are about as long and there are about `target` of them.  The lengths are on
// the device, so every wave works the cut out for itself.
struct AttendPlan {
  int32_t groups;  // column groups
  int32_t cols;    // columns of a group, at most 16 * NT
  int32_t target;  // blocks that fill the device
  int32_t splits;  // at most this many splits over all requests
  float* partials;
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
__device__ __forceinline__ int32_t tiles_of(const AttendArgs& a, int64_t b) {
  return queries_of(a, b) > 0 ? int32_t((length_of(a, b) + kTile - 1) / kTile) : 0;
}

template <class T>
__device__ __forceinline__ T wave_sum(T x) {
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// Tiles that a split has at most, by the whole call's tiles.
__device__ __forceinline__ int32_t split_tiles(const AttendArgs& a, const AttendPlan& p, int lane) {
  int64_t whole = 0;
  for (int64_t b = lane; b < a.rows; b += kWave) whole += tiles_of(a, b);
  whole = wave_sum(whole) * (a.kv_heads * p.groups);
  const int64_t per = (whole + p.target - 1) / p.target;
  return per < kWaves ? kWaves : int32_t(per);
}
__device__ __forceinline__ int32_t splits_of(int32_t tiles, int32_t most) {
  return tiles <= most ? 1 : (tiles + most - 1) / most;
}

// The request whose splits hold number `at`, the number of its first split,
// and its splits; false past the last.
__device__ __forceinline__ bool find_split(const AttendArgs& a, int32_t most, int32_t at, int lane, int64_t* row,
                                           int32_t* first, int32_t* splits) {
  int32_t before = 0;
  for (int64_t b0 = 0; b0 < a.rows; b0 += kWave) {
    const int32_t mine = b0 + lane < a.rows ? splits_of(tiles_of(a, b0 + lane), most) : 0;
    int32_t upto = mine;
    for (int o = 1; o < kWave; o <<= 1) {
      const int32_t y = __shfl_up(upto, o);
      if (lane >= o) upto += y;
    }
    const uint64_t m = __ballot(before + upto > at);
    if (m) {
      const int hit = __builtin_ctzll(m);
      *row = b0 + hit;
      *splits = __builtin_amdgcn_readlane(mine, hit);
      *first = before + __builtin_amdgcn_readlane(upto, hit) - *splits;
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return false;
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

// Two codes (byte B of w) times a scale, as two elements of the type: exact.
template <int DT, int B>
__device__ __forceinline__ uint32_t two_values(uint32_t w, float s) {
  if constexpr (DT == BPD_DTYPE_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, B));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, B));
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
template <int DT>
__device__ __forceinline__ uint32_t two_rounded(float x, float y) {
  if constexpr (DT == BPD_DTYPE_BF16) {
    const bf16x2 r = {static_cast<__bf16>(x), static_cast<__bf16>(y)};
    return __builtin_bit_cast(uint32_t, r);
  } else {
    const f16x2 r = {static_cast<_Float16>(x), static_cast<_Float16>(y)};
    return __builtin_bit_cast(uint32_t, r);
  }
}

// Byte `at` + `lane_at` of an array of words as a power of two (the float
// whose exponent it is); lane_at < 4 differs between lanes.
__device__ __forceinline__ float scale_at(const uint32_t* w, int at, int words, uint32_t sel) {
  const int i = at / 4, o = at % 4;
  const uint32_t hi = i + 1 < words ? w[i + 1] : 0;
  return bits_float(__builtin_amdgcn_perm(hi, w[i], sel + (uint32_t(o) << 24)) >> 1);
}

// One block per split of a unit, its tiles dealt to the waves in turn.
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
// The running maximum is followed loosely: weights may grow to 2^8 before the
// sums are scaled down, so most tiles cost no exchange between lanes.
template <int DT, int D, int NT>
__global__ __launch_bounds__(kWaves* kWave) void kv_attend_kernel(AttendArgs a, AttendPlan plan) {
  using Pt = Parts<D>;
  constexpr int G = D / kKvGroup, KW = D / 32, VT = D / 16;  // scales, key words of a lane, value tiles
  constexpr int kScaleWords = 4 * G;                          // of 16 tokens
  __shared__ float joined[(kWaves / 2) * (2 + 4 * VT) * kWave];

  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int m = lane & 15, g = lane >> 4;
  int64_t x = blockIdx.x;
  int32_t group = 0;
  if (plan.groups > 1) {  // a unit's groups read the same keys: blocks 8 apart, on one XCD
    const int64_t r = x % (8 * plan.groups);
    group = int32_t(r / 8);
    x = x / (8 * plan.groups) * 8 + r % 8;
  }
  const int32_t at = int32_t(x / a.kv_heads), kvh = int32_t(x % a.kv_heads);
  const int32_t most = split_tiles(a, plan, lane);
  int64_t b;
  int32_t first, splits;
  if (!find_split(a, most, at, lane, &b, &first, &splits)) return;

  const int32_t n_q = queries_of(a, b), share = a.heads / a.kv_heads;
  const int64_t end = length_of(a, b);
  const int32_t tiles = tiles_of(a, b), per = (tiles + splits - 1) / splits;
  const int32_t tile0 = (at - first) * per, tile1 = tile0 + per < tiles ? tile0 + per : tiles;
  if (a.err && n_q > 0 && a.lengths[b] > end && threadIdx.x == 0) atomicOr(a.err, BPD_FLAG_PAGE_RANGE);

  // this lane's columns: the queries, and how many tokens each sees
  Frag q[NT][KW];
  int32_t sees[NT];
  int32_t least = int32_t(end);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int32_t c = group * plan.cols + t * 16 + m;
    const int32_t i = c / share, h = kvh * share + c % share;
    const bool in = t * 16 + m < plan.cols && i < n_q;
    const int64_t s = in ? int64_t(a.lengths[b]) - n_q + 1 + i : 0;
    sees[t] = int32_t(s < 0 ? 0 : s < end ? s : end);
    if (in) least = min(least, sees[t]);
    const uint16_t* row = a.q + b * a.q_row + (in ? i : 0) * a.q_token + (in ? h : 0) * a.q_head;
#pragma unroll
    for (int p = 0; p < Pt::count; ++p)
#pragma unroll
      for (int k = 0; k < Pt::width(p) / 32; ++k) {
        const uint16_t* from = row + Pt::begin(p) + g * (Pt::width(p) / 4) + 8 * k;
        Frag f = {{0u, 0u, 0u, 0u}};
        if (in) __builtin_memcpy(&f, from, 16);  // at any element
        q[t][Pt::begin(p) / 32 + k] = f;
      }
  }
  for (int o = 1; o < 16; o <<= 1) least = min(least, __shfl_xor(least, o));

  const int32_t P = a.page.page_size;
  const int shift = __builtin_ctz(P);
  const int32_t* table = a.table.block_table + b * a.table.ld;
  // page of the chunk of 16 tokens that starts at t, -1: none
  const auto page_at = [&](int64_t t) -> int32_t { return t < end ? table[t >> shift] : -1; };
  const auto block_at = [&](int32_t page) -> const uint8_t* {
    const int64_t ok = page >= 0 && page < a.table.num_pages ? page : 0;  // a page outside the pool is masked below
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
  // which of 4 neighbouring scales a lane takes: as a key lane, as a value lane
  uint32_t ksel[Pt::count], vsel[Pt::count];
#pragma unroll
  for (int p = 0; p < Pt::count; ++p) {
    ksel[p] = uint32_t(g * Pt::width(p) / 128) << 24 | 0x0C0C0C;
    vsel[p] = uint32_t(m * Pt::width(p) / 512) << 24 | 0x0C0C0C;
  }

  f32x4 acc[NT][VT];
  float top[NT], sum[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    top[t] = -3e38f, sum[t] = 0.0f;
#pragma unroll
    for (int v = 0; v < VT; ++v) acc[t][v] = f32x4{0, 0, 0, 0};
  }
  int32_t nan_at[Pt::count];  // first token of the tail whose value group is bad, as a value lane
#pragma unroll
  for (int p = 0; p < Pt::count; ++p) nan_at[p] = kNever;
  const float to_log2 = a.scale * 1.44269504088896340736f;

  int32_t tile = tile0 + wave;
  int32_t kpage = -1, vpage = -1, knext = -1, vnext = -1;
  if (tile < tile1) {
    const int64_t t0 = int64_t(tile) * kTile;
    kpage = page_at(t0 + (m >> 2) * 16), vpage = page_at(t0 + g * 16);
    load_keys(block_at(kpage), int32_t((t0 + 4 * m) & (P - 1)));
    load_values(block_at(vpage), int32_t((t0 + 16 * g) & (P - 1)));
    const int64_t t1 = int64_t(tile + kWaves) * kTile;
    if (tile + kWaves < tile1) knext = page_at(t1 + (m >> 2) * 16), vnext = page_at(t1 + g * 16);
  }
  for (; tile < tile1; tile += kWaves) {
    const int64_t t0 = int64_t(tile) * kTile, t1 = t0 + kWaves * kTile;
    const bool more = tile + kWaves < tile1;
    f32x4 s[NT][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int t = 0; t < NT; ++t) s[t][j] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int p = 0; p < Pt::count; ++p) {
        // the scale of this token's group: byte G j + Pt::begin(p) / 32 + (g's share)
        const float sc = scale_at(ks, G * j + Pt::begin(p) / kKvGroup, G, ksel[p]);
#pragma unroll
        for (int k = 0; k < Pt::width(p) / 32; ++k) {
          const uint32_t w = kc[j][Pt::begin(p) / 32 + k];
          Frag f;
          f.u[0] = two_values<DT, 0>(w, sc);
          f.u[1] = two_values<DT, 1>(w, sc);
          f.u[2] = two_values<DT, 2>(w, sc);
          f.u[3] = two_values<DT, 3>(w, sc);
#pragma unroll
          for (int t = 0; t < NT; ++t) s[t][j] = mfma<DT>(f, q[t][Pt::begin(p) / 32 + k], s[t][j]);
        }
      }
    }
    if (more) load_keys(block_at(knext), int32_t((t1 + 4 * m) & (P - 1)));

    // scores in units of log 2; token 16 g + 4 i + j of the tile is s[t][j][i]
    const int64_t mine = t0 + 16 * g;
    const bool there = vpage >= 0 && vpage < a.table.num_pages;
    const bool tail = t0 + kTile > least;
    const bool masked = __any(!there || tail);
    uint32_t quiet[Pt::count] = {};  // value groups that are left out: one bit per token
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][j][i] *= to_log2;
    if (masked) {
      if (!there && mine < end && a.err) atomicOr(a.err, BPD_FLAG_PAGE_RANGE);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!there || mine + 4 * i + j >= sees[t]) s[t][j][i] = -INFINITY;
      // values that no query or not every query sees: nothing where there is
      // no token, and bad groups are noted, so that a weight of 0 meets no NaN
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        const bool gone = !there || mine + u >= end;
#pragma unroll
        for (int p = 0; p < Pt::count; ++p) {
          const int byte = G * u + Pt::begin(p) / kKvGroup;
          const uint32_t e = float_bits(scale_at(vs, byte, kScaleWords, vsel[p])) >> 23;
          if (e == kKvBadScale && !gone && tail) {
            const int32_t tok = int32_t(mine + u);
            nan_at[p] = tok < nan_at[p] ? tok : nan_at[p];
          }
          if (gone || (e == kKvBadScale && tail)) vc[u][p] = 0, quiet[p] |= 1u << u;
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
      if (__any(most_here > top[t] + 8.0f)) {
        float now = fmaxf(top[t], most_here);
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
          s[t][j][i] = __builtin_amdgcn_exp2f(s[t][j][i] - top[t]);
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
          for (int e = 0; e < 2; ++e) {
            sc[e] = scale_at(vs, G * (u + e) + Pt::begin(p) / kKvGroup, kScaleWords, vsel[p]);
            if (masked) sc[e] = quiet[p] >> (u + e) & 1u ? 1.0f : sc[e];
          }
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
    const int64_t t2 = t1 + kWaves * kTile;
    if (tile + 2 * kWaves < tile1) knext = page_at(t2 + (m >> 2) * 16), vnext = page_at(t2 + g * 16);
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

#pragma unroll
  for (int t = 0; t < NT; ++t) {
    sum[t] += __shfl_xor(sum[t], 16);
    sum[t] += __shfl_xor(sum[t], 32);
    // join the waves, the upper half to the lower
    for (int half = kWaves / 2; half; half /= 2) {
      float* to = joined + (wave % half) * ((2 + 4 * VT) * kWave) + lane;
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
        to[0] = top[t], to[kWave] = sum[t];
#pragma unroll
        for (int v = 0; v < VT; ++v)
#pragma unroll
          for (int i = 0; i < 4; ++i) to[(2 + 4 * v + i) * kWave] = acc[t][v][i];
      }
      __syncthreads();
      if (wave < half) {
        const float other = to[0], now = fmaxf(top[t], other);
        const float f0 = __builtin_amdgcn_exp2f(top[t] - now), f1 = __builtin_amdgcn_exp2f(other - now);
        top[t] = now;
        sum[t] = sum[t] * f0 + to[kWave] * f1;
#pragma unroll
        for (int v = 0; v < VT; ++v)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][v][i] = acc[t][v][i] * f0 + to[(2 + 4 * v + i) * kWave] * f1;
      }
    }
    if (wave) continue;
    if (splits == 1) {
      const int32_t c = group * plan.cols + t * 16 + m;
      const int32_t i = c / share, h = kvh * share + c % share;
      if (t * 16 + m >= plan.cols || i >= a.tokens) continue;
      uint16_t* out = a.out + ((b * a.tokens + i) * a.heads + h) * D;
      const float inv = sum[t] == 0.0f ? 0.0f : 1.0f / sum[t];
#pragma unroll
      for (int p = 0; p < Pt::count; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          uint16_t* at_row = out + Pt::begin(p) + (4 * g + r) * (Pt::width(p) / 16);
#pragma unroll
          for (int v = 0; v < Pt::width(p) / 16; v += 2)
            *reinterpret_cast<uint32_t*>(at_row + v) =
                two_rounded<DT>(acc[t][Pt::begin(p) / 16 + v][r] * inv, acc[t][Pt::begin(p) / 16 + v + 1][r] * inv);
        }
    } else {
      float* to = plan.partials + ((int64_t(at) * a.kv_heads + kvh) * plan.groups + group) * (NT * (2 + 4 * VT) * kWave) +
                  t * ((2 + 4 * VT) * kWave);
      to[lane] = top[t], to[kWave + lane] = sum[t];
#pragma unroll
      for (int v = 0; v < VT; ++v)
        *reinterpret_cast<f32x4*>(to + 2 * kWave + (v * kWave + lane) * 4) = acc[t][v];
    }
  }
}

// Joins a unit's splits: one block per unit, column tile and pair of value
// tiles, its waves over the splits.
template <int DT, int D, int NT>
__global__ __launch_bounds__(kWaves* kWave) void kv_attend_join_kernel(AttendArgs a, AttendPlan plan) {
  using Pt = Parts<D>;
  constexpr int VT = D / 16, kPiece = (2 + 4 * VT) * kWave;
  __shared__ float joined[kWaves][10][kWave];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int m = lane & 15, g = lane >> 4;
  int64_t x = blockIdx.x;
  const int v0 = int(x % (VT / 2)) * 2;
  x /= VT / 2;
  const int t = int(x % NT);
  x /= NT;
  const int32_t group = int32_t(x % plan.groups);
  x /= plan.groups;
  const int32_t kvh = int32_t(x % a.kv_heads);
  const int64_t b = x / a.kv_heads;
  const int32_t most = split_tiles(a, plan, lane);
  const int32_t splits = splits_of(tiles_of(a, b), most);
  if (splits == 1) return;
  int32_t first = 0;
  for (int64_t r = lane; r < b; r += kWave) first += splits_of(tiles_of(a, r), most);
  first = wave_sum(first);
  const float* from = plan.partials + ((int64_t(first) * a.kv_heads + kvh) * plan.groups + group) * (NT * kPiece) + t * kPiece;
  const int64_t step = int64_t(a.kv_heads) * plan.groups * (NT * kPiece);
  float top = -3e38f, sum = 0.0f;
  f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  for (int32_t i = wave; i < splits; i += kWaves) {
    const float* p = from + i * step;
    const float other = p[lane], now = fmaxf(top, other);
    const float f0 = __builtin_amdgcn_exp2f(top - now), f1 = __builtin_amdgcn_exp2f(other - now);
    top = now;
    sum = sum * f0 + p[kWave + lane] * f1;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(p + 2 * kWave + ((v0 + v) * kWave + lane) * 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[v][k] = acc[v][k] * f0 + y[k] * f1;
    }
  }
  joined[wave][0][lane] = top, joined[wave][1][lane] = sum;
#pragma unroll
  for (int k = 0; k < 4; ++k) joined[wave][2 + k][lane] = acc[0][k], joined[wave][6 + k][lane] = acc[1][k];
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    const float other = joined[w][0][lane], now = fmaxf(top, other);
    const float f0 = __builtin_amdgcn_exp2f(top - now), f1 = __builtin_amdgcn_exp2f(other - now);
    top = now;
    sum = sum * f0 + joined[w][1][lane] * f1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      acc[0][k] = acc[0][k] * f0 + joined[w][2 + k][lane] * f1;
      acc[1][k] = acc[1][k] * f0 + joined[w][6 + k][lane] * f1;
    }
  }
  const int32_t share = a.heads / a.kv_heads, c = group * plan.cols + t * 16 + m;
  const int32_t i = c / share, h = kvh * share + c % share;
  if (t * 16 + m >= plan.cols || i >= a.tokens) return;
  uint16_t* out = a.out + ((b * a.tokens + i) * a.heads + h) * D;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const int p = v0 * 16 < Pt::first ? 0 : 1;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    *reinterpret_cast<uint32_t*>(out + Pt::begin(p) + (4 * g + r) * (Pt::width(p) / 16) + v0 - Pt::begin(p) / 16) =
        two_rounded<DT>(acc[0][r] * inv, acc[1][r] * inv);
}

// Column tiles of a wave: every query column of a key head where they fit.
// More share the conversions of keys and values, but the registers of four
// (of two from 192 channels on) are the most that leave waves to hide loads.
constexpr int most_tiles(int dim) { return dim > 128 ? 2 : 4; }

struct AttendSizes {
  AttendPlan plan;
  int32_t nt;
  size_t piece;  // floats of one split's partial result
};

AttendSizes attend_sizes(int64_t rows, int32_t tokens, int32_t heads, int32_t kv_heads, int32_t dim, int64_t longest) {
  AttendSizes z{};
  const int64_t cols = int64_t(tokens) * (heads / kv_heads);
  const int64_t tiles = (cols + 15) / 16, most = most_tiles(dim);
  z.nt = tiles <= 1 ? 1 : tiles <= 2 || most == 2 ? 2 : 4;
  z.plan.groups = int32_t((tiles + z.nt - 1) / z.nt);
  z.plan.cols = int32_t((cols + z.plan.groups - 1) / z.plan.groups);
  z.plan.target = 2048;
  const int64_t units = int64_t(kv_heads) * z.plan.groups;
  // at least kWaves tiles each, and about `target` over all units
  const int64_t per_row = ((longest + kTile - 1) / kTile + kWaves - 1) / kWaves;
  const int64_t by_length = rows * (per_row < 1 ? 1 : per_row), by_target = z.plan.target / units + 1 + rows;
  z.plan.splits = int32_t(std::min(by_length, by_target));
  z.piece = size_t(z.nt) * (2 + dim / 4) * kWave;
  return z;
}

template <int DT, int D, int NT>
int launch_attend(const AttendArgs& a, const AttendSizes& z, hipStream_t s) {
  const int64_t units = int64_t(z.plan.splits) * a.kv_heads;
  const int64_t blocks = z.plan.groups == 1 ? units : (units + 7) / 8 * 8 * z.plan.groups;
  const int64_t joins = a.rows * a.kv_heads * z.plan.groups * NT * (D / 32);
  BPD_REQUIRE(blocks < (int64_t(1) << 31) && joins < (int64_t(1) << 31), "too many queries in one call");
  kv_attend_kernel<DT, D, NT><<<uint32_t(blocks), kWaves * kWave, 0, s>>>(a, z.plan);
  if (z.plan.splits > a.rows) kv_attend_join_kernel<DT, D, NT><<<uint32_t(joins), kWaves * kWave, 0, s>>>(a, z.plan);
  BPD_LAUNCHED();
  return BPD_OK;
}

template <int DT, int D>
int launch_attend_tiles(const AttendArgs& a, const AttendSizes& z, hipStream_t s) {
  if (z.nt == 1) return launch_attend<DT, D, 1>(a, z, s);
  if constexpr (most_tiles(D) == 4)
    if (z.nt == 4) return launch_attend<DT, D, 4>(a, z, s);
  return launch_attend<DT, D, 2>(a, z, s);
}

template <int DT>
int launch_attend_dim(const AttendArgs& a, const AttendSizes& z, hipStream_t s) {
  switch (a.page.dim) {
    case 64: return launch_attend_tiles<DT, 64>(a, z, s);
    case 96: return launch_attend_tiles<DT, 96>(a, z, s);
    case 128: return launch_attend_tiles<DT, 128>(a, z, s);
    case 192: return launch_attend_tiles<DT, 192>(a, z, s);
    default: return launch_attend_tiles<DT, 256>(a, z, s);
  }
}

template <int DT>
void host_attend(const AttendArgs& a) {
  const int32_t D = a.page.dim;
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
          const int64_t page = a.table.page_of(b, t, a.page.page_size);
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
          const int64_t page = a.table.page_of(b, t, a.page.page_size);
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
  BPD_REQUIRE(a.rows * int64_t(a.tokens) * a.heads < (int64_t(1) << 31), "too many queries in one call");
  return BPD_OK;
}

}  // namespace
}  // namespace bpd

using namespace bpd;

#define BPD_ATTEND_ARGS                                                                                    \
  AttendArgs a {                                                                                           \
    pages, KvPage{page_size, head_dim}, KvTable{block_table, table_ld, table_blocks, num_pages}, kv_heads, \
        heads, static_cast<const uint16_t*>(q), q_row, q_token, q_head, static_cast<uint16_t*>(out), rows, \
        tokens, lengths, query_lens, scale, err                                                            \
  }

extern "C" size_t bpd_kv_attend_workspace_bytes(int64_t rows, int32_t tokens, int32_t heads, int32_t kv_heads,
                                                int32_t head_dim, int64_t longest) {
  if (rows <= 0 || tokens <= 0 || kv_heads <= 0 || heads < kv_heads) return 0;
  const AttendSizes z = attend_sizes(rows, tokens, heads, kv_heads, head_dim, longest);
  return z.plan.splits > rows ? size_t(z.plan.splits) * kv_heads * z.plan.groups * z.piece * sizeof(float) : 0;
}

extern "C" int bpd_kv_attend(const uint8_t* pages, int64_t num_pages, int32_t page_size, int32_t kv_heads,
                             int32_t head_dim, int dtype, const void* q, int64_t q_row, int64_t q_token,
                             int64_t q_head, int32_t heads, void* out, int64_t rows, int32_t tokens,
                             const int32_t* block_table, int64_t table_ld, int32_t table_blocks,
                             const int32_t* lengths, const int32_t* query_lens, float scale, void* workspace,
                             size_t workspace_bytes, int32_t* err, void* stream) {
  BPD_ATTEND_ARGS;
  if (int rc = check_attend(a, dtype)) return rc;
  if (rows == 0 || tokens == 0) return BPD_OK;
  if (num_pages == 0) a.table.blocks = 0;  // no page to read: every length lies past the table
  const int64_t longest = int64_t(table_blocks) * page_size;
  AttendSizes z = attend_sizes(rows, tokens, heads, kv_heads, head_dim, longest);
  BPD_REQUIRE(workspace_bytes >= bpd_kv_attend_workspace_bytes(rows, tokens, heads, kv_heads, head_dim, longest) &&
                  (workspace || z.plan.splits <= rows),
              "the workspace is smaller than bpd_kv_attend_workspace_bytes");
  z.plan.partials = static_cast<float*>(workspace);
  return dtype == BPD_DTYPE_BF16 ? launch_attend_dim<BPD_DTYPE_BF16>(a, z, as_stream(stream))
                                 : launch_attend_dim<BPD_DTYPE_F16>(a, z, as_stream(stream));
}

extern "C" int bpd_host_kv_attend(const uint8_t* pages, int64_t num_pages, int32_t page_size, int32_t kv_heads,
                                  int32_t head_dim, int dtype, const void* q, int64_t q_row, int64_t q_token,
                                  int64_t q_head, int32_t heads, void* out, int64_t rows, int32_t tokens,
                                  const int32_t* block_table, int64_t table_ld, int32_t table_blocks,
                                  const int32_t* lengths, const int32_t* query_lens, float scale, int32_t* err) {
  BPD_ATTEND_ARGS;
  if (int rc = check_attend(a, dtype)) return rc;
  if (rows == 0 || tokens == 0) return BPD_OK;
  if (dtype == BPD_DTYPE_BF16)
    host_attend<BPD_DTYPE_BF16>(a);
  else
    host_attend<BPD_DTYPE_F16>(a);
  return BPD_OK;
}
