// The 4-bit paged cache (kv4.hpp): rotating a block's keys and queries to
// their positions and appending keys and values, reading tokens back, and
// the host forms of both.
#include <algorithm>
#include <type_traits>

#include "kv4.hpp"

namespace bpd {
namespace {

// Strides of q, k and v in elements: request, token, head (channels are next
// to each other).
struct Strides3 {
  int64_t row, token, head;
};

struct AppendArgs {
  uint8_t* pages;
  KvPage page;
  KvTable table;
  int32_t kv_heads, heads;
  const uint16_t *k, *v, *q;
  Strides3 ks, vs, qs;
  uint16_t* q_out;  // [rows, tokens, heads, dim]
  int64_t rows;
  int32_t tokens;
  const int32_t *starts, *counts;
  const float *cos, *sin;  // [positions, rotary / 2]
  int64_t positions;
  int32_t rotary;
  int32_t interleaved;
  int32_t* err;
  // positions apart from the place in the cache: of each token on `num_axes`
  // axes (0: none), and the axis of each channel pair (null: the first)
  const int32_t* places;
  int64_t place_axis, place_row, place_token;
  int32_t num_axes;
  const int32_t* axes;
};

// A token's rows of the rotation's tables, by axis.
struct Turns {
  int32_t first, second, third, fourth;
};
static_assert(BPD_MAX_AXES == 4, "as many as Turns holds");
// (an axis past the last is read as it, one below 0 as the first)
__host__ __device__ __forceinline__ int32_t turn_on(Turns t, int32_t axis) {
  // (sums: a choice between places to read from would put them into memory)
  return t.first + (axis > 0 ? t.second - t.first : 0) + (axis > 1 ? t.third - t.second : 0) +
         (axis > 2 ? t.fourth - t.third : 0);
}
// False where one lies outside the tables.
__host__ __device__ __forceinline__ bool turns_of(const AppendArgs& a, int64_t b, int32_t i, Turns* t) {
  const int32_t* place = a.places + b * a.place_row + i * a.place_token;
  const int32_t last = a.num_axes - 1;
  const auto at = [&](int32_t k) { return place[(k < last ? k : last) * a.place_axis]; };
  *t = Turns{at(0), at(1), at(2), at(3)};
  const auto in = [&](int32_t x) { return x >= 0 && x < a.positions; };
  return bool(int(in(t->first)) & int(in(t->second)) & int(in(t->third)) & int(in(t->fourth)));
}

// The axis of a pair; one that is not there is flagged.
__host__ __device__ __forceinline__ int32_t axis_of(const AppendArgs& a, int32_t pair) {
  const int32_t x = a.axes ? a.axes[pair] : 0;
  if ((x < 0 || x >= a.num_axes) && a.err) {
#ifdef __HIP_DEVICE_COMPILE__
    atomicOr(a.err, BPD_FLAG_PAGE_RANGE);
#else
    *a.err |= BPD_FLAG_PAGE_RANGE;
#endif
  }
  return x;
}

// Whether token i of request b is appended, and where; sets *bad where it
// should be and cannot.  *turn: its row of the rotation's tables (without axes
// of its own), or -1.  on_axes: whether the positions on axes are in the tables.
__host__ __device__ __forceinline__ int64_t append_place(const AppendArgs& a, int64_t b, int32_t i, int32_t start,
                                                         bool on_axes, int64_t* pos, int64_t* turn, bool* bad) {
  *bad = false;
  *turn = -1;
  if (a.counts && i >= a.counts[b]) return -1;
  *pos = int64_t(start) + i;
  if (*pos < 0 || (a.num_axes > 0 ? !on_axes : a.rotary > 0 && *pos >= a.positions)) {
    *bad = true;
    return -1;
  }
  *turn = *pos;
  const int64_t page = a.table.page_of(b, *pos, a.page.page_size);
  *bad = page < 0;
  return page;
}

constexpr int kKvThreads = 256;
constexpr int kKvWidth = 8;  // channels of a thread: four threads hold a group
// A block holds one token, a thread the same 8 channels of up to kKvPasses
// heads, all of them loaded before the first is used: the rotation's tables
// are read once, and the loads of a block are in flight together.
constexpr int kKvPasses = 4;

template <int D>
struct KvBlock {
  static constexpr int per_head = D / kKvWidth;               // threads of a head
  static constexpr int heads = kKvThreads / per_head;         // heads at a time
  static constexpr int blocks(int64_t n, int passes) { return int((n + heads * passes - 1) / (heads * passes)); }
};

// 8 neighbouring 16-bit elements at any address of theirs.
typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
typedef float floats4 __attribute__((ext_vector_type(4), aligned(4)));

template <int DT>
__device__ __forceinline__ void unpack8(words4 w, float (&x)[kKvWidth]) {
#pragma unroll
  for (int j = 0; j < kKvWidth; ++j) x[j] = elem16_float<DT>(uint16_t(w[j / 2] >> (16 * (j & 1))));
}

// How a thread finds the partners of its 8 channels: they are 8 channels half
// the rotated ones away, or its own, or anywhere (rotated channels that are no
// multiple of 16, of 8 for neighbours).
enum Partners { kHalves, kNeighbours, kAnywhere };

// Heads in the order queries, keys, values.  A rotation's products and sums are
// rounded one by one (kv4.hpp); the codes come from the hardware's conversion.
// Bound by memory: 49,000 tokens of 48 heads of 128, 1.2 GB with the rotated
// queries, in 276 us, 4.4 TB/s, where a large copy reaches 4.9.
// With Axes a pair's row of the tables goes by its axis; 8 pairs of one axis
// (blocks of them, as models with axes for time, height and width lay them out)
// are read as without, others one by one.  (12 prompts of 2,900 tokens, 36 heads
// of 128, three axes in blocks: 147 us, 4.0 TB/s, 128 without axes; 3 blocks of
// 1,533 tokens, 32 heads of 96, the axes of neighbouring pairs in turn: 22.)
template <int DT, int D, int Passes, int Mode, bool Axes>
__global__ __launch_bounds__(kKvThreads) void kv_append_kernel(AppendArgs a, uint32_t parts) {
  using B = KvBlock<D>;
  const int tid = threadIdx.x, slot = tid / B::per_head, d0 = tid % B::per_head * kKvWidth;
  const uint32_t token = blockIdx.x / parts, part = blockIdx.x - token * parts;
  const int64_t b = token / uint32_t(a.tokens);
  const int32_t i = int32_t(token - uint32_t(b) * uint32_t(a.tokens));
  // (the loads wait for the count alone, not for the token's place)
  const bool counted = !a.counts || i < a.counts[b];
  if (!counted && a.heads == 0) return;
  const int32_t total = a.heads + 2 * a.kv_heads, half = a.rotary / 2;
  const bool rotated = d0 < a.rotary;
  const bool upper = rotated && d0 >= half;

  // the axes of the thread's pairs, on their way first
  constexpr int kPairs = Mode == kHalves ? kKvWidth : kKvWidth / 2;
  const int32_t pair = Mode == kNeighbours ? d0 / 2 : upper ? d0 - half : d0;
  Turns own{};
  bool on_axes = false;
  int32_t axis[kPairs] = {};
  if constexpr (Axes) {
    if (Mode != kAnywhere && rotated && a.axes)
#pragma unroll
      for (int j = 0; j < kPairs; ++j) axis[j] = a.axes[pair + j];
  }
  const uint16_t* qs = a.q + b * a.qs.row + i * a.qs.token;
  const uint16_t* ks = a.k + b * a.ks.row + i * a.ks.token;
  const uint16_t* vs = a.v + b * a.vs.row + i * a.vs.token;
  words4 x[Passes], partner[Passes];
  int32_t kind[Passes], head[Passes];  // 0 queries, 1 keys, 2 values, 4 none
#pragma unroll
  for (int p = 0; p < Passes; ++p) {
    const int32_t h = (int32_t(part) * Passes + p) * B::heads + slot;
    kind[p] = slot >= B::heads || h >= total ? 4 : h < a.heads ? 0 : h < a.heads + a.kv_heads ? 1 : 2;
    head[p] = kind[p] == 2 ? h - a.heads - a.kv_heads : kind[p] == 1 ? h - a.heads : h;
    x[p] = partner[p] = words4{0u, 0u, 0u, 0u};
    if (!counted || kind[p] > 2) continue;
    const uint16_t* from = kind[p] == 0 ? qs : kind[p] == 1 ? ks : vs;
    from += head[p] * (kind[p] == 0 ? a.qs.head : kind[p] == 1 ? a.ks.head : a.vs.head) + d0;
    x[p] = *reinterpret_cast<const words4*>(from);
    if (Mode == kHalves && rotated && kind[p] != 2)
      partner[p] = *reinterpret_cast<const words4*>(upper ? from - half : from + half);
  }
  const int32_t start = a.starts[b];
  if constexpr (Axes) on_axes = turns_of(a, b, i, &own);
  int64_t pos, turn;
  bool bad;
  const int64_t page = append_place(a, b, i, start, on_axes, &pos, &turn, &bad);
  if (bad && a.err && tid == 0 && part == 0) atomicOr(a.err, BPD_FLAG_PAGE_RANGE);
  const bool turns = rotated && turn >= 0;
  float c[kKvWidth], sn[kKvWidth];
  bool apart = false;  // the pairs lie on several axes
  if (Axes && Mode != kAnywhere && turns) {
    bool outside = false;
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      apart |= axis[j] != axis[0];
      outside |= axis[j] < 0 || axis[j] >= a.num_axes;
    }
    if (outside && a.err) atomicOr(a.err, BPD_FLAG_PAGE_RANGE);
    turn = turn_on(own, axis[0]);
    if (apart) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const int64_t at = int64_t(turn_on(own, axis[j])) * half + pair + j;
        c[j] = a.cos[at], sn[j] = Mode == kHalves && !upper ? -a.sin[at] : a.sin[at];
      }
    }
  }
  if (Mode != kAnywhere && turns && !apart) {
    const int64_t at = turn * half + pair;
#pragma unroll
    for (int k = 0; k < (Mode == kHalves ? 2 : 1); ++k) {
      const floats4 y = *reinterpret_cast<const floats4*>(a.cos + at + 4 * k), z = *reinterpret_cast<const floats4*>(a.sin + at + 4 * k);
      // halves: x c - y s below, y c + x s above, each product and sum rounded
      // by itself; the sign goes with the sine
#pragma unroll
      for (int j = 0; j < 4; ++j) c[4 * k + j] = y[j], sn[4 * k + j] = Mode == kHalves && !upper ? -z[j] : z[j];
    }
  }
#pragma unroll
  for (int p = 0; p < Passes; ++p) {
    if (kind[p] > 2) continue;
    float val[kKvWidth];
    unpack8<DT>(x[p], val);
    if (turns && kind[p] < 2) {
      if constexpr (Mode == kHalves) {
        float other[kKvWidth];
        unpack8<DT>(partner[p], other);
#pragma unroll
        for (int j = 0; j < kKvWidth; ++j) val[j] = rot_second(other[j], val[j], c[j], sn[j]);
      } else if constexpr (Mode == kNeighbours) {
#pragma unroll
        for (int j = 0; j < kKvWidth; j += 2) {
          const float u = val[j], w = val[j + 1];
          val[j] = rot_first(u, w, c[j / 2], sn[j / 2]);
          val[j + 1] = rot_second(u, w, c[j / 2], sn[j / 2]);
        }
      } else {
        const uint16_t* from = kind[p] == 0 ? qs + head[p] * a.qs.head : ks + head[p] * a.ks.head;
#pragma unroll
        for (int j = 0; j < kKvWidth; ++j)
          val[j] = rotated_channel<DT>(from, d0 + j, a.rotary, a.interleaved, [&](int32_t pair, float* x, float* y) {
            const int64_t at = (Axes ? turn_on(own, axis_of(a, pair)) : turn) * half + pair;
            *x = a.cos[at], *y = a.sin[at];
          });
      }
    }
    if (kind[p] == 0) {
      uint4 w = {two_rounded<DT>(val[0], val[1]), two_rounded<DT>(val[2], val[3]), two_rounded<DT>(val[4], val[5]),
                 two_rounded<DT>(val[6], val[7])};
      if (turn < 0) w = uint4{0u, 0u, 0u, 0u};
      *reinterpret_cast<uint4*>(a.q_out + (int64_t(token) * a.heads + head[p]) * D + d0) = w;
      continue;
    }
    if (page < 0) continue;
    // the four threads of a group are neighbours in a wave
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < kKvWidth; ++j) most = max(most, float_bits(val[j]) & 0x7FFFFFFFu);
    most = max(most, uint32_t(__shfl_xor(int(most), 1)));
    most = max(most, uint32_t(__shfl_xor(int(most), 2)));
    const int32_t e = kv_scale_byte<DT>(most);
    // the conversion rounds as kv_code does; adding 0 clears the sign of -0
    const float sc = bits_float(uint32_t(e) << 23);
    uint32_t word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, val[0] + 0.0f, val[1] + 0.0f, sc, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, val[2] + 0.0f, val[3] + 0.0f, sc, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, val[4] + 0.0f, val[5] + 0.0f, sc, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, val[6] + 0.0f, val[7] + 0.0f, sc, 3);
    if (e == kKvBadScale) word = 0;
    uint8_t* block = a.pages + (page * a.kv_heads + head[p]) * int64_t(a.page.bytes());
    const int32_t t = int32_t(pos & (a.page.page_size - 1));
    *reinterpret_cast<uint32_t*>(block + (kind[p] == 2 ? a.page.v_codes() : 0) + t * (D / 2) + d0 / 2) = word;
    if ((d0 & (kKvGroup - 1)) == 0)
      block[(kind[p] == 2 ? a.page.v_scales() : a.page.k_scales()) + t * (D / kKvGroup) + d0 / kKvGroup] = uint8_t(e);
  }
}

template <int DT>
void host_append(const AppendArgs& a) {
  const int32_t D = a.page.dim;
  for (int64_t b = 0; b < a.rows; ++b)
    for (int32_t i = 0; i < a.tokens; ++i) {
      int64_t pos, turn;
      bool bad;
      Turns own{};
      const bool on_axes = a.num_axes > 0 && turns_of(a, b, i, &own);
      const int64_t page = append_place(a, b, i, a.starts[b], on_axes, &pos, &turn, &bad);
      if (bad && a.err) *a.err |= BPD_FLAG_PAGE_RANGE;
      const auto angle = [&](int32_t pair, float* c, float* s) {
        const int64_t at = (a.num_axes > 0 ? turn_on(own, axis_of(a, pair)) : turn) * (a.rotary / 2) + pair;
        *c = a.cos[at], *s = a.sin[at];
      };
      for (int32_t h = 0; h < a.heads; ++h) {
        const uint16_t* x = a.q + b * a.qs.row + i * a.qs.token + h * a.qs.head;
        uint16_t* out = a.q_out + ((b * a.tokens + i) * a.heads + h) * D;
        for (int32_t d = 0; d < D; ++d)
          out[d] = turn >= 0 ? float_elem16<DT>(rotated_channel<DT>(x, d, a.rotary, a.interleaved, angle)) : 0;
      }
      if (page < 0) continue;
      const int32_t t = int32_t(pos % a.page.page_size);
      for (int32_t h = 0; h < 2 * a.kv_heads; ++h) {
        const bool is_v = h >= a.kv_heads;
        const int32_t hh = is_v ? h - a.kv_heads : h;
        const uint16_t* x = is_v ? a.v + b * a.vs.row + i * a.vs.token + hh * a.vs.head
                                 : a.k + b * a.ks.row + i * a.ks.token + hh * a.ks.head;
        uint8_t* block = a.pages + (page * a.kv_heads + hh) * int64_t(a.page.bytes());
        uint8_t* codes = block + (is_v ? a.page.v_codes() : 0) + t * a.page.codes();
        uint8_t* scales = block + (is_v ? a.page.v_scales() : a.page.k_scales()) + t * a.page.groups();
        for (int32_t g = 0; g < a.page.groups(); ++g) {
          float val[kKvGroup];
          uint32_t most = 0;
          for (int32_t j = 0; j < kKvGroup; ++j) {
            val[j] = rotated_channel<DT>(x, g * kKvGroup + j, is_v ? 0 : a.rotary, a.interleaved, angle);
            most = std::max(most, float_bits(val[j]) & 0x7FFFFFFFu);
          }
          const int32_t e = kv_scale_byte<DT>(most);
          scales[g] = uint8_t(e);
          for (int32_t j = 0; j < kKvGroup; j += 2)
            codes[(g * kKvGroup + j) / 2] = uint8_t(kv_code(val[j], e) | kv_code(val[j + 1], e) << 4);
        }
      }
    }
}

struct ReadArgs {
  const uint8_t* pages;
  KvPage page;
  KvTable table;
  int32_t kv_heads;
  uint16_t *k, *v;  // [rows, tokens, kv_heads, dim]
  int64_t rows;
  int32_t tokens;
  const int32_t *starts, *counts;
  int32_t* err;
};

__host__ __device__ __forceinline__ int64_t read_place(const ReadArgs& a, int64_t b, int32_t i, int64_t* pos,
                                                       bool* bad) {
  *bad = false;
  if (a.counts && i >= a.counts[b]) return -1;
  *pos = int64_t(a.starts[b]) + i;
  const int64_t page = a.table.page_of(b, *pos, a.page.page_size);
  *bad = page < 0;
  return page;
}

// Heads in the order keys, values (320 MB in 85 us: 3.8 TB/s, mostly written).
// A block takes `parts`-th shares of the heads
// of one token, or, where all heads are one share, Passes tokens after another.
template <int DT, int D, int Passes>
__global__ __launch_bounds__(kKvThreads) void kv_read_kernel(ReadArgs a, uint32_t parts) {
  using B = KvBlock<D>;
  const int tid = threadIdx.x, slot = tid / B::per_head, d0 = tid % B::per_head * kKvWidth;
  const uint32_t first = blockIdx.x / parts * Passes, part = blockIdx.x % parts;
  const int32_t h = int32_t(part) * B::heads + slot;
  const bool is_v = h >= a.kv_heads, in = slot < B::heads && h < 2 * a.kv_heads;
  const int32_t head = is_v ? h - a.kv_heads : h;
  const uint32_t tokens = uint32_t(a.rows) * uint32_t(a.tokens);
  uint32_t word[Passes], e[Passes];
#pragma unroll
  for (int p = 0; p < Passes; ++p) {
    const uint32_t token = first + p;
    word[p] = 0, e[p] = 127;
    if (token >= tokens) continue;
    const uint32_t b = token / uint32_t(a.tokens);
    int64_t pos;
    bool bad;
    const int64_t page = read_place(a, b, int32_t(token - b * uint32_t(a.tokens)), &pos, &bad);
    if (bad && a.err && tid == 0 && part == 0) atomicOr(a.err, BPD_FLAG_PAGE_RANGE);
    if (page < 0 || !in) continue;
    const uint8_t* block = a.pages + (page * a.kv_heads + head) * int64_t(a.page.bytes());
    const int32_t t = int32_t(pos & (a.page.page_size - 1));
    word[p] = *reinterpret_cast<const uint32_t*>(block + (is_v ? a.page.v_codes() : 0) + t * (D / 2) + d0 / 2);
    e[p] = block[(is_v ? a.page.v_scales() : a.page.k_scales()) + t * (D / kKvGroup) + d0 / kKvGroup];
  }
#pragma unroll
  for (int p = 0; p < Passes; ++p) {
    const uint32_t token = first + p;
    if (token >= tokens || !in) break;
    uint16_t* out = (is_v ? a.v : a.k) + (int64_t(token) * a.kv_heads + head) * D + d0;
    const float s = bits_float(e[p] << 23);
    *reinterpret_cast<uint4*>(out) = uint4{two_values<DT, 0>(word[p], s), two_values<DT, 1>(word[p], s),
                                           two_values<DT, 2>(word[p], s), two_values<DT, 3>(word[p], s)};
  }
}

template <int DT>
void host_read(const ReadArgs& a) {
  const int32_t D = a.page.dim;
  for (int64_t b = 0; b < a.rows; ++b)
    for (int32_t i = 0; i < a.tokens; ++i) {
      int64_t pos;
      bool bad;
      const int64_t page = read_place(a, b, i, &pos, &bad);
      if (bad && a.err) *a.err |= BPD_FLAG_PAGE_RANGE;
      for (int32_t h = 0; h < 2 * a.kv_heads; ++h) {
        const bool is_v = h >= a.kv_heads;
        const int32_t hh = is_v ? h - a.kv_heads : h;
        uint16_t* out = (is_v ? a.v : a.k) + ((b * a.tokens + i) * a.kv_heads + hh) * D;
        if (page < 0) {
          std::fill(out, out + D, uint16_t(0));
          continue;
        }
        const uint8_t* block = a.pages + (page * a.kv_heads + hh) * int64_t(a.page.bytes());
        const int32_t t = int32_t(pos % a.page.page_size);
        const uint8_t* codes = block + (is_v ? a.page.v_codes() : 0) + t * a.page.codes();
        const uint8_t* scales = block + (is_v ? a.page.v_scales() : a.page.k_scales()) + t * a.page.groups();
        for (int32_t d = 0; d < D; ++d)
          out[d] = float_elem16<DT>(kv_value(uint32_t(codes[d / 2]) >> (4 * (d & 1)) & 15u, scales[d / kKvGroup]));
      }
    }
}

int check_append(const AppendArgs& a, int dtype) {
  if (int rc = check_kv_cache(a.pages, a.page, a.table, a.kv_heads, dtype)) return rc;
  BPD_REQUIRE(a.rows >= 0 && a.tokens >= 0, "negative sizes");
  BPD_REQUIRE(a.rotary >= 0 && a.rotary % 2 == 0 && a.rotary <= a.page.dim,
              "the rotated channels must be even and at most head_dim (got %d of %d)", a.rotary, a.page.dim);
  BPD_REQUIRE(a.rotary == 0 || (a.cos && a.sin && a.positions >= 0), "the rotation needs its tables");
  BPD_REQUIRE(a.num_axes >= 0 && a.num_axes <= BPD_MAX_AXES, "positions of 1 to %d axes (got %d)", BPD_MAX_AXES, a.num_axes);
  BPD_REQUIRE(a.num_axes == 0 || a.rotary > 0, "positions need the rotation's tables");
  BPD_REQUIRE(a.num_axes == 0 || a.places || a.rows * a.tokens == 0, "null positions");
  BPD_REQUIRE((reinterpret_cast<uintptr_t>(a.q_out) & 15u) == 0, "the output must lie at a multiple of 16 bytes");
  BPD_REQUIRE(a.heads >= 0 && (a.heads == 0 || (a.q && a.q_out) || a.rows * a.tokens == 0), "null query pointer");
  BPD_REQUIRE(a.rows * int64_t(a.tokens) == 0 || (a.k && a.v && a.table.block_table && a.starts),
              "null pointer argument");
  return BPD_OK;
}

int check_read(const ReadArgs& a, int dtype) {
  if (int rc = check_kv_cache(a.pages, a.page, a.table, a.kv_heads, dtype)) return rc;
  BPD_REQUIRE(a.rows >= 0 && a.tokens >= 0, "negative sizes");
  BPD_REQUIRE(((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 15u) == 0,
              "the outputs must lie at multiples of 16 bytes");
  BPD_REQUIRE(a.rows * int64_t(a.tokens) == 0 || (a.k && a.v && a.table.block_table && a.starts),
              "null pointer argument");
  return BPD_OK;
}

// Several passes to a block where the tokens fill the device by themselves (48
// heads of 128, appended and read back: 2,048 tokens 23.0 us, 25.6 with one
// pass to a block; 16,384: 104 and 109).
constexpr int64_t kKvFill = 512;

template <int DT, int D>
int launch_append(const AppendArgs& a, hipStream_t s) {
  using B = KvBlock<D>;
  const int64_t n = a.rows * a.tokens, total = a.heads + 2 * int64_t(a.kv_heads);
  const bool any = a.rotary % (a.interleaved ? 8 : 16) != 0, many = !any && n >= kKvFill;
  const int64_t parts = B::blocks(total, many ? kKvPasses : 1);
  BPD_REQUIRE(n * parts < (int64_t(1) << 31), "too many tokens in one call");
  const auto launch = [&](auto passes, auto mode) {
    if (a.num_axes > 0)
      kv_append_kernel<DT, D, passes(), mode(), true><<<uint32_t(n * parts), kKvThreads, 0, s>>>(a, uint32_t(parts));
    else
      kv_append_kernel<DT, D, passes(), mode(), false><<<uint32_t(n * parts), kKvThreads, 0, s>>>(a, uint32_t(parts));
  };
  const std::integral_constant<int, 1> one;
  const std::integral_constant<int, kKvPasses> more;
  const std::integral_constant<int, kHalves> halves;
  const std::integral_constant<int, kNeighbours> neighbours;
  if (any) launch(one, std::integral_constant<int, kAnywhere>());
  else if (a.interleaved && many) launch(more, neighbours);
  else if (a.interleaved) launch(one, neighbours);
  else if (many) launch(more, halves);
  else launch(one, halves);
  BPD_LAUNCHED();
  return BPD_OK;
}

template <int DT, int D>
int launch_read(const ReadArgs& a, hipStream_t s) {
  using B = KvBlock<D>;
  const int64_t n = a.rows * a.tokens, parts = B::blocks(2 * int64_t(a.kv_heads), 1);
  BPD_REQUIRE(n * parts < (int64_t(1) << 31), "too many tokens in one call");
  if (n * parts >= kKvFill)
    kv_read_kernel<DT, D, kKvPasses>
        <<<uint32_t((n + kKvPasses - 1) / kKvPasses * parts), kKvThreads, 0, s>>>(a, uint32_t(parts));
  else
    kv_read_kernel<DT, D, 1><<<uint32_t(n * parts), kKvThreads, 0, s>>>(a, uint32_t(parts));
  BPD_LAUNCHED();
  return BPD_OK;
}

// f(type code, head size) of a call.
template <class F>
int with_kv(int dtype, int32_t dim, F f) {
  const auto with_dim = [&](auto dt) -> int {
    switch (dim) {
      case 64: return f(dt, std::integral_constant<int, 64>());
      case 96: return f(dt, std::integral_constant<int, 96>());
      case 128: return f(dt, std::integral_constant<int, 128>());
      case 192: return f(dt, std::integral_constant<int, 192>());
      default: return f(dt, std::integral_constant<int, 256>());
    }
  };
  return dtype == BPD_DTYPE_BF16 ? with_dim(std::integral_constant<int, BPD_DTYPE_BF16>())
                                 : with_dim(std::integral_constant<int, BPD_DTYPE_F16>());
}

}  // namespace
}  // namespace bpd

using namespace bpd;

#define BPD_APPEND_ARGS                                                                                            \
  AppendArgs a {                                                                                                   \
    pages, KvPage{page_size, head_dim}, KvTable{block_table, table_ld, table_blocks, num_pages}, kv_heads, heads,  \
        static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), static_cast<const uint16_t*>(q),         \
        {k_row, k_token, k_head}, {v_row, v_token, v_head}, {q_row, q_token, q_head},                              \
        static_cast<uint16_t*>(q_out), rows, tokens, starts, counts, cos, sin, positions, rotary, interleaved, err, \
        nullptr, 0, 0, 0, 0, nullptr                                                                               \
  }
#define BPD_APPEND_AXES                                                                                           \
  a.places = places, a.place_axis = place_axis, a.place_row = place_row, a.place_token = place_token,             \
  a.num_axes = num_axes, a.axes = axes;                                                                           \
  BPD_REQUIRE(num_axes >= 1, "positions of 1 to %d axes (got %d)", BPD_MAX_AXES, num_axes)

extern "C" int bpd_kv_append(uint8_t* pages, int64_t num_pages, int32_t page_size, int32_t kv_heads, int32_t head_dim,
                             int dtype, const void* k, int64_t k_row, int64_t k_token, int64_t k_head, const void* v,
                             int64_t v_row, int64_t v_token, int64_t v_head, const void* q, int64_t q_row,
                             int64_t q_token, int64_t q_head, int32_t heads, void* q_out, int64_t rows,
                             int32_t tokens, const int32_t* block_table, int64_t table_ld, int32_t table_blocks,
                             const int32_t* starts, const int32_t* counts, const float* cos, const float* sin,
                             int64_t positions, int32_t rotary, int interleaved, int32_t* err, void* stream) {
  BPD_APPEND_ARGS;
  if (int rc = check_append(a, dtype)) return rc;
  if (rows == 0 || tokens == 0) return BPD_OK;
  return with_kv(dtype, head_dim, [&](auto dt, auto dim) { return launch_append<dt(), dim()>(a, as_stream(stream)); });
}

extern "C" int bpd_host_kv_append(uint8_t* pages, int64_t num_pages, int32_t page_size, int32_t kv_heads,
                                  int32_t head_dim, int dtype, const void* k, int64_t k_row, int64_t k_token,
                                  int64_t k_head, const void* v, int64_t v_row, int64_t v_token, int64_t v_head,
                                  const void* q, int64_t q_row, int64_t q_token, int64_t q_head, int32_t heads,
                                  void* q_out, int64_t rows, int32_t tokens, const int32_t* block_table,
                                  int64_t table_ld, int32_t table_blocks, const int32_t* starts,
                                  const int32_t* counts, const float* cos, const float* sin, int64_t positions,
                                  int32_t rotary, int interleaved, int32_t* err) {
  BPD_APPEND_ARGS;
  if (int rc = check_append(a, dtype)) return rc;
  if (rows == 0 || tokens == 0) return BPD_OK;
  if (dtype == BPD_DTYPE_BF16)
    host_append<BPD_DTYPE_BF16>(a);
  else
    host_append<BPD_DTYPE_F16>(a);
  return BPD_OK;
}

extern "C" int bpd_kv_append_axes(uint8_t* pages, int64_t num_pages, int32_t page_size, int32_t kv_heads,
                                  int32_t head_dim, int dtype, const void* k, int64_t k_row, int64_t k_token,
                                  int64_t k_head, const void* v, int64_t v_row, int64_t v_token, int64_t v_head,
                                  const void* q, int64_t q_row, int64_t q_token, int64_t q_head, int32_t heads,
                                  void* q_out, int64_t rows, int32_t tokens, const int32_t* block_table,
                                  int64_t table_ld, int32_t table_blocks, const int32_t* starts, const int32_t* counts,
                                  const float* cos, const float* sin, int64_t positions, int32_t rotary,
                                  int interleaved, const int32_t* places, int64_t place_axis, int64_t place_row,
                                  int64_t place_token, int32_t num_axes, const int32_t* axes, int32_t* err,
                                  void* stream) {
  BPD_APPEND_ARGS;
  BPD_APPEND_AXES;
  if (int rc = check_append(a, dtype)) return rc;
  if (rows == 0 || tokens == 0) return BPD_OK;
  return with_kv(dtype, head_dim, [&](auto dt, auto dim) { return launch_append<dt(), dim()>(a, as_stream(stream)); });
}

extern "C" int bpd_host_kv_append_axes(uint8_t* pages, int64_t num_pages, int32_t page_size, int32_t kv_heads,
                                       int32_t head_dim, int dtype, const void* k, int64_t k_row, int64_t k_token,
                                       int64_t k_head, const void* v, int64_t v_row, int64_t v_token, int64_t v_head,
                                       const void* q, int64_t q_row, int64_t q_token, int64_t q_head, int32_t heads,
                                       void* q_out, int64_t rows, int32_t tokens, const int32_t* block_table,
                                       int64_t table_ld, int32_t table_blocks, const int32_t* starts,
                                       const int32_t* counts, const float* cos, const float* sin, int64_t positions,
                                       int32_t rotary, int interleaved, const int32_t* places, int64_t place_axis,
                                       int64_t place_row, int64_t place_token, int32_t num_axes, const int32_t* axes,
                                       int32_t* err) {
  BPD_APPEND_ARGS;
  BPD_APPEND_AXES;
  if (int rc = check_append(a, dtype)) return rc;
  if (rows == 0 || tokens == 0) return BPD_OK;
  if (dtype == BPD_DTYPE_BF16)
    host_append<BPD_DTYPE_BF16>(a);
  else
    host_append<BPD_DTYPE_F16>(a);
  return BPD_OK;
}

#define BPD_READ_ARGS                                                                                   \
  ReadArgs a {                                                                                          \
    pages, KvPage{page_size, head_dim}, KvTable{block_table, table_ld, table_blocks, num_pages}, kv_heads, \
        static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out), rows, tokens, starts, counts, err \
  }

extern "C" int bpd_kv_read(const uint8_t* pages, int64_t num_pages, int32_t page_size, int32_t kv_heads,
                           int32_t head_dim, int dtype, void* k_out, void* v_out, int64_t rows, int32_t tokens,
                           const int32_t* block_table, int64_t table_ld, int32_t table_blocks, const int32_t* starts,
                           const int32_t* counts, int32_t* err, void* stream) {
  BPD_READ_ARGS;
  if (int rc = check_read(a, dtype)) return rc;
  if (rows == 0 || tokens == 0) return BPD_OK;
  return with_kv(dtype, head_dim, [&](auto dt, auto dim) { return launch_read<dt(), dim()>(a, as_stream(stream)); });
}

extern "C" int bpd_host_kv_read(const uint8_t* pages, int64_t num_pages, int32_t page_size, int32_t kv_heads,
                                int32_t head_dim, int dtype, void* k_out, void* v_out, int64_t rows, int32_t tokens,
                                const int32_t* block_table, int64_t table_ld, int32_t table_blocks,
                                const int32_t* starts, const int32_t* counts, int32_t* err) {
  BPD_READ_ARGS;
  if (int rc = check_read(a, dtype)) return rc;
  if (rows == 0 || tokens == 0) return BPD_OK;
  if (dtype == BPD_DTYPE_BF16)
    host_read<BPD_DTYPE_BF16>(a);
  else
    host_read<BPD_DTYPE_F16>(a);
  return BPD_OK;
}
