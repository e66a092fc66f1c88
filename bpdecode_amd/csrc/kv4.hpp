// The paged key/value cache held in 4 bits: layout of a page, and the
// conversion between values and codes, for the device and the host.
//
// A group of 32 neighbouring channels x of one token and head is kept as e2m1
// codes of x / s (levels 0, .5, 1, 1.5, 2, 3, 4, 6 and a sign; ties to the
// even code) and one byte e, s = 2^(e - 127).  s is the smallest power of two
// with max|x| <= 7 s: between 4 and 6 neighbouring levels are 2 s apart, so
// rounding is off by at most s there, and cutting 7 s to 6 s is off by no
// more.  (But for float16's last values: past 7 * 2^13 = 57,344 the scale stays
// 2^13, so 65,504 is kept as 49,152, two s below.)  A power of two keeps every value exact in bfloat16 and float16 (two
// significant bits), so reading the cache rounds nothing, and gfx950 converts
// two codes with their scale in one instruction.
// 4 + 8 / 32 = 4.25 bits per element.
#pragma once

#include "bpd_common.hpp"

namespace bpd {
namespace {

constexpr int kKvGroup = 32;
constexpr uint8_t kKvBadScale = 255;  // the group held an infinity or a NaN

// Sections of the block of one page and head: key codes, value codes, key
// scales, value scales, token after token.  Each starts at a multiple of 16
// bytes (page_size is a multiple of 16).
struct KvPage {
  int32_t page_size, dim;
  __host__ __device__ int32_t codes() const { return dim / 2; }      // bytes of a token's codes
  __host__ __device__ int32_t groups() const { return dim / kKvGroup; }
  __host__ __device__ int32_t v_codes() const { return page_size * codes(); }
  __host__ __device__ int32_t k_scales() const { return page_size * dim; }
  __host__ __device__ int32_t v_scales() const { return k_scales() + page_size * groups(); }
  __host__ __device__ int32_t bytes() const { return k_scales() + 2 * page_size * groups(); }
};

inline bool kv_dim_ok(int32_t dim) { return dim == 64 || dim == 96 || dim == 128 || dim == 192 || dim == 256; }
inline bool kv_page_ok(int32_t p) { return p >= 16 && p <= 256 && (p & (p - 1)) == 0; }

__host__ __device__ __forceinline__ uint32_t float_bits(float f) {
  uint32_t u;
  __builtin_memcpy(&u, &f, 4);
  return u;
}
__host__ __device__ __forceinline__ float bits_float(uint32_t u) {
  float f;
  __builtin_memcpy(&f, &u, 4);
  return f;
}

// 16-bit elements of the cache's type as float, and back (nearest even).
template <int DT>
__host__ __device__ __forceinline__ float elem16_float(uint16_t b) {
  if (DT == BPD_DTYPE_BF16) return bits_float(uint32_t(b) << 16);
  _Float16 h;
  __builtin_memcpy(&h, &b, 2);
  return float(h);
}
template <int DT>
__host__ __device__ __forceinline__ uint16_t float_elem16(float f) {
  if (DT == BPD_DTYPE_BF16) {
    uint32_t u = float_bits(f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0x7FC0;
    u += 0x7FFFu + ((u >> 16) & 1u);
    return uint16_t(u >> 16);
  }
  const _Float16 h = static_cast<_Float16>(f);
  uint16_t b;
  __builtin_memcpy(&b, &h, 2);
  return b;
}

// Scale byte of a group by the bits of its largest magnitude.  The smallest
// byte keeps half a step a normal bfloat16 number (in float16 its smallest
// subnormal), the largest keeps six steps finite: float16 ends at 6 * 2^13
// (4 * 2^14 would be an infinity), bfloat16 at 6 * 2^125.
template <int DT>
__host__ __device__ __forceinline__ int32_t kv_scale_byte(uint32_t most) {
  constexpr int32_t lo = DT == BPD_DTYPE_BF16 ? 2 : 104, hi = DT == BPD_DTYPE_BF16 ? 252 : 140;
  if (most >= 0x7F800000u) return kKvBadScale;
  const int32_t e = int32_t(most >> 23) - 2 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return e < lo ? lo : e > hi ? hi : e;
}

// Code of x at scale byte e (0 in a bad group): y = |x| / s is exact, the
// thresholds are the midpoints, each belonging to the even code beside it.
__host__ __device__ __forceinline__ uint32_t kv_code(float x, int32_t e) {
  if (e == kKvBadScale) return 0;
  const float y = bits_float(float_bits(x) & 0x7FFFFFFFu) * bits_float(uint32_t(254 - e) << 23);
  const uint32_t c = uint32_t(y > 0.25f) + uint32_t(y >= 0.75f) + uint32_t(y > 1.25f) + uint32_t(y >= 1.75f) +
                     uint32_t(y > 2.5f) + uint32_t(y >= 3.5f) + uint32_t(y > 5.0f);
  return c | (x < 0.0f ? 8u : 0u);
}

// Value of a 4-bit code at scale byte e, as gfx950 converts it: 2^(e - 127) is
// a normal float for every byte that kv_scale_byte gives, byte 0 a subnormal
// one.
__host__ __device__ __forceinline__ float kv_value(uint32_t code, uint32_t e) {
  if (e == kKvBadScale) return bits_float(0x7FC00000u);
  const uint32_t c = code & 7u;
  // levels: 0, then m * 2^k with m = 1 (even codes) or 1.5 (odd ones above 1)
  const float lv = c < 2 ? 0.5f * float(c) : bits_float((126u + (c >> 1)) << 23) * ((c & 1u) ? 1.5f : 1.0f);
  return (code & 8u ? -lv : lv) * bits_float(e ? e << 23 : 0x400000u);
}

// Two codes (byte B of w) times a scale, as two elements of the type: exact.
template <int DT, int B>
__device__ __forceinline__ uint32_t two_values(uint32_t w, float s) {
  if constexpr (DT == BPD_DTYPE_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, B));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, B));
}

// Two floats as two elements, rounded to nearest even.
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

// The rotation of a pair by its position's angle, each product and each sum
// rounded by itself (no fused multiply-add), so that the codes that follow
// from it do not depend on how a compiler joins them.
__host__ __device__ __forceinline__ float rot_first(float a, float b, float c, float s) {
#pragma clang fp contract(off)
  const float x = a * c, y = b * s;
  return x - y;
}
__host__ __device__ __forceinline__ float rot_second(float a, float b, float c, float s) {
#pragma clang fp contract(off)
  const float x = b * c, y = a * s;
  return x + y;
}

// Channel d of a head of `x`, rotated: pairs (d, d + rot / 2), or neighbours.
template <int DT>
__host__ __device__ __forceinline__ float rotated_channel(const uint16_t* x, int32_t d, int32_t rot,
                                                          bool interleaved, const float* cos, const float* sin) {
  const float v = elem16_float<DT>(x[d]);
  if (d >= rot) return v;
  const int32_t h = rot / 2;
  if (interleaved) {
    const float w = elem16_float<DT>(x[d ^ 1]);
    return (d & 1) ? rot_second(w, v, cos[d >> 1], sin[d >> 1]) : rot_first(v, w, cos[d >> 1], sin[d >> 1]);
  }
  if (d < h) return rot_first(v, elem16_float<DT>(x[d + h]), cos[d], sin[d]);
  return rot_second(elem16_float<DT>(x[d - h]), v, cos[d - h], sin[d - h]);
}

// Where token `pos` of a request lies: the index of its page's block of head
// 0 and its slot, or -1 for a position outside the request's table or a page
// outside the pool.
struct KvTable {
  const int32_t* block_table;
  int64_t ld;
  int32_t blocks;
  int64_t num_pages;
  __host__ __device__ __forceinline__ int64_t page_of(int64_t row, int64_t pos, int32_t page_size) const {
    if (pos < 0 || pos >= int64_t(blocks) * page_size) return -1;
    const int32_t page = block_table[row * ld + (pos >> __builtin_ctz(uint32_t(page_size)))];
    return page >= 0 && page < num_pages ? page : -1;
  }
};

// Host-side checks of a cache and a block table's shape.
inline int check_kv_cache(const void* pages, const KvPage& p, const KvTable& t, int32_t kv_heads, int dtype) {
  BPD_REQUIRE(dtype == BPD_DTYPE_BF16 || dtype == BPD_DTYPE_F16, "the cache takes float16 or bfloat16 (dtype code %d)",
              dtype);
  BPD_REQUIRE(kv_dim_ok(p.dim), "head_dim must be 64, 96, 128, 192 or 256 (got %d)", p.dim);
  BPD_REQUIRE(kv_page_ok(p.page_size), "page_size must be a power of two from 16 to 256 (got %d)", p.page_size);
  BPD_REQUIRE(kv_heads >= 1 && t.num_pages >= 0, "the cache needs at least one head");
  BPD_REQUIRE(pages || t.num_pages == 0, "null cache pointer");
  BPD_REQUIRE((reinterpret_cast<uintptr_t>(pages) & 15u) == 0, "the pages must lie at a multiple of 16 bytes");
  BPD_REQUIRE(t.blocks >= 0 && t.ld >= t.blocks, "a block table's rows overlap (%d blocks, row stride %lld)", t.blocks,
              (long long)t.ld);
  return BPD_OK;
}

}  // namespace
}  // namespace bpd
