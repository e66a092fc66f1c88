// Sums, scans and extremes over a wave of 64 lanes by data-parallel moves: a
// step within a row of 16 lanes or to the next rows takes a few cycles, where
// an exchange through LDS takes about a hundred.
#pragma once

#include "bpd_common.hpp"

namespace bpd {
namespace {

// x of the lane that Ctrl names, `none` where there is none or the row is not
// in Rows.
template <int Ctrl, int Rows>
__device__ __forceinline__ int32_t moved(int32_t x, int32_t none) {
  return __builtin_amdgcn_update_dpp(none, x, Ctrl, Rows, 0xF, false);
}
template <int Ctrl, int Rows, class T>
__device__ __forceinline__ T moved_as(T x, T none) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, moved<Ctrl, Rows>(__builtin_bit_cast(int32_t, x), __builtin_bit_cast(int32_t, none)));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, x), n = __builtin_bit_cast(uint64_t, none);
    const uint32_t lo = uint32_t(moved<Ctrl, Rows>(int32_t(uint32_t(u)), int32_t(uint32_t(n))));
    const uint32_t hi = uint32_t(moved<Ctrl, Rows>(int32_t(uint32_t(u >> 32)), int32_t(uint32_t(n >> 32))));
    return __builtin_bit_cast(T, uint64_t(hi) << 32 | lo);
  }
}

// Lane i gets op over lanes 0 .. i (all lanes active).
template <class T, class Op>
__device__ __forceinline__ T wave_scan(T x, T none, Op op) {
  x = op(moved_as<0x111, 0xF>(x, none), x);  // 1, 2, 4, 8 lanes before, within 16
  x = op(moved_as<0x112, 0xF>(x, none), x);
  x = op(moved_as<0x114, 0xF>(x, none), x);
  x = op(moved_as<0x118, 0xF>(x, none), x);
  x = op(moved_as<0x142, 0xA>(x, none), x);  // the last lane of 16 to the next 16
  x = op(moved_as<0x143, 0xC>(x, none), x);  // the last lane of 32 to the next 32
  return x;
}
template <class T>
__device__ __forceinline__ T wave_scan_sum(T x) {
  return wave_scan(x, T(0), [](T a, T b) { return a + b; });
}

// Lane `from`'s value, on every lane.
template <class T>
__device__ __forceinline__ T of_lane(T x, int from) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int32_t, x), from));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int32_t(uint32_t(u)), from));
    const uint32_t hi = uint32_t(__builtin_amdgcn_readlane(int32_t(uint32_t(u >> 32)), from));
    return __builtin_bit_cast(T, uint64_t(hi) << 32 | lo);
  }
}

template <class T>
__device__ __forceinline__ T wave_sum(T x) {
  return of_lane(wave_scan_sum(x), 63);
}
__device__ __forceinline__ float wave_max(float x) {
  return of_lane(wave_scan(x, -INFINITY, [](float a, float b) { return fmaxf(a, b); }), 63);
}
__device__ __forceinline__ int32_t wave_min(int32_t x) {
  return of_lane(wave_scan(x, int32_t(0x7FFFFFFF), [](int32_t a, int32_t b) { return a < b ? a : b; }), 63);
}

}  // namespace
}  // namespace bpd
