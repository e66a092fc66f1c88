// Rows of logits as runs of 8 neighbouring tokens, at any alignment of their
// type, and the exponential in 64 bits: what verification and sampling share.
#pragma once

#include "bpd_common.hpp"

namespace bpd {
namespace {

constexpr int kWave = 64;
constexpr int kRun = 8;  // neighbouring tokens of a thread
constexpr double kLog2E = 1.4426950408889634;

__host__ __device__ __forceinline__ float load_elem(const void* p, int dtype, int64_t i) {
  if (dtype == BPD_DTYPE_F32) return static_cast<const float*>(p)[i];
  const uint16_t b = static_cast<const uint16_t*>(p)[i];
  if (dtype == BPD_DTYPE_BF16) {
    const uint32_t u = uint32_t(b) << 16;
    float f;
    __builtin_memcpy(&f, &u, 4);
    return f;
  }
  _Float16 h;
  __builtin_memcpy(&h, &b, 2);
  return float(h);
}

__host__ __device__ __forceinline__ bool allowed(const uint32_t* bits, int64_t t) {
  return !bits || (bits[t >> 5] >> (t & 31) & 1u);
}

// exp2(y) for y <= 0; 0 from -1075 on and for -inf: 2^k times a polynomial of
// degree 8 on [-1/2, 1/2] (least largest relative error, 7.7e-13, computed by
// exchange).
__device__ __forceinline__ double exp2_down(double y) {
  // no lower than -1100, by the high word: larger for a more negative number
  uint64_t u = __builtin_bit_cast(uint64_t, y);
  u = uint64_t(min(uint32_t(u >> 32), 0xC0913000u)) << 32 | uint32_t(u);
  y = __builtin_bit_cast(double, u);
  const double t = y + 0x1.8p52;  // the low word is y's nearest whole number
  const double r = y - (t - 0x1.8p52);
  double p = 1.3175877963987601e-06;
  p = __builtin_fma(p, r, 1.530970905613007e-05);
  p = __builtin_fma(p, r, 0.00015403851427779082);
  p = __builtin_fma(p, r, 0.0013333452167635066);
  p = __builtin_fma(p, r, 0.009618128543707452);
  p = __builtin_fma(p, r, 0.05550410939233352);
  p = __builtin_fma(p, r, 0.2402265069887445);
  p = __builtin_fma(p, r, 0.6931471805465407);
  p = __builtin_fma(p, r, 0.999999999999763);
  return __builtin_amdgcn_ldexp(p, int32_t(uint32_t(__builtin_bit_cast(uint64_t, t))));
}

typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));

// kRun neighbouring elements as they lie in memory; any alignment of the type's
// own.
template <int DT>
struct Raw {
  words4 w[DT == BPD_DTYPE_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ void unpack(const Raw<DT>& x, float (&z)[kRun]) {
#pragma unroll
  for (int j = 0; j < kRun; ++j) {
    if constexpr (DT == BPD_DTYPE_F32)
      z[j] = __builtin_bit_cast(float, uint32_t(x.w[j / 4][j % 4]));
    else if constexpr (DT == BPD_DTYPE_BF16)
      z[j] = __builtin_bit_cast(float, j & 1 ? x.w[0][j / 2] & 0xFFFF0000u : x.w[0][j / 2] << 16);
    else
      z[j] = float(__builtin_bit_cast(_Float16, uint16_t(x.w[0][j / 2] >> (16 * (j & 1)))));
  }
}

// The run of a thread that begins at token `t` (a multiple of kRun).  Where it
// would pass the vocabulary it is moved back to end there, and the tokens
// before t that it then holds are not its own.  (A vocabulary of fewer than
// kRun tokens is read from its first on.)
struct Run {
  int64_t t;      // first token it reads
  uint32_t own;   // which of its tokens count, before the grammar
  int32_t shift;  // t moved back by this
};
__device__ __forceinline__ Run run_at(int64_t t, int64_t vocab) {
  if (t + kRun <= vocab) return Run{t, 0xFFu, 0};
  if (t >= vocab) return Run{vocab >= kRun ? vocab - kRun : 0, 0u, 0};
  if (vocab < kRun) return Run{0, (1u << vocab) - 1u, 0};
  const int32_t shift = int32_t(t + kRun - vocab);
  return Run{t - shift, 0xFFu << shift & 0xFFu, shift};
}
template <int DT>
__device__ __forceinline__ Raw<DT> load_raw(const void* from, const Run& run, int64_t vocab) {
  Raw<DT> x;
  if (vocab >= kRun) {
    const char* p = static_cast<const char*>(from) + run.t * (DT == BPD_DTYPE_F32 ? 4 : 2);
    __builtin_memcpy(&x, __builtin_assume_aligned(p, DT == BPD_DTYPE_F32 ? 4 : 2), sizeof(x));
    return x;
  }
#pragma unroll
  for (int j = 0; j < kRun; ++j) {
    const int64_t t = j < vocab ? j : 0;
    if constexpr (DT == BPD_DTYPE_F32)
      x.w[j / 4][j % 4] = static_cast<const uint32_t*>(from)[t];
    else
      x.w[0][j / 2] = (j & 1 ? uint32_t(x.w[0][j / 2]) : 0u) | uint32_t(static_cast<const uint16_t*>(from)[t]) << (16 * (j & 1));
  }
  return x;
}
template <int DT>
__device__ __forceinline__ void load_run(const void* from, const Run& run, int64_t vocab, float (&z)[kRun]) {
  unpack<DT>(load_raw<DT>(from, run, vocab), z);
}
template <int DT, int N>
__device__ __forceinline__ void load_runs(const void* from, const Run (&runs)[N], int64_t vocab, float (&z)[N][kRun]) {
#pragma unroll
  for (int k = 0; k < N; ++k) load_run<DT>(from, runs[k], vocab, z[k]);
}

// -inf for tokens whose bit is not set.
__device__ __forceinline__ float masked(float z, uint32_t bits, int j) {
  const uint32_t keep = uint32_t(int32_t(bits << (31 - j)) >> 31);
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, z) & keep) | (0xFF800000u & ~keep));
}

}  // namespace
}  // namespace bpd
