// Sampling with temperature, top-k, top-p and min-p from given uniform
// numbers, truncation of logits by the same cuts, and their host forms.
//
// With z the logits that the row's grammar state allows (those of -inf left
// out), top the largest and w = exp((z - top) / temperature), tokens stand in
// the order of falling z, equal ones in that of their index.  top-k keeps the
// first k, top-p of these the first whose sum of w is top_p of theirs at
// least, min-p those with z - top >= temperature * log(min_p): each is a first
// part of the order, and so is what all of them keep.  The token drawn is the
// first of the order whose running sum passes u times the whole sum of what
// is kept; truncation writes -inf over everything else.  At temperature 0
// (or where it is not positive and finite) the first token alone is kept.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>
#include <vector>

#include "runs.hpp"
#include "wave.hpp"

namespace bpd {
namespace {

struct SampleArgs {
  const void* logits;
  int dtype;
  int64_t rows, vocab, ld;
  const float* temperature;  // per row, or temperature_all; the same below
  float temperature_all;
  const int32_t* top_k;
  int32_t top_k_all;
  const float* top_p;
  float top_p_all;
  const float* min_p;
  float min_p_all;
  const uint32_t* allow_bits;
  int64_t words;
  int32_t num_states;
  int32_t* states;
  const int64_t* slots;
  // a draw
  const float* uniforms;
  const int32_t* tok_next;
  int write_back;
  int32_t* token;
  float* logprob;
  int32_t* next_state;
  // a truncation
  void* out;
  int64_t cols, out_ld;
  int32_t* err;
};

// What a row asks for.
struct Asked {
  double temp;   // 0: the first largest
  int64_t top_k; // 0: all
  float top_p;   // 1: all
  double min_p;  // 0: all
};
__host__ __device__ __forceinline__ Asked asked_of(const SampleArgs& a, int64_t b) {
  const float t = a.temperature ? a.temperature[b] : a.temperature_all;
  const int32_t k = a.top_k ? a.top_k[b] : a.top_k_all;
  const float p = a.top_p ? a.top_p[b] : a.top_p_all, m = a.min_p ? a.min_p[b] : a.min_p_all;
  return Asked{t > 0.0f && t < INFINITY ? double(t) : 0.0, k > 0 ? k : 0, p < 1.0f ? (p > 0.0f ? p : 0.0f) : 1.0f,
               m > 0.0f ? (m < 1.0f ? double(m) : 1.0) : 0.0};
}

__host__ __device__ __forceinline__ int32_t state_of(const SampleArgs& a, int64_t b) {
  return a.allow_bits ? a.states[a.slots ? a.slots[b] : b] : 0;
}

__host__ __device__ __forceinline__ void store_drawn(const SampleArgs& a, int64_t b, int32_t state, int64_t token,
                                                     float logprob) {
  a.token[b] = int32_t(token);
  a.logprob[b] = logprob;
  if (!a.tok_next) return;
  const int32_t s = token < 0 ? -1 : a.tok_next[int64_t(state) * a.vocab + token];
  if (a.next_state) a.next_state[b] = s;
  if (a.write_back) a.states[a.slots ? a.slots[b] : b] = s;
}

// ------------------------------------------------------------- the device --
// One block per row.  Sums of weights are whole numbers of 64 bits: a weight
// is its nearest multiple of 2^-scale of the largest, so that no sum depends
// on its order, equal logits weigh the same, and a border that lies between
// two sums is decided as the sums themselves are.  Off by half of that per
// token, a row of 2^17 tokens is off by 2^-37 of its largest weight or so,
// where a row's 10^5 borders want 10^-12 of its sum.
typedef unsigned long long u64;

// A row of normal logits and 150,000 tokens has 470 in its fullest bin at a
// standard deviation of one temperature, 240 at two: few enough to be put in
// order at once, each counted against all others.  Rows that are flatter, or hold
// many equal logits, take the bin apart by key, 2,048 parts and a pass at a
// time.  (8,192 bins take longer to clear and to sum, 74.6 us for 70.5 below.)
constexpr int kBins = 4096, kSubBins = 2048;  // of the first table, and of a part of one bin of it
constexpr int kListed = 512;                  // tokens of a bin that are put in order
constexpr int kMostScale = 50;  // a weight is read off the bits of its sum with 2^52

// Bits of a weight: the sum of a row's fits 63.
__host__ __device__ __forceinline__ int scale_of(int64_t vocab) {
  const int bits = vocab > 1 ? 64 - __builtin_clzll(uint64_t(vocab) - 1) : 0;
  return 62 - bits < kMostScale ? 62 - bits : kMostScale;
}

struct Row {
  const char* logits;
  const uint8_t* bits;  // of its state, null: every token
  int64_t vocab;        // 0: its state allows nothing
};

// Which tokens of a run are the thread's own and allowed.
__device__ __forceinline__ uint32_t run_bits(const Row& r, const Run& run) {
  if (!r.bits || run.own == 0) return run.own;
  return uint32_t(r.bits[(run.t + run.shift) / 8]) << run.shift & run.own;
}

// A logit as a number that orders as it does (-0 as 0), and back.
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t u = __builtin_bit_cast(uint32_t, z + 0.0f);
  return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// What the logits of a row are measured by.
struct Measure {
  double top, to_log2;  // y = (z - top) * to_log2, w = 2^y
  double bins;          // bins of the first table to an octave
  int scale;
  __device__ __forceinline__ double y(float z) const { return (double(z) - top) * to_log2; }
  __device__ __forceinline__ u64 weight(double y) const {
    const double w = __builtin_fma(exp2_down(y), __builtin_ldexp(1.0, scale), 0x1p52);
    return __builtin_bit_cast(u64, w) & ((u64(1) << 52) - 1);
  }
  __device__ __forceinline__ int32_t bin(double y) const { return int32_t(fmin(-y * bins, double(kBins - 1))); }
};

// A first part of the order: all tokens with larger keys, and the first `rank`
// of those with this one, the last of them at `last` (-1: not yet known).
struct Cut {
  uint32_t key;
  u64 rank, sum;  // sum: of its weights
  int64_t last;
};

template <int Bins>
struct Table {
  u64 sums[Bins];
  uint32_t counts[Bins];
};
struct Listed {
  u64 place;  // larger for one that stands before: its key and its index, the other way round
  u64 weight;
};
template <int N>  // threads
struct Scratch {
  static constexpr int waves = N / kWave;
  Table<kBins> first;  // by weight
  union {
    Table<kSubBins> sub;  // by key
    Listed list[kListed];
  };
  uint32_t listed;
  Cut hit;
  u64 sums[waves], counts[waves];
  u64 hit_count, hit_sum;
  int64_t found;
  float tops[waves];
  int32_t bad[waves], hit_bin;
};

template <int N, int Bins>
__device__ __forceinline__ void clear(Table<Bins>& t) {
  for (int i = threadIdx.x; i < Bins; i += N) t.sums[i] = 0, t.counts[i] = 0;
}

// A thread's neighbouring bins: what lies before them, and with them.
struct Span {
  u64 count, count_end, sum, sum_end;
};
// *count and *sum become those of the whole table.
template <int N, int Bins>
__device__ __forceinline__ Span span_of(const Table<Bins>& t, u64* count, u64* sum, Scratch<N>& s) {
  constexpr int kMine = Bins / N, kWaves = N / kWave;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  u64 c = 0, x = 0;
#pragma unroll
  for (int k = 0; k < kMine; ++k) c += t.counts[tid * kMine + k], x += t.sums[tid * kMine + k];
  Span p{0, wave_scan_sum(c), 0, wave_scan_sum(x)};
  if (lane == kWave - 1) s.counts[wave] = p.count_end, s.sums[wave] = p.sum_end;
  __syncthreads();
  *count = *sum = 0;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    if (k == wave) p.count_end += *count, p.sum_end += *sum;
    *count += s.counts[k], *sum += s.sums[k];
  }
  p.count = p.count_end - c, p.sum = p.sum_end - x;
  __syncthreads();
  return p;
}
// The bin in which the running count or sum passes `target` (less than the
// whole); *count and *sum become what lies before it.
template <int N, int Bins>
__device__ __forceinline__ int32_t find_bin(const Table<Bins>& t, const Span& p, u64 target, bool by_count, u64* count,
                                            u64* sum, Scratch<N>& s) {
  constexpr int kMine = Bins / N;
  const int tid = threadIdx.x;
  if (tid == 0) s.hit_bin = Bins - 1, s.hit_count = s.hit_sum = 0;
  __syncthreads();
  if (by_count ? p.count <= target && target < p.count_end : p.sum <= target && target < p.sum_end) {
    u64 c = p.count, x = p.sum;
#pragma unroll 1
    for (int k = tid * kMine;; ++k) {
      const u64 nc = c + t.counts[k], nx = x + t.sums[k];
      if (k == tid * kMine + kMine - 1 || target < (by_count ? nc : nx)) {
        s.hit_bin = k, s.hit_count = c, s.hit_sum = x;
        break;
      }
      c = nc, x = nx;
    }
  }
  __syncthreads();
  *count = s.hit_count, *sum = s.hit_sum;
  const int32_t bin = s.hit_bin;
  __syncthreads();
  return bin;
}

// f(z, valid, t) for the runs of tokens [begin, end) that threads take from
// `first` on, `step` tokens apart: t is the token of z[0], `valid` says which
// are the thread's own and allowed.
template <int DT, int kAtOnce, class F>  // runs on their way together
__device__ __forceinline__ void each_run(const Row& r, int64_t first, int64_t end, int64_t step, F f) {
#pragma unroll 1
  for (int64_t t0 = first; t0 < end; t0 += kAtOnce * step) {
    Raw<DT> raw[kAtOnce];
    uint32_t valid[kAtOnce];
    int64_t at[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const Run run = run_at(t0 + k * step, r.vocab);  // (past the row: none of its own)
      const bool in = t0 + k * step < end;
      raw[k] = load_raw<DT>(r.logits, run, r.vocab);
      valid[k] = in ? run_bits(r, run) : 0u;
      at[k] = run.t;
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      float z[kRun];
      unpack<DT>(raw[k], z);
      f(z, valid[k], at[k]);
    }
  }
}

// The token of rank `rank` (from 1) among those with this key, by index.
template <int DT, int N>
__device__ __forceinline__ int64_t nth_token(const Row& r, uint32_t key, u64 rank, Scratch<N>& s) {
  constexpr int kWaves = N / kWave, kStep = N * kRun;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  // a wave takes neighbouring tokens
  const int64_t part = (r.vocab + kStep - 1) / kStep * (kWave * kRun);
  const int64_t begin = part * wave, end = begin + part < r.vocab ? begin + part : r.vocab;
  const auto same = [&](const float(&z)[kRun], uint32_t valid) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kRun; ++j) m |= uint32_t(key_of(z[j]) == key) << j;
    return m & valid;
  };
  u64 n = 0;
  each_run<DT, 4>(r, begin + lane * kRun, end, kWave * kRun,
               [&](const float(&z)[kRun], uint32_t valid, int64_t) { n += __popc(same(z, valid)); });
  n = wave_sum(n);
  if (lane == 0) s.counts[wave] = n;
  if (threadIdx.x == 0) s.found = -1;
  __syncthreads();
  u64 before = 0;
  int hit = 0;
  for (; hit < kWaves - 1 && before + s.counts[hit] < rank; ++hit) before += s.counts[hit];
  if (wave == hit) {
    for (int64_t t0 = begin; t0 < end; t0 += kWave * kRun) {
      const Run run = run_at(t0 + lane * kRun, r.vocab);
      const int64_t at = run.t;
      float z[kRun];
      load_run<DT>(r.logits, run, r.vocab, z);
      uint32_t m = t0 + lane * kRun < end ? same(z, run_bits(r, run)) : 0u;
      const u64 upto = before + wave_scan_sum(u64(__popc(m)));
      if (upto >= rank && upto - __popc(m) < rank) {
        for (u64 k = upto - __popc(m) + 1; k < rank; ++k) m &= m - 1;
        s.found = at + __builtin_ctz(m);
      }
      before = of_lane(upto, kWave - 1);
      if (before >= rank) break;
    }
  }
  __syncthreads();
  const int64_t found = s.found;
  __syncthreads();
  return found;
}

// floor(x * f) for f in [0, 1), exactly; `ceil_less_one`: ceil(x * f) - 1, no
// less than 0.
__device__ __forceinline__ u64 share_of(u64 x, float f, bool ceil_less_one) {
  if (!(f > 0.0f)) return 0;
  int e;
  const u64 m = u64(frexpf(f, &e) * 0x1p24f);  // f = m 2^(e - 24)
  const int down = 24 - e;                      // at least 24
  u64 lo = x * m, hi = __umul64hi(x, m);
  if (lo == 0 && hi == 0) return 0;
  if (ceil_less_one) hi -= lo == 0, lo -= 1;
  if (down >= 128) return 0;
  if (down >= 64) return hi >> (down - 64);
  return hi << (64 - down) | lo >> down;
}

template <int DT, int N>
__device__ __forceinline__ void sample_row(const SampleArgs& a, const Row& r, const Asked& want, int64_t b, bool draw, Scratch<N>& s,
                           Cut* cut_out, int64_t* last_out, float* logprob, bool* bad_out) {
  constexpr int kWaves = N / kWave, kStep = N * kRun;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  float top = -INFINITY;
  bool bad = false;
  each_run<DT, 4>(r, tid * kRun, r.vocab, kStep, [&](const float(&z)[kRun], uint32_t valid, int64_t) {
    if (__all(valid == 0xFFu)) {
#pragma unroll
      for (int j = 0; j < kRun; ++j) bad |= !(z[j] < INFINITY), top = fmaxf(top, z[j]);
    } else {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        const float x = valid >> j & 1 ? z[j] : -INFINITY;
        bad |= !(x < INFINITY), top = fmaxf(top, x);
      }
    }
  });
  const float own = top;  // the thread's
  top = wave_max(top);
  bad = __any(bad);
  if (lane == 0) s.tops[wave] = top, s.bad[wave] = bad;
  __syncthreads();
  bad = false;
  for (int k = 0; k < kWaves; ++k) top = fmaxf(top, s.tops[k]), bad |= s.bad[k] != 0;
  *bad_out = bad;
  *last_out = -1;
  *logprob = -INFINITY;
  if (bad || top == -INFINITY) return;
  const uint32_t top_key = key_of(top);
  Cut cut{top_key, 1, 1, -1};
  Measure m{double(top), want.temp > 0.0 ? kLog2E / want.temp : 0.0, 0.0, scale_of(r.vocab)};
  m.bins = double(kBins) / (m.scale + 2);
  const bool whole = want.temp > 0.0 && want.top_k == 0 && want.top_p >= 1.0f && want.min_p <= 0.0;
  if (!draw && whole) {
    cut.key = cut.rank = 0;
  } else if (want.temp > 0.0) {
    // keys that bin i can hold, generously
    const auto keys_of = [&](int32_t i, uint32_t* lo, uint32_t* hi) {
      const double per = m.bins * m.to_log2;
      const double from = m.top - i / per, to = m.top - (i + 1) / per;
      const double off = fabs(m.top) * 0x1p-50 + (m.top - to) * 0x1p-50;
      *hi = top_key, *lo = key_of(-3.402823466e38f);
      if (from + off < m.top) *hi = min(*hi, key_of(float(from + off)) + 2);
      if (i < kBins - 1 && to - off > -3.4e38) *lo = max(*lo, key_of(float(to - off)) - 2);
    };
    // the least key that min-p keeps
    uint32_t likely = 0;
    if (want.min_p > 0.0) {
      const double least = want.temp * log(want.min_p);
      uint32_t out = 0;
      likely = top_key;
      while (likely - out > 1) {
        const uint32_t mid = out + (likely - out) / 2;
        if (mid > 0x007FFFFFu && double(logit_of(mid)) - m.top >= least) likely = mid;
        else out = mid;
      }
    }
    // What lies below `from` is not needed: min-p's border, where top-p does not
    // want the sum of more, and the bin that holds the k-th of the threads'
    // largest logits, which is not before that of the k-th of all.
    uint32_t from = want.top_p < 1.0f ? 0 : likely;
    clear<N>(s.first);
    __syncthreads();
    if (want.top_k > 0 && want.top_k <= N) {
      if (own > -INFINITY) atomicAdd(&s.first.counts[m.bin(m.y(own))], 1u);
      __syncthreads();
      u64 c, x;
      const Span span = span_of(s.first, &c, &x, s);
      const int32_t i = find_bin(s.first, span, u64(want.top_k) - 1, true, &c, &x, s);
      if (c < u64(want.top_k) && c + s.first.counts[i] >= u64(want.top_k)) {
        uint32_t lo, hi;
        keys_of(i, &lo, &hi);
        from = max(from, lo);
      }
      __syncthreads();
      clear<N>(s.first);
      __syncthreads();
    }
    const float floor_z = from > 0x007FFFFFu ? logit_of(from) : -3.402823466e38f;  // (-inf lies below)
    const bool counts = want.top_k > 0;
    each_run<DT, 2>(r, tid * kRun, r.vocab, kStep, [&](const float(&z)[kRun], uint32_t valid, int64_t) {
      const auto add = [&](float x) {
        const double y = m.y(x);
        const int32_t i = m.bin(y);
        if (counts) atomicAdd(&s.first.counts[i], 1u);
        atomicAdd(&s.first.sums[i], m.weight(y));
      };
#pragma unroll
      for (int j = 0; j < kRun; ++j)
        if (z[j] < floor_z) valid &= ~(1u << j);
      if (__all(valid == 0xFFu)) {  // (no branches: the exponentials of eight tokens interleave)
#pragma unroll
        for (int j = 0; j < kRun; ++j) add(z[j]);
      } else if (__any(valid != 0)) {
#pragma unroll
        for (int j = 0; j < kRun; ++j)
          if (valid >> j & 1) add(z[j]);
      }
    });
    __syncthreads();
    u64 count, sum;
    const Span span = span_of(s.first, &count, &sum, s);
    // (all that min-p keeps, or all of the row)
    cut = want.top_p < 1.0f || likely == 0 ? Cut{0, 0, sum, -1} : Cut{likely - 1, 0, sum, -1};
    // the first part of the order that ends where the running count or sum passes `target`
    const auto select = [&](u64 target, bool by_count) {
      u64 c, x;
      const int32_t bin = find_bin(s.first, span, target, by_count, &c, &x, s);
      uint32_t lo, hi;
      keys_of(bin, &lo, &hi);
      lo = max(lo, from);
      // the bin's tokens, put in order where they are few
      const float least = logit_of(lo), most = logit_of(hi);
      const float middle = 0.5f * least + 0.5f * most, half = (0.5f * most - 0.5f * least) * (1.0f + 0x1p-20f) + fabsf(middle) * 0x1p-20f + 1e-38f;
      if (tid == 0) s.listed = 0;
      __syncthreads();
      each_run<DT, 4>(r, tid * kRun, r.vocab, kStep, [&](const float(&z)[kRun], uint32_t valid, int64_t t) {
        uint32_t near = 0;
#pragma unroll
        for (int j = 0; j < kRun; ++j) near |= fabsf(z[j] - middle) <= half ? 1u << j : 0u;
        near &= valid;
        while (__any(near != 0)) {  // few: read again one by one
          if (near == 0) continue;
          const int64_t i = t + __builtin_ctz(near);
          near &= near - 1;
          const float x = load_elem(r.logits, DT, i);
          const double y = m.y(x);
          if (!(x >= least && x <= most) || m.bin(y) != bin) continue;
          const uint32_t at = atomicAdd(&s.listed, 1u);
          if (at < kListed) s.list[at] = Listed{u64(key_of(x)) << 32 | uint32_t(~uint32_t(i)), m.weight(y)};
        }
      });
      __syncthreads();
      const uint32_t listed = s.listed;
      if (listed <= uint32_t(kListed)) {
        if (tid == 0) s.hit = Cut{hi, 1, x + 1, -1};
        __syncthreads();
        for (uint32_t i = tid; i < listed; i += N) {
          const Listed mine = s.list[i];
          u64 bc = c, bx = x, rank = 1;
#pragma unroll 4
          for (uint32_t e = 0; e < listed; ++e) {
            const Listed other = s.list[e];
            const bool before = other.place > mine.place;
            bc += before, bx += before ? other.weight : 0;
            rank += before && (other.place ^ mine.place) >> 32 == 0;
          }
          if (by_count ? bc == target : bx <= target && target < bx + mine.weight)
            s.hit = Cut{uint32_t(mine.place >> 32), rank, bx + mine.weight, int64_t(uint32_t(~uint32_t(mine.place)))};
        }
        __syncthreads();
        const Cut found = s.hit;
        __syncthreads();
        return found;
      }
      for (;;) {
        const uint32_t range = hi - lo;
        const int shift = range < uint32_t(kSubBins) ? 0 : 32 - __builtin_clz(range) - __builtin_ctz(uint32_t(kSubBins));
        __syncthreads();
        clear<N>(s.sub);
        __syncthreads();
        each_run<DT, 4>(r, tid * kRun, r.vocab, kStep, [&](const float(&z)[kRun], uint32_t valid, int64_t) {
#pragma unroll
          for (int j = 0; j < kRun; ++j) {
            const uint32_t key = key_of(z[j]);
            if (!(valid >> j & 1) || key < lo || key > hi) continue;
            const double y = m.y(z[j]);
            if (m.bin(y) != bin) continue;
            atomicAdd(&s.sub.counts[(hi - key) >> shift], 1u);
            atomicAdd(&s.sub.sums[(hi - key) >> shift], m.weight(y));
          }
        });
        __syncthreads();
        u64 dc, dx;
        const Span part = span_of(s.sub, &dc, &dx, s);
        const uint32_t i = uint32_t(find_bin(s.sub, part, target - (by_count ? c : x), by_count, &dc, &dx, s));
        c += dc, x += dx;
        hi -= i << shift;
        if (shift == 0 || hi <= lo) break;
        lo = max(lo, hi - ((1u << shift) - 1));
      }
      const u64 w = m.weight(m.y(logit_of(hi)));
      const u64 rank = by_count ? target - c + 1 : (target - x) / w + 1;
      return Cut{hi, rank, x + rank * w, -1};
    };
    if (want.top_k > 0 && u64(want.top_k) <= count) cut = select(u64(want.top_k) - 1, true);
    if (want.top_p < 1.0f) cut = select(share_of(cut.sum, want.top_p, true), false);
    if (likely > cut.key && !(cut.rank == 0 && cut.key == likely - 1)) {
      // (behind top-p: its sum is not known yet)
      u64 x = 0;
      each_run<DT, 4>(r, tid * kRun, r.vocab, kStep, [&](const float(&z)[kRun], uint32_t valid, int64_t) {
#pragma unroll
        for (int j = 0; j < kRun; ++j)
          if ((valid >> j & 1) && key_of(z[j]) >= likely) x += m.weight(m.y(z[j]));
      });
      x = wave_sum(x);
      if (lane == 0) s.sums[wave] = x;
      __syncthreads();
      cut = Cut{likely - 1, 0, 0, -1};
      for (int k = 0; k < kWaves; ++k) cut.sum += s.sums[k];
      __syncthreads();
    }
    if (draw) {
      const float u = a.uniforms[b];
      u64 target = u < 1.0f ? share_of(cut.sum, u, false) : cut.sum;
      if (target >= cut.sum) target = cut.sum - 1;
      const u64 kept = cut.sum;
      cut = select(target, false);
      *logprob = float((double(logit_of(cut.key)) - m.top) / want.temp - log(double(kept) * __builtin_ldexp(1.0, -m.scale)));
    }
  } else {
    *logprob = 0.0f;
  }
  *cut_out = cut;
  if (cut.rank > 0) *last_out = cut.last >= 0 ? cut.last : nth_token<DT, N>(r, cut.key, cut.rank, s);
}

__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t b, int32_t* state, int32_t* flags) {
  *state = state_of(a, b);
  *flags = a.allow_bits && *state >= a.num_states ? BPD_FLAG_STATE_RANGE : 0;
  const bool some = !a.allow_bits || (*state >= 0 && *state < a.num_states);
  return Row{static_cast<const char*>(a.logits) + b * a.ld * (a.dtype == BPD_DTYPE_F32 ? 4 : 2),
             a.allow_bits && some ? reinterpret_cast<const uint8_t*>(a.allow_bits + int64_t(*state) * a.words) : nullptr,
             some ? a.vocab : 0};
}

// All of a row's work, by a block of N threads.
template <int DT, bool Draw, int N>
__device__ __forceinline__ void general_row(const SampleArgs& a, const Row& r, const Asked& want, int64_t b, int32_t state, int32_t flags,
                            Scratch<N>& s) {
  Cut cut{0xFFFFFFFFu, 0, 0, -1};
  int64_t last = -1;
  float logprob = -INFINITY;
  bool bad = false;
  sample_row<DT, N>(a, r, want, b, Draw, s, &cut, &last, &logprob, &bad);
  if (bad) flags |= BPD_FLAG_LOGITS;
  if (flags && a.err && threadIdx.x == 0) atomicOr(a.err, flags);
  if constexpr (Draw) {
    if (threadIdx.x == 0) store_drawn(a, b, state, last, logprob);
    return;
  }
  constexpr int kBytes = DT == BPD_DTYPE_F32 ? 4 : 2;
  const uint32_t none = DT == BPD_DTYPE_F32 ? 0xFF800000u : DT == BPD_DTYPE_BF16 ? 0xFF80u : 0xFC00u;
  char* out = static_cast<char*>(a.out) + b * a.out_ld * kBytes;
  const auto put = [&](int64_t t, uint32_t x) {
    if (kBytes == 4) reinterpret_cast<uint32_t*>(out)[t] = x;
    else reinterpret_cast<uint16_t*>(out)[t] = uint16_t(x);
  };
  for (int64_t t = threadIdx.x * kRun; t < a.vocab; t += N * kRun) {
    const Run run = run_at(t, a.vocab);
    uint32_t keep = r.vocab ? run_bits(r, run) : 0;
    const Raw<DT> raw = load_raw<DT>(r.logits, run, a.vocab);
    float z[kRun];
    unpack<DT>(raw, z);
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      const uint32_t key = key_of(z[j]);
      const bool in = key > cut.key || (key == cut.key && run.t + j <= last);
      const uint32_t x = kBytes == 4 ? raw.w[kBytes == 4 ? j / 4 : 0][j % 4] : raw.w[0][j / 2] >> (16 * (j & 1)) & 0xFFFFu;
      if (run.own >> j & 1) put(run.t + j, in && (keep >> j & 1) ? x : none);
    }
  }
  for (int64_t t = a.vocab + threadIdx.x; t < a.cols; t += N) put(t, none);
}

// Rows of 32-bit logits (97 of 100,003 under all three cuts: 70.5 us, with 512
// threads 2 us more).  What bounds it: 64-bit instructions, 26 us of it in the
// pass that sums weights (an exponential and an addition to 64 bits in LDS for
// each token that the cuts can reach), on the CUs that have a row; a maximum
// takes 6 us, tables' sums 3, each cut's or the draw's pass over the row 8, from
// the cache.  Of the five steps the maximum and the sums, 32 us, would need one
// join each if a row were dealt over the CUs that have none, the cuts one each;
// rows are not dealt.
constexpr int kThreads = 1024;
template <int DT, bool Draw>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ Scratch<kThreads> s;
  const int64_t b = blockIdx.x;
  int32_t state, flags;
  const Row r = row_of(a, b, &state, &flags);
  general_row<DT, Draw, kThreads>(a, r, asked_of(a, b), b, state, flags, s);
}

// ---------------------------------------------- rows of 16-bit logits --
// A 16-bit type has few values, and a weight follows from the value: a row is
// counted by value, once, and all sums are those of counts times weights.  The
// counts lie in LDS, a word to a magnitude: tokens of both signs in its lower
// half, the negative ones in its upper.  The row stays in registers, where its
// equal tokens are told apart by index and the kept ones written.  Values stand
// at positions in falling order.
//
// What bounds it: 256 rows of 151,936 in bfloat16, one to a CU, take 36 us where
// reading them takes 13.5.  16 us are the counting (five vector instructions a
// token, and an addition in LDS that takes 7.3 cycles for 64 tokens at random
// words), 6 the sums of counts and of the weights that the cuts need, 2.6 the cuts
// themselves, which one wave finds, 5 the search for the token among its equals.
// Truncation writes the row from its registers (160 rows under a grammar: 49
// us, a copy takes 20).  A grammar's row costs what one without does: it is loaded
// and counted whole, however few tokens the state allows.
//
// Rows past the registers take as long for a token (256 of 262,144: 66 us, 0.25 ns
// for each token of a row, as with 151,936; 48 of 200,064: 38 us).
// One finite value that most of a row holds is the slowest input: lanes that add
// to one word take 128 cycles, and past 65,535 tokens the row starts over in the
// form for 32 bits.  48 rows of 151,936 with 99 of 100 logits at the type's lowest
// number, as a mask with a finite fill leaves them: 300 us under top-p, 204 with
// top-k of 50 (50,000 tokens: 55), with -inf in their place 28, unmasked 30; 32-bit
// rows 161, 57, 63 and 95.
constexpr int kMagnitudes = 32768;
// Half the threads that a CU holds, with twice the registers: 40 runs are the
// row of a vocabulary of 163,840, longer ones are read once more.  (1,024
// threads and 24 runs: 256 draws 51.6 us for 37.4, 160 truncations 48.5 for 50.6.)
constexpr int kThreads16 = 512, kWaves16 = kThreads16 / kWave, kStep16 = kThreads16 * kRun, kHeld = 40;
constexpr int kWaveRun = kWave * kRun;  // tokens of a wave's run
constexpr int kAhead = 8;  // runs on their way while one is counted (4 or 16: 0 to 3 us more)
constexpr int kChunk = 4 * kWave;       // words of counts that a wave takes at a time
constexpr int kChunks = 2 * kMagnitudes / kChunk;

template <int DT>
struct Half {
  static constexpr uint32_t inf = DT == BPD_DTYPE_BF16 ? 0x7F80u : 0x7C00u, none = inf | 0x8000u;
};
template <int DT>
__device__ __forceinline__ float value_of(uint32_t magnitude) {
  if (DT == BPD_DTYPE_BF16) return __builtin_bit_cast(float, magnitude << 16);
  return float(__builtin_bit_cast(_Float16, uint16_t(magnitude)));
}
template <int DT>
__device__ __forceinline__ float value_at(int32_t position) {
  return position < kMagnitudes ? value_of<DT>(uint32_t(kMagnitudes - 1 - position))
                                : -value_of<DT>(uint32_t(position - kMagnitudes));
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pair_max(uint32_t x, uint32_t y) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, x), __builtin_bit_cast(u16x2, y)));
}
__device__ __forceinline__ uint32_t pair_signed_max(uint32_t x, uint32_t y) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(i16x2, x), __builtin_bit_cast(i16x2, y)));
}
__device__ __forceinline__ uint32_t pair_min(uint32_t x, uint32_t y) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, x), __builtin_bit_cast(u16x2, y)));
}

// f(k) for k = 0 .. N - 1 as constants: arrays that it indexes stay in registers.
template <class F, int... K>
__device__ __forceinline__ void each_of(std::integer_sequence<int, K...>, F f) {
  (f(std::integral_constant<int, K>()), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F f) {
  each_of(std::make_integer_sequence<int, N>(), f);
}

struct Counted {
  uint32_t words[kMagnitudes];
  uint32_t left_out[kWave];  // what a lane does not count goes to its own word
  u64 sums[kChunks];  // by chunks of positions
  uint32_t counts[kChunks];
  uint32_t added[kWaves16], found[kWaves16];
  int32_t tops[kWaves16], bad[kWaves16];
  // what the first wave comes to
  int32_t position;
  uint32_t rank;  // 0: all of the position
  float logprob;
  int64_t last;
};

// A first part of the order, as Cut, by position.
struct Place16 {
  int32_t position;
  uint32_t rank;
  u64 sum;
};

// A lane's four positions of chunk `c`: counts, and weights of one each.
template <int DT>
__device__ __forceinline__ void chunk_positions(const Counted& s, const Measure& m, int c, int lane, uint32_t (&n)[4],
                                                u64 (&w)[4]) {
  const int32_t at = c * kChunk + 4 * lane;
  const bool below = c >= kChunks / 2;
  const uint4 q = *reinterpret_cast<const uint4*>(s.words + (below ? at - kMagnitudes : kMagnitudes - 4 - at));
  const uint32_t x[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    n[k] = below ? x[k] >> 16 : (x[3 - k] & 0xFFFFu) - (x[3 - k] >> 16);
    w[k] = m.weight(m.y(value_at<DT>(at + k)));
  }
}

// The first wave's view of the chunks: each lane has four of them.
template <int DT>
struct Chunks {
  const Counted& s;
  const Measure& m;
  int lane;
  u64 sum_before, sum_mine;
  uint32_t count_before, count_mine;
  __device__ __forceinline__ Chunks(const Counted& s_, const Measure& m_, int lane_) : s(s_), m(m_), lane(lane_) {
    sum_mine = 0, count_mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) sum_mine += s.sums[4 * lane + k], count_mine += s.counts[4 * lane + k];
    sum_before = wave_scan_sum(sum_mine) - sum_mine;
    count_before = wave_scan_sum(count_mine) - count_mine;
  }
  __device__ __forceinline__ u64 sum() const { return of_lane(sum_before + sum_mine, kWave - 1); }
  __device__ __forceinline__ uint32_t count() const { return of_lane(count_before + count_mine, kWave - 1); }
  // what stands before chunk `c`
  __device__ __forceinline__ void before(int c, uint32_t* count, u64* sum) const {
    *count = of_lane(count_before, c / 4), *sum = of_lane(sum_before, c / 4);
    for (int k = c / 4 * 4; k < c; ++k) *count += s.counts[k], *sum += s.sums[k];
  }
  // where the running count (of tokens) or sum (of weights) passes `target`
  template <bool ByCount>
  __device__ __forceinline__ Place16 find(u64 target) const {
    const u64 from = ByCount ? count_before : sum_before, own = ByCount ? count_mine : sum_mine;
    const int l = __builtin_ctzll(__ballot(from <= target && target < from + own) | u64(1) << 63);
    const uint4 four = *reinterpret_cast<const uint4*>(s.counts + 4 * l);
    const ulonglong2 two[2] = {reinterpret_cast<const ulonglong2*>(s.sums + 4 * l)[0],
                               reinterpret_cast<const ulonglong2*>(s.sums + 4 * l)[1]};
    const uint32_t fc[3] = {four.x, four.y, four.z};
    const u64 fs[3] = {two[0].x, two[0].y, two[1].x};
    int c = 4 * l;
    uint32_t cb = of_lane(count_before, l);
    u64 sb = of_lane(sum_before, l);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const uint32_t nc = cb + fc[k];
      const u64 ns = sb + fs[k];
      if (c != 4 * l + k || target < (ByCount ? nc : ns)) continue;
      cb = nc, sb = ns, ++c;
    }
    uint32_t n[4];
    u64 w[4];
    chunk_positions<DT>(s, m, c, lane, n, w);
    uint32_t nc = 0;
    u64 ns = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) nc += n[k], ns += n[k] * w[k];
    const uint32_t upto_c = cb + wave_scan_sum(nc);
    const u64 upto_s = sb + wave_scan_sum(ns);
    const u64 hits = __ballot(target < (ByCount ? upto_c : upto_s));
    const int hit = hits ? __builtin_ctzll(hits) : kWave - 1;
    cb = of_lane(upto_c - nc, hit), sb = of_lane(upto_s - ns, hit);
    Place16 p{c * kChunk + 4 * hit, 1, 0};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t kn = of_lane(n[k], hit);
      const u64 kw = of_lane(w[k], hit), end_s = sb + kn * kw;
      if (kn && target < (ByCount ? u64(cb + kn) : end_s)) {
        p.position += k;
        if (ByCount) {
          p.rank = uint32_t(target) - cb + 1;
        } else {  // the quotient, by its nearest float of 64 bits
          p.rank = uint32_t(double(target - sb) / double(kw));
          p.rank += (p.rank + u64(1)) * kw <= target - sb ? 1u : p.rank * kw > target - sb ? -1u : 0u;
          ++p.rank;
        }
        p.sum = sb + p.rank * kw;
        // zeros of both signs are equal: those of the first position count too
        if (p.position == kMagnitudes) p.rank += (s.words[0] & 0xFFFFu) - (s.words[0] >> 16);
        return p;
      }
      cb += kn, sb = end_s;
    }
    return p;
  }
  // the sum of all positions up to this one
  __device__ __forceinline__ u64 sum_upto(int32_t position) const {
    const int c = position / kChunk;
    uint32_t cb, n[4];
    u64 sb, w[4], x = 0;
    before(c, &cb, &sb);
    chunk_positions<DT>(s, m, c, lane, n, w);
#pragma unroll
    for (int k = 0; k < 4; ++k) x += c * kChunk + 4 * lane + k <= position ? n[k] * w[k] : 0;
    return sb + wave_sum(x);
  }
};

// One block per row.
template <int DT, bool Draw, bool Grammar>
__global__ __launch_bounds__(kThreads16) void sample16_kernel(SampleArgs a) {
  __shared__ union {
    Counted s;
    Scratch<kThreads16> general;
  } shared;
  Counted& s = shared.s;
  constexpr uint32_t kNone = Half<DT>::none;
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int64_t b = blockIdx.x, V = a.vocab;
  const char* row = static_cast<const char*>(a.logits) + b * a.ld * 2;
  // A wave takes neighbouring tokens: runs that lie whole in the row, the first
  // of them held, and maybe one that does not.
  const int32_t runs = int32_t((V + kStep16 - 1) / kStep16);
  const int64_t begin = int64_t(wave) * runs * kWaveRun, left = V - begin;
  const int32_t full = left <= 0 ? 0 : left < int64_t(runs) * kWaveRun ? int32_t(left / kWaveRun) : runs;
  const bool tail = left > int64_t(full) * kWaveRun && full < runs;
  const int32_t held = full < kHeld ? full : kHeld;
  // (formed anew at each use: the registers hold the row instead)
  const auto token_of = [&](int32_t k) {
    int32_t l = lane;
    asm volatile("" : "+v"(l));
    return begin + int64_t(k) * kWaveRun + l * kRun;
  };
  const char* mine = row + (begin + lane * kRun) * 2;
  const auto load = [&](int32_t k) {
    Raw<DT> x;
    __builtin_memcpy(&x, __builtin_assume_aligned(mine + int64_t(k) * (kWaveRun * 2), 2), sizeof(x));
    return x;
  };
  Raw<DT> raw[kHeld];
  each<kAhead>([&](auto k) {
    if (k < held) raw[k] = load(k);
  });
  int32_t state, flags;
  const Row r = row_of(a, b, &state, &flags);
  const uint8_t* allow = Grammar && r.bits ? r.bits + (begin + lane * kRun) / 8 : nullptr;
  const auto load_bits = [&](int32_t k) -> uint32_t { return allow ? allow[k * (kWaveRun / 8)] : 0u; };
  uint32_t bits[kAhead];
  if constexpr (Grammar)
    each<kAhead>([&](auto k) {
      if (k < held) bits[k] = load_bits(k);
    });
  const Asked want = asked_of(a, b);
  Measure m{0.0, want.temp > 0.0 ? kLog2E / want.temp : 0.0, 0.0, scale_of(V)};
  for (int i = tid; i < kMagnitudes / 4; i += kThreads16) reinterpret_cast<uint4*>(s.words)[i] = uint4{0, 0, 0, 0};
  if (tid < kChunks) s.counts[tid] = 0, s.sums[tid] = 0;
  __syncthreads();

  // -inf for tokens whose bit is not set
  const auto mask = [&](Raw<DT>& x, uint32_t valid) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = uint32_t(int32_t(valid << (31 - 2 * i)) >> 31), hi = uint32_t(int32_t(valid << (30 - 2 * i)) >> 31);
      const uint32_t keep = (lo & 0xFFFFu) | (hi & 0xFFFF0000u);
      x.w[0][i] = (x.w[0][i] & keep) | ((kNone << 16 | kNone) & ~keep);
    }
  };
  // Counts a run, and follows the largest of the values that are not negative.
  // Five instructions a token, and two for its run's part: what bounds this,
  // beside the LDS, which takes 7.3 cycles for 64 additions at random words.
  uint32_t most = 0xFFFFFFFFu, not_counted = 0;
  char* words = reinterpret_cast<char*>(s.words);
  const auto count = [&](const Raw<DT>& x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = x.w[0][i];
      most = pair_signed_max(most, w);
      atomicAdd(reinterpret_cast<uint32_t*>(words + (w << 2 & 0x1FFFCu)), (w << 1 & 0x10000u) | 1u);
      atomicAdd(reinterpret_cast<uint32_t*>(words + (w >> 14 & 0x1FFFCu)), (w >> 15 & 0x10000u) | 1u);
    }
  };
  // the same, but for tokens of -inf
  const uint32_t apart = uint32_t(reinterpret_cast<char*>(s.left_out + lane) - words);
  const auto count_some = [&](const Raw<DT>& x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = x.w[0][i];
      most = pair_signed_max(most, w);
      const bool lo = (w & 0xFFFFu) == kNone, hi = w >> 16 == kNone;
      atomicAdd(reinterpret_cast<uint32_t*>(words + (lo ? apart : w << 2 & 0x1FFFCu)), (w << 1 & 0x10000u) | 1u);
      atomicAdd(reinterpret_cast<uint32_t*>(words + (hi ? apart : w >> 14 & 0x1FFFCu)), (w >> 15 & 0x10000u) | 1u);
      not_counted += uint32_t(lo) + uint32_t(hi);
    }
  };
  const auto is_none = [&](const Raw<DT>& x) {  // some of the run is -inf (or a negative NaN)
    const uint32_t u = pair_max(pair_max(x.w[0][0], x.w[0][1]), pair_max(x.w[0][2], x.w[0][3]));
    return u >= kNone << 16 || (u & 0xFFFFu) >= kNone;
  };
  const auto take = [&](Raw<DT>& x, uint32_t valid) {
    if constexpr (Grammar) {
      mask(x, valid);
      if (__any(valid != 0)) count_some(x);
      else not_counted += kRun;
    } else {
      if (__builtin_expect(__any(is_none(x)), 0)) count_some(x);
      else count(x);
    }
  };
  each<kHeld>([&](auto k) {
    if (k >= held) return;
    uint32_t valid = 0;
    if constexpr (Grammar) valid = bits[k % kAhead];
    if constexpr (k + kAhead < kHeld) {
      if (k + kAhead < held) {
        raw[k + kAhead] = load(k + kAhead);
        if constexpr (Grammar) bits[k % kAhead] = load_bits(k + kAhead);
      }
    }
    take(raw[k], valid);
  });
  const auto again = [&](int32_t k) {  // a run past those held
    Raw<DT> x = load(k);
    if constexpr (Grammar) mask(x, load_bits(k));
    return x;
  };
#pragma unroll 1
  for (int32_t k = held; k < full; ++k) count_some(again(k));
  Raw<DT> end{};  // the run that is not whole
  if (tail) {
    const Run run = run_at(token_of(full), V);
    end = load_raw<DT>(row, run, V);
    mask(end, r.vocab ? run_bits(r, run) : 0u);
    count_some(end);
  }
  int32_t top_bits = max(int32_t(most) >> 16, int32_t(most << 16) >> 16);
  top_bits = -wave_min(-top_bits);
  const uint32_t added = wave_sum(uint32_t(full + tail) * kRun - not_counted);
  if (lane == 0) s.added[wave] = added, s.tops[wave] = top_bits;
  __syncthreads();
  uint32_t all = 0, counted = 0;
  for (int k = 0; k < kWaves16; ++k) all += s.added[k], top_bits = max(top_bits, s.tops[k]);
  float top = value_of<DT>(uint32_t(top_bits));
  if (top_bits < 0) {  // no value but negative ones (and -0): the smallest magnitude
    int32_t least = kMagnitudes - 1;
#pragma unroll 1
    for (int i = tid; i < kMagnitudes; i += kThreads16)
      if (s.words[i] != 0) {
        least = i;
        break;
      }
    least = wave_min(least);
    __syncthreads();
    if (lane == 0) s.tops[wave] = least;
    __syncthreads();
    for (int k = 0; k < kWaves16; ++k) least = min(least, s.tops[k]);
    top = 0.0f - value_of<DT>(uint32_t(least));
  }

  // counts of the chunks; whether all are numbers, and whether all were counted: a
  // count past 16 bits leaves fewer
  m.top = double(top);
  bool bad = false;
  constexpr int kMine = kChunks / 2 / kWaves16;  // of a wave, every kWaves16-th
  uint32_t some = 0;
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const uint4 q = reinterpret_cast<const uint4*>(s.words)[(i * kWaves16 + wave) * kWave + lane];
    some |= uint32_t(__any((q.x | q.y | q.z | q.w) != 0)) << i;
  }
  while (some) {
    const int32_t c = __builtin_ctz(some) * kWaves16 + wave, at = c * kChunk + 4 * lane;
    some &= some - 1;
    const uint4 q = reinterpret_cast<const uint4*>(s.words)[c * kWave + lane];
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    uint32_t n[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t below = w[k] >> 16, above = (w[k] & 0xFFFFu) - below;
      counted += w[k] & 0xFFFFu;
      n[0] += above, n[1] += below;
      bad |= at + k >= int32_t(Half<DT>::inf) && (at + k == int32_t(Half<DT>::inf) ? above : w[k]) != 0;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) n[e] = wave_scan_sum(n[e]);
    if (lane == kWave - 1) s.counts[kChunks / 2 - 1 - c] = n[0], s.counts[kChunks / 2 + c] = n[1];
  }
  counted = wave_sum(counted);
  bad = __any(bad);
  if (lane == 0) s.found[wave] = counted, s.bad[wave] = bad;
  __syncthreads();
  counted = 0;
  for (int k = 0; k < kWaves16; ++k) counted += s.found[k], bad |= s.bad[k] != 0;
  if (__builtin_expect(counted != all, 0)) {
    __syncthreads();
    general_row<DT, Draw, kThreads16>(a, r, want, b, state, flags, shared.general);
    return;
  }
  const bool none = bad || all == 0;
  if (bad) flags |= BPD_FLAG_LOGITS;
  int64_t last = -1;
  float border = INFINITY, logprob = -INFINITY;  // what lies above it is kept, and of what equals it all up to `last`
  if (!none) {
    const uint32_t magnitude = DT == BPD_DTYPE_BF16 ? __builtin_bit_cast(uint32_t, fabsf(top)) >> 16
                                                    : __builtin_bit_cast(uint16_t, _Float16(fabsf(top)));
    const int32_t first = top < 0.0f ? kMagnitudes + int32_t(magnitude) : kMagnitudes - 1 - int32_t(magnitude);
    const bool whole = want.temp > 0.0 && want.top_k == 0 && want.top_p >= 1.0f && want.min_p <= 0.0;
    if (want.temp > 0.0 && (Draw || !whole)) {
      // the last position that min-p keeps
      int32_t likely = kChunks * kChunk - 1;
      if (want.min_p > 0.0) {
        const double least = want.temp * log(want.min_p);
        int32_t out = kMagnitudes + int32_t(Half<DT>::inf);
        likely = first;
        while (out - likely > 1) {
          const int32_t mid = (likely + out) / 2;
          if (double(value_at<DT>(mid)) - m.top >= least) likely = mid;
          else out = mid;
        }
      }
      // Sums of the chunks, dealt to the waves in turn: of those that hold the
      // first top_k tokens, or what min-p keeps (top-p is a share of more than that).
      const uint4 four = *reinterpret_cast<const uint4*>(s.counts + 4 * lane);
      const uint32_t here[4] = {four.x, four.y, four.z, four.w};
      int32_t last_chunk = want.top_p < 1.0f ? kChunks - 1 : likely / kChunk;
      if (want.top_k > 0) {
        const uint32_t own = (here[0] + here[1]) + (here[2] + here[3]), upto = wave_scan_sum(own);
        const uint64_t past = __ballot(int64_t(upto) >= want.top_k);
        if (past) last_chunk = min(last_chunk, 4 * __builtin_ctzll(past) + 3);
      }
      uint32_t turn = 0;
#pragma unroll 1
      for (int k = 0; k < 4; ++k) {
        uint64_t chunks = __ballot((k == 0 ? here[0] : k == 1 ? here[1] : k == 2 ? here[2] : here[3]) != 0);
        while (chunks) {
          const int32_t o = 4 * __builtin_ctzll(chunks) + k;
          chunks &= chunks - 1;
          if (o > last_chunk) break;
          if (turn++ % kWaves16 != uint32_t(wave)) continue;
          uint32_t n[4];
          u64 w[4];
          chunk_positions<DT>(s, m, o, lane, n, w);
          const u64 sum = wave_scan_sum((n[0] * w[0] + n[1] * w[1]) + (n[2] * w[2] + n[3] * w[3]));
          if (lane == kWave - 1) s.sums[o] = sum;
        }
      }
      __syncthreads();
      if (wave == 0) {
        const Chunks<DT> chunks(s, m, lane);
        Place16 cut{kChunks * kChunk - 1, 0, chunks.sum()};
        if (want.top_k > 0 && want.top_k < int64_t(chunks.count())) cut = chunks.template find<true>(u64(want.top_k) - 1);
        if (want.top_p < 1.0f) cut = chunks.template find<false>(share_of(cut.sum, want.top_p, true));
        if (likely < cut.position) cut = Place16{likely, 0, chunks.sum_upto(likely)};
        if (Draw) {
          const float u = a.uniforms[b];
          u64 target = u < 1.0f ? share_of(cut.sum, u, false) : cut.sum;
          if (target >= cut.sum) target = cut.sum - 1;
          const u64 kept = cut.sum;
          cut = chunks.template find<false>(target);
          if (lane == 0)
            s.logprob = float((double(value_at<DT>(cut.position)) - m.top) / want.temp - log(double(kept) * __builtin_ldexp(1.0, -m.scale)));
        }
        if (lane == 0) s.position = cut.position, s.rank = cut.rank;
      }
    } else if (tid == 0) {
      s.position = whole ? kChunks * kChunk - 1 : first, s.rank = whole ? 0 : 1, s.logprob = 0.0f;
    }
    __syncthreads();
    const uint32_t rank = s.rank;
    border = s.position == kChunks * kChunk - 1 ? -INFINITY : value_at<DT>(s.position);
    logprob = s.logprob;
    last = INT64_MAX;
    if (rank > 0) {
      // The token of that rank among those that equal the border: halves that
      // differ from it are counted two at a time.
      const uint32_t h = uint32_t(s.position < kMagnitudes ? kMagnitudes - 1 - s.position : s.position - kMagnitudes) |
                         (s.position < kMagnitudes ? 0u : 0x8000u);
      const bool zero = (h & 0x7FFFu) == 0;
      const uint32_t both = zero ? 0u : h << 16 | h, sign = zero ? 0x7FFF7FFFu : 0xFFFFFFFFu;
      const auto other = [&](uint32_t w) {  // 1 in halves that differ
        return pair_min((w & sign) ^ both, 0x00010001u);
      };
      const auto others = [&](const Raw<DT>& x) { return (other(x.w[0][0]) + other(x.w[0][1])) + (other(x.w[0][2]) + other(x.w[0][3])); };
      const auto none_of = [&](const Raw<DT>& x) {  // no token equals the border
        const uint32_t least = pair_min(pair_min((x.w[0][0] & sign) ^ both, (x.w[0][1] & sign) ^ both),
                                        pair_min((x.w[0][2] & sign) ^ both, (x.w[0][3] & sign) ^ both));
        return pair_min(least, 0x00010001u) == 0x00010001u;
      };
      uint32_t same = 0;
      uint64_t equal = 0;  // held runs in which some token does
      const auto add_some = [&](const Raw<DT>& x) {
        const uint32_t d = others(x);
        same += kRun - (d & 0xFFFFu) - (d >> 16);
      };
      each<kHeld>([&](auto k) {
        if (k >= held || !__any(!none_of(raw[k]))) return;
        equal |= uint64_t(1) << k;
        add_some(raw[k]);
      });
#pragma unroll 1
      for (int32_t k = held; k < full; ++k) add_some(again(k));
      if (tail) add_some(end);
      same = wave_sum(same);
      if (lane == 0) s.found[wave] = same;
      if (tid == 0) s.last = -1;
      __syncthreads();
      uint32_t before = 0;
#pragma unroll
      for (int k = 0; k < kWaves16; ++k) before += k < wave ? s.found[k] : 0;
      if (before < rank && rank <= before + same) {
        const auto look = [&](const Raw<DT>& x, int32_t k) {
          if (before >= rank) return;
          uint32_t e = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t d = other(x.w[0][i]);
            e |= (~d & 1u) << (2 * i) | (~(d >> 16) & 1u) << (2 * i + 1);
          }
          const uint32_t own = __popc(e), upto = before + wave_scan_sum(own);
          if (upto - own < rank && rank <= upto) {
            for (uint32_t i = upto - own + 1; i < rank; ++i) e &= e - 1;
            s.last = run_at(token_of(k), V).t + __builtin_ctz(e);
          }
          before = of_lane(upto, kWave - 1);
        };
        each<kHeld / 8>([&](auto k8) {
          if ((equal >> (8 * k8) & 0xFF) == 0) return;
          each<8>([&](auto k) {
            if (__builtin_expect(equal >> (8 * k8 + k) & 1, 0)) look(raw[8 * k8 + k], 8 * k8 + k);
          });
        });
#pragma unroll 1
        for (int32_t k = held; k < full && before < rank; ++k) look(again(k), k);
        if (tail) look(end, full);
      }
      __syncthreads();
      last = s.last;
    }
  }
  if (flags && a.err && tid == 0) atomicOr(a.err, flags);
  if constexpr (Draw) {
    if (tid == 0) store_drawn(a, b, state, last, logprob);
    return;
  }
  uint16_t* out = static_cast<uint16_t*>(a.out) + b * a.out_ld;
  const auto cut = [&](Raw<DT>& x, int64_t t) {
    float z[kRun];
    unpack<DT>(x, z);
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      const bool in = z[j] > border || (z[j] == border && t + j <= last);
      if (!in) x.w[0][j / 2] = j & 1 ? (x.w[0][j / 2] & 0xFFFFu) | kNone << 16 : (x.w[0][j / 2] & 0xFFFF0000u) | kNone;
    }
  };
  const auto put = [&](Raw<DT> x, int32_t k) {
    const int64_t t = token_of(k);
    cut(x, t);
    __builtin_memcpy(__builtin_assume_aligned(out + t, 2), &x, sizeof(x));
  };
  each<kHeld>([&](auto k) {
    if (k < held) put(raw[k], k);
  });
#pragma unroll 1
  for (int32_t k = held; k < full; ++k) put(again(k), k);
  if (tail) {
    const Run run = run_at(token_of(full), V);
    cut(end, run.t);
#pragma unroll
    for (int j = 0; j < kRun; ++j)
      if (run.own >> j & 1) out[run.t + j] = uint16_t(end.w[0][j / 2] >> (16 * (j & 1)));
  }
  for (int64_t t = V + tid; t < a.cols; t += kThreads16) out[t] = uint16_t(kNone);
}

template <int DT, bool Draw>
int launch_sample_rows(const SampleArgs& a, hipStream_t s) {
  if constexpr (DT == BPD_DTYPE_F32) {
    sample_kernel<DT, Draw><<<uint32_t(a.rows), kThreads, 0, s>>>(a);
  } else {
    if (a.allow_bits)
      sample16_kernel<DT, Draw, true><<<uint32_t(a.rows), kThreads16, 0, s>>>(a);
    else
      sample16_kernel<DT, Draw, false><<<uint32_t(a.rows), kThreads16, 0, s>>>(a);
  }
  BPD_LAUNCHED();
  return BPD_OK;
}
template <bool Draw>
int launch_sample(const SampleArgs& a, hipStream_t s) {
  if (a.dtype == BPD_DTYPE_BF16) return launch_sample_rows<BPD_DTYPE_BF16, Draw>(a, s);
  if (a.dtype == BPD_DTYPE_F16) return launch_sample_rows<BPD_DTYPE_F16, Draw>(a, s);
  return launch_sample_rows<BPD_DTYPE_F32, Draw>(a, s);
}

// --------------------------------------------------------------- the host --
void host_sample(const SampleArgs& a, bool draw) {
  int32_t flags = 0;
  std::vector<int32_t> order;
  std::vector<double> w;
  for (int64_t b = 0; b < a.rows; ++b) {
    const Asked want = asked_of(a, b);
    const int32_t state = state_of(a, b);
    if (a.allow_bits && state >= a.num_states) flags |= BPD_FLAG_STATE_RANGE;
    const bool some = !a.allow_bits || (state >= 0 && state < a.num_states);
    const uint32_t* bits = a.allow_bits && some ? a.allow_bits + int64_t(state) * a.words : nullptr;
    const auto z = [&](int64_t t) { return load_elem(a.logits, a.dtype, b * a.ld + t); };
    bool bad = false;
    order.clear();
    for (int64_t t = 0; t < (some ? a.vocab : 0); ++t) {
      if (!allowed(bits, t) || z(t) == -INFINITY) continue;
      bad |= !(z(t) < INFINITY);
      order.push_back(int32_t(t));
    }
    if (bad) flags |= BPD_FLAG_LOGITS, order.clear();
    int64_t n = int64_t(order.size());
    double whole = 1.0;
    if (n > 0) {
      std::sort(order.begin(), order.end(), [&](int32_t x, int32_t y) { return z(x) > z(y) || (z(x) == z(y) && x < y); });
      const double top = z(order[0]);
      if (!(want.temp > 0.0)) n = 1;
      else if (want.top_k > 0) n = std::min(n, want.top_k);
      w.resize(size_t(n));
      whole = 0.0;
      for (int64_t i = 0; i < n; ++i) whole += w[i] = want.temp > 0.0 ? std::exp((z(order[i]) - top) / want.temp) : 1.0;
      if (want.top_p < 1.0f) {
        const double most = double(want.top_p) * whole;
        double upto = 0.0;
        int64_t i = 0;
        while (i < n && (i == 0 || upto < most)) upto += w[i++];
        n = i, whole = upto;
      }
      if (want.min_p > 0.0 && want.temp > 0.0) {
        const double least = want.temp * std::log(want.min_p);
        int64_t i = n;
        while (z(order[i - 1]) - top < least) --i;
        if (i < n) {
          n = i, whole = 0.0;
          for (int64_t k = 0; k < n; ++k) whole += w[k];
        }
      }
    }
    if (draw) {
      int64_t at = -1;
      if (n > 0) {
        const float u = a.uniforms[b];
        const double target = u > 0.0f ? double(u) * whole : 0.0;
        double upto = 0.0;
        for (int64_t i = 0; i < n; ++i) {
          if (!(w[i] > 0.0)) break;
          upto += w[i], at = i;
          if (upto > target) break;
        }
      }
      store_drawn(a, b, state, at < 0 ? -1 : order[at],
                  at < 0 ? -INFINITY
                         : float((want.temp > 0.0 ? (z(order[at]) - double(z(order[0]))) / want.temp : 0.0) - std::log(whole)));
      continue;
    }
    std::vector<char> keep(size_t(a.vocab), 0);
    for (int64_t i = 0; i < n; ++i) keep[order[i]] = 1;
    for (int64_t t = 0; t < a.cols; ++t) {
      const bool in = t < a.vocab && keep[t];
      if (a.dtype == BPD_DTYPE_F32) {
        float* out = static_cast<float*>(a.out) + b * a.out_ld + t;
        *out = in ? static_cast<const float*>(a.logits)[b * a.ld + t] : -INFINITY;
      } else {
        uint16_t* out = static_cast<uint16_t*>(a.out) + b * a.out_ld + t;
        *out = in ? static_cast<const uint16_t*>(a.logits)[b * a.ld + t] : a.dtype == BPD_DTYPE_BF16 ? 0xFF80 : 0xFC00;
      }
    }
  }
  if (flags && a.err) *a.err |= flags;
}

int check_sample(const SampleArgs& a, bool draw) {
  BPD_REQUIRE(elem_bytes(a.dtype) != 0, "unknown logits dtype code %d", a.dtype);
  BPD_REQUIRE(a.rows >= 0 && a.rows < (int64_t(1) << 21), "at most 2^21 - 1 rows in one call");
  BPD_REQUIRE(a.vocab >= 1 && a.vocab < (int64_t(1) << 31), "a vocabulary of 1 to 2^31 - 1 tokens (got %lld)",
              (long long)a.vocab);
  if (a.rows == 0) return BPD_OK;
  BPD_REQUIRE(a.logits, "null pointer argument");
  BPD_REQUIRE(a.temperature || (std::isfinite(a.temperature_all) && a.temperature_all >= 0.0f),
              "the temperature must be finite and not negative");
  BPD_REQUIRE(a.top_k || a.top_k_all >= 0, "top_k must not be negative");
  BPD_REQUIRE(a.top_p || (a.top_p_all >= 0.0f && a.top_p_all <= 1.0f), "top_p must lie between 0 and 1");
  BPD_REQUIRE(a.min_p || (a.min_p_all >= 0.0f && a.min_p_all <= 1.0f), "min_p must lie between 0 and 1");
  BPD_REQUIRE(!a.allow_bits || (a.states && a.num_states >= 0 && a.words >= (a.vocab + 31) / 32),
              "allow bits need states, and a row of ceil(vocab / 32) words");
  if (draw) {
    BPD_REQUIRE(a.uniforms && a.token && a.logprob, "null pointer argument");
    BPD_REQUIRE(!a.tok_next || a.allow_bits, "a grammar needs its allow bits");
    BPD_REQUIRE(!(a.write_back || a.next_state) || a.tok_next, "states are advanced through tok_next only");
  } else {
    BPD_REQUIRE(a.out && a.cols >= a.vocab && (a.rows == 1 || a.out_ld >= a.cols), "the output's rows overlap or are too short");
  }
  return BPD_OK;
}

}  // namespace
}  // namespace bpd

using namespace bpd;

#define BPD_SAMPLE_ARGS                                                                                               \
  SampleArgs a {}; /* by name: two calls share it */                                                                  \
  a.logits = logits, a.dtype = dtype, a.rows = rows, a.vocab = vocab, a.ld = ld, a.temperature = temperature,         \
  a.temperature_all = temperature_all, a.top_k = top_k, a.top_k_all = top_k_all, a.top_p = top_p,                     \
  a.top_p_all = top_p_all, a.min_p = min_p, a.min_p_all = min_p_all, a.allow_bits = allow_bits, a.words = words,      \
  a.num_states = num_states, a.slots = slots, a.err = err
#define BPD_DRAW_ARGS                                                                                                 \
  BPD_SAMPLE_ARGS, a.states = states, a.uniforms = uniforms, a.tok_next = tok_next, a.write_back = write_back,        \
                   a.token = token, a.logprob = logprob, a.next_state = next_state
#define BPD_TRUNCATE_ARGS \
  BPD_SAMPLE_ARGS, a.states = const_cast<int32_t*>(states), a.out = out, a.cols = cols, a.out_ld = out_ld

extern "C" int bpd_sample(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, const float* uniforms,
                          const float* temperature, float temperature_all, const int32_t* top_k, int32_t top_k_all,
                          const float* top_p, float top_p_all, const float* min_p, float min_p_all,
                          const uint32_t* allow_bits, int64_t words, int32_t num_states, const int32_t* tok_next,
                          int32_t* states, const int64_t* slots, int write_back, int32_t* token, float* logprob,
                          int32_t* next_state, int32_t* err, void* stream) {
  BPD_DRAW_ARGS;
  if (int rc = check_sample(a, true)) return rc;
  return rows == 0 ? BPD_OK : launch_sample<true>(a, as_stream(stream));
}

extern "C" int bpd_host_sample(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld,
                               const float* uniforms, const float* temperature, float temperature_all,
                               const int32_t* top_k, int32_t top_k_all, const float* top_p, float top_p_all,
                               const float* min_p, float min_p_all, const uint32_t* allow_bits, int64_t words,
                               int32_t num_states, const int32_t* tok_next, int32_t* states, const int64_t* slots,
                               int write_back, int32_t* token, float* logprob, int32_t* next_state, int32_t* err) {
  BPD_DRAW_ARGS;
  if (int rc = check_sample(a, true)) return rc;
  if (rows > 0) host_sample(a, true);
  return BPD_OK;
}

extern "C" int bpd_truncate(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, void* out,
                            int64_t cols, int64_t out_ld, const float* temperature, float temperature_all,
                            const int32_t* top_k, int32_t top_k_all, const float* top_p, float top_p_all,
                            const float* min_p, float min_p_all, const uint32_t* allow_bits, int64_t words,
                            int32_t num_states, const int32_t* states, const int64_t* slots, int32_t* err,
                            void* stream) {
  BPD_TRUNCATE_ARGS;
  if (int rc = check_sample(a, false)) return rc;
  return rows == 0 ? BPD_OK : launch_sample<false>(a, as_stream(stream));
}

extern "C" int bpd_host_truncate(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, void* out,
                                 int64_t cols, int64_t out_ld, const float* temperature, float temperature_all,
                                 const int32_t* top_k, int32_t top_k_all, const float* top_p, float top_p_all,
                                 const float* min_p, float min_p_all, const uint32_t* allow_bits, int64_t words,
                                 int32_t num_states, const int32_t* states, const int64_t* slots, int32_t* err) {
  BPD_TRUNCATE_ARGS;
  if (int rc = check_sample(a, false)) return rc;
  if (rows > 0) host_sample(a, false);
  return BPD_OK;
}
