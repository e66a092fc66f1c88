// Verification of a block of drafted tokens against the target's logits, and
// its host form.
//
// With p_i the softmax of position i's logits at the request's temperature
// over the tokens that its grammar state allows (at temperature 0 all on the
// first largest) and q_i the probabilities that draft i was sampled from (all
// on the drafted token where the draft gives none), draft i stands while
//   u_i q_i(x_i) < p_i(x_i),
// which happens with probability min(1, p / q).  At the first position n that
// does not stand the next token is drawn from max(p_n - q_n, 0), after a
// whole block from p_n: the first token whose running sum passes u_T times
// the whole sum.  A token emitted this way is distributed as p.
#include <algorithm>
#include <cmath>

#include "runs.hpp"
#include "wave.hpp"

namespace bpd {
namespace {

constexpr int kMaxPositions = BPD_MAX_DRAFTS + 1;

struct VerifyArgs {
  const void* logits;
  int dtype;
  int64_t rows;
  int32_t drafts;
  int64_t vocab, ld_row, ld_pos;
  const void* tokens;
  int token_dtype;
  int64_t tokens_ld;
  const int32_t* draft_lens;
  const void* probs;
  int probs_dtype;
  int64_t probs_row, probs_pos;
  const float* uniforms;
  int64_t uniforms_ld;
  const float* temperature;  // per request, or temperature_all
  float temperature_all;
  const uint32_t* allow_bits;
  int64_t words;
  int32_t num_states;
  const int32_t* tok_next;
  int32_t* states;
  const int64_t* slots;
  const int32_t* bit_rows;  // [rows, drafts + 1]: row of allow_bits per position
  int write_back;
  int32_t *accepted, *next_token, *next_state;
  int32_t* err;
};

__host__ __device__ __forceinline__ int32_t draft_len(const VerifyArgs& a, int64_t b) {
  if (!a.draft_lens) return a.drafts;
  const int32_t n = a.draft_lens[b];
  return n < 0 ? 0 : n < a.drafts ? n : a.drafts;
}

// 0 (the largest logit) unless positive and finite.
__host__ __device__ __forceinline__ double temperature_of(const VerifyArgs& a, int64_t b) {
  const float t = a.temperature ? a.temperature[b] : a.temperature_all;
  return t > 0.0f && t < INFINITY ? t : 0.0;
}

// What a position's row comes to.  `empty`: the grammar allows nothing, every
// allowed logit is -inf, or one is +inf or NaN and the row has no softmax.
struct RowStat {
  double sum;   // of exp((z - top) / temperature)
  float top;
  int32_t first;  // first token with the largest logit
  int32_t empty;
  int32_t bad;    // an allowed logit is +inf or NaN
  int32_t state;  // row of allow_bits; outside of its rows: allows nothing
};

// The weight of token t: what it is drawn by, before the draft is taken off.
__host__ __device__ __forceinline__ double weight(const RowStat& st, double temp, float z, int64_t t) {
  if (!(temp > 0.0)) return t == st.first ? 1.0 : 0.0;
  return exp((double(z) - double(st.top)) / temp);
}

__host__ __device__ __forceinline__ const uint32_t* bits_of(const VerifyArgs& a, int32_t state) {
  return a.allow_bits ? a.allow_bits + int64_t(state) * a.words : nullptr;
}

__host__ __device__ __forceinline__ int64_t row_at(const VerifyArgs& a, int64_t b, int32_t i) {
  return b * a.ld_row + i * a.ld_pos;
}

__host__ __device__ __forceinline__ double prob_of(const VerifyArgs& a, int64_t b, int32_t i, int64_t t, int64_t drafted) {
  if (!a.probs) return t == drafted ? 1.0 : 0.0;
  return load_elem(a.probs, a.probs_dtype, b * a.probs_row + i * a.probs_pos + t);
}

// The state of position i of request b by that of the position before (i = 0:
// by the request's); -1 where it allows nothing.
__host__ __device__ __forceinline__ int32_t state_at(const VerifyArgs& a, int64_t b, int32_t i, int32_t before) {
  if (a.bit_rows) return a.bit_rows[b * (a.drafts + 1) + i];
  if (!a.tok_next) return 0;
  if (i == 0) return a.states[a.slots ? a.slots[b] : b];
  const int64_t x = read_token(a.tokens, a.token_dtype, b * a.tokens_ld + i - 1);
  if (x < 0 || x >= a.vocab || before < 0 || before >= a.num_states) return -1;
  return a.tok_next[int64_t(before) * a.vocab + x];
}

// What the row that decides a request's block is to flag: its state, the
// token drafted there, an allowed logit without a softmax.
__host__ __device__ __forceinline__ int32_t flags_of(const VerifyArgs& a, int64_t b, int32_t n, int32_t len, int32_t state,
                                                     bool bad) {
  int32_t f = bad ? BPD_FLAG_LOGITS : 0;
  if (a.allow_bits && state >= a.num_states) f |= BPD_FLAG_STATE_RANGE;
  if (n < len) {
    const int64_t x = read_token(a.tokens, a.token_dtype, b * a.tokens_ld + n);
    if (x < 0 || x >= a.vocab) f |= BPD_FLAG_TOKEN_RANGE;
  }
  return f;
}

// Whether draft i of request b stands.
__host__ __device__ __forceinline__ bool stands(const VerifyArgs& a, int64_t b, int32_t i, const RowStat& st) {
  const int64_t x = read_token(a.tokens, a.token_dtype, b * a.tokens_ld + i);
  if (st.empty || x < 0 || x >= a.vocab || !allowed(bits_of(a, st.state), x)) return false;
  const double p = weight(st, temperature_of(a, b), load_elem(a.logits, a.dtype, row_at(a, b, i) + x), x) / st.sum;
  return double(a.uniforms[b * a.uniforms_ld + i]) * prob_of(a, b, i, x, x) < p;
}

// What token t is drawn by at position n; `less`: the draft's share taken off.
__host__ __device__ __forceinline__ double share(const VerifyArgs& a, int64_t b, int32_t n, const RowStat& st, double temp,
                                                 const uint32_t* bits, bool less, int64_t drafted, int64_t t) {
  if (!allowed(bits, t)) return 0.0;
  const double p = weight(st, temp, load_elem(a.logits, a.dtype, row_at(a, b, n) + t), t) / st.sum;
  if (!less) return p;
  const double r = p - prob_of(a, b, n, t, drafted);
  return r > 0.0 ? r : 0.0;
}

__host__ __device__ __forceinline__ void finish(const VerifyArgs& a, int64_t b, int32_t n, const RowStat& st, int64_t token) {
  a.accepted[b] = n;
  a.next_token[b] = int32_t(token);
  if (!a.tok_next) return;
  const int32_t s = token < 0 || st.state < 0 || st.state >= a.num_states ? -1 : a.tok_next[int64_t(st.state) * a.vocab + token];
  if (a.next_state) a.next_state[b] = s;
  if (a.write_back) a.states[a.slots ? a.slots[b] : b] = s;
}

// ------------------------------------------------------------- the device --
// Every position's row is read once, for its largest logit and the sum of its
// weights in 32 bits: within kSumError of the sum, which decides all but about
// one verdict in 10^5 (those are summed anew in 64 bits).  The draw needs the
// running sum of one row per request in 64 bits: a token's border there moves
// by the sum's relative error, and a row has 10^5 borders.  That row is read a
// second time, with the draft's probabilities, in chunks: a chunk leaves the
// sum of its weights w, and over the tokens with w > q W (W the row's sum)
// those of w and of q, so that the chunk's part of the sum of max(w - q W, 0)
// follows for the W in 64 bits that all chunks together give.  Tokens so near
// to w = q W that the 32-bit W may put them on the wrong side are summed too:
// they are off by kSumError of themselves at most, and where that is not
// nothing beside the whole, the chunks are formed anew.  A last launch finds
// the chunk that the token lies in, and the token.
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
// Runs of a thread: a wave's part of a row is kWave, a block's chunk kThreads
// threads with that many runs each.
constexpr int kLongRuns = 4, kShortRuns = 1;
// Of the 32-bit sum, if every rounding goes the same way, in units of 2^-24 of a
// term.  Its exponent y is off by 3 |y| (a difference in float's normal range,
// the factor and their product rounded; with every change of the maximum y is the sum of pieces of
// one sign), which is 3 ln 2 |y| of the term; over the row |y| has a mean of
// log2 of the vocabulary at most, below 31, because the entropy of p is no
// more than that and no less than this mean.  Each of its exponentials is off
// by 2 (one for itself, one for every later run's maximum, one for the wave's),
// each of their products by 1.  It passes 3 sums of its run, one for every later
// run and 6 of the wave's.
constexpr double kSumUnits = 3 * 0.69314718056 * 31 + 2 * (kLongRuns + 1) + kLongRuns + 3 + (kLongRuns - 1) + 6;
constexpr double kSumError = 5.5e-6;
static_assert(kRun == 8 && kWave == 64 && kSumUnits * 0x1p-24 < kSumError, "the row's sum is off by more");
// What tokens near their border may move of the whole, if all of them lie on
// the wrong side by all of kSumError.
constexpr double kNearly = 1e-9;

struct Part {  // of one wave's share of a position's row
  float top;   // NaN: an allowed logit is +inf or NaN
  float sum;   // of exp((z - top) / temperature); at temperature 0 the bits of the first token with the largest logit
};

struct ChunkSum {
  double all;   // sum of w = exp((z - top) / temperature)
  double over;  // of those with w > q W
  double take;  // their sum of q
  double near;  // sum of w close to q W
};

struct Space {
  Part* parts;       // [rows, drafts + 1, parts of a row]
  ChunkSum* chunks;  // [rows, chunks] of the deciding row
  int32_t* states;   // [rows, drafts + 1]
  RowStat* finals;   // [rows]: the deciding row
  int32_t* decided;  // [rows]: its position, -1: not yet found
  int32_t runs, row_parts, row_chunks;
  size_t bytes;
};

// Long runs share out what a wave does besides its tokens, short ones spread a
// small call over more of the device and need no launch of their own for the
// verdicts (five positions of 151,936 bf16: one request 30 us with long runs,
// 25 with short ones; 8: 33.3 and 32.6; 12: 35 and 37; 32: 45 and 62).
constexpr int64_t kLongFrom = int64_t(8) << 20;  // tokens of all positions

Space verify_space(int64_t rows, int32_t drafts, int64_t vocab, void* at = nullptr) {
  Space w{};
  w.runs = rows * (drafts + 1) * vocab >= kLongFrom ? kLongRuns : kShortRuns;
  w.row_parts = int32_t((vocab + kWave * kRun * w.runs - 1) / (kWave * kRun * w.runs));
  w.row_chunks = int32_t((vocab + kThreads * kRun * w.runs - 1) / (kThreads * kRun * w.runs));
  char* p = static_cast<char*>(at);
  const auto take = [&](size_t n) {
    char* q = p + w.bytes;
    w.bytes += (n + 15) / 16 * 16;
    return q;
  };
  const size_t positions = size_t(rows) * size_t(drafts + 1);
  w.parts = reinterpret_cast<Part*>(take(positions * w.row_parts * sizeof(Part)));
  w.chunks = reinterpret_cast<ChunkSum*>(take(size_t(rows) * w.row_chunks * sizeof(ChunkSum)));
  w.states = reinterpret_cast<int32_t*>(take(positions * 4));
  w.finals = reinterpret_cast<RowStat*>(take(size_t(rows) * sizeof(RowStat)));
  w.decided = reinterpret_cast<int32_t*>(take(size_t(rows) * 4));
  return w;
}

// Which of a run's tokens are its own and allowed.
__device__ __forceinline__ uint32_t run_bits(const VerifyArgs& a, int32_t state, const Run& run) {
  if (!a.allow_bits) return run.own;
  if (state < 0 || state >= a.num_states || run.own == 0) return 0u;
  const uint32_t bits = reinterpret_cast<const uint8_t*>(bits_of(a, state))[(run.t + run.shift) / 8];
  return bits << run.shift & run.own;
}
__device__ __forceinline__ const char* row_of(const VerifyArgs& a, int64_t b, int32_t i) {
  return static_cast<const char*>(a.logits) + row_at(a, b, i) * (a.dtype == BPD_DTYPE_F32 ? 4 : 2);
}

// One wave per part, position (`count` from `from` on) and request, in this
// order.  The positions before `from` have been judged.  About 14 vector
// instructions a token, half of the time, and the read: the first position of
// 256 rows of 151,936 bf16 takes 23 us (78 MB, 3.4 TB/s).  A lane keeps its own
// largest logit and the sum relative to it; all its runs are on their way before
// the first is summed.  (Two or four such sets per wave, the next on its way
// while one is summed: 23 -> 26 us for the first position of 256 rows.)
template <int DT, int Runs>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(VerifyArgs a, Space w, int32_t from, int32_t count) {
  const int lane = threadIdx.x % kWave;
  const uint32_t id = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + threadIdx.x / kWave);
  const uint32_t at = id / uint32_t(w.row_parts);
  if (at >= uint32_t(a.rows) * uint32_t(count)) return;
  const int32_t part = int32_t(id - at * uint32_t(w.row_parts));
  const int64_t b = at / uint32_t(count);
  const int32_t i = from + int32_t(at - uint32_t(b) * uint32_t(count));
  if (i > draft_len(a, b) || (from > 0 && w.decided[b] >= 0)) return;
  int32_t* states = w.states + b * (a.drafts + 1);
  const char* row = row_of(a, b, i);
  Raw<DT> raw[Runs];
  uint32_t bits[Runs];
  const auto run_of = [&](int k) { return run_at((int64_t(part) * Runs + k) * (kWave * kRun) + lane * kRun, a.vocab); };
  // the logits, before the walk to this position's state is waited for
#pragma unroll
  for (int k = 0; k < Runs; ++k) raw[k] = load_raw<DT>(row, run_of(k), a.vocab);
  int32_t state = from > 0 ? states[from - 1] : 0;
  for (int32_t k = a.bit_rows ? i : from; k <= i; ++k) state = state_at(a, b, k, state);
  if (part == 0 && lane == 0) states[i] = state;
#pragma unroll
  for (int k = 0; k < Runs; ++k) bits[k] = run_bits(a, state, run_of(k));
  const double temp = temperature_of(a, b);
  // half the difference does not pass the type's range; a factor past it (of a
  // subnormal temperature) would only make a zero of the largest logit's
  // difference a NaN
  const float to_log2 = temp > 0.0 ? float(fmin(2.0 * kLog2E / temp, 3e38)) : 0.0f;
  bool bad = false;
  float top = -INFINITY, sum = 0.0f;
  int32_t first = 0x7FFFFFFF;
#pragma unroll
  for (int k = 0; k < Runs; ++k) {
    if (!__any(bits[k] != 0)) continue;
    float z[kRun], here = -INFINITY;
    unpack<DT>(raw[k], z);
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      z[j] = masked(z[j], bits[k], j);
      bad |= !(z[j] < INFINITY);
      here = fmaxf(here, z[j]);
    }
    if (temp > 0.0) {
      if (__any(here > top)) {
        const float now = fmaxf(top, here);
        sum *= top > -INFINITY ? __builtin_amdgcn_exp2f(__builtin_fmaf(top, 0.5f, -0.5f * now) * to_log2) : 0.0f;
        top = now;
      }
      const float half = -0.5f * (top > -INFINITY ? top : 0.0f);
#pragma unroll
      for (int j = 0; j < kRun; ++j) z[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[j], 0.5f, half) * to_log2);
      sum += ((z[0] + z[1]) + (z[2] + z[3])) + ((z[4] + z[5]) + (z[6] + z[7]));
    } else if (here > top) {
      top = here;
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j)
        if (z[j] == top) first = int32_t(run_of(k).t) + j;
    }
  }
  // the lanes' parts as one
  const float whole = wave_max(top);
  Part p{__any(bad) ? NAN : whole, 0.0f};
  if (p.top > -INFINITY && temp > 0.0) {
    p.sum = wave_sum(sum * __builtin_amdgcn_exp2f(__builtin_fmaf(top, 0.5f, -0.5f * whole) * to_log2));
  } else if (p.top > -INFINITY) {
    if (top != whole) first = 0x7FFFFFFF;
    p.sum = __builtin_bit_cast(float, wave_min(first));
  }
  if (lane == 0) w.parts[(b * (a.drafts + 1) + i) * w.row_parts + part] = p;
}

// A position's row from its parts, by one wave.
__device__ __forceinline__ RowStat whole_row(const VerifyArgs& a, const Space& w, int64_t b, int32_t i, int lane) {
  const int64_t at = b * (a.drafts + 1) + i;
  const Part* parts = w.parts + at * w.row_parts;
  RowStat st{0.0, -INFINITY, 0x7FFFFFFF, 0, 0, w.states[at]};
  const double temp = temperature_of(a, b);
  bool bad = false;
  for (int32_t c = lane; c < w.row_parts; c += kWave) {
    bad |= parts[c].top != parts[c].top;
    st.top = fmaxf(st.top, parts[c].top);
  }
  st.top = wave_max(st.top);
  st.bad = __any(bad);
  st.empty = st.bad || st.top == -INFINITY;
  if (st.empty) return st;
  if (temp > 0.0) {
    const double to_log2 = kLog2E / temp;
    for (int32_t c = lane; c < w.row_parts; c += kWave)
      if (parts[c].top > -INFINITY)
        st.sum += double(parts[c].sum) * exp2_down((double(parts[c].top) - double(st.top)) * to_log2);
    st.sum = wave_sum(st.sum);
    return st;
  }
  for (int32_t c = lane; c < w.row_parts; c += kWave)
    if (parts[c].top == st.top) st.first = min(st.first, __builtin_bit_cast(int32_t, parts[c].sum));
  st.first = wave_min(st.first);
  st.sum = 1.0;
  return st;
}

// Sum over a block of N waves, on every thread; `sums` is shared memory.
template <int N>
__device__ __forceinline__ double block_sum(double x, double* sums) {
  x = wave_sum(x);
  __syncthreads();
  if (threadIdx.x % kWave == 0) sums[threadIdx.x / kWave] = x;
  __syncthreads();
  x = sums[0];
#pragma unroll
  for (int k = 1; k < N; ++k) x += sums[k];
  return x;
}

// A position's sum of weights in 64 bits, by a block.
template <int DT, int N>
__device__ double exact_sum(const VerifyArgs& a, int64_t b, int32_t i, float top, int32_t state, double* sums) {
  const double to_log2 = kLog2E / temperature_of(a, b);
  const char* row = row_of(a, b, i);
  double sum = 0.0;
#pragma unroll 1
  for (int64_t t = threadIdx.x * kRun; t < a.vocab; t += N * kWave * kRun) {
    const Run run = run_at(t, a.vocab);
    float z[kRun];
    load_run<DT>(row, run, a.vocab, z);
    const uint32_t bits = run_bits(a, state, run);
#pragma unroll
    for (int j = 0; j < kRun; ++j) sum += exp2_down((double(masked(z[j], bits, j)) - double(top)) * to_log2);
  }
  return block_sum<N>(sum, sums);
}

// The deciding position: the first that does not stand (a request's last has
// no draft and never stands), among those from `from` on and before `to`; -1
// where they all stand.  By a whole block of N waves, a wave per position; *v
// (the rows) and `sums` are shared memory.
struct Verdict {
  RowStat rows[kMaxPositions];
  double weight[kMaxPositions], least[kMaxPositions];  // of the drafted token, and u q
  int32_t holds[kMaxPositions];                        // 2: too near to tell
};
template <int DT, int N>
__device__ __forceinline__ int32_t verdict(const VerifyArgs& a, const Space& w, int64_t b, int32_t from, int32_t to,
                                           Verdict* v, double* sums) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int32_t len = draft_len(a, b);
  if (to > len + 1) to = len + 1;
  for (int32_t i = from + wave; i < to; i += N) {
    // what the draft asks for, before the row's sums are waited for
    bool in = false;
    float z = 0.0f;
    double uq = 0.0;
    int64_t x = -1;
    if (i < len) {
      x = read_token(a.tokens, a.token_dtype, b * a.tokens_ld + i);
      in = x >= 0 && x < a.vocab;
      if (in) {
        z = load_elem(a.logits, DT, row_at(a, b, i) + x);
        uq = double(a.uniforms[b * a.uniforms_ld + i]) * prob_of(a, b, i, x, x);
      }
    }
    const RowStat row = whole_row(a, w, b, i, lane);
    const double temp = temperature_of(a, b);
    in = in && !row.empty && allowed(bits_of(a, row.state), x);
    if (lane != 0) continue;
    const double weight = temp > 0.0 ? exp2_down((double(z) - double(row.top)) * (kLog2E / temp)) : x == row.first ? 1.0 : 0.0;
    const double off = uq * row.sum - weight;
    v->rows[i] = row, v->weight[i] = weight, v->least[i] = uq;
    v->holds[i] = !in ? 0 : temp > 0.0 && fabs(off) <= kSumError * weight ? 2 : off < 0.0;
  }
  __syncthreads();
  for (int32_t n = from; n < to; ++n) {
    int32_t holds = v->holds[n];
    if (holds == 2) holds = v->least[n] * exact_sum<DT, N>(a, b, n, v->rows[n].top, v->rows[n].state, sums) < v->weight[n];
    if (!holds) return n;
  }
  return -1;
}

// The verdicts by themselves, one block per request.
constexpr int kJudgeWaves = 16;
template <int DT>
__global__ __launch_bounds__(kJudgeWaves* kWave) void verify_judge_kernel(VerifyArgs a, Space w, int32_t from,
                                                                           int32_t to) {
  __shared__ Verdict v;
  __shared__ double sums[kJudgeWaves];
  const int64_t b = blockIdx.x;
  if (from > 0 && w.decided[b] >= 0) return;
  const int32_t n = verdict<DT, kJudgeWaves>(a, w, b, from, to, &v, sums);
  if (threadIdx.x != 0) return;
  w.decided[b] = n;
  if (n >= 0) w.finals[b] = v.rows[n];
}

// What the chunks of the deciding row are formed from.
struct Deciding {
  const char *row, *probs;  // probs: null where nothing comes off, or all of one token
  int64_t drafted;          // that token, -1
  int32_t state;
  double top, to_log2;
};

// The draft's probabilities of a run.  A certain draft counts as 2: never less
// than a weight, and not near one.
template <int N>
__device__ __forceinline__ void draft_runs(const VerifyArgs& a, const Deciding& d, const Run (&runs)[N], float (&q)[N][kRun]) {
  if (d.probs) {
    if (a.probs_dtype == BPD_DTYPE_BF16) load_runs<BPD_DTYPE_BF16>(d.probs, runs, a.vocab, q);
    else if (a.probs_dtype == BPD_DTYPE_F16) load_runs<BPD_DTYPE_F16>(d.probs, runs, a.vocab, q);
    else load_runs<BPD_DTYPE_F32>(d.probs, runs, a.vocab, q);
    return;
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int j = 0; j < kRun; ++j) q[k][j] = runs[k].t + j == d.drafted ? 2.0f : 0.0f;
}

__device__ __forceinline__ Deciding deciding(const VerifyArgs& a, int64_t b, int32_t n, const RowStat& st) {
  Deciding d{row_of(a, b, n), nullptr, -1, st.state, double(st.top), kLog2E / temperature_of(a, b)};
  if (n < draft_len(a, b)) {
    if (a.probs)
      d.probs = static_cast<const char*>(a.probs) + (b * a.probs_row + n * a.probs_pos) * (a.probs_dtype == BPD_DTYPE_F32 ? 4 : 2);
    else
      d.drafted = read_token(a.tokens, a.token_dtype, b * a.tokens_ld + n);
  }
  return d;
}

// The sums of a chunk of a request's deciding row, one block each: about 40
// vector instructions a token, most of them in 64 bits, which is its bound.
// Where a grammar leaves every lane of a wave at most a quarter of its tokens,
// these alone are loaded, all at once, and summed one by one (256 rows of 151,936
// bf16 with bf16 probabilities under grammars that allow 0.0002 to 0.95 of the
// tokens: 39 us, and 53 where every lane sums all of them).  With few requests
// (kShortRuns) every block forms the verdicts for itself: a launch less.
template <int DT, int Runs>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs a, Space w) {
  __shared__ double sums[kWaves][4];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int64_t b = blockIdx.x / uint32_t(w.row_chunks);
  const int32_t chunk = int32_t(blockIdx.x - uint32_t(b) * uint32_t(w.row_chunks));
  RowStat st;
  int32_t n;
  if constexpr (Runs == kShortRuns) {
    __shared__ Verdict v;
    n = verdict<DT, kWaves>(a, w, b, 0, a.drafts + 1, &v, &sums[0][0]);
    st = v.rows[n];
    if (chunk == 0 && tid == 0) w.decided[b] = n, w.finals[b] = st;
    __syncthreads();
  } else {
    n = w.decided[b], st = w.finals[b];
  }
  if (st.empty || !(temperature_of(a, b) > 0.0)) return;
  const Deciding d = deciding(a, b, n, st);
  const bool less = n < draft_len(a, b);
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  // a token's weight, and where the draft's probabilities come off, its p
  const auto add = [&](double x, double p) {
    const double y = x - p * st.sum;
    s[1] += y > 0.0 ? x : 0.0;
    s[2] += y > 0.0 ? p : 0.0;
    s[3] += fabs(y) <= kSumError * x ? x : 0.0;
  };
  uint32_t all_bits = 0;  // of the runs, eight each
#pragma unroll
  for (int k = 0; k < Runs; ++k)
    all_bits |= run_bits(a, d.state, run_at((int64_t(chunk) * Runs + k) * (kThreads * kRun) + tid * kRun, a.vocab))
                << (8 * k);
  constexpr int kFew = 2 * Runs;
  const int allowed_here = __popc(all_bits);
  const bool few = a.allow_bits && !__any(allowed_here > kFew);
  if (few && __any(allowed_here > 0)) {
    float z[kFew], q[kFew];
#pragma unroll
    for (int k = 0; k < kFew; ++k) {
      const bool on = all_bits != 0;
      const int bit = on ? __builtin_ctz(all_bits) : 0;
      all_bits &= all_bits - 1;
      const int64_t t = run_at((int64_t(chunk) * Runs + bit / 8) * (kThreads * kRun) + tid * kRun, a.vocab).t + bit % 8;
      z[k] = on ? load_elem(d.row, DT, t) : -INFINITY;
      q[k] = !on ? 0.0f : d.probs ? load_elem(d.probs, a.probs_dtype, t) : t == d.drafted ? 2.0f : 0.0f;
    }
#pragma unroll 1
    for (int k = 0; k < kFew; ++k) {
      if (!__any(k < allowed_here)) break;
      const double x = exp2_down((double(z[0]) - d.top) * d.to_log2);
      s[0] += x;
      if (less) add(x, q[0]);
#pragma unroll
      for (int l = 1; l < kFew; ++l) z[l - 1] = z[l], q[l - 1] = q[l];
    }
  }
  // One run at a time leaves seven waves on a SIMD, which hide its loads better
  // than two or four runs in flight do (57, 60 and 66 us: 256 rows of 151,936
  // bf16 with bf16 probabilities, every token summed).
#pragma unroll 1
  for (int k0 = 0; k0 < Runs && !few; ++k0, all_bits >>= 8) {
    const Run run[1] = {run_at((int64_t(chunk) * Runs + k0) * (kThreads * kRun) + tid * kRun, a.vocab)};
    const uint32_t bits = all_bits & 0xFFu;
    if (!__any(bits != 0)) continue;
    float z[1][kRun], q[1][kRun];
    load_runs<DT>(d.row, run, a.vocab, z);
    if (d.probs) draft_runs(a, d, run, q);
    double x[kRun];
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      x[j] = exp2_down((double(masked(z[0][j], bits, j)) - d.top) * d.to_log2);
      s[0] += x[j];
    }
    if (d.probs) {
#pragma unroll
      for (int j = 0; j < kRun; ++j) add(x[j], q[0][j]);
    } else if (less) {  // all but the drafted token
#pragma unroll
      for (int j = 0; j < kRun; ++j) s[1] += run[0].t + j == d.drafted ? 0.0 : x[j];
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k > 0 && !less) break;
    s[k] = wave_sum(s[k]);
    if (lane == 0) sums[wave][k] = s[k];
  }
  __syncthreads();
  if (tid >= 4) return;
  double x = 0.0;
  if (tid == 0 || (less && (tid == 1 || d.probs)))
    for (int k = 0; k < kWaves; ++k) x += sums[k][tid];
  reinterpret_cast<double*>(w.chunks + b * w.row_chunks + chunk)[tid] = x;
}

// The next token, one block per request, a run of the chunk per thread: a chain
// of loads that wait for each other (5 us for a short chunk, 8 to 10 for a long
// one; 40 to 60 us more where it forms the chunks of 151,936 tokens anew).
template <int DT, int Runs>
__global__ __launch_bounds__(kThreads* Runs) void verify_pick_kernel(VerifyArgs a, Space w) {
  constexpr int N = kWaves * Runs;
  __shared__ double sums[N], before, target, row_sum;
  __shared__ int32_t where, found, last, take_off;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int64_t b = blockIdx.x;
  const int32_t n = w.decided[b], len = draft_len(a, b);
  const RowStat st = w.finals[b];
  if (tid == 0) {
    const int32_t f = flags_of(a, b, n, len, st.state, st.bad);
    if (f && a.err) atomicOr(a.err, f);
  }
  if (st.empty || !(temperature_of(a, b) > 0.0)) {
    if (tid == 0) finish(a, b, n, st, st.empty ? -1 : st.first);
    return;
  }
  const bool less = n < len;
  const Deciding d = deciding(a, b, n, st);
  ChunkSum* chunks = w.chunks + b * w.row_chunks;
  // max(w - q W, 0) of a run of a chunk (w without q)
  const auto shares = [&](int32_t c, bool off, double whole, double (&x)[kRun]) -> int64_t {
    const Run run[1] = {run_at((int64_t(c) * (kThreads * Runs) + tid) * kRun, a.vocab)};
    float z[1][kRun], q[1][kRun];
    load_runs<DT>(d.row, run, a.vocab, z);
    draft_runs(a, d, run, q);
    const uint32_t bits = run_bits(a, d.state, run[0]);
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      const double y = exp2_down((double(masked(z[0][j], bits, j)) - d.top) * d.to_log2) - (off ? double(q[0][j]) * whole : 0.0);
      x[j] = y > 0.0 ? y : 0.0;
    }
    return run[0].t;
  };
  // First with the sums as they are; where tokens near their border weigh too
  // much, or none is found, with sums formed anew.
#pragma unroll 1
  for (int anew = 0;; ++anew) {
    if (wave == 0) {
      const double u = a.uniforms[b * a.uniforms_ld + a.drafts];
      ChunkSum s{0.0, 0.0, 0.0, 0.0};
      if (lane < w.row_chunks) s = chunks[lane];
      const ChunkSum near_by = s;
      for (int32_t c = lane + kWave; c < w.row_chunks; c += kWave) {
        const ChunkSum y = chunks[c];
        s.all += y.all, s.over += y.over, s.take += y.take, s.near += y.near;
      }
      s.all = wave_sum(s.all), s.over = wave_sum(s.over), s.take = wave_sum(s.take), s.near = wave_sum(s.near);
      const double rest = s.over - s.take * s.all;
      const bool sure = anew || !less || !(s.near * kSumError > kNearly * rest), off = less && rest > 0.0;
      // the chunk in which the share u of the whole lies, or the last that has
      // any of it; the whole is summed in the order of the running sum
      double whole = 0.0, run = 0.0, at = 0.0;
      int32_t hit = -1;
      bool past_it = false;
#pragma unroll 1
      for (int pass = 0; pass < 2 && sure; ++pass) {
        run = 0.0;
        for (int32_t c0 = 0; c0 < w.row_chunks && !past_it; c0 += kWave) {
          double mine = 0.0;
          if (c0 + lane < w.row_chunks) {
            const ChunkSum y = c0 == 0 ? near_by : chunks[c0 + lane];
            mine = off ? y.over - y.take * s.all : y.all;
            mine = mine > 0.0 ? mine : 0.0;
          }
          const double upto = run + wave_scan_sum(mine);
          run = of_lane(upto, kWave - 1);
          const uint64_t any = pass == 0 ? 0 : __ballot(mine > 0.0), past = __ballot(mine > 0.0 && upto > u * whole);
          if (any) {
            past_it = (any & past) != 0;
            const int l = past_it ? __builtin_ctzll(past) : 63 - __builtin_clzll(any);
            hit = c0 + l, at = of_lane(upto - mine, l);
          }
        }
        if (pass == 0) whole = run;
      }
      if (lane == 0) where = hit, before = at, target = u * whole, take_off = off, row_sum = s.all, found = 0x7FFFFFFF, last = -1;
    }
    __syncthreads();
    if (where >= 0) {
      double x[kRun], own = 0.0;
      const int64_t t = shares(where, take_off != 0, row_sum, x);
#pragma unroll
      for (int j = 0; j < kRun; ++j) own += x[j];
      const double upto = wave_scan_sum(own);
      if (lane == kWave - 1) sums[wave] = upto;
      __syncthreads();
      double at = before + (upto - own);
      for (int k = 0; k < wave; ++k) at += sums[k];
      int32_t hit = 0x7FFFFFFF, end = -1;
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        at += x[j];
        if (!(x[j] > 0.0)) continue;
        end = int32_t(t) + j;
        if (at > target && hit == 0x7FFFFFFF) hit = end;
      }
      // tokens rise with the lanes: one of a wave speaks for it
      const uint64_t hits = __ballot(hit != 0x7FFFFFFF), some = __ballot(end >= 0);
      if (hits && lane == __builtin_ctzll(hits)) atomicMin(&found, hit);
      if (some && lane == 63 - __builtin_clzll(some)) atomicMax(&last, end);
      __syncthreads();
      if (last >= 0) break;
    }
    if (anew) break;
#pragma unroll 1
    for (int32_t c = 0; c < w.row_chunks; ++c) {
      double x[kRun], own = 0.0;
      shares(c, true, row_sum, x);
#pragma unroll
      for (int j = 0; j < kRun; ++j) own += x[j];
      own = block_sum<N>(own, sums);
      if (tid == 0) chunks[c].over = own, chunks[c].take = 0.0;
    }
    __syncthreads();
  }
  if (tid == 0) finish(a, b, n, st, found != 0x7FFFFFFF ? found : last);
}

// Bytes of one position of every request from which the positions are read in
// three steps (the first, the second, the others), each for the requests whose
// drafts stand so far (half of them at each; five positions of 151,936 bf16:
// 128 requests 96 us in steps, 92 at once; 160: 108 and 106; 256: 178 and 188).
constexpr int64_t kStepBytes = int64_t(48) << 20;

template <int DT, int Runs>
int launch_verify_runs(const VerifyArgs& a, const Space& w, hipStream_t s) {
  const int32_t all = a.drafts + 1;
  const bool steps = Runs != kShortRuns && a.rows * a.vocab * elem_bytes(DT) >= kStepBytes;
  for (int32_t from = 0, to; from < all; from = to) {
    to = steps && from < 2 ? from + 1 : all;
    const int64_t waves = a.rows * (to - from) * w.row_parts;
    verify_rows_kernel<DT, Runs><<<uint32_t((waves + kWaves - 1) / kWaves), kThreads, 0, s>>>(a, w, from, to - from);
    if (Runs != kShortRuns) verify_judge_kernel<DT><<<uint32_t(a.rows), kJudgeWaves * kWave, 0, s>>>(a, w, from, to);
  }
  verify_sums_kernel<DT, Runs><<<uint32_t(a.rows * w.row_chunks), kThreads, 0, s>>>(a, w);
  verify_pick_kernel<DT, Runs><<<uint32_t(a.rows), kThreads * Runs, 0, s>>>(a, w);
  BPD_LAUNCHED();
  return BPD_OK;
}

template <int DT>
int launch_verify_dtype(const VerifyArgs& a, const Space& w, hipStream_t s) {
  return w.runs == kLongRuns ? launch_verify_runs<DT, kLongRuns>(a, w, s) : launch_verify_runs<DT, kShortRuns>(a, w, s);
}

int launch_verify(const VerifyArgs& a, void* workspace, hipStream_t s) {
  const Space w = verify_space(a.rows, a.drafts, a.vocab, workspace);
  BPD_REQUIRE(a.rows * int64_t(a.drafts + 1) * w.row_parts < (int64_t(1) << 31), "too many positions in one call");
  if (a.dtype == BPD_DTYPE_BF16) return launch_verify_dtype<BPD_DTYPE_BF16>(a, w, s);
  if (a.dtype == BPD_DTYPE_F16) return launch_verify_dtype<BPD_DTYPE_F16>(a, w, s);
  return launch_verify_dtype<BPD_DTYPE_F32>(a, w, s);
}

void host_verify(const VerifyArgs& a) {
  int32_t flags = 0;
  for (int64_t b = 0; b < a.rows; ++b) {
    const int32_t len = draft_len(a, b);
    const double temp = temperature_of(a, b);
    RowStat st{};
    int32_t n = 0;
    for (;; ++n) {
      st = RowStat{0.0, -INFINITY, 0, 0, 0, state_at(a, b, n, st.state)};
      const bool some = !a.allow_bits || (st.state >= 0 && st.state < a.num_states);
      const uint32_t* bits = some ? bits_of(a, st.state) : nullptr;
      const int64_t V = some ? a.vocab : 0;
      for (int64_t t = 0; t < V; ++t) {
        if (!allowed(bits, t)) continue;
        const float z = load_elem(a.logits, a.dtype, row_at(a, b, n) + t);
        if (!(z < INFINITY)) st.empty = st.bad = 1;
        if (z > st.top) st.top = z, st.first = int32_t(t);
      }
      if (st.top == -INFINITY) st.empty = 1;
      for (int64_t t = 0; t < V && !st.empty; ++t)
        if (allowed(bits, t)) st.sum += weight(st, temp, load_elem(a.logits, a.dtype, row_at(a, b, n) + t), t);
      if (n == len || !stands(a, b, n, st)) break;
    }
    flags |= flags_of(a, b, n, len, st.state, st.bad);
    int64_t token = -1;
    if (!st.empty) {
      const uint32_t* bits = bits_of(a, st.state);
      const int64_t drafted = n < len ? read_token(a.tokens, a.token_dtype, b * a.tokens_ld + n) : -1;
      bool less = n < len;
      double whole = 0.0;
      for (;;) {
        whole = 0.0;
        for (int64_t t = 0; t < a.vocab; ++t) whole += share(a, b, n, st, temp, bits, less, drafted, t);
        if (whole > 0.0 || !less) break;
        less = false;
      }
      const double target = double(a.uniforms[b * a.uniforms_ld + a.drafts]) * whole;
      double run = 0.0;
      for (int64_t t = 0; t < a.vocab; ++t) {
        const double r = share(a, b, n, st, temp, bits, less, drafted, t);
        if (!(r > 0.0)) continue;
        run += r;
        token = t;
        if (run > target) break;
      }
    }
    finish(a, b, n, st, token);
  }
  if (flags && a.err) *a.err |= flags;
}

int check_verify(const VerifyArgs& a) {
  BPD_REQUIRE(elem_bytes(a.dtype) != 0, "unknown logits dtype code %d", a.dtype);
  BPD_REQUIRE(a.rows >= 0 && a.drafts >= 0 && a.drafts <= BPD_MAX_DRAFTS, "at most %d drafted tokens (got %d)",
              BPD_MAX_DRAFTS, a.drafts);
  BPD_REQUIRE(a.vocab >= 1 && a.vocab < (int64_t(1) << 31), "a vocabulary of 1 to 2^31 - 1 tokens (got %lld)",
              (long long)a.vocab);
  BPD_REQUIRE(!a.probs || elem_bytes(a.probs_dtype) != 0, "unknown dtype code %d of the draft's probabilities",
              a.probs_dtype);
  BPD_REQUIRE(token_dtype_ok(a.token_dtype), "unknown token dtype code %d", a.token_dtype);
  if (a.rows == 0) return BPD_OK;
  BPD_REQUIRE(a.logits && a.uniforms && a.accepted && a.next_token && (a.drafts == 0 || a.tokens),
              "null pointer argument");
  BPD_REQUIRE(a.temperature || (std::isfinite(a.temperature_all) && a.temperature_all >= 0.0f),
              "the temperature must be finite and not negative");
  BPD_REQUIRE(!(a.tok_next && a.bit_rows), "states come from tok_next or from bit_rows, not both");
  BPD_REQUIRE(!(a.tok_next || a.bit_rows) || a.allow_bits, "a grammar needs its allow bits");
  BPD_REQUIRE(!a.allow_bits || ((a.tok_next || a.bit_rows) && a.num_states >= 0 && a.words >= (a.vocab + 31) / 32),
              "allow bits need states, and a row of ceil(vocab / 32) words");
  BPD_REQUIRE(!a.tok_next || a.states, "tok_next needs the requests' states");
  BPD_REQUIRE(!(a.write_back || a.next_state) || a.tok_next, "states are advanced through tok_next only");
  BPD_REQUIRE(a.rows * int64_t(a.drafts + 1) < (int64_t(1) << 31), "too many positions in one call");
  return BPD_OK;
}

}  // namespace
}  // namespace bpd

using namespace bpd;

#define BPD_VERIFY_ARGS                                                                                          \
  VerifyArgs a {                                                                                                 \
    logits, dtype, rows, drafts, vocab, ld_row, ld_pos, tokens, token_dtype, tokens_ld, draft_lens, probs,       \
        probs_dtype, probs_row, probs_pos, uniforms, uniforms_ld, temperature, temperature_all, allow_bits,      \
        words, num_states, tok_next, states, slots, bit_rows, write_back, accepted, next_token, next_state, err \
  }

extern "C" size_t bpd_verify_workspace_bytes(int64_t rows, int32_t drafts, int64_t vocab) {
  return rows <= 0 || drafts < 0 || vocab <= 0 ? 0 : verify_space(rows, drafts, vocab).bytes;
}

extern "C" int bpd_verify(const void* logits, int dtype, int64_t rows, int32_t drafts, int64_t vocab, int64_t ld_row,
                          int64_t ld_pos, const void* tokens, int token_dtype, int64_t tokens_ld,
                          const int32_t* draft_lens, const void* probs, int probs_dtype, int64_t probs_row,
                          int64_t probs_pos, const float* uniforms, int64_t uniforms_ld, const float* temperature,
                          float temperature_all, const uint32_t* allow_bits, int64_t words, int32_t num_states,
                          const int32_t* tok_next, int32_t* states, const int64_t* slots, const int32_t* bit_rows,
                          int write_back, int32_t* accepted, int32_t* next_token, int32_t* next_state,
                          void* workspace, size_t workspace_bytes, int32_t* err, void* stream) {
  BPD_VERIFY_ARGS;
  if (int rc = check_verify(a)) return rc;
  if (rows == 0) return BPD_OK;
  BPD_REQUIRE(workspace && workspace_bytes >= bpd_verify_workspace_bytes(rows, drafts, vocab),
              "the workspace is smaller than bpd_verify_workspace_bytes");
  return launch_verify(a, workspace, as_stream(stream));
}

extern "C" int bpd_host_verify(const void* logits, int dtype, int64_t rows, int32_t drafts, int64_t vocab,
                               int64_t ld_row, int64_t ld_pos, const void* tokens, int token_dtype,
                               int64_t tokens_ld, const int32_t* draft_lens, const void* probs, int probs_dtype,
                               int64_t probs_row, int64_t probs_pos, const float* uniforms, int64_t uniforms_ld,
                               const float* temperature, float temperature_all, const uint32_t* allow_bits,
                               int64_t words, int32_t num_states, const int32_t* tok_next, int32_t* states,
                               const int64_t* slots, const int32_t* bit_rows, int write_back, int32_t* accepted,
                               int32_t* next_token, int32_t* next_state, int32_t* err) {
  BPD_VERIFY_ARGS;
  if (int rc = check_verify(a)) return rc;
  if (rows > 0) host_verify(a);
  return BPD_OK;
}
