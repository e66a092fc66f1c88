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
#include <vector>

#include "bpd_common.hpp"

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

__host__ __device__ __forceinline__ bool allowed(const uint32_t* bits, int64_t t) {
  return !bits || (bits[t >> 5] >> (t & 31) & 1u);
}

// What a position's row comes to.  `empty`: the grammar allows nothing, every
// allowed logit is -inf, or one is +inf or NaN and the row has no softmax.
struct RowStat {
  double sum;   // of exp((z - top) / temperature)
  float top;
  int32_t first;  // first token with the largest logit
  int32_t empty;
  int32_t state;  // row of allow_bits, -1: allows nothing
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

// The state of each position of request b, walked along its drafted tokens.
__host__ __device__ __forceinline__ void walk_states(const VerifyArgs& a, int64_t b, RowStat* st, int32_t* flags) {
  const int32_t n = draft_len(a, b);
  int32_t s = 0;
  if (a.tok_next) s = a.states[a.slots ? a.slots[b] : b];
  for (int32_t i = 0; i <= n; ++i) {
    if (a.bit_rows) s = a.bit_rows[b * (a.drafts + 1) + i];
    if (a.allow_bits && s >= a.num_states) {
      *flags |= BPD_FLAG_STATE_RANGE;
      s = -1;
    }
    if (s < 0) s = -1;
    st[i].state = s;
    if (i == n) break;
    const int64_t x = read_token(a.tokens, a.token_dtype, b * a.tokens_ld + i);
    if (x < 0 || x >= a.vocab) {
      *flags |= BPD_FLAG_TOKEN_RANGE;
      s = a.tok_next ? -1 : s;
    } else if (a.tok_next && s >= 0) {
      s = a.tok_next[int64_t(s) * a.vocab + x];
    }
  }
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
  const int32_t s = token < 0 || st.state < 0 ? -1 : a.tok_next[int64_t(st.state) * a.vocab + token];
  if (a.next_state) a.next_state[b] = s;
  if (a.write_back) a.states[a.slots ? a.slots[b] : b] = s;
}

__global__ void verify_walk_kernel(VerifyArgs a, RowStat* stats) {
  const int64_t b = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (b >= a.rows) return;
  int32_t flags = 0;
  walk_states(a, b, stats + b * (a.drafts + 1), &flags);
  if (flags && a.err) atomicOr(a.err, flags);
}

constexpr int kRowThreads = 1024;

// One block per position: the largest logit and its first token, then the
// sum of the weights.
__global__ __launch_bounds__(kRowThreads) void verify_rows_kernel(VerifyArgs a, RowStat* stats) {
  const int64_t b = blockIdx.x / (a.drafts + 1);
  const int32_t i = int32_t(blockIdx.x - b * (a.drafts + 1));
  if (i > draft_len(a, b)) return;
  RowStat& st = stats[blockIdx.x];
  __shared__ float tops[kRowThreads];
  __shared__ int64_t firsts[kRowThreads];
  __shared__ double sums[kRowThreads];
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  const int32_t state = a.allow_bits ? st.state : 0;
  const uint32_t* bits = state < 0 ? nullptr : bits_of(a, state);
  const int64_t V = state < 0 ? 0 : a.vocab;
  const int64_t row = row_at(a, b, i);
  float top = -INFINITY;
  int64_t first = a.vocab;
  for (int64_t t = threadIdx.x; t < V; t += kRowThreads) {
    if (!allowed(bits, t)) continue;
    const float z = load_elem(a.logits, a.dtype, row + t);
    if (!(z < INFINITY)) bad = 1;
    if (z > top) top = z, first = t;
  }
  tops[threadIdx.x] = top;
  firsts[threadIdx.x] = first;
  __syncthreads();
  for (int o = kRowThreads / 2; o; o >>= 1) {
    if (threadIdx.x < o) {
      const float y = tops[threadIdx.x + o];
      const int64_t f = firsts[threadIdx.x + o];
      if (y > tops[threadIdx.x] || (y == tops[threadIdx.x] && f < firsts[threadIdx.x])) {
        tops[threadIdx.x] = y;
        firsts[threadIdx.x] = f;
      }
    }
    __syncthreads();
  }
  RowStat mine{0.0, tops[0], int32_t(firsts[0]), tops[0] == -INFINITY || bad, st.state};
  const double temp = temperature_of(a, b);
  double sum = 0.0;
  if (!mine.empty)
    for (int64_t t = threadIdx.x; t < V; t += kRowThreads)
      if (allowed(bits, t)) sum += weight(mine, temp, load_elem(a.logits, a.dtype, row + t), t);
  sums[threadIdx.x] = sum;
  __syncthreads();
  for (int o = kRowThreads / 2; o; o >>= 1) {
    if (threadIdx.x < o) sums[threadIdx.x] += sums[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    mine.sum = sums[0];
    st = mine;
    if (bad && a.err) atomicOr(a.err, BPD_FLAG_LOGITS);
  }
}

// One block per request: how many drafts stand, and the next token.  Each
// thread sums a run of neighbouring tokens; the thread whose run the share
// falls into walks it again.
__global__ __launch_bounds__(kRowThreads) void verify_draw_kernel(VerifyArgs a, const RowStat* stats) {
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x;
  __shared__ int32_t count;
  __shared__ double sums[kRowThreads];
  __shared__ long long found, last;
  stats += b * (a.drafts + 1);
  const int32_t len = draft_len(a, b);
  if (tid == 0) {
    int32_t n = 0;
    while (n < len && stands(a, b, n, stats[n])) ++n;
    count = n;
  }
  __syncthreads();
  const int32_t n = count;
  const RowStat st = stats[n];
  if (st.empty) {
    if (tid == 0) finish(a, b, n, st, -1);
    return;
  }
  const double temp = temperature_of(a, b);
  const uint32_t* bits = bits_of(a, st.state);
  const int64_t drafted = n < len ? read_token(a.tokens, a.token_dtype, b * a.tokens_ld + n) : -1;
  const int64_t per = (a.vocab + kRowThreads - 1) / kRowThreads;
  const int64_t t0 = tid * per, t1 = t0 + per < a.vocab ? t0 + per : a.vocab;
  double mine = 0.0, whole = 0.0;
  bool less = n < len;
  for (;;) {
    mine = 0.0;
    for (int64_t t = t0; t < t1; ++t) mine += share(a, b, n, st, temp, bits, less, drafted, t);
    sums[tid] = mine;
    __syncthreads();
    for (int o = 1; o < kRowThreads; o <<= 1) {
      const double y = tid >= o ? sums[tid - o] : 0.0;
      __syncthreads();
      sums[tid] += y;
      __syncthreads();
    }
    whole = sums[kRowThreads - 1];
    if (whole > 0.0 || !less) break;
    less = false;
    __syncthreads();
  }
  const double target = double(a.uniforms[b * a.uniforms_ld + a.drafts]) * whole;
  if (tid == 0) found = a.vocab, last = -1;
  __syncthreads();
  double run = tid ? sums[tid - 1] : 0.0;
  if (mine > 0.0) {
    int64_t hit = -1, end = -1;
    for (int64_t t = t0; t < t1; ++t) {
      const double r = share(a, b, n, st, temp, bits, less, drafted, t);
      if (!(r > 0.0)) continue;
      end = t;
      run += r;
      if (hit < 0 && run > target) hit = t;
    }
    if (hit >= 0) atomicMin(&found, (long long)hit);
    atomicMax(&last, (long long)end);
  }
  __syncthreads();
  if (tid == 0) finish(a, b, n, st, found < a.vocab ? found : last);
}

void host_verify(const VerifyArgs& a) {
  std::vector<RowStat> stats(size_t(a.drafts) + 1);
  int32_t flags = 0;
  for (int64_t b = 0; b < a.rows; ++b) {
    walk_states(a, b, stats.data(), &flags);
    const int32_t len = draft_len(a, b);
    const double temp = temperature_of(a, b);
    int32_t n = 0;
    for (;; ++n) {
      RowStat& st = stats[n];
      const uint32_t* bits = a.allow_bits && st.state >= 0 ? bits_of(a, st.state) : nullptr;
      const int64_t V = a.allow_bits && st.state < 0 ? 0 : a.vocab;
      st.top = -INFINITY, st.first = 0, st.empty = 0, st.sum = 0.0;
      for (int64_t t = 0; t < V; ++t) {
        if (!allowed(bits, t)) continue;
        const float z = load_elem(a.logits, a.dtype, row_at(a, b, n) + t);
        if (!(z < INFINITY)) st.empty = 1, flags |= BPD_FLAG_LOGITS;
        if (z > st.top) st.top = z, st.first = int32_t(t);
      }
      if (st.top == -INFINITY) st.empty = 1;
      for (int64_t t = 0; t < V && !st.empty; ++t)
        if (allowed(bits, t)) st.sum += weight(st, temp, load_elem(a.logits, a.dtype, row_at(a, b, n) + t), t);
      if (n == len || !stands(a, b, n, st)) break;
    }
    const RowStat& st = stats[n];
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
  (void)vocab;
  return rows <= 0 || drafts < 0 ? 0 : size_t(rows) * size_t(drafts + 1) * sizeof(RowStat);
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
  RowStat* stats = static_cast<RowStat*>(workspace);
  hipStream_t s = as_stream(stream);
  verify_walk_kernel<<<uint32_t((rows + 63) / 64), 64, 0, s>>>(a, stats);
  verify_rows_kernel<<<uint32_t(rows * (drafts + 1)), kRowThreads, 0, s>>>(a, stats);
  verify_draw_kernel<<<uint32_t(rows), kRowThreads, 0, s>>>(a, stats);
  BPD_LAUNCHED();
  return BPD_OK;
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
