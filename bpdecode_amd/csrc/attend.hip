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

// One wave per query token and head, 64 cache tokens at a time: a lane scores
// one of them, then the lanes share out the channels.  The running maximum
// and sum are held in float.
template <int DT>
__global__ __launch_bounds__(kWave) void kv_attend_kernel(AttendArgs a) {
  __shared__ float qs[256], ps[kWave];
  __shared__ int64_t at[kWave];  // offset of each token's page block, -1: not there
  const int lane = threadIdx.x;
  const int64_t x = blockIdx.x;
  const int32_t h = int32_t(x % a.heads);
  const int32_t i = int32_t(x / a.heads % a.tokens);
  const int64_t b = x / a.heads / a.tokens;
  const int32_t D = a.page.dim, kvh = h / (a.heads / a.kv_heads);
  const uint16_t* q = a.q + b * a.q_row + i * a.q_token + h * a.q_head;
  for (int32_t d = lane; d < D; d += kWave) qs[d] = elem16_float<DT>(q[d]);
  bool past;
  const int64_t n = seen_tokens(a, b, i, &past);
  if (past && a.err && lane == 0) atomicOr(a.err, BPD_FLAG_PAGE_RANGE);
  float m = -INFINITY, l = 0.0f, acc[4] = {0, 0, 0, 0};
  for (int64_t t0 = 0; t0 < n; t0 += kWave) {
    __syncthreads();
    const int64_t t = t0 + lane;
    const int64_t page = t < n ? a.table.page_of(b, t, a.page.page_size) : -1;
    if (t < n && page < 0 && a.err) atomicOr(a.err, BPD_FLAG_PAGE_RANGE);
    const int64_t base = page < 0 ? -1 : (page * a.kv_heads + kvh) * int64_t(a.page.bytes());
    float s = -INFINITY;
    if (base >= 0) {
      const int32_t slot = int32_t(t % a.page.page_size);
      const uint8_t* codes = a.pages + base + slot * a.page.codes();
      const uint8_t* scales = a.pages + base + a.page.k_scales() + slot * a.page.groups();
      s = 0.0f;
      for (int32_t d = 0; d < D; d += 2) {
        const uint32_t c = codes[d / 2], e = scales[d / kKvGroup];
        s += qs[d] * kv_value(c & 15u, e) + qs[d + 1] * kv_value(c >> 4, e);
      }
      s *= a.scale;
    }
    at[lane] = base;
    float top = s;
    bool nan = s != s;
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (__any(nan)) top = NAN;
    const float m1 = top > m || top != top ? top : m;
    const float keep = m1 == -INFINITY ? 1.0f : expf(m - m1);
    const float p = m1 == -INFINITY ? 0.0f : expf(s - m1);
    float sum = p;
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    l = l * keep + sum;
    m = m1;
    ps[lane] = p;
    __syncthreads();
    const int32_t cnt = int32_t(n - t0 < kWave ? n - t0 : kWave);
    for (int u = 0; u < 4; ++u) {
      const int32_t d = u * kWave + lane;
      if (d >= D) continue;
      float o = acc[u] * keep;
      for (int32_t j = 0; j < cnt; ++j) {
        if (at[j] < 0) continue;
        const int32_t slot = int32_t((t0 + j) % a.page.page_size);
        const uint8_t* block = a.pages + at[j];
        const uint32_t c = block[a.page.v_codes() + slot * a.page.codes() + d / 2];
        o += ps[j] * kv_value(c >> (4 * (d & 1)) & 15u, block[a.page.v_scales() + slot * a.page.groups() + d / kKvGroup]);
      }
      acc[u] = o;
    }
  }
  uint16_t* out = a.out + x * D;
  for (int u = 0; u < 4; ++u) {
    const int32_t d = u * kWave + lane;
    if (d < D) out[d] = float_elem16<DT>(l == 0.0f ? 0.0f : acc[u] / l);
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
  (void)rows, (void)tokens, (void)heads, (void)kv_heads, (void)head_dim, (void)longest;
  return 0;
}

extern "C" int bpd_kv_attend(const uint8_t* pages, int64_t num_pages, int32_t page_size, int32_t kv_heads,
                             int32_t head_dim, int dtype, const void* q, int64_t q_row, int64_t q_token,
                             int64_t q_head, int32_t heads, void* out, int64_t rows, int32_t tokens,
                             const int32_t* block_table, int64_t table_ld, int32_t table_blocks,
                             const int32_t* lengths, const int32_t* query_lens, float scale, void* workspace,
                             size_t workspace_bytes, int32_t* err, void* stream) {
  BPD_ATTEND_ARGS;
  (void)workspace, (void)workspace_bytes;
  if (int rc = check_attend(a, dtype)) return rc;
  if (rows == 0 || tokens == 0) return BPD_OK;
  const uint32_t blocks = uint32_t(rows * tokens * heads);
  if (dtype == BPD_DTYPE_BF16)
    kv_attend_kernel<BPD_DTYPE_BF16><<<blocks, kWave, 0, as_stream(stream)>>>(a);
  else
    kv_attend_kernel<BPD_DTYPE_F16><<<blocks, kWave, 0, as_stream(stream)>>>(a);
  BPD_LAUNCHED();
  return BPD_OK;
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
