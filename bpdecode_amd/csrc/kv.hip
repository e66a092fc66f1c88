// The 4-bit paged cache (kv4.hpp): rotating a block's keys and queries to
// their positions and appending keys and values, reading tokens back, and
// the host forms of both.
#include <algorithm>

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
};

// Whether token i of request b is appended, and where; sets *bad where it
// should be and cannot.  *turn: its row of the rotation's tables, or -1.
__host__ __device__ __forceinline__ int64_t append_place(const AppendArgs& a, int64_t b, int32_t i, int64_t* pos,
                                                         int64_t* turn, bool* bad) {
  *bad = false;
  *turn = -1;
  if (a.counts && i >= a.counts[b]) return -1;
  *pos = int64_t(a.starts[b]) + i;
  if (*pos < 0 || (a.rotary > 0 && *pos >= a.positions)) {
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

// A thread takes 8 channels of one head of one token: the query heads first
// (where there are queries), then the key heads, then the value heads.
template <int DT>
__global__ __launch_bounds__(kKvThreads) void kv_append_kernel(AppendArgs a) {
  const int32_t per_head = a.page.dim / kKvWidth;
  const int32_t slots = (a.heads + 2 * a.kv_heads) * per_head;
  const int64_t at = int64_t(blockIdx.x) * kKvThreads + threadIdx.x;
  const int64_t token = at / slots;
  if (token >= a.rows * a.tokens) return;
  const int32_t slot = int32_t(at - token * slots);
  const int64_t b = token / a.tokens;
  const int32_t i = int32_t(token - b * a.tokens);
  const int32_t head = slot / per_head, d0 = (slot - head * per_head) * kKvWidth;
  int64_t pos, turn;
  bool bad;
  const int64_t page = append_place(a, b, i, &pos, &turn, &bad);
  if (bad && a.err && slot == 0) atomicOr(a.err, BPD_FLAG_PAGE_RANGE);
  const bool is_q = head < a.heads, is_v = head >= a.heads + a.kv_heads;
  const int32_t h = is_q ? head : is_v ? head - a.heads - a.kv_heads : head - a.heads;
  const Strides3& s = is_q ? a.qs : is_v ? a.vs : a.ks;
  const uint16_t* x = (is_q ? a.q : is_v ? a.v : a.k) + b * s.row + i * s.token + h * s.head;
  float val[kKvWidth];
  const bool read = is_q ? turn >= 0 : page >= 0;
#pragma unroll
  for (int j = 0; j < kKvWidth; ++j) {
    val[j] = 0.0f;
    if (read)
      val[j] = rotated_channel<DT>(x, d0 + j, is_v ? 0 : a.rotary, a.interleaved, a.cos + turn * (a.rotary / 2),
                                   a.sin + turn * (a.rotary / 2));
  }
  if (is_q) {
    uint16_t* out = a.q_out + (token * a.heads + h) * a.page.dim + d0;
#pragma unroll
    for (int j = 0; j < kKvWidth; ++j) out[j] = float_elem16<DT>(val[j]);
  }
  // the four threads of a group are neighbours in a wave and take one branch
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < kKvWidth; ++j) most = max(most, float_bits(val[j]) & 0x7FFFFFFFu);
  most = max(most, uint32_t(__shfl_xor(int(most), 1)));
  most = max(most, uint32_t(__shfl_xor(int(most), 2)));
  if (is_q || page < 0) return;
  const int32_t e = kv_scale_byte<DT>(most);
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < kKvWidth; ++j) word |= kv_code(val[j], e) << (4 * j);
  uint8_t* block = a.pages + (page * a.kv_heads + h) * int64_t(a.page.bytes());
  const int32_t t = int32_t(pos % a.page.page_size);
  *reinterpret_cast<uint32_t*>(block + (is_v ? a.page.v_codes() : 0) + t * a.page.codes() + d0 / 2) = word;
  if ((d0 & (kKvGroup - 1)) == 0)
    block[(is_v ? a.page.v_scales() : a.page.k_scales()) + t * a.page.groups() + d0 / kKvGroup] = uint8_t(e);
}

template <int DT>
void host_append(const AppendArgs& a) {
  const int32_t D = a.page.dim;
  for (int64_t b = 0; b < a.rows; ++b)
    for (int32_t i = 0; i < a.tokens; ++i) {
      int64_t pos, turn;
      bool bad;
      const int64_t page = append_place(a, b, i, &pos, &turn, &bad);
      if (bad && a.err) *a.err |= BPD_FLAG_PAGE_RANGE;
      const float *cos = a.cos + std::max<int64_t>(turn, 0) * (a.rotary / 2),
                  *sin = a.sin + std::max<int64_t>(turn, 0) * (a.rotary / 2);
      for (int32_t h = 0; h < a.heads; ++h) {
        const uint16_t* x = a.q + b * a.qs.row + i * a.qs.token + h * a.qs.head;
        uint16_t* out = a.q_out + ((b * a.tokens + i) * a.heads + h) * D;
        for (int32_t d = 0; d < D; ++d)
          out[d] = turn >= 0 ? float_elem16<DT>(rotated_channel<DT>(x, d, a.rotary, a.interleaved, cos, sin)) : 0;
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
            val[j] = rotated_channel<DT>(x, g * kKvGroup + j, is_v ? 0 : a.rotary, a.interleaved, cos, sin);
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

// A thread takes 8 channels of one head of one token, keys before values.
template <int DT>
__global__ __launch_bounds__(kKvThreads) void kv_read_kernel(ReadArgs a) {
  const int32_t per_head = a.page.dim / kKvWidth;
  const int32_t slots = 2 * a.kv_heads * per_head;
  const int64_t at = int64_t(blockIdx.x) * kKvThreads + threadIdx.x;
  const int64_t token = at / slots;
  if (token >= a.rows * a.tokens) return;
  const int32_t slot = int32_t(at - token * slots);
  const int64_t b = token / a.tokens;
  int64_t pos;
  bool bad;
  const int64_t page = read_place(a, b, int32_t(token - b * a.tokens), &pos, &bad);
  if (bad && a.err && slot == 0) atomicOr(a.err, BPD_FLAG_PAGE_RANGE);
  const int32_t head = slot / per_head, d0 = (slot - head * per_head) * kKvWidth;
  const bool is_v = head >= a.kv_heads;
  const int32_t h = is_v ? head - a.kv_heads : head;
  uint32_t word = 0, e = 127;
  if (page >= 0) {
    const uint8_t* block = a.pages + (page * a.kv_heads + h) * int64_t(a.page.bytes());
    const int32_t t = int32_t(pos % a.page.page_size);
    word = *reinterpret_cast<const uint32_t*>(block + (is_v ? a.page.v_codes() : 0) + t * a.page.codes() + d0 / 2);
    e = block[(is_v ? a.page.v_scales() : a.page.k_scales()) + t * a.page.groups() + d0 / kKvGroup];
  }
  uint16_t* out = (is_v ? a.v : a.k) + (token * a.kv_heads + h) * a.page.dim + d0;
#pragma unroll
  for (int j = 0; j < kKvWidth; ++j) out[j] = float_elem16<DT>(kv_value(word >> (4 * j) & 15u, e));
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
  BPD_REQUIRE(a.heads >= 0 && (a.heads == 0 || (a.q && a.q_out) || a.rows * a.tokens == 0), "null query pointer");
  BPD_REQUIRE(a.rows * int64_t(a.tokens) == 0 || (a.k && a.v && a.table.block_table && a.starts),
              "null pointer argument");
  return BPD_OK;
}

int check_read(const ReadArgs& a, int dtype) {
  if (int rc = check_kv_cache(a.pages, a.page, a.table, a.kv_heads, dtype)) return rc;
  BPD_REQUIRE(a.rows >= 0 && a.tokens >= 0, "negative sizes");
  BPD_REQUIRE(a.rows * int64_t(a.tokens) == 0 || (a.k && a.v && a.table.block_table && a.starts),
              "null pointer argument");
  return BPD_OK;
}

int grid_of(int64_t threads, uint32_t* blocks) {
  const int64_t n = (threads + kKvThreads - 1) / kKvThreads;
  BPD_REQUIRE(n < (int64_t(1) << 31), "too many tokens in one call");
  *blocks = uint32_t(n);
  return BPD_OK;
}

}  // namespace
}  // namespace bpd

using namespace bpd;

#define BPD_APPEND_ARGS                                                                                            \
  AppendArgs a {                                                                                                   \
    pages, KvPage{page_size, head_dim}, KvTable{block_table, table_ld, table_blocks, num_pages}, kv_heads, heads,  \
        static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), static_cast<const uint16_t*>(q),         \
        {k_row, k_token, k_head}, {v_row, v_token, v_head}, {q_row, q_token, q_head},                              \
        static_cast<uint16_t*>(q_out), rows, tokens, starts, counts, cos, sin, positions, rotary, interleaved, err \
  }

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
  uint32_t blocks = 0;
  if (int rc = grid_of(rows * tokens * int64_t(heads + 2 * kv_heads) * (head_dim / kKvWidth), &blocks)) return rc;
  if (dtype == BPD_DTYPE_BF16)
    kv_append_kernel<BPD_DTYPE_BF16><<<blocks, kKvThreads, 0, as_stream(stream)>>>(a);
  else
    kv_append_kernel<BPD_DTYPE_F16><<<blocks, kKvThreads, 0, as_stream(stream)>>>(a);
  BPD_LAUNCHED();
  return BPD_OK;
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
  uint32_t blocks = 0;
  if (int rc = grid_of(rows * tokens * int64_t(2 * kv_heads) * (head_dim / kKvWidth), &blocks)) return rc;
  if (dtype == BPD_DTYPE_BF16)
    kv_read_kernel<BPD_DTYPE_BF16><<<blocks, kKvThreads, 0, as_stream(stream)>>>(a);
  else
    kv_read_kernel<BPD_DTYPE_F16><<<blocks, kKvThreads, 0, as_stream(stream)>>>(a);
  BPD_LAUNCHED();
  return BPD_OK;
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
