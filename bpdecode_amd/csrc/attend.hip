// Attention of a block of query tokens over the 4-bit paged cache (kv4.hpp),
// and its host form.
//
// Query token i of a block of n sees the request's first length - n + 1 + i
// tokens (the block's own keys are already in the cache), so a single token
// sees all of them; out = softmax(scale q k^T) v over those, zeros where
// there are none.  Query heads share key heads in order: head h reads key
// head h / (heads / kv_heads).
#include "attend.hpp"

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
  const AttendSizes z = attend_sizes(rows, tokens, heads, kv_heads, head_dim, longest, longest);
  return 2 * size_t(attend_runs(z, rows)) * z.piece * sizeof(float);
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
  AttendSizes z = attend_sizes(rows, tokens, heads, kv_heads, head_dim, longest, longest);
  BPD_REQUIRE(workspace_bytes >= bpd_kv_attend_workspace_bytes(rows, tokens, heads, kv_heads, head_dim, longest) &&
                  (workspace || z.plan.blocks == 0),
              "the workspace is smaller than bpd_kv_attend_workspace_bytes");
  z.plan.partials = static_cast<float*>(workspace);
  return with_attend(head_dim, z.nt, [&](auto d, auto nt) {
    return dtype == BPD_DTYPE_BF16 ? launch_attend<BPD_DTYPE_BF16, d(), nt()>(a, z, NoPrefix{}, as_stream(stream))
                                   : launch_attend<BPD_DTYPE_F16, d(), nt()>(a, z, NoPrefix{}, as_stream(stream));
  });
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
