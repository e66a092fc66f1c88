// Attention over the 4-bit paged cache (kv4.hpp) of a batch that shares a
// prefix, and its host form.
//
// The first tokens of every request lie in the same pages.  Queries of all
// requests are columns of one product with them: a softmax's numerator and
// denominator are sums over keys, so those of the prefix and of a request's
// own tokens are formed apart, each relative to its own maximum m, and joined
// as sum_i exp(m_i - max m) (numerator_i, denominator_i).
#include "attend.hpp"

namespace bpd {
namespace {

// The prefix's whole tiles for all requests.  A block takes one key head, a
// chunk of the tiles and W * NT * 16 columns (request, query, head that shares
// the key head), a wave NT tiles of 16 columns.  The codes of a tile are
// converted once for the block, a fourth by each of four waves, into operands
// as the products' lanes take them (attend.hpp's order, which keeps the weights
// in their lane), and read from LDS by all; the next W / 4 tiles are converted
// while as many are multiplied.  Every column sees every token: a request with
// a query that does not is left to kv_attend_kernel, and what its columns come
// to here is not read.
//
// Scores, maximum, sums and accumulated values are floats; weights are rounded
// to the cache's type, half a step, as kv_attend_kernel's are and for the same
// reason (attend.hpp states what other choices cost).  Their sum is of the rounded
// weights, so numerator and denominator err alike.  With bfloat16 outputs are off
// by 0.00176 and 0.00177 of themselves (6 requests behind 1,000 tokens, 128 behind
// 32,768), in float16 by 0.000217 (48 of four drafts), where rounding exact
// results alone makes 0.00166 and 0.000204.
//
// What bounds it: dependent steps.  Products take 70,000 of a SIMD's 217,000
// cycles, vector instructions (conversions, the exponentials and roundings of
// weights) about as many, and the two waves of a SIMD cover the waits between
// them in part.  128 requests of 32 heads, 8 key heads of 128, behind 32,768
// tokens: 69 GFLOP in 90 us, 760 of the 1,197 TFLOP/s that a large product
// reaches.  (The whole call takes 114 us where kv_attend_kernel over whole tables,
// which name the same pages, takes 560.)  A block's
// conversions shared by eight waves instead of four took it from 99 us to 90;
// scores formed a tile ahead of their exponentials, for 248 registers, from 99
// to 110; loads that go around the registers do not fit codes that have to be
// converted.
template <int DT, int D, int NT, int W>
__global__ __launch_bounds__(W* kWave, D <= 128 ? 2 : 1) void kv_prefix_kernel(AttendArgs a, Prefix px, uint32_t groups) {
  using Pt = Parts<D>;
  constexpr int G = D / kKvGroup, KW = D / 32, VT = D / 16, kStep = W / 4;
  __shared__ Frag keys[2][kStep][4 * KW][kWave], values[2][kStep][2 * VT][kWave];
  __shared__ int32_t pages_there[2][kStep][4];
  const int lane = threadIdx.x % kWave, number = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wave = number % 4, part = number / 4;  // its share of a tile, and which tile of a step
  const int m = lane & 15, g = lane >> 4;
  const uint32_t group = blockIdx.x % groups, kvh = blockIdx.x / groups % uint32_t(a.kv_heads);
  const int32_t chunk = int32_t(blockIdx.x / groups / uint32_t(a.kv_heads));
  bool past;
  const Spans sp = px.spans(a.page.page_size, &past);
  if (past && a.err && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(a.err, BPD_FLAG_PAGE_RANGE);
  const int32_t tiles = sp.whole / kTile, per = (tiles + px.chunks - 1) / px.chunks;
  const int32_t tile0 = chunk * per, tile1 = tile0 + per < tiles ? tile0 + per : tiles;

  const int32_t share = a.heads / a.kv_heads, per_request = a.tokens * share;
  const int64_t first = (int64_t(group) * W + number) * (NT * 16);  // of the wave's columns
  const int64_t at = (int64_t(chunk) * a.kv_heads + kvh) * px.columns;
  const float to_log2 = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.44269504088896340736f;
  Frag q[NT][KW];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t c = first + t * 16 + m;
    const bool there = c < px.columns;
    const int32_t b = there ? int32_t(uint32_t(c) / uint32_t(per_request)) : 0;
    const int32_t r = there ? int32_t(c) - b * per_request : 0, i = r / share, h = int32_t(kvh) * share + r % share;
    const bool in = there && i < queries_of(a, b);
    const uint16_t* row = a.q + int64_t(b) * a.q_row + (in ? i : 0) * a.q_token + h * a.q_head;
#pragma unroll
    for (int p = 0; p < Pt::count; ++p)
#pragma unroll
      for (int k = 0; k < Pt::width(p) / 32; ++k) {
        Frag f = {{0u, 0u, 0u, 0u}};
        if (in && a.scale != 0.0f) __builtin_memcpy(&f, row + Pt::begin(p) + g * (Pt::width(p) / 4) + 8 * k, 16);
        if (a.scale < 0.0f)
#pragma unroll
          for (int j = 0; j < 4; ++j) f.u[j] ^= 0x80008000u;
        q[t][Pt::begin(p) / 32 + k] = f;
      }
  }
  // The sums of weights are a product with ones, of the rounded weights that the
  // values are weighted by: four products of 16 cycles for 32 additions.
  constexpr uint32_t kOnes = DT == BPD_DTYPE_BF16 ? 0x3F803F80u : 0x3C003C00u;
  const Frag ones = {{kOnes, kOnes, kOnes, kOnes}};
  f32x4 acc[NT][VT], sum[NT];  // (rows of sum are equal)
  float top[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    top[t] = -3e38f, sum[t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < VT; ++v) acc[t][v] = f32x4{0, 0, 0, 0};
  }

  uint32_t vsel[Pt::count];
#pragma unroll
  for (int p = 0; p < Pt::count; ++p) vsel[p] = uint32_t(m * Pt::width(p) / 512) << 24 | 0x0C0C0C;
  const int32_t P = a.page.page_size;
  const int shift = __builtin_ctz(P);
  // a wave's share of a tile: keys of tokens 4 m + wave, values of tokens 16 g + 4 wave + 0..3
  uint32_t kc[KW], ks[Pt::count], vc[4][Pt::count], vs[G];
  int32_t kpage = -1, vpage = -1;  // of the tile to be loaded next
  // (a wave whose tile lies past the last converts that once more, for nobody)
  const auto first_of = [&](int32_t tile) { return (tile + part < tile1 ? tile + part : tile1 - 1) * kTile; };
  const auto load_pages = [&](int32_t tile) {
    const int32_t t0 = first_of(tile);
    kpage = px.table[(t0 + (m >> 2) * 16) >> shift];
    vpage = px.table[(t0 + g * 16) >> shift];
  };
  const auto is_page = [&](int32_t page) { return page >= 0 && page < a.table.num_pages; };
  const auto block_at = [&](int32_t page) -> const uint8_t* {
    return a.pages + (int64_t(is_page(page) ? page : 0) * a.kv_heads + kvh) * int64_t(a.page.bytes());
  };
  const auto load = [&](int32_t tile) {
    const int32_t t0 = first_of(tile);
    const uint8_t* block = block_at(kpage);
    int32_t slot = ((t0 + 4 * m) & (P - 1)) + wave;
#pragma unroll
    for (int p = 0; p < Pt::count; ++p) {
      const uint32_t* from =
          reinterpret_cast<const uint32_t*>(block + slot * (D / 2) + Pt::begin(p) / 2 + g * (Pt::width(p) / 8));
#pragma unroll
      for (int k = 0; k < Pt::width(p) / 32; ++k) kc[Pt::begin(p) / 32 + k] = from[k];
      ks[p] = block[a.page.k_scales() + slot * G + Pt::begin(p) / kKvGroup + g * Pt::width(p) / 128];
    }
    block = block_at(vpage);
    slot = ((t0 + 16 * g) & (P - 1)) + 4 * wave;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int p = 0; p < Pt::count; ++p) {
        const uint8_t* from = block + a.page.v_codes() + (slot + u) * (D / 2) + Pt::begin(p) / 2 + m * (Pt::width(p) / 32);
        if (Pt::width(p) == 128) vc[u][p] = *reinterpret_cast<const uint32_t*>(from);
        if (Pt::width(p) == 64) vc[u][p] = *reinterpret_cast<const uint16_t*>(from);
        if (Pt::width(p) == 32) vc[u][p] = *from;
      }
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(block + a.page.v_scales() + slot * G);
#pragma unroll
    for (int k = 0; k < G; ++k) vs[k] = scales[k];
  };
  const auto convert = [&](int to, bool there) {
#pragma unroll
    for (int p = 0; p < Pt::count; ++p) {
      const float sc = bits_float(ks[p] << 23);
#pragma unroll
      for (int k = 0; k < Pt::width(p) / 32; ++k) {
        const uint32_t w = kc[Pt::begin(p) / 32 + k];
        keys[to][part][wave * KW + Pt::begin(p) / 32 + k][lane] =
            Frag{{two_values<DT, 0>(w, sc), two_values<DT, 1>(w, sc), two_values<DT, 2>(w, sc), two_values<DT, 3>(w, sc)}};
      }
    }
    if (wave == 0 && m == 0) pages_there[to][part][g] = there;
    if (!there) {  // no page: zeros, at a scale of one
#pragma unroll
      for (int k = 0; k < G; ++k) vs[k] = 0x7F7F7F7Fu;
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int p = 0; p < Pt::count; ++p) vc[u][p] = 0;
    }
#pragma unroll
    for (int p = 0; p < Pt::count; ++p) {
      uint32_t x[8][2];  // of each value tile, the tokens' two pairs
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float s0 = scale_at(vs, G * (2 * k) + Pt::begin(p) / kKvGroup, G, vsel[p]);
        const float s1 = scale_at(vs, G * (2 * k + 1) + Pt::begin(p) / kKvGroup, G, vsel[p]);
        const auto pair = [&](auto byte) {
          constexpr int B = decltype(byte)::value;
          const uint32_t x0 = two_values<DT, B>(vc[2 * k][p], s0), x1 = two_values<DT, B>(vc[2 * k + 1][p], s1);
          x[2 * B][k] = __builtin_amdgcn_perm(x1, x0, 0x05040100);
          x[2 * B + 1][k] = __builtin_amdgcn_perm(x1, x0, 0x07060302);
        };
        pair(std::integral_constant<int, 0>());
        if (Pt::width(p) >= 64) pair(std::integral_constant<int, 1>());
        if (Pt::width(p) >= 128) pair(std::integral_constant<int, 2>()), pair(std::integral_constant<int, 3>());
      }
#pragma unroll
      for (int v = 0; v < Pt::width(p) / 16; ++v)
        *reinterpret_cast<uint2*>(&values[to][part][(wave >> 1) * VT + Pt::begin(p) / 16 + v][lane].u[2 * (wave & 1)]) =
            uint2{x[v][0], x[v][1]};
    }
  };

  bool there_next = false;  // this lane's 16 tokens of the tile loaded
  if (tile0 < tile1) {
    load_pages(tile0);
    load(tile0);
    const bool there = is_page(vpage);
    if (tile0 + kStep < tile1) load_pages(tile0 + kStep);
    convert(0, there);
    if (tile0 + kStep < tile1) {
      load(tile0 + kStep);
      there_next = is_page(vpage);
      if (tile0 + 2 * kStep < tile1) load_pages(tile0 + 2 * kStep);
    }
  }
  int now_at = 0;
  bool missing = false;
  for (int32_t tile = tile0; tile < tile1; tile += kStep, now_at ^= 1) {
    __syncthreads();  // these tiles are converted, and the other buffer has been read
    if (tile + kStep < tile1) {
      convert(now_at ^ 1, there_next);
      if (tile + 2 * kStep < tile1) {
        load(tile + 2 * kStep);
        there_next = is_page(vpage);
        if (tile + 3 * kStep < tile1) load_pages(tile + 3 * kStep);
      }
    }
    if (first >= px.columns) continue;
#pragma unroll 1
    for (int e = 0; e < kStep && tile + e < tile1; ++e) {
      const bool here_valid = pages_there[now_at][e][g] != 0;
      f32x4 s[NT][4];
#pragma unroll
      for (int k = 0; k < KW; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const Frag f = keys[now_at][e][j * KW + k][lane];
#pragma unroll
          for (int t = 0; t < NT; ++t) s[t][j] = mfma<DT>(f, q[t][k], k == 0 ? f32x4{0, 0, 0, 0} : s[t][j]);
        }
      if (__any(!here_valid)) {
        missing = true;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][j][i] = here_valid ? s[t][j][i] : -INFINITY;
      }
      Frag w[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float most = s[t][0][0];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) most = fmaxf(most, s[t][j][i]);
        most *= to_log2;
        // the running maximum is followed loosely, as in kv_attend_kernel
        if (__any(most > top[t] + (kLift<DT> + 8.0f))) {
          float now = fmaxf(top[t], most - kLift<DT>);
          now = fmaxf(now, __shfl_xor(now, 16));
          now = fmaxf(now, __shfl_xor(now, 32));
          const float keep = __builtin_amdgcn_exp2f(top[t] - now);
          top[t] = now;
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[t][i] *= keep;
#pragma unroll
          for (int v = 0; v < VT; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][v][i] *= keep;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[t][j][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][j][i], to_log2, -top[t]));
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[t][h].u[k] = two_rounded<DT>(s[t][2 * (k & 1)][2 * h + (k >> 1)], s[t][2 * (k & 1) + 1][2 * h + (k >> 1)]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t) sum[t] = mfma<DT>(ones, w[t][h], sum[t]);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int v = 0; v < VT; ++v) {
          const Frag f = values[now_at][e][h * VT + v][lane];
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[t][v] = mfma<DT>(f, w[t][h], acc[t][v]);
        }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t c = first + t * 16 + m;
    if (c >= px.columns) continue;
    if (missing && a.err) {
      // noted where some query sees it: requests whose queries do not all see the
      // prefix are looked after by kv_attend_kernel
      const int64_t b = c / per_request;
      if (int32_t(c - b * per_request) / share < queries_of(a, b) && begin_of(a, sp, b) > 0)
        atomicOr(a.err, BPD_FLAG_PAGE_RANGE);
    }
    if (g == 0) px.stats[at + c] = float2{top[t], sum[t][0]};
    if (tile0 >= tile1) continue;
    f32x4* to = reinterpret_cast<f32x4*>(px.values + (at + c) * D) + g * VT;
#pragma unroll
    for (int v = 0; v < VT; ++v) to[v] = acc[t][v];
  }
}

struct SharedSizes {
  AttendSizes own;
  int32_t nt, waves, chunks;
  int64_t columns, groups;
  size_t partials, stats, bytes;
};

// How many blocks of four waves the device is to have: two a CU, which is what
// their registers and LDS allow (128 requests behind 32,768 tokens: 99 us, with
// 256 blocks 128, with 1,024 108; 12 requests: 15.3, 17.7, 15.3).
constexpr int kPrefixBlocks = 512;

// Wide blocks share what they convert, and narrow ones are more: the widest
// that still come to a block for each place with chunks of four tiles.  (us of
// narrow, 128 columns, 256 columns: 128 requests behind 32,768 tokens 128, 99,
// 90; 48 of four drafts, heads of 64, behind 4,096 15.3, 17.0, 15.0; 40 behind
// 2,048 13.5, 16.5, 15.7; 6 behind 1,000, which fill one narrow block, 9.1, 11.6.)
// Heads past 128 have no LDS for the widest.  A chunk has four tiles, as what it
// leaves is written and read once more, but where that makes fewer than eight
// chunks, two for each wave that joins them.  (6 requests behind 1,000 tokens,
// both kernels: 4 chunks 17.6 us, 8 16.0, 15 15.7; 40 behind 2,048: 8 chunks
// 27.3, 16 30.3, 32 39; with eight tiles a chunk 40 behind 2,048 take 21.2 for
// 16.5 in this kernel, 48 of four drafts 19.0 for 17.3.)

SharedSizes shared_sizes(int64_t rows, int32_t tokens, int32_t heads, int32_t kv_heads, int32_t dim, int64_t longest,
                         int64_t prefix) {
  SharedSizes z{};
  z.own = attend_sizes(rows, tokens, heads, kv_heads, dim, longest, longest > prefix ? longest - prefix : longest);
  z.columns = rows * tokens * (heads / kv_heads);
  const int64_t tiles = std::min<int64_t>(prefix, 0x7FFFFFFF) / kTile;
  const auto groups = [&](int64_t of) { return (z.columns + of - 1) / of; };
  const auto fills = [&](int64_t of) { return groups(of) * kv_heads * ((tiles + 3) / 4) * (of / 64) >= 2 * kPrefixBlocks; };
  z.waves = dim <= 128 && z.columns > 128 && fills(256) ? 8 : 4;
  z.nt = z.waves == 8 || (z.columns > 64 && fills(128)) ? 2 : 1;
  z.groups = groups(z.waves * 16 * z.nt);
  const int64_t room = kPrefixBlocks * 4 / z.waves / (z.groups * kv_heads);
  z.chunks = int32_t(std::max<int64_t>(1, std::min<int64_t>(room, std::max<int64_t>((tiles + 3) / 4, std::min<int64_t>(tiles, 8)))));
  z.partials = (2 * size_t(attend_runs(z.own, rows)) * z.own.piece * sizeof(float) + 15) / 16 * 16;
  const size_t all = size_t(z.chunks) * kv_heads * size_t(z.columns);
  z.stats = (all * sizeof(float2) + 15) / 16 * 16;
  z.bytes = z.partials + z.stats + all * dim * sizeof(float);
  return z;
}

template <int DT, int D>
int launch_prefix(const AttendArgs& a, const SharedSizes& z, const Prefix& px, hipStream_t s) {
  const int64_t blocks = z.groups * a.kv_heads * z.chunks;
  BPD_REQUIRE(blocks < (int64_t(1) << 31), "too many queries in one call");
  if constexpr (D <= 128)
    if (z.waves == 8) {
      kv_prefix_kernel<DT, D, 2, 8><<<uint32_t(blocks), 8 * kWave, 0, s>>>(a, px, uint32_t(z.groups));
      BPD_LAUNCHED();
      return BPD_OK;
    }
  if (z.nt == 1)
    kv_prefix_kernel<DT, D, 1, 4><<<uint32_t(blocks), 4 * kWave, 0, s>>>(a, px, uint32_t(z.groups));
  else
    kv_prefix_kernel<DT, D, 2, 4><<<uint32_t(blocks), 4 * kWave, 0, s>>>(a, px, uint32_t(z.groups));
  BPD_LAUNCHED();
  return BPD_OK;
}

int check_shared(const AttendArgs& a, const Prefix& px, int dtype) {
  if (int rc = check_attend(a, dtype)) return rc;
  BPD_REQUIRE(px.blocks >= 0 && (px.table || px.blocks == 0), "null prefix table");
  BPD_REQUIRE(px.shared || (px.shared_all >= 0 && px.shared_all <= int64_t(px.blocks) * a.page.page_size),
              "%d shared tokens in a prefix of %d pages of %d", px.shared_all, px.blocks, a.page.page_size);
  BPD_REQUIRE(int64_t(px.blocks) * a.page.page_size < (int64_t(1) << 31), "too long a prefix");
  return BPD_OK;
}

}  // namespace
}  // namespace bpd

using namespace bpd;

#define BPD_SHARED_ARGS                                                                                    \
  AttendArgs a {                                                                                           \
    pages, KvPage{page_size, head_dim}, KvTable{block_table, table_ld, table_blocks, num_pages}, kv_heads, \
        heads, static_cast<const uint16_t*>(q), q_row, q_token, q_head, static_cast<uint16_t*>(out), rows, \
        tokens, lengths, query_lens, scale, err                                                            \
  };                                                                                                       \
  Prefix px { prefix_table, prefix_blocks, shared, shared_all, 0, 0, nullptr, nullptr }

extern "C" size_t bpd_kv_attend_shared_workspace_bytes(int64_t rows, int32_t tokens, int32_t heads, int32_t kv_heads,
                                                       int32_t head_dim, int64_t longest, int64_t prefix) {
  if (rows <= 0 || tokens <= 0 || kv_heads <= 0 || heads < kv_heads || head_dim <= 0) return 0;
  return shared_sizes(rows, tokens, heads, kv_heads, head_dim, longest, prefix).bytes;
}

extern "C" int bpd_kv_attend_shared(const uint8_t* pages, int64_t num_pages, int32_t page_size, int32_t kv_heads,
                                    int32_t head_dim, int dtype, const void* q, int64_t q_row, int64_t q_token,
                                    int64_t q_head, int32_t heads, void* out, int64_t rows, int32_t tokens,
                                    const int32_t* prefix_table, int32_t prefix_blocks, const int32_t* shared,
                                    int32_t shared_all, const int32_t* block_table, int64_t table_ld,
                                    int32_t table_blocks, const int32_t* lengths, const int32_t* query_lens,
                                    float scale, void* workspace, size_t workspace_bytes, int32_t* err, void* stream) {
  BPD_SHARED_ARGS;
  if (int rc = check_shared(a, px, dtype)) return rc;
  if (rows == 0 || tokens == 0) return BPD_OK;
  const int64_t longest = int64_t(table_blocks) * page_size;
  if (num_pages == 0) a.table.blocks = px.blocks = 0;  // no page to read: every length lies past the table
  SharedSizes z = shared_sizes(rows, tokens, heads, kv_heads, head_dim, longest, int64_t(prefix_blocks) * page_size);
  BPD_REQUIRE(workspace && workspace_bytes >= z.bytes && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0,
              "the workspace is smaller than bpd_kv_attend_shared_workspace_bytes, or not at a multiple of 16 bytes");
  char* at = static_cast<char*>(workspace);
  z.own.plan.partials = reinterpret_cast<float*>(at);
  px.chunks = z.chunks, px.columns = z.columns;
  px.stats = reinterpret_cast<float2*>(at + z.partials);
  px.values = reinterpret_cast<float*>(at + z.partials + z.stats);
  return with_attend(head_dim, z.own.nt, [&](auto d, auto nt) {
    const auto launch = [&](auto dt) {
      if (int rc = launch_prefix<dt(), d()>(a, z, px, as_stream(stream))) return rc;
      return launch_attend<dt(), d(), nt()>(a, z.own, px, as_stream(stream));
    };
    return dtype == BPD_DTYPE_BF16 ? launch(std::integral_constant<int, BPD_DTYPE_BF16>())
                                   : launch(std::integral_constant<int, BPD_DTYPE_F16>());
  });
}

extern "C" int bpd_host_kv_attend_shared(const uint8_t* pages, int64_t num_pages, int32_t page_size, int32_t kv_heads,
                                         int32_t head_dim, int dtype, const void* q, int64_t q_row, int64_t q_token,
                                         int64_t q_head, int32_t heads, void* out, int64_t rows, int32_t tokens,
                                         const int32_t* prefix_table, int32_t prefix_blocks, const int32_t* shared,
                                         int32_t shared_all, const int32_t* block_table, int64_t table_ld,
                                         int32_t table_blocks, const int32_t* lengths, const int32_t* query_lens,
                                         float scale, int32_t* err) {
  BPD_SHARED_ARGS;
  if (int rc = check_shared(a, px, dtype)) return rc;
  if (rows == 0 || tokens == 0) return BPD_OK;
  bool past;
  const Spans sp = px.spans(page_size, &past);
  if (past && err) *err |= BPD_FLAG_PAGE_RANGE;
  if (dtype == BPD_DTYPE_BF16)
    host_attend<BPD_DTYPE_BF16>(a, prefix_table, sp.paged);
  else
    host_attend<BPD_DTYPE_F16>(a, prefix_table, sp.paged);
  return BPD_OK;
}
