// Attention over a paged cache that holds 8-bit values, or under a sliding window with first tokens that stay visible
// (sinks), or both.  Formulas: query i of a sequence with Lq new tokens and Lk keys stands at position P = Lk - Lq + i;
//
//   key j is visible  iff  j <= P + right  and  (j >= P - left  or  j < sinks)
//   t = scale * s_k[b, h] * (q . c_j)   or   cap * tanh(that / cap)
//   out = s_v[b, h] * sum_j softmax(t)_j * c'_j        lse = log sum_j exp(t_j)
//
// c, c' are the cached K and V values as they stand, s the scales they were written with (1 for a 16-bit cache).
#include <limits.h>
#include "fg_common.h"

namespace {

#include "attn_cache.h"
#include "attn_stream.h"
#include "attn_tile.h"

template <typename T, int FMT, int DP>
int stream_rows(const CacheAttnArgs& a, int nq, bool narrow, hipStream_t st) {
  if (narrow) return launch_stream<T, FMT, DP, 1, true>(a, st);
  if constexpr (DP < 256) {
    if (nq == 2) return launch_stream<T, FMT, DP, 2, false>(a, st);
  }
  return launch_stream<T, FMT, DP, 1, false>(a, st);
}
template <typename T, int FMT>
int stream_dims(const CacheAttnArgs& a, int nq, bool narrow, hipStream_t st) {
  const int D = a.p.base.D;
  if (D <= 64) return stream_rows<T, FMT, 64>(a, nq, narrow, st);
  if (D <= 128) return stream_rows<T, FMT, 128>(a, nq, narrow, st);
  return stream_rows<T, FMT, 256>(a, nq, narrow, st);
}
template <typename T>
int stream_formats(const CacheAttnArgs& a, int nq, bool narrow, hipStream_t st) {
  if (a.p.cache_format == FG_CACHE_E4M3) return stream_dims<T, FG_CACHE_E4M3>(a, nq, narrow, st);
  if (a.p.cache_format == FG_CACHE_E5M2) return stream_dims<T, FG_CACHE_E5M2>(a, nq, narrow, st);
  return stream_dims<T, FG_CACHE_SAME>(a, nq, narrow, st);
}

template <typename T>
int tile_formats(const CacheAttnArgs& a, hipStream_t st) {
  const bool small = a.p.base.D <= 64;
  if (a.p.cache_format == FG_CACHE_E4M3) return small ? launch_tile<T, FG_CACHE_E4M3, 64>(a, st) : launch_tile<T, FG_CACHE_E4M3, 128>(a, st);
  if (a.p.cache_format == FG_CACHE_E5M2) return small ? launch_tile<T, FG_CACHE_E5M2, 64>(a, st) : launch_tile<T, FG_CACHE_E5M2, 128>(a, st);
  return small ? launch_tile<T, FG_CACHE_SAME, 64>(a, st) : launch_tile<T, FG_CACHE_SAME, 128>(a, st);
}

int num_cu() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 0;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
  return n;
}

struct Plan {
  int stream_q;     // sequences with up to so many new tokens take the stream kernel (0: none)
  bool tile;        // the others take the tile kernel
  int nq;           // stream kernel: 16-row tiles of a row block
  bool narrow;      // stream kernel: pages of a size that is not a multiple of 8
  int splits;       // stream kernel: key ranges
  size_t workspace;
};

int padded_dim(int D) { return D <= 64 ? 64 : (D <= 128 ? 128 : 256); }

// Which kernels run, and how the rows and the keys are cut.
Plan make_plan(const FgCacheAttnParams& c) {
  const FgFlashParams& p = c.base;
  const int G = p.Hq / p.Hk;
  Plan plan;
  const int few = 32 / G > 1 ? 32 / G : 1;
  plan.tile = p.D <= 128 && p.max_seqlen_q > few;
  plan.stream_q = plan.tile ? few : p.max_seqlen_q;
  // every sequence as long as the longest: the stream kernel has none to take
  if (plan.tile && (int64_t)p.total_q >= (int64_t)p.batch * p.max_seqlen_q) plan.stream_q = 0;
  plan.narrow = p.page_size % 8 != 0;
  plan.nq = !plan.narrow && p.D <= 128 && (int64_t)plan.stream_q * G > 16 ? 2 : 1;
  // the most keys that one row block may see
  int64_t keys = p.max_seqlen_k > 0 ? p.max_seqlen_k : 1;
  if (p.window_left >= 0) {
    const int64_t window = (int64_t)p.window_left + plan.stream_q + c.num_sink_tokens + 2 * kTile;
    keys = window < keys ? window : keys;
  }
  const int64_t tiles = fg_cdiv(keys, kTile);
  const int64_t row_blocks = fg_cdiv((int64_t)plan.stream_q * G, 16 * plan.nq);
  const int64_t groups = (row_blocks > 0 ? row_blocks : 1) * p.batch * p.Hk;
  int64_t splits = fg_cdiv(2 * (int64_t)num_cu(), groups);
  const int64_t most = tiles / 16 > 1 ? tiles / 16 : 1;
  if (splits > most) splits = most;
  plan.splits = (int)splits;
  plan.workspace = splits > 1 ? (size_t)splits * p.batch * plan.stream_q * p.Hq * (padded_dim(p.D) + 2) * sizeof(float) : 0;
  return plan;
}

int check_params(const FgCacheAttnParams* c) {
  FG_REQUIRE(c != nullptr, FG_ERR_INVALID, "cache_attn_fwd: null params");
  const FgFlashParams& p = c->base;
  FG_REQUIRE(p.dtype == FG_F16 || p.dtype == FG_BF16, FG_ERR_INVALID, "cache_attn_fwd: only fp16 and bf16 queries are supported (dtype %d)", p.dtype);
  FG_REQUIRE(c->cache_format == FG_CACHE_SAME || c->cache_format == FG_CACHE_E4M3 || c->cache_format == FG_CACHE_E5M2, FG_ERR_INVALID,
             "cache_attn_fwd: cache format %d", c->cache_format);
  FG_REQUIRE(p.batch >= 0 && p.total_q >= 0 && c->num_sink_tokens >= 0 && c->table_width >= 0, FG_ERR_INVALID, "cache_attn_fwd: negative size");
  if (p.batch == 0 || p.total_q == 0) return FG_OK;
  FG_REQUIRE(p.q && p.k_cache && p.v_cache && p.out && p.cu_seqlens_q && p.seqused_k && p.block_table, FG_ERR_INVALID,
             "cache_attn_fwd: null pointer (q, k, v, out, cu_seqlens_q, seqused_k and block_table are required)");
  const bool narrow8 = c->cache_format != FG_CACHE_SAME;
  FG_REQUIRE(p.D > 0 && p.D <= 256 && p.D % (narrow8 ? 16 : 8) == 0, FG_ERR_INVALID,
             "cache_attn_fwd: head dim %d must be a multiple of %d and at most 256", p.D, narrow8 ? 16 : 8);
  FG_REQUIRE(p.Hq > 0 && p.Hk > 0 && p.Hq % p.Hk == 0, FG_ERR_INVALID,
             "cache_attn_fwd: %d query heads are not a multiple of %d kv heads", p.Hq, p.Hk);
  FG_REQUIRE(p.page_size > 0 && p.max_seqlen_q > 0, FG_ERR_INVALID, "cache_attn_fwd: page size and max_seqlen_q must be positive");
  FG_REQUIRE(c->num_pages > 0 && c->num_pages < ((int64_t)1 << 31), FG_ERR_INVALID, "cache_attn_fwd: the cache has %lld pages",
             (long long)c->num_pages);
  FG_REQUIRE(p.alibi_slopes == nullptr, FG_ERR_UNSUPPORTED, "cache_attn_fwd: alibi_slopes are not supported with an 8-bit cache or sink tokens");
  auto al = [](const void* q, int64_t n, int64_t s1, int64_t s2, int64_t s3) {
    return fg_aligned(q, 16) && s1 % n == 0 && s2 % n == 0 && s3 % n == 0;
  };
  const int64_t n = narrow8 ? 16 : 8;
  FG_REQUIRE(al(p.q, 8, p.q_row_stride, p.q_head_stride, 0) && al(p.k_cache, n, p.k_row_stride, p.k_head_stride, p.k_page_stride) &&
                 al(p.v_cache, n, p.v_row_stride, p.v_head_stride, p.v_page_stride),
             FG_ERR_UNSUPPORTED, "cache_attn_fwd: q/k/v rows must be 16-byte aligned");
  FG_REQUIRE(p.batch < 65536 && p.Hk < 65536, FG_ERR_UNSUPPORTED, "cache_attn_fwd: batch/heads exceed the grid");
  return FG_OK;
}

}  // namespace

extern "C" size_t fg_cache_attn_workspace_bytes(const FgCacheAttnParams* c, int device) {
  (void)device;
  if (c == nullptr || c->base.batch <= 0 || c->base.total_q <= 0 || check_params(c) != FG_OK) return 0;
  return make_plan(*c).workspace;
}

extern "C" int fg_cache_attn_fwd(const FgCacheAttnParams* c, void* stream) {
  const int rc = check_params(c);
  if (rc != FG_OK) return rc;
  const FgFlashParams& p = c->base;
  if (p.batch == 0 || p.total_q == 0) return FG_OK;
  CacheAttnArgs a;
  a.p = *c;
  if (c->cache_format == FG_CACHE_SAME) a.p.k_scale = a.p.v_scale = nullptr;
  const float log2e = 1.4426950408889634f;
  a.scale_log2 = p.softmax_scale * log2e;
  a.cap_in = p.softcap > 0.f ? p.softmax_scale / p.softcap : 0.f;
  a.cap_out_log2 = p.softcap * log2e;
  a.group = p.Hq / p.Hk;
  a.left = p.window_left >= 0 ? p.window_left : INT_MAX;
  a.right = p.is_causal ? 0 : (p.window_right >= 0 ? p.window_right : INT_MAX);
  int s = 0;
  while (((int64_t)1 << s) < p.page_size) ++s;
  a.page_magic = (uint32_t)(((uint64_t)1 << (31 + s)) / (uint64_t)p.page_size + 1);
  a.page_shift = 31 + s;
  a.page_bits = ((int64_t)1 << s) == p.page_size ? s : -1;
  const Plan plan = make_plan(*c);
  a.splits = plan.splits;
  if (plan.splits > 1 && (p.workspace == nullptr || (size_t)p.workspace_bytes < plan.workspace || !fg_aligned(p.workspace, 16))) a.splits = 1;
  a.min_tiles = 16;
  a.part_o = (float*)p.workspace;
  a.part_ml = a.part_o + (size_t)a.splits * p.batch * plan.stream_q * p.Hq * padded_dim(p.D);
  hipStream_t st = (hipStream_t)stream;
  if (plan.stream_q > 0) {
    a.min_q = 1;
    a.max_q = plan.stream_q;
    const int done = p.dtype == FG_F16 ? stream_formats<f16_t>(a, plan.nq, plan.narrow, st) : stream_formats<bf16_t>(a, plan.nq, plan.narrow, st);
    if (done != FG_OK || !plan.tile) return done;
  }
  a.min_q = plan.stream_q + 1;
  a.max_q = p.max_seqlen_q;
  return p.dtype == FG_F16 ? tile_formats<f16_t>(a, st) : tile_formats<bf16_t>(a, st);
}
