// Attention over a paged cache that holds 8-bit values, or under a sliding window with first tokens that stay visible
// (sinks), or both.  Formulas: query i of a sequence with Lq new tokens and Lk keys stands at position P = Lk - Lq + i;
//
//   key j is visible  iff  j <= P + right  and  (j >= P - left  or  j < sinks)
//   t = scale * s_k[b, h] * (q . c_j)   or   cap * tanh(that / cap)
//   out = s_v[b, h] * sum_j softmax(t)_j * c'_j        lse = log sum_j exp(t_j)
//
// c, c' are the cached K and V values as they stand, s the scales they were written with (1 for a 16-bit cache).
#include <limits.h>
#include <algorithm>
#include <atomic>
#include "fg_common.h"

namespace {

#include "attn_cache.h"
#include "attn_stream.h"
#include "attn_tile.h"

template <typename T, int FMT, int DP>
int stream_pages(const CacheAttnArgs& a, int nq, int pages, hipStream_t st) {
  if (pages == kKeys) return launch_stream<T, FMT, DP, 1, kKeys>(a, st);
  if constexpr (DP < 256) {
    if (nq == 2) return pages == kHalves ? launch_stream<T, FMT, DP, 2, kHalves>(a, st) : launch_stream<T, FMT, DP, 2, kGroups>(a, st);
  }
  return pages == kHalves ? launch_stream<T, FMT, DP, 1, kHalves>(a, st) : launch_stream<T, FMT, DP, 1, kGroups>(a, st);
}
template <typename T, int FMT>
int stream_dims(const CacheAttnArgs& a, int nq, int pages, hipStream_t st) {
  const int D = a.p.base.D;
  if (D <= 64) return stream_pages<T, FMT, 64>(a, nq, pages, st);
  if (D <= 128) return stream_pages<T, FMT, 128>(a, nq, pages, st);
  return stream_pages<T, FMT, 256>(a, nq, pages, st);
}
template <typename T>
int stream_formats(const CacheAttnArgs& a, int nq, int pages, hipStream_t st) {
  if (a.p.cache_format == FG_CACHE_E4M3) return stream_dims<T, FG_CACHE_E4M3>(a, nq, pages, st);
  if (a.p.cache_format == FG_CACHE_E5M2) return stream_dims<T, FG_CACHE_E5M2>(a, nq, pages, st);
  return stream_dims<T, FG_CACHE_SAME>(a, nq, pages, st);
}

template <typename T, int FMT>
int tile_dims(const CacheAttnArgs& a, int nq, hipStream_t st) {
  if (a.p.base.D <= 64) return nq == 1 ? launch_tile<T, FMT, 64, 1>(a, st) : launch_tile<T, FMT, 64, 2>(a, st);
  return nq == 1 ? launch_tile<T, FMT, 128, 1>(a, st) : launch_tile<T, FMT, 128, 2>(a, st);
}
template <typename T>
int tile_formats(const CacheAttnArgs& a, int nq, hipStream_t st) {
  if (a.p.cache_format == FG_CACHE_E4M3) return tile_dims<T, FG_CACHE_E4M3>(a, nq, st);
  if (a.p.cache_format == FG_CACHE_E5M2) return tile_dims<T, FG_CACHE_E5M2>(a, nq, st);
  return tile_dims<T, FG_CACHE_SAME>(a, nq, st);
}

int num_cu() {
  static std::atomic<int> known[64];             // by device; two queries of the runtime a call otherwise
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 0;
  if (dev >= 0 && dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
  if (dev >= 0 && dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

struct Plan {
  int stream_q;     // sequences with up to so many new tokens take the stream kernel (0: none)
  bool tile;        // the others take the tile kernel
  int nq, tile_nq;  // 16-row tiles of a row block (stream), of a wave (tile)
  int tile_batch;   // sequences of a launch of the tile kernel (0: one of them alone is too long for one)
  int pages;        // stream kernel: how pages are found
  int splits, min_tiles, tile_splits, tile_min_tiles;
  size_t stream_bytes, tile_bytes;  // scratch for the key ranges; one after the other
};

// Most scratch for the key ranges of chunks: their partial results grow with the tokens of the call (1.5 GiB for 16384 tokens of 32
// heads of 128 in 6 ranges) and lie next to a cache that may fill the card.  1 GiB keeps the speed where it was measured: 8 chunks of up to
// 4096 tokens over up to 131072 keys 24.2 ms in 3 ranges, 24.0 in 6, 46.4 unsplit (row blocks of sequences of different length start at
// different times, and no longer share what the L2 holds); one of 8200 over 131072 18.4 ms in 3, 18.3 in 9, 21.0 unsplit.  The
// stream kernel's ranges need no bound: there are some for fewer than 512 row blocks only, and then at most 52 MB.
constexpr size_t kMostScratch = (size_t)1 << 30;

int padded_dim(int D) { return D <= 64 ? 64 : (D <= 128 ? 128 : 256); }

// Microseconds that a launch of the tile kernel takes with row blocks of 64 * nq rows and `splits` key ranges, from what was
// measured on MI355X: the steps of a tile on a CU that holds one workgroup or two, start and end of a workgroup, and the merge
// (its launch, and 2 * (DP + 2) * 4 bytes for each range, token and head at 5 TB/s).  `even`: all sequences as long as the
// longest; otherwise their blocks are taken to be 0.6 of the longest on average, and a long one to begin among the last.  Whole
// calls, chunks of (1024, 765, 284, 14) tokens over (8192, 4816, 3212, 2548) keys, 32/8 heads: blocks of 128 rows 588 us unsplit, 305 in
// 2 ranges, 303 in 3, 309 in 4 (taken), 328 in 6, 518 in 12; of 64 rows 826, 391 in 2, 400 in 4.  One chunk of 1000 over 1000: blocks
// of 64 rows 33 us (taken), of 128 rows 42, in 2 ranges 48 and 51.  What the model leaves out is workgroups for rows that are not
// there, which uneven batches have many of: the merge of the chunks above takes 45 us, its bytes 28.
double tile_cost(int64_t blocks, double tiles, int nq, int dp, int64_t cus, int splits, bool even, double merge_bytes) {
  const double dim = dp == 64 ? 0.72 : 1.0;
  const double alone = (nq == 1 ? 1.32 : 1.7) * dim, shared = (nq == 1 ? 1.54 : 2.3) * dim;
  const int64_t wgs = blocks * splits;
  const double range = tiles / splits < 1 ? 1 : tiles / splits;
  double us = 6;
  if (wgs <= cus) us += range * alone;
  else if (wgs <= 2 * cus) us += range * shared;
  else if (even) us += (double)fg_cdiv(wgs, 2 * cus) * range * shared;
  else us += (0.6 * (double)blocks * tiles / (double)(2 * cus) + 0.75 * range) * shared;
  if (splits > 1) us += 4 + splits * merge_bytes * 2 / 5e6;
  return us;
}

// Which kernels run, and how the rows and the keys are cut.
Plan make_plan(const FgCacheAttnParams& c) {
  const FgFlashParams& p = c.base;
  const int G = p.Hq / p.Hk;
  const int64_t cus = num_cu();
  Plan plan = {};
  // the most keys that one row block of `q` tokens may see
  auto keys_of = [&](int64_t q, int tile) {
    int64_t keys = p.max_seqlen_k > 0 ? p.max_seqlen_k : 1;
    const int64_t window = (int64_t)p.window_left + q + c.num_sink_tokens + 2 * tile;
    return p.window_left >= 0 && window < keys ? window : keys;
  };
  const int few = 32 / G > 1 ? 32 / G : 1;
  // The tile kernel's offsets are 32 bits of 16-byte pieces: inside a page, and from one page to the next.
  const int bytes = c.cache_format == FG_CACHE_SAME ? 2 : 1;
  auto near = [&](int64_t page, int64_t row) {
    const int64_t most = (int64_t)1 << 32;
    return (p.page_size == 1 || row * bytes / 16 <= (most - 1) / (p.page_size - 1)) && (c.num_pages == 1 || page * bytes / 16 < most);
  };
  plan.tile = p.D <= 128 && p.max_seqlen_q > few && near(p.k_page_stride, p.k_row_stride) && near(p.v_page_stride, p.v_row_stride);
  plan.stream_q = plan.tile ? few : p.max_seqlen_q;
  // The tile kernel takes the short sequences too where all are as long as the longest, so that there are none, and where no row
  // sees more than 1024 keys: a launch of its own mostly costs more than such sequences do here.  A chunk of 512 and three tokens over
  // 512 keys each, 32/8 heads: 38 us here, 48 in two launches; 300 and 15 tokens over up to 900: 53 and 57; 24 sequences of up to 100
  // over up to 700, 8/2 heads: 25 and 35; 300 and 15 over up to 2000: 77 and 78.  (100 and 63 tokens over 1000: 94 and 79.)
  const bool even = (int64_t)p.total_q >= (int64_t)p.batch * p.max_seqlen_q;
  if (plan.tile && (even || keys_of(fg_cdiv(64, G), kTileKeys) <= 1024)) plan.stream_q = 0;
  const bool pow2 = (p.page_size & (p.page_size - 1)) == 0;
  plan.pages = pow2 && p.page_size >= 16 ? kHalves : (p.page_size % 8 == 0 ? kGroups : kKeys);
  plan.nq = plan.pages != kKeys && p.D <= 128 && (int64_t)plan.stream_q * G > 16 ? 2 : 1;
  const size_t row = (size_t)p.Hq * (padded_dim(p.D) + 2) * sizeof(float);
  plan.splits = 1;
  if (plan.stream_q > 0) {
    const int64_t tiles = fg_cdiv(keys_of(fg_cdiv(16 * plan.nq, G), kTile), kTile);
    const int64_t groups = fg_cdiv((int64_t)plan.stream_q * G, 16 * plan.nq) * p.batch * p.Hk;
    // Two workgroups per CU fill the card.  Below that the keys are cut into ranges for up to four per CU (sequences differ, and
    // the ranges of a short one end early) of at least 16 tiles, or for one per CU of at least 4.  Whole calls: 24 groups of up to
    // 4096 tiles take 984 us unsplit, 111 cut in 16 and 107 in 43; 8 groups of 62 tiles 21 us unsplit, 17 cut in 12; 512 groups of
    // 128 tiles 98 us unsplit, 98 cut in 3.  Up to 32 tiles the launch that merges costs more than the ranges save: 8 groups of 32
    // take 13.5 us unsplit, 17.3 in 4 or in 8.
    plan.min_tiles = 4;
    int64_t splits = 1;
    if (groups < 2 * cus && tiles > 32) {
      const int64_t many = std::min(fg_cdiv(4 * cus, groups), tiles / 16), few_keys = std::min(fg_cdiv(cus, groups), tiles / 4);
      splits = std::max(std::max(many, few_keys), (int64_t)1);
    }
    plan.splits = (int)splits;
    if (plan.splits > 1) plan.stream_bytes = (plan.splits * row * p.batch * plan.stream_q + 15) / 16 * 16;
  }
  if (plan.tile) {
    const int dp = padded_dim(p.D);
    double best = 0;
    for (int nq = 1; nq <= 2; ++nq) {
      const int rows = 64 * nq;
      // even: exact; otherwise half a block is left over in a sequence on average
      const int64_t blocks = p.Hk * (even ? fg_cdiv((int64_t)p.max_seqlen_q * G, rows) * p.batch : (int64_t)p.total_q * G / rows + p.batch / 2 + 1);
      const int64_t tiles = fg_cdiv(keys_of(fg_cdiv(rows, G), kTileKeys), kTileKeys);
      for (int splits = 1; splits <= 64 && (splits == 1 || (tiles >= 2 * splits && splits * row * p.total_q <= kMostScratch)); ++splits) {
        if (tile_blocks(p, p.max_seqlen_q, nq, splits, p.batch) >= kMostBlocks) break;
        const double us = tile_cost(blocks, (double)tiles, nq, dp, cus, splits, even, (double)row * (double)p.total_q);
        if (plan.tile_splits == 0 || us < best) best = us, plan.tile_nq = nq, plan.tile_splits = splits;
      }
    }
    plan.tile_batch = p.batch;
    if (plan.tile_splits == 0) {  // more than a launch holds in any cut: unsplit, a few sequences at a time
      plan.tile_nq = 2, plan.tile_splits = 1;
      const int64_t eights = (kMostBlocks - 1) / tile_blocks(p, p.max_seqlen_q, 2, 1, 1) * fg_cdiv(p.Hk, 8);
      plan.tile_batch = (int)(eights * 8 / p.Hk);
    }
    plan.tile_min_tiles = 2;
    if (plan.tile_splits > 1) plan.tile_bytes = plan.tile_splits * row * p.total_q;
  }
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
  // (key numbers, a tile or a few past the last one too, are 32-bit integers in the kernels)
  FG_REQUIRE((int64_t)c->table_width * p.page_size <= INT_MAX - 65536, FG_ERR_UNSUPPORTED,
             "cache_attn_fwd: a row of the block table spans %lld keys", (long long)c->table_width * p.page_size);
  return FG_OK;
}

// The call with its longest sequence no longer than all tokens together: the grids and the scratch go by it.
FgCacheAttnParams bounded(const FgCacheAttnParams& given) {
  FgCacheAttnParams c = given;
  c.base.max_seqlen_q = (int)std::min((int64_t)c.base.max_seqlen_q, (int64_t)c.base.total_q);
  return c;
}

}  // namespace

extern "C" size_t fg_cache_attn_workspace_bytes(const FgCacheAttnParams* c, int device) {
  (void)device;
  if (c == nullptr || c->base.batch <= 0 || c->base.total_q <= 0 || check_params(c) != FG_OK) return 0;
  const Plan plan = make_plan(bounded(*c));
  return plan.stream_bytes + plan.tile_bytes;
}

extern "C" int fg_cache_attn_fwd(const FgCacheAttnParams* c, void* stream) {
  const int rc = check_params(c);
  if (rc != FG_OK) return rc;
  if (c->base.batch == 0 || c->base.total_q == 0) return FG_OK;
  CacheAttnArgs a;
  a.p = bounded(*c);
  const FgFlashParams& p = a.p.base;
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
  const Plan plan = make_plan(a.p);
  const bool scratch = p.workspace != nullptr && fg_aligned(p.workspace, 16) && (size_t)p.workspace_bytes >= plan.stream_bytes + plan.tile_bytes;
  FG_REQUIRE(!plan.tile || plan.tile_batch > 0, FG_ERR_UNSUPPORTED, "cache_attn_fwd: too many query rows for one launch");
  const int dp = padded_dim(p.D);
  hipStream_t st = (hipStream_t)stream;
  if (plan.stream_q > 0) {
    a.min_q = 1;
    a.max_q = plan.stream_q;
    a.splits = scratch ? plan.splits : 1;
    a.min_tiles = plan.min_tiles;
    a.part_q = plan.stream_q;
    a.part_rows = (int64_t)p.batch * plan.stream_q;
    a.part_o = (float*)p.workspace;
    a.part_ml = a.part_o + (size_t)a.splits * a.part_rows * p.Hq * dp;
    const int done = p.dtype == FG_F16 ? stream_formats<f16_t>(a, plan.nq, plan.pages, st) : stream_formats<bf16_t>(a, plan.nq, plan.pages, st);
    if (done != FG_OK || !plan.tile) return done;
  }
  a.min_q = plan.stream_q + 1;
  a.max_q = p.max_seqlen_q;
  a.splits = scratch ? plan.tile_splits : 1;
  a.min_tiles = plan.tile_min_tiles;
  a.part_q = 0;
  a.part_rows = p.total_q;
  a.part_o = (float*)((char*)p.workspace + plan.stream_bytes);
  a.part_ml = a.part_o + (size_t)a.splits * a.part_rows * p.Hq * dp;
  const int batch = p.batch;
  for (int b = 0; b < batch; b += plan.tile_batch) {
    CacheAttnArgs s = a;
    s.p.base.batch = std::min(plan.tile_batch, batch - b);
    s.p.base.cu_seqlens_q += b;
    s.p.base.seqused_k += b;
    s.p.base.block_table += b * p.block_table_stride;
    if (s.p.k_scale != nullptr) s.p.k_scale += b * s.p.k_scale_batch_stride;
    if (s.p.v_scale != nullptr) s.p.v_scale += b * s.p.v_scale_batch_stride;
    const int done = p.dtype == FG_F16 ? tile_formats<f16_t>(s, plan.tile_nq, st) : tile_formats<bf16_t>(s, plan.tile_nq, st);
    if (done != FG_OK) return done;
  }
  return FG_OK;
}
