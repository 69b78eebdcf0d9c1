// What the attention kernels over a paged cache share: arguments, the cache's element types, which keys a block of rows sees.
// Included by attn_cache.hip inside its unnamed namespace, in front of attn_stream.h and attn_tile.h.
#pragma once

constexpr int64_t kMostBlocks = (int64_t)1 << 24;  // of 256 threads: a launch counts threads in 32 bits

struct CacheAttnArgs {
  FgCacheAttnParams p;
  float scale_log2;            // softmax_scale * log2(e)             (softcap == 0)
  float cap_in, cap_out_log2;  // softcap: t = cap_out_log2 * tanh(S * cap_in)
  int group;                   // query heads per KV head
  int left, right;             // window bounds, INT32_MAX where unbounded
  int splits;                  // key ranges per row block
  int min_tiles;               // fewest tiles of a range
  int min_q, max_q;            // sequences with min_q..max_q new tokens are taken, others are left alone
  uint32_t page_magic;         // page number of key k: (k * page_magic) >> page_shift
  int page_shift;
  int page_bits;               // log2(page_size) where it is a power of two, else -1
  // splits > 1: partial results, fp32.  Rows are tokens: part_q of each sequence, or all tokens of the call (part_q == 0)
  int part_q;
  int64_t part_rows;           // batch * part_q, or total_q
  float* part_o;               // [splits][part_rows][Hq][DP], not divided by the sum
  float* part_ml;              // [splits][part_rows][Hq][2]: maximum (base 2), sum
};

// ---- element types of the cache ------------------------------------------------------------------------------------------
template <typename T, int FMT> struct Widen;  // two 8-bit elements of a 32-bit word -> two T in 32 bits
template <> struct Widen<bf16_t, FG_CACHE_E4M3> {
  template <bool HI> static __device__ __forceinline__ uint32_t two(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  }
};
template <> struct Widen<bf16_t, FG_CACHE_E5M2> {
  template <bool HI> static __device__ __forceinline__ uint32_t two(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, HI));
  }
};
template <> struct Widen<f16_t, FG_CACHE_E4M3> {
  template <bool HI> static __device__ __forceinline__ uint32_t two(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  }
};
template <> struct Widen<f16_t, FG_CACHE_E5M2> {
  template <bool HI> static __device__ __forceinline__ uint32_t two(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, HI));
  }
};

template <typename T> struct Mma16;
template <> struct Mma16<bf16_t> {
  typedef bf16x8 Frag;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mma16<f16_t> {
  typedef f16x8 Frag;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// ---- what a row block sees ---------------------------------------------------------------------------------------------
struct Seen {
  int lo, hi;       // keys [lo, hi) may be seen by some row
  int sinks;        // and keys [0, sinks), where they lie in front of lo
  int sink_tiles;   // tiles that hold them
  int first_tile;   // tile of lo
  int tiles;        // sink tiles + tiles of [lo, hi)
};

// Tokens tok_lo..tok_hi of a sequence with q_len new tokens and k_len keys (the last new token sits on the last key).
template <int TILE>
__device__ __forceinline__ Seen seen_by(const CacheAttnArgs& a, int q_len, int k_len, int tok_lo, int tok_hi) {
  Seen s;
  const int shift = k_len - q_len;
  const int64_t hi = (int64_t)shift + tok_hi + 1 + a.right, lo = (int64_t)shift + tok_lo - a.left;
  s.hi = hi < k_len ? (hi > 0 ? (int)hi : 0) : k_len;
  s.lo = lo > 0 ? (int)lo : 0;
  s.lo = s.lo < s.hi ? s.lo : s.hi;
  s.first_tile = s.lo / TILE;
  const int front = s.first_tile * TILE;  // whole tiles in front of lo
  s.sinks = a.p.num_sink_tokens < s.hi ? a.p.num_sink_tokens : s.hi;
  s.sink_tiles = ((s.sinks < front ? s.sinks : front) + TILE - 1) / TILE;
  s.tiles = s.sink_tiles + (s.lo < s.hi ? (s.hi + TILE - 1) / TILE - s.first_tile : 0);
  return s;
}
template <int TILE>
__device__ __forceinline__ int tile_key(const Seen& s, int t) {
  return (t < s.sink_tiles ? t : s.first_tile + t - s.sink_tiles) * TILE;
}
__device__ __forceinline__ int page_of(const CacheAttnArgs& a, int key) {
  return (int)(((uint64_t)(uint32_t)key * a.page_magic) >> a.page_shift);
}
__device__ __forceinline__ float seq_scale(const float* s, int64_t bs, int64_t hs, int b, int h) {
  return s == nullptr ? 1.0f : s[b * bs + h * hs];
}

// Keys that token `tok` sees: [lo, hi) and [0, min(sinks, hi)).
__device__ __forceinline__ void row_bounds(const CacheAttnArgs& a, int q_len, int k_len, int tok, int& lo, int& hi) {
  const int64_t at = (int64_t)(k_len - q_len) + tok;
  const int64_t h = at + 1 + a.right, l = at - a.left;
  hi = h < k_len ? (h > 0 ? (int)h : 0) : k_len;
  lo = l > 0 ? (l < k_len ? (int)l : k_len) : 0;
}
// A sequence as a workgroup takes it; `mine` is false where it is not for this launch.
struct Sequence {
  int q_bos, q_len, k_len;
  float k_scale, v_scale;
  bool mine, too_long;  // longer than its row of the block table: nothing is read behind the row, its output is NaN
};
// Everything that does not depend on other loads is requested at once: each trip to memory is about a microsecond, and a
// short call is little else.
__device__ __forceinline__ Sequence sequence(const CacheAttnArgs& a, int b, int kvh) {
  const FgFlashParams& p = a.p.base;
  Sequence s;
  const int end = p.cu_seqlens_q[b + 1];
  const int k_said = p.seqused_k[b];
  s.q_bos = p.cu_seqlens_q[b];
  s.k_scale = seq_scale(a.p.k_scale, a.p.k_scale_batch_stride, a.p.k_scale_head_stride, b, kvh);
  s.v_scale = seq_scale(a.p.v_scale, a.p.v_scale_batch_stride, a.p.v_scale_head_stride, b, kvh);
  s.q_len = end - s.q_bos;
  s.mine = s.q_len >= a.min_q && s.q_len <= a.max_q && s.q_bos >= 0 && end <= p.total_q;
  const int64_t reach = (int64_t)a.p.table_width * p.page_size;
  s.too_long = k_said > reach;
  s.k_len = k_said < 0 ? 0 : (k_said < reach ? k_said : (int)reach);
  return s;
}
// tanh to about 4 roundings: its series near 0, (1 - e) / (1 + e) with e = exp(-2x) elsewhere.
__device__ __forceinline__ float tanh_of(float x) {
  const float ax = fabsf(x), x2 = x * x;
  const float near0 = x + x * x2 * (-1.f / 3 + x2 * (2.f / 15 + x2 * (-17.f / 315 + x2 * (62.f / 2835))));
  const float far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(ax * 2.8853900817779268f));
  return ax < 0.25f ? near0 : copysignf(far, x);
}
// In every 16 lanes: lanes 8-15 of `lo` and lanes 0-7 of `hi` change places.
__device__ __forceinline__ void swap_half_rows(uint32_t& lo, uint32_t& hi) {
  constexpr int kRor8 = 0x128;  // the lane 8 further on, round the 16
  const int a = (int)lo, b = (int)hi;
  lo = (uint32_t)__builtin_amdgcn_update_dpp(a, b, kRor8, 0xF, 0xC, false);
  hi = (uint32_t)__builtin_amdgcn_update_dpp(b, a, kRor8, 0xF, 0x3, false);
}
// ds_read_b64_tr_b16: the 16 lanes of a group read four rows of 16 elements; lane i receives element i of the four rows.
__device__ __forceinline__ u32x2 read_tr(const char* at) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4* lds_ptr;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)at));
}

// ---- key ranges ----------------------------------------------------------------------------------------------------------
// A row block's tiles are spread over all `splits` ranges, whatever the host knew of the sequence's length, but a range has at
// least min_tiles of them, and a multiple of UNIT.
template <int UNIT>
__device__ __forceinline__ int range_tiles(const CacheAttnArgs& a, int tiles) {
  const int t = ((tiles + a.splits - 1) / a.splits + UNIT - 1) / UNIT * UNIT;
  return t < a.min_tiles && a.splits > 1 ? a.min_tiles : t;
}
__device__ __forceinline__ int64_t part_row(const CacheAttnArgs& a, int split, int b, int q_bos, int tok) {
  return split * a.part_rows + (a.part_q > 0 ? (int64_t)b * a.part_q : q_bos) + tok;
}

// Merges the key ranges of a row (token, head), which belongs to a block of ROWS rows whose tiles have TILE keys.  WHOLE: a
// workgroup for each row (many ranges), else a wave.  A lane holds four elements; what lanes are left take other ranges.
template <typename T, int DP, int TILE, int ROWS, int UNIT, bool WHOLE>
__global__ __launch_bounds__(256) void attn_merge_kernel(CacheAttnArgs a) {
  constexpr int LR = DP / 4;                     // lanes of a row
  constexpr int NG = (WHOLE ? 256 : 64) / LR;    // groups of ranges
  __shared__ __attribute__((aligned(16))) float parts[WHOLE ? 4 : 1][DP + 4];
  const FgFlashParams& p = a.p.base;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t th = WHOLE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;  // token * Hq + head
  const int b = blockIdx.y;
  const int tok = (int)(th / p.Hq), head = (int)(th - (int64_t)tok * p.Hq);
  const Sequence seq = sequence(a, b, head / a.group);
  const int q_bos = seq.q_bos, q_len = seq.q_len, k_len = seq.k_len;
  if (!seq.mine || tok >= q_len) return;         // (the same for all threads of a row)
  const int rows = q_len * a.group;
  const int row0 = (tok * a.group + head % a.group) / ROWS * ROWS;
  const int last_row = row0 + ROWS < rows ? row0 + ROWS - 1 : rows - 1;
  const Seen seen = seen_by<TILE>(a, q_len, k_len, row0 / a.group, last_row / a.group);
  const int per = range_tiles<UNIT>(a, seen.tiles);
  int ns = per > 0 ? (seen.tiles + per - 1) / per : 1;  // ranges that were written
  ns = ns < 1 ? 1 : (ns > a.splits ? a.splits : ns);
  const int64_t step = a.part_rows * p.Hq, at = part_row(a, 0, b, q_bos, tok) * p.Hq + head;
  // a lane's own ranges, four at a time, under their running maximum
  const int mine = (WHOLE ? tid : lane) / LR, d = (tid % LR) * 4;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f, m = -INFINITY;
  for (int s0 = mine; s0 < ns; s0 += 4 * NG) {
    f32x2 ml[4];
    f32x4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {                // (a range past the last one: the last one, with no weight)
      const int s = s0 + i * NG < ns ? s0 + i * NG : ns - 1;
      ml[i] = *reinterpret_cast<const f32x2*>(a.part_ml + (s * step + at) * 2);
      x[i] = *reinterpret_cast<const f32x4*>(a.part_o + (s * step + at) * DP + d);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[i][0]);
    const float use = top == -INFINITY ? 0.f : top;
    const float old = __builtin_amdgcn_exp2f(m - use);
    l *= old;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= old;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (s0 + i * NG >= ns) continue;
      const float f = __builtin_amdgcn_exp2f(ml[i][0] - use);
      l += ml[i][1] * f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += x[i][e] * f;
    }
    m = top;
  }
  // the groups of a wave, then the waves
  float all = m;
#pragma unroll
  for (int x = LR; x < 64; x *= 2) all = fmaxf(all, __shfl_xor(all, x, 64));
  float m_use = all == -INFINITY ? 0.f : all;
  const float own = __builtin_amdgcn_exp2f(m - m_use);
  l *= own;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= own;
#pragma unroll
  for (int x = LR; x < 64; x *= 2) {
    l += __shfl_xor(l, x, 64);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x, 64);
  }
  if constexpr (WHOLE) {
    if (lane < LR) *reinterpret_cast<f32x4*>(&parts[wave][d]) = o;
    if (lane == 0) parts[wave][DP] = l, parts[wave][DP + 1] = all;
    __syncthreads();
    if (tid >= LR) return;
    all = fmaxf(fmaxf(parts[0][DP + 1], parts[1][DP + 1]), fmaxf(parts[2][DP + 1], parts[3][DP + 1]));
    m_use = all == -INFINITY ? 0.f : all;
    o = f32x4{0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(parts[w][DP + 1] - m_use);
      l += parts[w][DP] * f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += parts[w][d + e] * f;
    }
  } else if (lane >= LR) {
    return;
  }
  const bool empty = l == 0.f;
  const float f = empty ? 0.f : seq.v_scale / l;
  T* const out = (T*)p.out + (int64_t)(q_bos + tok) * p.o_row_stride + (int64_t)head * p.o_head_stride;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (d + e < p.D) out[d + e] = (T)(empty ? 0.f : o[e] * f);
  if (d == 0 && p.lse != nullptr)
    p.lse[(int64_t)head * p.total_q + q_bos + tok] = empty ? INFINITY : m_use * 0.6931471805599453f + logf(l);
}

template <typename T, int DP, int TILE, int ROWS, int UNIT>
int launch_merge(const CacheAttnArgs& a, hipStream_t st) {
  const FgFlashParams& p = a.p.base;
  const int64_t rows = (int64_t)a.max_q * p.Hq;
  FG_REQUIRE(rows < kMostBlocks, FG_ERR_UNSUPPORTED, "cache_attn_fwd: too many query rows for one launch");
  if (a.splits > 8)
    hipLaunchKernelGGL((attn_merge_kernel<T, DP, TILE, ROWS, UNIT, true>), dim3((unsigned)rows, (unsigned)p.batch), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((attn_merge_kernel<T, DP, TILE, ROWS, UNIT, false>), dim3((unsigned)fg_cdiv(rows, 4), (unsigned)p.batch), dim3(256), 0, st, a);
  return fg_check_launch("cache_attn_fwd");
}
