// What the attention kernels over a paged cache share: arguments, the cache's element types, which keys a block of rows sees.
// Included by attn_cache.hip inside its unnamed namespace, in front of attn_stream.h and attn_tile.h.
#pragma once

struct CacheAttnArgs {
  FgCacheAttnParams p;
  float scale_log2;            // softmax_scale * log2(e)             (softcap == 0)
  float cap_in, cap_out_log2;  // softcap: t = cap_out_log2 * tanh(S * cap_in)
  int group;                   // query heads per KV head
  int left, right;             // window bounds, INT32_MAX where unbounded
  int splits;                  // key ranges per row block (grid x = splits * row blocks)
  int min_tiles;               // fewest tiles of a range, a multiple of 4
  int min_q, max_q;            // sequences with min_q..max_q new tokens are taken, others are left alone
  uint32_t page_magic;         // page number of key k: (k * page_magic) >> page_shift
  int page_shift;
  int page_bits;               // log2(page_size) where it is a power of two, else -1
  float* part_o;               // [splits][batch][max_q][Hq][DP] fp32, not divided by the sum   (splits > 1)
  float* part_ml;              // [splits][batch][max_q][Hq][2] fp32: maximum (base 2), sum
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
// ds_read_b64_tr_b16: the 16 lanes of a group read four rows of 16 elements; lane i receives element i of the four rows.
__device__ __forceinline__ u32x2 read_tr(const char* at) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4* lds_ptr;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)at));
}
