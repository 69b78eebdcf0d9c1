// The 8-bit paged KV cache: rows quantised as they are scattered into it, and read back as packed rows of sequences.
//
//   write:  c = rn8(clamp(x / s[h], -max, max))     s fp32, one number or one for each KV head; c in e4m3 or e5m2
//   read:   x = rn(c * s[h])                         one rounding, to fp16, bf16 or fp32 (16- and 32-bit caches: a copy)
//
// The quotient is rounded to fp32 before it is rounded to 8 bits (see Quotient), so a value whose quotient is half way between
// two 8-bit numbers goes to the even one.  Numbers beyond the format's largest are cut
// to it, infinities too (the conversion instruction itself would turn them into NaN or infinity); NaN stays NaN.
//
// Both kernels are bound by HBM.
#include "fg_common.h"

namespace {

enum { kE4M3 = FG_CACHE_E4M3, kE5M2 = FG_CACHE_E5M2 };
constexpr int64_t kMostBlocks = (int64_t)1 << 24;  // of 256 threads: a launch counts threads in 32 bits

template <int FMT> struct Fp8;
template <> struct Fp8<kE4M3> {
  static constexpr float kMax = 448.0f;
  static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  }
  template <bool HI> static __device__ __forceinline__ f32x2 unpack2(uint32_t w) {
    return __builtin_amdgcn_cvt_pk_f32_fp8((int)w, HI);
  }
};
template <> struct Fp8<kE5M2> {
  static constexpr float kMax = 57344.0f;
  static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
  }
  template <bool HI> static __device__ __forceinline__ f32x2 unpack2(uint32_t w) {
    return __builtin_amdgcn_cvt_pk_f32_bf8((int)w, HI);
  }
};

// x / s in fp32, cut to the format's range; NaN stays NaN.
//   q = x * r,  r = 1 / s rounded to nearest;   q' = q + (x - q * s) * r
// (the residual x - q * s is exact in one fused operation, so q' is x / s with a relative error of 2^-46 in front of its one
// rounding: a quotient that is an fp32 number, such as a middle between two 8-bit ones, comes out as it is).  x is cut to
// twice the range first, so that nothing overflows.  Seven plain operations an element instead of the eighteen of a division, which
// alone would keep the vector ALU busy for 40 of the 76 us below.  Scales outside [2^-60, 2^100] are divided by (the residual of a
// smaller one would lose bits below 2^-149).
template <int FMT> struct Quotient {
  float s, r, most;
  bool plain;
  __device__ __forceinline__ explicit Quotient(float scale) : s(scale), r(1.0f / scale) {
    const float a = fabsf(scale);
    plain = a >= 0x1p-60f && a <= 0x1p100f;     // false for NaN
    most = 2.0f * Fp8<FMT>::kMax * a;
  }
  __device__ __forceinline__ float operator()(float x) const {
    float q;
    if (plain) {
      const float c = __builtin_amdgcn_fmed3f(x, -most, most);
      q = c * r;
      q = fmaf(fmaf(-q, s, c), r, q);
    } else {
      q = x / s;
      if (q != q) return q;
    }
    q = __builtin_amdgcn_fmed3f(q, -Fp8<FMT>::kMax, Fp8<FMT>::kMax);
    return x != x ? x : q;
  }
};

struct WriteArgs {
  const void* src[2];      // key, value rows
  char* cache[2];
  const float* scale[2];   // NULL: 1
  int64_t scale_stride[2]; // 0: one number, 1: one for each head
  int64_t src_stride[2];   // elements between tokens
  int64_t block_stride[2]; // bytes between pages
  const void* slots;
  int64_t num_tokens, num_slots;
  int row, D, block_size;  // row = H * D elements
  int waves_log2;          // waves of a row: 1, 2 or 4
};

// One to four waves take a (token, K or V) row, CH elements per lane and piece: 16 bytes are loaded and 4 or 8 stored, both in
// one stretch over a wave.  A piece lies in one head (CH divides D), so it has one scale.  Two pieces per lane are in flight.
// [16384, 32, 128] K and V, bf16 to e4m3, random slots: 76 us = 5.3 TB/s (a large copy on this card: 5.0 to 5.4); one
// wave per row with eight pieces in flight 86.
template <typename T, int FMT, int CH, typename SLOT>
__global__ __launch_bounds__(256) void cache_write8_kernel(WriteArgs a) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t row = w >> a.waves_log2;
  const int64_t tok = row >> 1;
  if (tok >= a.num_tokens) return;
  const int which = (int)(row & 1);
  const int64_t slot = (int64_t)((const SLOT*)a.slots)[tok];
  if (slot < 0 || slot >= a.num_slots) return;  // a padding token; a slot outside the cache is dropped
  const int64_t blk = slot / a.block_size;
  const int64_t off = slot - blk * a.block_size;
  const T* src = (const T*)(which ? a.src[1] : a.src[0]) + tok * (which ? a.src_stride[1] : a.src_stride[0]);
  char* dst = (which ? a.cache[1] : a.cache[0]) + blk * (which ? a.block_stride[1] : a.block_stride[0]) + off * a.row;
  const float* sc = which ? a.scale[1] : a.scale[0];
  const int64_t ss = which ? a.scale_stride[1] : a.scale_stride[0];
  constexpr int U = 2;
  const int step = (64 * CH) << a.waves_log2;
  for (int i0 = (int)(w & ((1 << a.waves_log2) - 1)) * 64 * CH + (threadIdx.x & 63) * CH; i0 < a.row; i0 += step * U) {
    Pack<T, CH> x[U];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * step;
      if (i < a.row) {
        x[u] = ld_pack_nt<T, CH>(src + i);
        s[u] = sc == nullptr ? 1.0f : sc[(i / a.D) * ss];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * step;
      if (i >= a.row) continue;
      const Quotient<FMT> quotient(s[u]);
      if constexpr (CH == 1) {
        const float q = quotient((float)x[u].v[0]);
        dst[i] = (char)(Fp8<FMT>::pack4(q, q, q, q) & 0xff);
      } else {
        uint32_t o[CH / 4];
#pragma unroll
        for (int j = 0; j < CH / 4; ++j) {
          float q[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) q[e] = quotient((float)x[u].v[j * 4 + e]);
          o[j] = Fp8<FMT>::pack4(q[0], q[1], q[2], q[3]);
        }
        if constexpr (CH == 8)
          __builtin_nontemporal_store(*reinterpret_cast<u32x2*>(o), reinterpret_cast<u32x2*>(dst + i));
        else
          __builtin_nontemporal_store(o[0], reinterpret_cast<uint32_t*>(dst + i));
      }
    }
  }
}

template <typename T, int FMT, int CH>
int write_launch(WriteArgs a, int slot_is_i64, hipStream_t st) {
  a.waves_log2 = a.row > 256 * CH ? 2 : (a.row > 128 * CH ? 1 : 0);
  const int64_t grid64 = fg_cdiv((a.num_tokens * 2) << a.waves_log2, 4);
  FG_REQUIRE(grid64 < kMostBlocks, FG_ERR_UNSUPPORTED, "reshape_and_cache_flash_8bit: problem too large for one launch");
  const unsigned grid = (unsigned)grid64;
  if (slot_is_i64) hipLaunchKernelGGL((cache_write8_kernel<T, FMT, CH, int64_t>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((cache_write8_kernel<T, FMT, CH, int32_t>), dim3(grid), dim3(256), 0, st, a);
  return fg_check_launch("reshape_and_cache_flash_8bit");
}

template <typename T, int FMT>
int write_pieces(const WriteArgs& a, int slot_is_i64, hipStream_t st) {
  constexpr int CH = 16 / (int)sizeof(T);
  bool fits = a.D % CH == 0;
  for (int i = 0; i < 2; ++i)
    fits = fits && fg_aligned(a.src[i], 16) && a.src_stride[i] % CH == 0 && fg_aligned(a.cache[i], CH) && a.block_stride[i] % CH == 0;
  return fits ? write_launch<T, FMT, CH>(a, slot_is_i64, st) : write_launch<T, FMT, 1>(a, slot_is_i64, st);
}

struct ReadArgs {
  const char* cache[2];
  char* out[2];
  const float* scale[2];
  int64_t scale_stride[2];
  int64_t page_stride[2];  // bytes
  int64_t out_stride[2];   // elements between output rows
  const int32_t* table;
  int64_t table_stride;
  int table_width;
  const int32_t* cu;       // [batch + 1]
  const int32_t* first;    // [batch] position of a sequence's first row, NULL: 0
  int64_t num_rows, num_pages;
  int batch, row, D, page_size;
};

template <int PB> __device__ __forceinline__ Pack<char, PB> ld_bytes_nt(const char* p) {
  if constexpr (PB >= 8) {
    return ld_pack_nt<char, PB>(p);
  } else {
    Pack<char, PB> v;
    __builtin_memcpy(&v, __builtin_assume_aligned(p, PB), PB);
    return v;
  }
}

// One wave takes one output row, K and V.  Its sequence is the last one that starts at or before the row: 64 starts are
// compared at once.  Rows in front of the first and behind the last sequence are left alone; a page that the cache does
// not have, or a position behind the table, gives zeros.
template <typename U, int FMT, int CH>
__global__ __launch_bounds__(256) void cache_read_kernel(ReadArgs a) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= a.num_rows) return;
  const int lane = threadIdx.x & 63;
  int b = -1;
  for (int i = 0; i <= a.batch; i += 64) {
    const int at = i + lane <= a.batch ? i + lane : a.batch;
    const bool begun = i + lane <= a.batch && (int64_t)a.cu[at] <= r;
    b += __builtin_popcountll(__builtin_amdgcn_ballot_w64(begun));
  }
  if (b < 0 || b >= a.batch) return;
  const int64_t pos = r - a.cu[b] + (a.first == nullptr ? 0 : a.first[b]);
  const int64_t page_at = pos / a.page_size;
  const int64_t slot = pos - page_at * a.page_size;
  const int64_t page = pos >= 0 && page_at < a.table_width ? (int64_t)a.table[(int64_t)b * a.table_stride + page_at] : -1;
  const bool known = page >= 0 && page < a.num_pages;
  constexpr int IB = FMT == FG_CACHE_SAME ? (int)sizeof(U) : 1;  // bytes of a cached element
  constexpr int PB = CH * IB;                                    // of a piece
  const char* src[2];
  U* dst[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    src[k] = a.cache[k] + (known ? page * a.page_stride[k] + slot * (int64_t)a.row * IB : 0);
    dst[k] = (U*)a.out[k] + r * a.out_stride[k];
  }
  constexpr int N = 4;  // pieces of K and of V in flight
  for (int i0 = lane * CH; i0 < a.row; i0 += 64 * CH * N) {
    Pack<char, PB> c[N][2];
    float s[N][2];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = i0 + n * 64 * CH;
      if (i < a.row) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          c[n][k] = ld_bytes_nt<PB>(src[k] + (int64_t)i * IB);
          s[n][k] = FMT == FG_CACHE_SAME || a.scale[k] == nullptr ? 1.0f : a.scale[k][(i / a.D) * a.scale_stride[k]];
        }
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = i0 + n * 64 * CH;
      if (i >= a.row) continue;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        Pack<U, CH> o;
        if constexpr (FMT == FG_CACHE_SAME) {
          __builtin_memcpy(&o, &c[n][k], PB);
          if (!known) o = Pack<U, CH>{};
        } else if constexpr (CH == 1) {
          const f32x2 x = Fp8<FMT>::template unpack2<false>((uint8_t)c[n][k].v[0]);
          o.v[0] = (U)(known ? x[0] * s[n][k] : 0.f);
        } else {
          uint32_t w[CH / 4];
          __builtin_memcpy(w, &c[n][k], PB);
#pragma unroll
          for (int j = 0; j < CH / 4; ++j) {
            const f32x2 lo = Fp8<FMT>::template unpack2<false>(w[j]), hi = Fp8<FMT>::template unpack2<true>(w[j]);
            o.v[j * 4] = (U)(known ? lo[0] * s[n][k] : 0.f);
            o.v[j * 4 + 1] = (U)(known ? lo[1] * s[n][k] : 0.f);
            o.v[j * 4 + 2] = (U)(known ? hi[0] * s[n][k] : 0.f);
            o.v[j * 4 + 3] = (U)(known ? hi[1] * s[n][k] : 0.f);
          }
        }
        st_pack_nt<U, CH>(dst[k] + i, o);
      }
    }
  }
}

template <typename U, int FMT, int CH>
int read_launch(const ReadArgs& a, hipStream_t st) {
  FG_REQUIRE(fg_cdiv(a.num_rows, 4) < kMostBlocks, FG_ERR_UNSUPPORTED, "gather_cache_flash: problem too large for one launch");
  hipLaunchKernelGGL((cache_read_kernel<U, FMT, CH>), dim3((unsigned)fg_cdiv(a.num_rows, 4)), dim3(256), 0, st, a);
  return fg_check_launch("gather_cache_flash");
}

// 85 thousand rows of [8, 128], K and V, e4m3 to bf16: 90 us = 5.8 TB/s (two thirds of it stores, which alone reach 6.8).
// Pieces of 16 output bytes, one stretch over the wave (pieces of 32 bytes were a fifth slower), where everything is aligned for
// them, else single elements.
template <typename U, int FMT>
int read_pieces(const ReadArgs& a, hipStream_t st) {
  constexpr int CH = 16 / (int)sizeof(U), IB = FMT == FG_CACHE_SAME ? (int)sizeof(U) : 1;
  bool fits = a.D % CH == 0;
  for (int i = 0; i < 2; ++i)
    fits = fits && fg_aligned(a.cache[i], CH * IB) && a.page_stride[i] % (CH * IB) == 0 && fg_aligned(a.out[i], 16) &&
           a.out_stride[i] % CH == 0;
  return fits ? read_launch<U, FMT, CH>(a, st) : read_launch<U, FMT, 1>(a, st);
}

template <typename U>
int read_formats(const ReadArgs& a, int fmt, hipStream_t st) {
  if (fmt == FG_CACHE_E4M3) return read_pieces<U, kE4M3>(a, st);
  if (fmt == FG_CACHE_E5M2) return read_pieces<U, kE5M2>(a, st);
  return read_pieces<U, FG_CACHE_SAME>(a, st);
}

bool scale_ok(const float* s, int64_t stride) { return s == nullptr || ((stride == 0 || stride == 1) && fg_aligned(s, 4)); }

}  // namespace

extern "C" int fg_reshape_and_cache_flash_8bit(const void* key, const void* value, void* key_cache, void* value_cache,
                                               const void* slot_mapping, int slot_is_i64, int64_t num_tokens, int H, int D,
                                               int block_size, int64_t num_blocks, int64_t key_stride, int64_t value_stride,
                                               int64_t key_block_stride, int64_t value_block_stride, const float* k_scale,
                                               int64_t k_scale_stride, const float* v_scale, int64_t v_scale_stride,
                                               int dtype, int cache_format, void* stream) {
  FG_REQUIRE(num_tokens >= 0 && H >= 0 && D >= 0 && num_blocks >= 0, FG_ERR_INVALID, "reshape_and_cache_flash_8bit: negative size");
  FG_REQUIRE(block_size > 0, FG_ERR_INVALID, "reshape_and_cache_flash_8bit: block_size must be positive");
  FG_REQUIRE(dtype == FG_F16 || dtype == FG_BF16 || dtype == FG_F32, FG_ERR_INVALID, "reshape_and_cache_flash_8bit: dtype %d", dtype);
  FG_REQUIRE(cache_format == FG_CACHE_E4M3 || cache_format == FG_CACHE_E5M2, FG_ERR_INVALID,
             "reshape_and_cache_flash_8bit: cache format %d is not e4m3 or e5m2", cache_format);
  if (num_tokens == 0 || (int64_t)H * D == 0 || num_blocks == 0) return FG_OK;
  FG_REQUIRE(key && value && key_cache && value_cache && slot_mapping, FG_ERR_INVALID,
             "reshape_and_cache_flash_8bit: null pointer");
  FG_REQUIRE((int64_t)H * D < ((int64_t)1 << 30) && num_tokens < ((int64_t)1 << 29), FG_ERR_UNSUPPORTED,
             "reshape_and_cache_flash_8bit: problem too large for one launch");
  FG_REQUIRE(key_block_stride >= (int64_t)block_size * H * D && value_block_stride >= (int64_t)block_size * H * D, FG_ERR_INVALID,
             "reshape_and_cache_flash_8bit: block stride smaller than a page (%d x %d x %d)", block_size, H, D);
  FG_REQUIRE(scale_ok(k_scale, k_scale_stride) && scale_ok(v_scale, v_scale_stride), FG_ERR_INVALID,
             "reshape_and_cache_flash_8bit: a scale is one number (stride 0) or one for each head (stride 1)");
  WriteArgs a;
  a.src[0] = key, a.src[1] = value;
  a.cache[0] = (char*)key_cache, a.cache[1] = (char*)value_cache;
  a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.scale_stride[0] = k_scale_stride, a.scale_stride[1] = v_scale_stride;
  a.src_stride[0] = key_stride, a.src_stride[1] = value_stride;
  a.block_stride[0] = key_block_stride, a.block_stride[1] = value_block_stride;
  a.slots = slot_mapping;
  a.num_tokens = num_tokens;
  a.num_slots = num_blocks * block_size;
  a.row = H * D, a.D = D, a.block_size = block_size;
  hipStream_t st = (hipStream_t)stream;
#define FG_WRITE(T)                                                                        \
  return cache_format == FG_CACHE_E4M3 ? write_pieces<T, kE4M3>(a, slot_is_i64, st) \
                                       : write_pieces<T, kE5M2>(a, slot_is_i64, st)
  if (dtype == FG_F16) FG_WRITE(f16_t);
  if (dtype == FG_BF16) FG_WRITE(bf16_t);
  FG_WRITE(float);
#undef FG_WRITE
}

extern "C" int fg_gather_cache_flash(const void* key_cache, const void* value_cache, void* key, void* value,
                                     const int32_t* block_table, int64_t block_table_stride, int table_width,
                                     const int32_t* cu_seqlens, const int32_t* seq_starts, int batch, int64_t num_rows, int H,
                                     int D, int page_size, int64_t num_pages, int64_t key_page_stride,
                                     int64_t value_page_stride, int64_t key_stride, int64_t value_stride,
                                     const float* k_scale, int64_t k_scale_stride, const float* v_scale,
                                     int64_t v_scale_stride, int dtype, int cache_format, void* stream) {
  FG_REQUIRE(num_rows >= 0 && H >= 0 && D >= 0 && num_pages >= 0 && batch >= 0 && table_width >= 0, FG_ERR_INVALID,
             "gather_cache_flash: negative size");
  FG_REQUIRE(page_size > 0, FG_ERR_INVALID, "gather_cache_flash: page size must be positive");
  FG_REQUIRE(dtype == FG_F16 || dtype == FG_BF16 || dtype == FG_F32, FG_ERR_INVALID, "gather_cache_flash: dtype %d", dtype);
  FG_REQUIRE(cache_format == FG_CACHE_SAME || cache_format == FG_CACHE_E4M3 || cache_format == FG_CACHE_E5M2, FG_ERR_INVALID,
             "gather_cache_flash: cache format %d", cache_format);
  if (num_rows == 0 || batch == 0 || (int64_t)H * D == 0) return FG_OK;
  FG_REQUIRE(key_cache && value_cache && key && value && block_table && cu_seqlens, FG_ERR_INVALID,
             "gather_cache_flash: null pointer");
  FG_REQUIRE((int64_t)H * D < ((int64_t)1 << 30), FG_ERR_UNSUPPORTED, "gather_cache_flash: problem too large for one launch");
  FG_REQUIRE(num_pages > 0, FG_ERR_INVALID, "gather_cache_flash: the cache has no pages");  // (there is nothing that could be read)
  FG_REQUIRE(key_page_stride >= (int64_t)page_size * H * D && value_page_stride >= (int64_t)page_size * H * D, FG_ERR_INVALID,
             "gather_cache_flash: page stride smaller than a page (%d x %d x %d)", page_size, H, D);
  FG_REQUIRE(key_stride >= (int64_t)H * D && value_stride >= (int64_t)H * D, FG_ERR_INVALID,
             "gather_cache_flash: row stride smaller than a row (%d x %d)", H, D);
  FG_REQUIRE(scale_ok(k_scale, k_scale_stride) && scale_ok(v_scale, v_scale_stride), FG_ERR_INVALID,
             "gather_cache_flash: a scale is one number (stride 0) or one for each head (stride 1)");
  const int eb = cache_format == FG_CACHE_SAME ? (dtype == FG_F32 ? 4 : 2) : 1;
  ReadArgs a;
  a.cache[0] = (const char*)key_cache, a.cache[1] = (const char*)value_cache;
  a.out[0] = (char*)key, a.out[1] = (char*)value;
  a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.scale_stride[0] = k_scale_stride, a.scale_stride[1] = v_scale_stride;
  a.page_stride[0] = key_page_stride * eb, a.page_stride[1] = value_page_stride * eb;
  a.out_stride[0] = key_stride, a.out_stride[1] = value_stride;
  a.table = block_table, a.table_stride = block_table_stride, a.table_width = table_width;
  a.cu = cu_seqlens, a.first = seq_starts;
  a.num_rows = num_rows, a.num_pages = num_pages;
  a.batch = batch, a.row = H * D, a.D = D, a.page_size = page_size;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == FG_F16) return read_formats<f16_t>(a, cache_format, st);
  if (dtype == FG_BF16) return read_formats<bf16_t>(a, cache_format, st);
  return read_formats<float>(a, cache_format, st);
}
