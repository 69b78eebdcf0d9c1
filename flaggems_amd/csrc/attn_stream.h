// Attention of a few query rows over a long paged cache: single tokens (decode), a few proposed tokens, and any batch
// that no other kernel takes.
//
// Rows.  The query tokens of a sequence and the G = Hq / Hk query heads that share a KV head form rows r = token * G + g;
// a workgroup takes R = 16 * NQ of them (a row block) for one (sequence, KV head, key range), so that every byte of the
// cache is read once for up to R rows.
//
// Keys.  The keys that some row of the block may see are [lo, hi) and, in front of them, the first `sinks` ones.  They are
// walked in tiles of 32 keys: first the tiles of the sinks (where lo lies behind them), then those of [lo, hi); what lies
// between is not touched, neither its keys nor its entries of the block table.  A sequence's tiles are dealt out over
// `splits` key ranges (grid x), the tiles of a range to the four waves in turn; each wave keeps its own running maximum,
// sum and output, merged through LDS at the end, and a second kernel merges the ranges.
//
// Products, transposed so that a lane owns one query row (lane % 16) and four lanes share it:
//   S^T[key, r] = K[key, :] . Q[r, :]     A: lane (m, g) holds elements of one key row, B: lane (n, g) of query row n;
//   O^T[d, r] += V^T[d, key] . P^T[key, r].
// Both operands come from global memory straight into registers: no LDS, no barrier in the loop.
//   K: MFMA row m of half tile t is key (m / 4) * 8 + t * 4 + m % 4, so the accumulators of lane (r, g) are the scores of
//      keys g * 8 + 0..7: exactly the k-slots that lane supplies to the second product.  P never moves between lanes.
//   V: lane (i, g) loads, for keys g * 8 + 0..7, the same VC = DP / 16 consecutive elements d = i * VC + j.  An 8 x VC
//      transpose inside the lane (v_perm) makes fragment j: keys g * 8 + 0..7 of element i * VC + j.  Output sub-tile j
//      then holds elements j, VC + j, 2 VC + j, ...: a permutation that the epilogue undoes for free, since a lane ends
//      with consecutive elements.
// 8-bit caches: v_cvt_scalef32_pk_{bf16,f16}_{fp8,bf8} widens two elements at a time; every e4m3 and e5m2 value is exact in
// bf16 and in fp16.  The scale of K goes into the softmax scale, the scale of V into the last division.
//
// Softmax in base 2, fp32 statistics; the reference maximum follows the true one only when a score exceeds it by 2^8.
// P is rounded to the query type for the second product, as is usual; the sum is taken before the rounding.
//
// What is masked: keys past the sequence, causal and window bounds by row.  K of a key that no row of the block sees is read
// from a visible key's place instead; its V is replaced by zero (0 * NaN would be NaN).  Rows that see nothing give
// out = 0, lse = +inf.  A block table entry that names no page of the cache makes the rows that need it NaN.
//
// Bound: HBM (2 * D bytes a key for 8 bits, against 4 * D * rows flop).
#pragma once

constexpr int kTile = 32;  // keys per tile

// Tiles per key range: the tiles spread over all ranges, a multiple of the four waves, at least min_tiles.
__device__ __forceinline__ int range_tiles(const CacheAttnArgs& a, int tiles) {
  int t = ((tiles + a.splits - 1) / a.splits + 3) & ~3;
  return t < a.min_tiles && a.splits > 1 ? a.min_tiles : t;
}

// NARROW: pages of a size that is not a multiple of 8 keys (every key looks its page up).
template <typename T, int FMT, int DP, int NQ, bool NARROW>
__global__ __launch_bounds__(256, 2) void attn_stream_kernel(CacheAttnArgs a) {
  typedef typename Mma16<T>::Frag Frag;
  constexpr bool WIDE = FMT == FG_CACHE_SAME;    // the cache holds T
  constexpr int EB = WIDE ? 2 : 1;               // bytes of a cached element
  constexpr int KS = DP / 32;                    // k-steps of the first product
  constexpr int EPL = 16 / EB;                   // elements of a 16-byte load
  constexpr int KL = DP / (4 * EPL);             // 16-byte loads per key row and lane
  constexpr int VC = DP / 16;                    // elements of a value row per lane = output sub-tiles
  constexpr int VW = VC * EB / 4;                // 32-bit words of them
  // 16-bit rows of 256 elements do not fit in the registers while the others are at work: keys and values are loaded where
  // they are used, values 16 bytes a lane at a time
  constexpr bool LATE = WIDE && DP == 256;
  constexpr int VP = LATE ? 2 : 1;             // parts of a value row
  constexpr int VWP = VW / VP;                   // words of a part
  constexpr int R = 16 * NQ;
  constexpr int EH = DP == 256 ? 2 : 4;          // accumulator elements merged at once
  constexpr int MD = 16 * VC * EH / 4;           // row elements merged at once: DP, or half of 256
  constexpr int PITCH = MD + 4;
  __shared__ float part[4 * 16 * PITCH];         // [wave][row][element]
  __shared__ float ml[4 * 16 * 2];               // [wave][row]: maximum, sum

  const FgFlashParams& p = a.p.base;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rl = lane & 15, g = lane >> 4;       // row / key / element index of the lane, its group
  const int b = blockIdx.y, kvh = blockIdx.z;
  const int G = a.group;
  // rotated per (sequence, head): workgroups go round-robin to the XCDs, and short sequences fill the first ranges only
  const int split = (int)((blockIdx.x + (unsigned)(b * 5 + kvh * 3)) % (unsigned)a.splits);
  const int row0 = (int)(blockIdx.x / (unsigned)a.splits) * R;

  const int q_bos = p.cu_seqlens_q[b];
  const int q_len = p.cu_seqlens_q[b + 1] - q_bos;
  const int rows = q_len * G;
  if (q_len < a.min_q || q_len > a.max_q || row0 >= rows) return;
  if (q_bos < 0 || (int64_t)q_bos + q_len > p.total_q) return;
  // a sequence longer than its row of the block table: nothing is read behind the row, its output is NaN
  const int64_t reach = (int64_t)a.p.table_width * p.page_size;
  const int k_said = p.seqused_k[b];
  const int k_len = k_said < 0 ? 0 : (k_said < reach ? k_said : (int)reach);
  const int last_row = row0 + R < rows ? row0 + R - 1 : rows - 1;
  const Seen seen = seen_by<kTile>(a, q_len, k_len, row0 / G, last_row / G);
  const int per = range_tiles(a, seen.tiles);
  const int t_begin = split * per;
  const int t_end = t_begin + per < seen.tiles ? t_begin + per : seen.tiles;
  if (split > 0 && t_begin >= t_end) return;     // range 0 always reports

  // ---- query rows: lane (r, g), step s holds elements of the same place as the key fragments below ------------------------
  int lo_r[NQ], hi_r[NQ];                        // keys the lane's row sees: [lo_r, hi_r) and [0, min(sinks, hi_r))
  Frag qf[NQ][KS];
  const int D = p.D;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = row0 + n * 16 + rl;
    const bool ok = row < rows;
    const int tok = (ok ? row : row0) / G, head = kvh * G + (ok ? row : row0) % G;
    row_bounds(a, q_len, k_len, tok, lo_r[n], hi_r[n]);
    const T* q = (const T*)p.q + (int64_t)(q_bos + tok) * p.q_row_stride + (int64_t)head * p.q_head_stride;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = WIDE ? s * 32 + g * 8 : (s >> 1) * 64 + g * 16 + (s & 1) * 8;
      u32x4 v = {0u, 0u, 0u, 0u};
      if (ok && d < D) v = *reinterpret_cast<const u32x4*>(q + d);
      qf[n][s] = __builtin_bit_cast(Frag, v);
    }
  }
  f32x4 acc[NQ][VC];
  float m_run[NQ], l_run[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m_run[n] = -INFINITY, l_run[n] = 0.f;
#pragma unroll
    for (int j = 0; j < VC; ++j) acc[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const float k_scale = seq_scale(a.p.k_scale, a.p.k_scale_batch_stride, a.p.k_scale_head_stride, b, kvh);
  const float sc = a.scale_log2 * k_scale, cap_in = a.cap_in * k_scale;
  const bool capped = p.softcap > 0.f;
  const char* const kbase = (const char*)p.k_cache + (int64_t)kvh * p.k_head_stride * EB;
  const char* const vbase = (const char*)p.v_cache + (int64_t)kvh * p.v_head_stride * EB;
  const int32_t* const table = p.block_table + (int64_t)b * p.block_table_stride;
  bool bad = k_said > reach;                     // or a page that the cache does not have was asked for

  // a key that some row of the block sees
  auto any_sees = [&](int key) { return key < seen.hi && (key >= seen.lo || key < seen.sinks); };
  // the group of 8 keys that starts at `key`, or one that is seen where none of them is
  auto usable = [&](int key) {
    const bool some = key < seen.hi && (key + 8 > seen.lo || key < seen.sinks);
    return some ? key : (seen.hi - 1) & ~7;
  };
  auto checked = [&](int page) {
    const bool ok = (uint32_t)page < (uint32_t)a.p.num_pages;
    bad |= !ok;
    return ok ? page : 0;
  };

  u32x4 xk[2][KL];                               // the wave's tile
  uint32_t xv[8][VWP];
  const int kg = rl >> 2;                        // K: the lane's group of 8 keys
  // byte offsets of the lane's pieces inside a row; pieces past the head dim read the row's start (K: zeroed, V: not stored)
  int k_at[KL];
#pragma unroll
  for (int c = 0; c < KL; ++c) {
    const int d = (c * 4 + g) * EPL;
    k_at[c] = d < D ? d * EB : 0;
  }
  const bool ragged = D < DP;
  const int v_at = rl * VC < D ? rl * VC * EB : 0;
  const int v_second = rl * VC + 8 < D ? 16 : 0;  // second part of a value row, where it lies inside the row

  auto load_words = [](uint32_t (&dst)[VWP], const char* src) {
    if constexpr (VWP == 1) {
      dst[0] = __builtin_nontemporal_load((const uint32_t*)src);
    } else if constexpr (VWP == 2) {
      const u32x2 w = __builtin_nontemporal_load((const u32x2*)src);
      dst[0] = w[0], dst[1] = w[1];
    } else {
      const u32x4 w = __builtin_nontemporal_load((const u32x4*)src);
      dst[0] = w[0], dst[1] = w[1], dst[2] = w[2], dst[3] = w[3];
    }
  };

  const int64_t krow = p.k_row_stride * EB, vrow = p.v_row_stride * EB;
  auto place = [&](int key, const char* base, int64_t page_stride, int64_t row) {  // of one key (NARROW)
    const int k = any_sees(key) ? key : seen.hi - 1;
    const int pg = page_of(a, k);
    return base + checked(table[pg]) * page_stride * EB + (k - pg * p.page_size) * row;
  };
  auto load_k = [&](int key0, int page) {
    const int k = usable(key0 + kg * 8);
    const char* at = kbase + checked(page) * p.k_page_stride * EB + (k - page_of(a, k) * p.page_size + (rl & 3)) * krow;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (NARROW) at = place(key0 + kg * 8 + t * 4 + (rl & 3), kbase, p.k_page_stride, krow);
#pragma unroll
      for (int c = 0; c < KL; ++c) xk[t][c] = __builtin_nontemporal_load((const u32x4*)(at + k_at[c]));
      if constexpr (!NARROW) at += 4 * krow;
    }
  };
  auto load_v = [&](int key0, int page, int vp) {
    const int k = usable(key0 + g * 8);
    const char* at = vbase + checked(page) * p.v_page_stride * EB + (k - page_of(a, k) * p.page_size) * vrow + v_at + vp * v_second;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (NARROW) at = place(key0 + g * 8 + j, vbase, p.v_page_stride, vrow) + v_at + vp * v_second;
      load_words(xv[j], at);
      if constexpr (!NARROW) at += vrow;
    }
  };

  // ---- the wave's tiles.  The keys of the next tile are requested as soon as the scores have taken those of this one, its
  // values as soon as the output has: one tile in flight per wave and one set of registers for it; the page numbers of a
  // tile are requested two tiles ahead. ---------------------------------------------------------------------------------
  auto page_at = [&](int t, int group) -> int {
    if constexpr (NARROW) return 0;
    return table[page_of(a, usable(tile_key<kTile>(seen, t < t_end ? t : t_end - 1) + group * 8))];
  };
  int t = t_begin + wave;
  int k_page = 0, v_page = 0, k_now = 0, v_now = 0;
  if (t < t_end) {
    const int kp = page_at(t, kg), vp = page_at(t, g);
    k_page = page_at(t + 4, kg), v_page = page_at(t + 4, g);
    if constexpr (!LATE) {
      load_k(tile_key<kTile>(seen, t), kp);
      load_v(tile_key<kTile>(seen, t), vp, 0);
    }
    k_now = kp, v_now = vp;
  }
  for (; t < t_end; t += 4) {
    const int key0 = tile_key<kTile>(seen, t), key1 = tile_key<kTile>(seen, t + 4 < t_end ? t + 4 : t);
    const bool more = t + 4 < t_end;
    const int k_page2 = page_at(t + 8, kg), v_page2 = page_at(t + 8, g);
    // a tile that every row sees in full needs no mask
    bool full = true;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
      full = full && key0 + kTile <= hi_r[n] && (key0 >= lo_r[n] || key0 + kTile <= seen.sinks);
    full = __builtin_amdgcn_ballot_w64(full) == ~0ull;
    if constexpr (LATE) load_k(key0, k_now);
    if (ragged) {
#pragma unroll
      for (int c = 0; c < KL; ++c)
        if ((c * 4 + g) * EPL >= D) xk[0][c] = xk[1][c] = u32x4{0u, 0u, 0u, 0u};
    }
    // ---- scores -----------------------------------------------------------------------------------------------------
    f32x4 s[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) s[n][0] = s[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        u32x4 w;
        if constexpr (WIDE) {
          w = xk[t][st];
        } else {
          const u32x4 raw = xk[t][st >> 1];
          const uint32_t r0 = raw[(st & 1) * 2], r1 = raw[(st & 1) * 2 + 1];
          w = u32x4{Widen<T, FMT>::template two<false>(r0), Widen<T, FMT>::template two<true>(r0),
                    Widen<T, FMT>::template two<false>(r1), Widen<T, FMT>::template two<true>(r1)};
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][t] = Mma16<T>::mma(__builtin_bit_cast(Frag, w), qf[n][st], s[n][t]);
      }
    if constexpr (!LATE)
      if (more) load_k(key1, k_page);
    // ---- softmax: element e of half t is key key0 + g * 8 + t * 4 + e ---------------------------------------------------
    Frag pf[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = s[n][e >> 2][e & 3];
      if (capped) {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = a.cap_out_log2 * tanhf(z[e] * cap_in);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] *= sc;
      }
      if (!full) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = key0 + g * 8 + e;
          const bool sees = key < hi_r[n] && (key >= lo_r[n] || key < seen.sinks);
          z[e] = sees ? z[e] : -INFINITY;
        }
      }
      float top = z[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, z[e]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const bool moved = top > m_run[n] + 8.0f;
      const float m_new = moved ? top : m_run[n];
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      T pr[8];
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = __builtin_amdgcn_exp2f(z[e] - m_use);
        sum += v;
        pr[e] = (T)v;
      }
      pf[n] = *reinterpret_cast<Frag*>(pr);
      if (__builtin_amdgcn_ballot_w64(moved) != 0) {
        const float alpha = moved ? __builtin_amdgcn_exp2f(m_run[n] - m_use) : 1.0f;
        l_run[n] *= alpha;
#pragma unroll
        for (int j = 0; j < VC; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][j][e] *= alpha;
      }
      l_run[n] += sum;                           // of the lane's own keys; the four lanes of a row meet at the end
      m_run[n] = m_new;
    }
    // ---- output: words of 2 elements per key -> fragments of 8 keys per element -----------------------------------------
#pragma unroll
    for (int vp = 0; vp < VP; ++vp) {
      if constexpr (LATE) load_v(key0, v_now, vp);
      if (!full) {  // values of keys that no row sees: zero
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!any_sees(key0 + g * 8 + j)) {
#pragma unroll
            for (int w = 0; w < VWP; ++w) xv[j][w] = 0u;
          }
      }
#pragma unroll
      for (int hp = 0; hp < VC / 2 / VP; ++hp) {
        const int h = vp * (VC / 2 / VP) + hp;
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (WIDE) w[j] = xv[j][hp];
          else if (hp & 1) w[j] = Widen<T, FMT>::template two<true>(xv[j][hp >> 1]);
          else w[j] = Widen<T, FMT>::template two<false>(xv[j][hp >> 1]);
        }
        u32x4 f0, f1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f0[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x05040100);
          f1[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302);
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          acc[n][2 * h] = Mma16<T>::mma(__builtin_bit_cast(Frag, f0), pf[n], acc[n][2 * h]);
          acc[n][2 * h + 1] = Mma16<T>::mma(__builtin_bit_cast(Frag, f1), pf[n], acc[n][2 * h + 1]);
        }
      }
    }
    if constexpr (!LATE)
      if (more) load_v(key1, v_page, 0);
    k_now = k_page, v_now = v_page;
    k_page = k_page2, v_page = v_page2;
  }
  const bool broken = __builtin_amdgcn_ballot_w64(bad) != 0;

  // ---- merge of the four waves: 16 rows at a time -------------------------------------------------------------------------
  const float v_scale = seq_scale(a.p.v_scale, a.p.v_scale_batch_stride, a.p.v_scale_head_stride, b, kvh);
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int live = rows - (row0 + n * 16) < 16 ? rows - (row0 + n * 16) : 16;
    if (live <= 0) break;                              // (the same for all waves)
    float l = l_run[n];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (broken) l = NAN;
#pragma unroll
    for (int e0 = 0; e0 < 4; e0 += EH) {
      if (n > 0 || e0 > 0) __syncthreads();
      if (g == 0 && e0 == 0) {
        ml[(wave * 16 + rl) * 2] = m_run[n];
        ml[(wave * 16 + rl) * 2 + 1] = l;
      }
#pragma unroll
      for (int e = 0; e < EH; ++e)                     // element (g * 4 + e0 + e) * VC + j of the row
#pragma unroll
        for (int j = 0; j < VC; ++j) part[(wave * 16 + rl) * PITCH + (g * EH + e) * VC + j] = acc[n][j][e0 + e];
      __syncthreads();
      for (int i = tid; i < live * MD; i += 256) {
        const int r = i / MD, x = i - r * MD;
        const int d = (x / (EH * VC) * 4 + e0) * VC + x % (EH * VC);
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[(w * 16 + r) * 2]);
        const float m_use = m == -INFINITY ? 0.f : m;
        float sum = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float f = __builtin_amdgcn_exp2f(ml[(w * 16 + r) * 2] - m_use);
          sum += ml[(w * 16 + r) * 2 + 1] * f;
          o += part[(w * 16 + r) * PITCH + x] * f;
        }
        const int row = row0 + n * 16 + r;
        const int tok = row / G, head = kvh * G + row % G;
        if (a.splits == 1) {
          const bool empty = sum == 0.f;
          if (d < D)
            ((T*)p.out)[(int64_t)(q_bos + tok) * p.o_row_stride + (int64_t)head * p.o_head_stride + d] =
                (T)(empty ? 0.f : o * (v_scale / sum));
          if (d == 0 && p.lse != nullptr)
            p.lse[(int64_t)head * p.total_q + q_bos + tok] = empty ? INFINITY : m_use * 0.6931471805599453f + logf(sum);
        } else {
          const int64_t at = (((int64_t)split * p.batch + b) * a.max_q + tok) * p.Hq + head;
          a.part_o[at * DP + d] = o;
          if (d == 0) a.part_ml[at * 2] = m, a.part_ml[at * 2 + 1] = sum;
        }
      }
    }
  }
}

// Merges the key ranges: one thread per (sequence, token, head, element).
template <typename T, int DP, int NQ>
__global__ __launch_bounds__(256) void attn_stream_merge_kernel(CacheAttnArgs a) {
  const FgFlashParams& p = a.p.base;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int d = (int)(i % DP);
  const int64_t bth = i / DP;
  const int head = (int)(bth % p.Hq);
  const int tok = (int)(bth / p.Hq % a.max_q);
  const int64_t b64 = bth / p.Hq / a.max_q;
  if (b64 >= p.batch) return;
  const int b = (int)b64;
  const int q_bos = p.cu_seqlens_q[b];
  const int q_len = p.cu_seqlens_q[b + 1] - q_bos;
  if (q_len < a.min_q || q_len > a.max_q || tok >= q_len || d >= p.D) return;
  if (q_bos < 0 || (int64_t)q_bos + q_len > p.total_q) return;
  const int64_t reach = (int64_t)a.p.table_width * p.page_size;
  const int k_said = p.seqused_k[b];
  const int k_len = k_said < 0 ? 0 : (k_said < reach ? k_said : (int)reach);
  // the ranges of the row's block that were written
  const int row = tok * a.group + head % a.group;
  const int row0 = row / (16 * NQ) * (16 * NQ), rows = q_len * a.group;
  const int last_row = row0 + 16 * NQ < rows ? row0 + 16 * NQ - 1 : rows - 1;
  const Seen seen = seen_by<kTile>(a, q_len, k_len, row0 / a.group, last_row / a.group);
  const int per = range_tiles(a, seen.tiles);
  int ns = per > 0 ? (seen.tiles + per - 1) / per : 1;
  ns = ns < 1 ? 1 : (ns > a.splits ? a.splits : ns);
  const int64_t step = (int64_t)p.batch * a.max_q * p.Hq, at = ((int64_t)b * a.max_q + tok) * p.Hq + head;
  float m = -INFINITY;
  for (int s = 0; s < ns; ++s) m = fmaxf(m, a.part_ml[(s * step + at) * 2]);
  const float m_use = m == -INFINITY ? 0.f : m;
  float l = 0.f, o = 0.f;
  for (int s = 0; s < ns; ++s) {
    const float f = __builtin_amdgcn_exp2f(a.part_ml[(s * step + at) * 2] - m_use);
    l += a.part_ml[(s * step + at) * 2 + 1] * f;
    o += a.part_o[(s * step + at) * DP + d] * f;
  }
  const bool empty = l == 0.f;
  const float v_scale = seq_scale(a.p.v_scale, a.p.v_scale_batch_stride, a.p.v_scale_head_stride, b, head / a.group);
  ((T*)p.out)[(int64_t)(q_bos + tok) * p.o_row_stride + (int64_t)head * p.o_head_stride + d] =
      (T)(empty ? 0.f : o * (v_scale / l));
  if (d == 0 && p.lse != nullptr)
    p.lse[(int64_t)head * p.total_q + q_bos + tok] = empty ? INFINITY : m_use * 0.6931471805599453f + logf(l);
}

template <typename T, int FMT, int DP, int NQ, bool NARROW>
int launch_stream(const CacheAttnArgs& a, hipStream_t st) {
  const FgFlashParams& p = a.p.base;
  const int64_t blocks = fg_cdiv((int64_t)a.max_q * a.group, 16 * NQ) * a.splits;
  FG_REQUIRE(blocks < ((int64_t)1 << 31), FG_ERR_UNSUPPORTED, "cache_attn_fwd: too many query rows for one launch");
  hipLaunchKernelGGL((attn_stream_kernel<T, FMT, DP, NQ, NARROW>), dim3((unsigned)blocks, (unsigned)p.batch, (unsigned)p.Hk),
                     dim3(256), 0, st, a);
  if (a.splits > 1) {
    const int64_t total = (int64_t)p.batch * a.max_q * p.Hq * DP;
    hipLaunchKernelGGL((attn_stream_merge_kernel<T, DP, NQ>), dim3((unsigned)fg_cdiv(total, 256)), dim3(256), 0, st, a);
  }
  return fg_check_launch("cache_attn_fwd");
}
