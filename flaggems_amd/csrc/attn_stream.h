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
//      transpose inside the lane (v_perm, in front of the widening) makes fragment j: keys g * 8 + 0..7 of element i * VC + j.  Output sub-tile j
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
// Bound: HBM (2 * D bytes a key for 8 bits, against 4 * D * rows flop; without its arithmetic the loop takes the same time).
// 32/8 heads of 128, one token: 64 sequences of 4096 keys, e4m3, 98 us = 5.5 TB/s; 256 of them 326 = 6.6; three of 131072 keys at most,
// in ranges, 102 us and 5 for the merge = 5.4 TB/s; 128 of 4096, 16 bits, 329 = 6.5 (a large copy on this card: 4.8 to 5.4).  Head
// dim 256, 64 of 4096: e4m3 179 us = 6.0 TB/s, 16 bits (loaded where they are used) 459 = 4.7.  Chunks of head dims above 128 come
// here too and read the keys again for every 16 rows: 1024 tokens over 8192, dim 256, 744 us = 0.35 PFLOP/s, 16 bits 2.65 ms = 0.10.
// One workgroup draws 22 to 28 GB/s on its own, with four waves or eight: a short sequence is bound by that and by the trips
// to memory one after another (lengths and table, keys, output), 12 us for 513 keys in 8 workgroups.
// What the loads are made of decides: 32 bytes a lane at a stretch, in place of whole 128-byte lines, cost a fifth.
#pragma once

constexpr int kTile = 32;  // keys per tile

// How a wave finds the pages of a tile.
enum {
  kHalves,  // power-of-two pages of at least 16 keys: half a tile lies in one page; table entries and page addresses are scalar
  kGroups,  // pages of a multiple of 8 keys: a lane looks up its group of 8 keys
  kKeys,    // any page size: a lane looks up each of its keys
};

template <typename T, int FMT, int DP, int NQ, int PAGES>
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
  // tiles in flight per wave: two where the registers of a wave (256 at two waves per SIMD) hold them
  constexpr int NB = DP == 256 || (DP == 128 && (WIDE || NQ == 2)) ? 1 : 2;
  // Loads that take whole 128-byte lines, eight rows at a time: one lane bit then says which piece of the row the lane holds
  // where the fragment wants it to say which row, and the two loads of a pair exchange halves (swap_half_rows).
  constexpr bool SWAP_K = KL >= 2, SWAP_V = VW <= 2;
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

  const Sequence seq = sequence(a, b, kvh);
  const int q_bos = seq.q_bos, q_len = seq.q_len, k_len = seq.k_len;
  const int rows = q_len * G;
  if (!seq.mine || row0 >= rows) return;
  const int last_row = row0 + R < rows ? row0 + R - 1 : rows - 1;
  const Seen seen = seen_by<kTile>(a, q_len, k_len, row0 / G, last_row / G);
  const int per = range_tiles<4>(a, seen.tiles);
  const int t_begin = split * per;
  const int t_end = t_begin + per < seen.tiles ? t_begin + per : seen.tiles;
  if (split > 0 && t_begin >= t_end) return;     // range 0 always reports

  // ---- query rows: lane (r, g), step s holds elements of the same place as the key fragments below ------------------------
  // t = sc * S with sc > 0, so that the largest t is sc times the largest S: the sign goes into the query (0: a query of 0)
  const bool capped = p.softcap > 0.f;
  const float given = (capped ? a.cap_in : a.scale_log2) * seq.k_scale;
  const uint32_t q_keep = given == 0.f ? 0u : ~0u, q_flip = given < 0.f ? 0x80008000u : 0u;
  const float inner = given == 0.f ? 1.0f : fabsf(given);
  const float sc = capped ? a.cap_out_log2 : inner;  // of S, or of tanh(inner * S)
  int lo_r[NQ], hi_r[NQ];                        // keys the lane's row sees: [lo_r, hi_r) and [0, min(sinks, hi_r))
  u32x4 q_raw[NQ][KS];
  uint32_t q_mask[NQ];
  const int D = p.D;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = row0 + n * 16 + rl;
    const bool ok = row < rows;
    q_mask[n] = ok ? q_keep : 0u;
    const int tok = (ok ? row : row0) / G, head = kvh * G + (ok ? row : row0) % G;
    row_bounds(a, q_len, k_len, tok, lo_r[n], hi_r[n]);
    const T* q = (const T*)p.q + (int64_t)(q_bos + tok) * p.q_row_stride + (int64_t)head * p.q_head_stride;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = WIDE ? s * 32 + g * 8 : (s >> 1) * 64 + g * 16 + (s & 1) * 8;
      q_raw[n][s] = *reinterpret_cast<const u32x4*>(q + (d < D ? d : 0));  // (made a fragment behind the first tile's loads)
    }
  }
  auto q_inside = [&](int s) { return (WIDE ? s * 32 + g * 8 : (s >> 1) * 64 + g * 16 + (s & 1) * 8) < D; };
  f32x4 acc[NQ][VC];
  float m_run[NQ], l_run[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m_run[n] = -INFINITY, l_run[n] = 0.f;
#pragma unroll
    for (int j = 0; j < VC; ++j) acc[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const char* const kbase = (const char*)p.k_cache + (int64_t)kvh * p.k_head_stride * EB;
  const char* const vbase = (const char*)p.v_cache + (int64_t)kvh * p.v_head_stride * EB;
  const int32_t* const table = p.block_table + (int64_t)b * p.block_table_stride;
  bool bad = seq.too_long, bad_half = false;     // or a page that the cache does not have was asked for

  // a key that some row of the block sees
  auto any_sees = [&](int key) { return (key < seen.hi) & ((key >= seen.lo) | (key < seen.sinks)); };
  // the group of 8 keys that starts at `key`, or one that is seen where none of them is
  auto usable = [&](int key) {
    const bool some = (key < seen.hi) & ((key + 8 > seen.lo) | (key < seen.sinks));
    return some ? key : (seen.hi - 1) & ~7;
  };
  auto checked = [&](int page) {
    const bool ok = (uint32_t)page < (uint32_t)a.p.num_pages;
    bad |= !ok;
    return ok ? page : 0;
  };

  u32x4 xk[NB][2][KL];                           // the wave's tiles, as loaded
  uint32_t xv[NB][8][VWP];
  // the group of 8 keys of the lane's MFMA row (SWAP_K: of its row in the first load of a pair; in the second, two further)
  const int kg = SWAP_K ? (rl >> 2) & 1 : rl >> 2;
  // byte offsets of the lane's pieces inside a row; pieces past the head dim read the row's start (K: zeroed, V: not stored)
  int k_at[KL];
#pragma unroll
  for (int c = 0; c < KL; ++c) {
    const int d = SWAP_K ? (((c & ~1) + ((rl >> 3) & 1)) * 4 + g) * EPL : (c * 4 + g) * EPL;
    k_at[c] = d < D ? d * EB : 0;
  }
  const bool ragged = D < DP;
  const int v_first = SWAP_V ? (rl & 7) * 2 * VC : rl * VC;  // first element that the lane loads of a value row
  const int v_at = v_first < D ? v_first * EB : 0;
  const int v_second = v_first + 8 < D ? 16 : 0;  // second part of a value row, where it lies inside the row

  const int64_t krow = p.k_row_stride * EB, vrow = p.v_row_stride * EB;
  const int64_t kpage = p.k_page_stride * EB, vpage = p.v_page_stride * EB;
  auto place = [&](int key, const char* base, int64_t page_stride, int64_t row) {  // of one key (kKeys)
    const int k = any_sees(key) ? key : seen.hi - 1;
    const int pg = page_of(a, k);
    return base + checked(table[pg]) * page_stride + (k - pg * p.page_size) * row;
  };
  // kHalves: the 16 keys from `key` on, or 16 of which one is seen (scalar)
  const int half_mask = p.page_size - 1;
  auto usable_half = [&](int key) {
    const bool some = (key < seen.hi) & ((key + 16 > seen.lo) | (key < seen.sinks));
    return some ? key : (seen.hi - 1) & ~15;
  };
  // page numbers of a tile.  kHalves: of its halves (scalar); kGroups: of the lane's groups for K (SWAP_K: two) and V
  struct Pages {
    int a, b, c;
  };
  typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
  // Tiles past the wave's last one are the range's last one again: loads are never skipped, so that the waits of the loop are
  // for the loads they mean and not for all of them.
  auto key_of = [&](int t) { return tile_key<kTile>(seen, t < t_end ? t : t_end - 1); };
  auto pages_of = [&](int t) {
    const int key0 = key_of(t);
    if constexpr (PAGES == kHalves) {
      const scalar_ptr entries = (scalar_ptr)(uintptr_t)table;
      return Pages{entries[usable_half(key0) >> a.page_bits], entries[usable_half(key0 + 16) >> a.page_bits], 0};
    } else if constexpr (PAGES == kGroups) {
      return Pages{table[page_of(a, usable(key0 + kg * 8))], SWAP_K ? table[page_of(a, usable(key0 + (kg + 2) * 8))] : 0,
                   table[page_of(a, usable(key0 + g * 8))]};
    } else {
      return Pages{0, 0, 0};
    }
  };
  auto half_at = [&](int key, int page, int64_t page_stride, int64_t row) {
    const bool ok = (uint32_t)page < (uint32_t)a.p.num_pages;
    bad_half |= !ok;
    return (ok ? page : 0) * page_stride + (usable_half(key) & half_mask) * row;
  };
  // the lane's row in its half tile (kHalves) or in its group
  const int64_t k_lane = ((PAGES == kHalves ? (kg & 1) * 8 : 0) + (rl & 3)) * krow;
  const int v_bit = SWAP_V ? (rl >> 3) & 1 : 0;  // SWAP_V: which key of a pair the lane loads
  const int64_t v_lane = ((PAGES == kHalves ? (g & 1) * 8 : 0) + v_bit) * vrow + v_at;
  auto group_at = [&](int key, int page, int64_t page_stride, int64_t row) {
    const int k = usable(key);
    return checked(page) * page_stride + (k - page_of(a, k) * p.page_size) * row;
  };
  auto load_k = [&](u32x4 (&x)[2][KL], int key0, Pages pg) {
    int64_t at[SWAP_K ? 2 : 1];                  // of the lane's row in half tile 0, for the loads of a pair
    if constexpr (PAGES == kHalves) {
      const int64_t h0 = half_at(key0, pg.a, kpage, krow), h1 = half_at(key0 + 16, pg.b, kpage, krow);
      if constexpr (SWAP_K) at[0] = h0, at[1] = h1;
      else at[0] = kg >= 2 ? h1 : h0;
    } else if constexpr (PAGES == kGroups) {
      at[0] = group_at(key0 + kg * 8, pg.a, kpage, krow);
      if constexpr (SWAP_K) at[1] = group_at(key0 + (kg + 2) * 8, pg.b, kpage, krow);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < (SWAP_K ? 2 : 1); ++i) {
        const char* row;
        if constexpr (PAGES == kKeys) row = place(key0 + (kg + 2 * i) * 8 + t * 4 + (rl & 3), kbase, kpage, krow);
        else row = kbase + at[i] + (k_lane + t * 4 * krow);
#pragma unroll
        for (int c = i; c < KL; c += SWAP_K ? 2 : 1) x[t][c] = __builtin_nontemporal_load((const u32x4*)(row + k_at[c]));
      }
  };
  auto load_v = [&](uint32_t (&x)[8][VWP], int key0, Pages pg, int vp) {
    int64_t at = 0;
    if constexpr (PAGES == kHalves) {
      const int64_t h0 = half_at(key0, pg.a, vpage, vrow), h1 = half_at(key0 + 16, pg.b, vpage, vrow);
      at = g >= 2 ? h1 : h0;
    } else if constexpr (PAGES == kGroups) {
      at = group_at(key0 + g * 8, pg.c, vpage, vrow);
    }
    const char* row = vbase + at + (v_lane + vp * v_second);
#pragma unroll
    for (int j = 0; j < 8; j += SWAP_V ? 2 : 1) {
      if constexpr (PAGES == kKeys) row = place(key0 + g * 8 + j + v_bit, vbase, vpage, vrow) + v_at + vp * v_second;
      constexpr int W = SWAP_V ? 2 * VWP : VWP;  // words of the load: two blocks of the row, or one
      uint32_t w[W];
      if constexpr (W == 2) *reinterpret_cast<u32x2*>(w) = __builtin_nontemporal_load((const u32x2*)row);
      else *reinterpret_cast<u32x4*>(w) = __builtin_nontemporal_load((const u32x4*)row);
#pragma unroll
      for (int i = 0; i < W; ++i) x[j + i / VWP][i % VWP] = w[i];
      row += (SWAP_V ? 2 : 1) * vrow;
    }
  };

  // ---- the wave's tiles, NB in flight.  As soon as the scores have taken the keys of a tile, those of the tile NB further
  // on are requested into the same registers, and its values as soon as the output has taken them; the page numbers of a tile
  // are requested another NB tiles ahead. ---------------------------------------------------------------------------------
  Frag qf[NQ][KS];
  Pages now = {0, 0};
  auto body = [&](int t, u32x4 (&xk)[2][KL], uint32_t (&xv)[8][VWP], Pages& next) {
    const int key0 = key_of(t);
    const bool live = NB == 1 || t < t_end;
    const int key1 = key_of(t + 4 * NB);
    const Pages later = pages_of(t + 8 * NB);
    // a tile that every row sees in full needs no mask
    bool full = live;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
      full = full & (key0 + kTile <= hi_r[n]) & ((key0 >= lo_r[n]) | (key0 + kTile <= seen.sinks));
    full = __builtin_amdgcn_ballot_w64(full) == ~0ull;
    if constexpr (LATE) load_k(xk, key0, now);
    if constexpr (SWAP_K) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int c = 0; c < KL; c += 2)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t lo = xk[t][c][w], hi = xk[t][c + 1][w];
            swap_half_rows(lo, hi);
            xk[t][c][w] = lo, xk[t][c + 1][w] = hi;
          }
    }
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
    if constexpr (!LATE) load_k(xk, key1, next);
    // ---- softmax: element e of half t is key key0 + g * 8 + t * 4 + e ---------------------------------------------------
    float z[NQ][8], top[NQ];
    bool moves = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int e = 0; e < 8; ++e) z[n][e] = s[n][e >> 2][e & 3];
      if (capped) {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[n][e] = tanh_of(z[n][e] * inner);
      }
      if (!full) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = key0 + g * 8 + e;
          const bool sees = live & (key < hi_r[n]) & ((key >= lo_r[n]) | (key < seen.sinks));
          z[n][e] = sees ? z[n][e] : -INFINITY;
        }
      }
      top[n] = z[n][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top[n] = fmaxf(top[n], z[n][e]);
      top[n] *= sc;
      moves = moves | (top[n] > m_run[n] + 8.0f);
    }
    if (__builtin_amdgcn_ballot_w64(moves) != 0) {  // rare: only now do the four lanes of a row compare
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float m = fmaxf(top[n], __shfl_xor(top[n], 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        m = m > m_run[n] + 8.0f ? m : m_run[n];
        const float alpha = m == m_run[n] ? 1.0f : __builtin_amdgcn_exp2f(m_run[n] - m);
        m_run[n] = m;
        l_run[n] *= alpha;
#pragma unroll
        for (int j = 0; j < VC; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][j][e] *= alpha;
      }
    }
    Frag pf[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float m_use = m_run[n] == -INFINITY ? 0.f : m_run[n];
      T pr[8];
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = __builtin_amdgcn_exp2f(fmaf(z[n][e], sc, -m_use));
        sum += v;
        pr[e] = (T)v;
      }
      pf[n] = *reinterpret_cast<Frag*>(pr);
      l_run[n] += sum;                           // of the lane's own keys; the four lanes of a row meet at the end
    }
    // ---- output: words of 2 elements per key -> fragments of 8 keys per element -----------------------------------------
#pragma unroll
    for (int vp = 0; vp < VP; ++vp) {
      if constexpr (LATE) load_v(xv, key0, now, vp);
      if constexpr (SWAP_V) {
#pragma unroll
        for (int j = 0; j < 8; j += 2)
#pragma unroll
          for (int w = 0; w < VWP; ++w) swap_half_rows(xv[j][w], xv[j + 1][w]);
      }
      if (!full) {  // values of keys that no row sees: zero
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(live & any_sees(key0 + g * 8 + j))) {
#pragma unroll
            for (int w = 0; w < VWP; ++w) xv[j][w] = 0u;
          }
      }
      auto product = [&](int j, u32x4 f) {       // element j of the lane's VC, keys g * 8 + 0..7
#pragma unroll
        for (int n = 0; n < NQ; ++n) acc[n][j] = Mma16<T>::mma(__builtin_bit_cast(Frag, f), pf[n], acc[n][j]);
      };
#pragma unroll
      for (int i = 0; i < VWP; ++i) {
        if constexpr (WIDE) {                    // a word is two elements of a key
          const int j = (vp * VWP + i) * 2;
          u32x4 f0, f1;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            f0[k] = __builtin_amdgcn_perm(xv[2 * k + 1][i], xv[2 * k][i], 0x05040100);
            f1[k] = __builtin_amdgcn_perm(xv[2 * k + 1][i], xv[2 * k][i], 0x07060302);
          }
          product(j, f0);
          product(j + 1, f1);
        } else {                                 // four: bytes of two keys side by side first, widened as pairs of keys
          u32x4 f0, f1, f2, f3;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t lo = __builtin_amdgcn_perm(xv[2 * k + 1][i], xv[2 * k][i], 0x05010400);
            const uint32_t hi = __builtin_amdgcn_perm(xv[2 * k + 1][i], xv[2 * k][i], 0x07030602);
            f0[k] = Widen<T, FMT>::template two<false>(lo);
            f1[k] = Widen<T, FMT>::template two<true>(lo);
            f2[k] = Widen<T, FMT>::template two<false>(hi);
            f3[k] = Widen<T, FMT>::template two<true>(hi);
          }
          product(i * 4, f0);
          product(i * 4 + 1, f1);
          product(i * 4 + 2, f2);
          product(i * 4 + 3, f3);
        }
      }
    }
    if constexpr (!LATE) load_v(xv, key1, next, 0);
    now = next;
    next = later;
  };
  const int t0 = t_begin + wave;
  if (t0 < t_end) {
    Pages ahead[NB];
#pragma unroll
    for (int u = 0; u < NB; ++u) ahead[u] = pages_of(t0 + 4 * u);
    now = ahead[0];
    if constexpr (!LATE) {
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        // (in the order of the loop: a wait counts what was requested later)
        load_k(xk[u], key_of(t0 + 4 * u), ahead[u]);
        __builtin_amdgcn_sched_barrier(0);
        load_v(xv[u], key_of(t0 + 4 * u), ahead[u], 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int u = 0; u < NB; ++u) ahead[u] = pages_of(t0 + 4 * (NB + u));
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int s = 0; s < KS; ++s)
        qf[n][s] = __builtin_bit_cast(Frag, (q_raw[n][s] & (q_inside(s) ? q_mask[n] : 0u)) ^ q_flip);
    // (an odd tile out is computed with every key masked: with a way round it in the loop the compiler waits for all loads)
    for (int t = t0; t < t_end; t += 4 * NB) {
      body(t, xk[0], xv[0], ahead[0]);
      if constexpr (NB == 2) body(t + 4, xk[1], xv[1], ahead[1]);
    }
  }
  const bool broken = __builtin_amdgcn_ballot_w64(bad || bad_half) != 0;

  // ---- merge of the four waves: 16 rows at a time -------------------------------------------------------------------------
  const float v_scale = seq.v_scale;
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
      for (int e = 0; e < EH; ++e) {                   // output row m = g * 4 + e0 + e is a block of VC elements
        const int m = g * 4 + e;
        const int block = SWAP_V ? (m & 7) * 2 + (m >> 3) : g * EH + e;
#pragma unroll
        for (int j = 0; j < VC; ++j) part[(wave * 16 + rl) * PITCH + block * VC + j] = acc[n][j][e0 + e];
      }
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
          const int64_t at = part_row(a, split, b, q_bos, tok) * p.Hq + head;
          a.part_o[at * DP + d] = o;
          if (d == 0) a.part_ml[at * 2] = m, a.part_ml[at * 2 + 1] = sum;
        }
      }
    }
  }
}

template <typename T, int FMT, int DP, int NQ, int PAGES>
int launch_stream(const CacheAttnArgs& a, hipStream_t st) {
  const FgFlashParams& p = a.p.base;
  const int64_t blocks = fg_cdiv((int64_t)a.max_q * a.group, 16 * NQ) * a.splits;
  FG_REQUIRE(blocks < kMostBlocks, FG_ERR_UNSUPPORTED, "cache_attn_fwd: too many query rows for one launch");
  hipLaunchKernelGGL((attn_stream_kernel<T, FMT, DP, NQ, PAGES>), dim3((unsigned)blocks, (unsigned)p.batch, (unsigned)p.Hk),
                     dim3(256), 0, st, a);
  if (a.splits > 1) return launch_merge<T, DP, kTile, 16 * NQ, 4>(a, st);
  return fg_check_launch("cache_attn_fwd");
}
