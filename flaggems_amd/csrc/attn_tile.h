// Attention of chunks of new tokens over a paged cache.
//
// Rows r = token * G + g as in attn_stream.h; a workgroup takes a block of 64 * NQ rows of one (sequence, KV head) and key range,
// each of its four waves 16 * NQ of them, and walks the tiles of 64 keys that some row of the block may see (the tiles of the sinks, then
// those of [lo, hi)).  The workgroup stages a tile once for all its rows: global memory -> registers -> LDS, 8-bit values
// widened to the query's type on the way, so that the widening costs each wave a quarter of the tile.  Two tile buffers:
// the loads of the next tile are in flight while this one is computed, one barrier per tile.
//
// Products as in attn_stream.h (transposed; P stays in the lane), the fragments read from LDS.
//   K tile: [key][d], 16-byte chunks XOR-swizzled by the key's place in its fragment (k_swz), so that the 16 rows of a
//     fragment read lie in different banks;
//   V tile: [key][d], read transposed by ds_read_b64_tr_b16 (four keys of one element per lane), swizzled (v_swz) so that the
//     eight rows of half a read do.  Output sub-tile j is elements 16 j + m.
//
// Softmax in base 2 with fp32 statistics; the common path tests in the lane whether a score exceeds the reference maximum by
// 2^8, and only then reduces over the four lanes of a row and rescales.
//
// Bound: matrix pipe and vector ALU together (32 MFMA of 16 clocks against 16 exponentials of 16 clocks and some 40 plain
// instructions of 4 per wave and 32 keys); two workgroups per CU, so that one wave's softmax runs under another's products.
// 32/8 heads of 128, e4m3: 8 x 2048 tokens over 8192 keys 2.10 ms = 0.92 PFLOP/s, 8192 over themselves 625 us = 0.88; four chunks of
// up to 1024 over up to 8192, in four ranges, 262 us = 0.76 and 45 for the merge (0.64 with everything; uneven, one round of workgroups).
// 16 bits, 8192 tokens under a window of 1024 keys and 4 sinks: 246 us = 0.53 PFLOP/s of visible keys (19 tiles a block, of which
// two or three are partly masked).  (After a third of a second of such calls; the first ones after a pause take a sixth longer.)
// Counters there: matrix pipe busy 22 % of the time, no LDS conflicts.  With 8 bits a quarter of the LDS cycles are conflicts of the staging writes; places without them (the halves of a row apart) gain 1 % there
// and cost the 16-bit reads 7 %.
#pragma once

constexpr int kTileKeys = 64;

// POW2: the page size is a power of two.
// NQ: 16-row tiles of a wave; the workgroup's block has 64 * NQ rows.
template <typename T, int FMT, int DP, bool POW2, int NQ>
__global__ __launch_bounds__(256, 2) void attn_tile_kernel(CacheAttnArgs a) {
  typedef typename Mma16<T>::Frag Frag;
  constexpr bool WIDE = FMT == FG_CACHE_SAME;
  constexpr int EB = WIDE ? 2 : 1;
  constexpr int EPL = 16 / EB;                   // elements of a 16-byte load
  constexpr int KS = DP / 32;
  constexpr int DT = DP / 16;                    // output sub-tiles
  constexpr int ROWS = 64 * NQ;
  constexpr int RB = DP * 2;                     // bytes of a tile row
  constexpr int CPR = RB / 16;                   // 16-byte chunks of it: 16 or 8
  constexpr int TB = kTileKeys * RB;
  constexpr int TPR = DP / EPL;                  // threads per cached row while staging
  constexpr int RPP = 256 / TPR;                 // rows per pass
  constexpr int NP = kTileKeys / RPP;            // passes
  constexpr int CW = WIDE ? 1 : 2;               // LDS chunks of one load
  __shared__ __attribute__((aligned(16))) char lds[2][2][TB];  // [buffer][K, V]

  const FgFlashParams& p = a.p.base;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rl = lane & 15, g = lane >> 4;
  // Workgroup id -> (sequence, KV head), row block, key range.  Workgroups go round-robin to the 8 XCDs; what a pair has runs on
  // one, whose L2 then holds its keys.  Unsplit: the last rows of the sequences, which see the most, come first.  Split: the
  // row blocks that share a range run next to each other.
  const int pairs = p.batch * p.Hk;
  const int xcd = blockIdx.x & 7, turn = blockIdx.x >> 3;
  const int per_xcd = (pairs + 7) >> 3;
  const int blocks = (a.max_q * a.group + ROWS - 1) / ROWS;
  const int place = a.splits > 1 ? turn / blocks : turn;
  const int pair = xcd + 8 * (place % per_xcd);
  if (pair >= pairs) return;
  const int split = a.splits > 1 ? place / per_xcd : 0;
  const int from_last = a.splits > 1 ? turn % blocks : place / per_xcd;
  const int b = pair / p.Hk, kvh = pair - b * p.Hk;
  const int G = a.group;
  const Sequence seq = sequence(a, b, kvh);
  const int q_bos = seq.q_bos, q_len = seq.q_len, k_len = seq.k_len;
  const int rows = q_len * G;
  const int row0 = ((rows + ROWS - 1) / ROWS - 1 - from_last) * ROWS;
  if (!seq.mine || row0 < 0) return;
  const int last_row = row0 + ROWS < rows ? row0 + ROWS - 1 : rows - 1;
  const Seen seen = seen_by<kTileKeys>(a, q_len, k_len, row0 / G, last_row / G);
  bool bad = seq.too_long;
  const int per = range_tiles<1>(a, seen.tiles);
  const int t_begin = split * per;
  const int t_end = t_begin + per < seen.tiles ? t_begin + per : seen.tiles;
  if (split > 0 && t_begin >= t_end) return;     // range 0 always reports

  // t = sc * S with sc > 0, so that the largest t is sc times the largest S: the sign goes into the query (0: a query of 0)
  const bool capped = p.softcap > 0.f;
  const float given = (capped ? a.cap_in : a.scale_log2) * seq.k_scale;
  const uint32_t q_keep = given == 0.f ? 0u : ~0u, q_flip = given < 0.f ? 0x80008000u : 0u;
  const float inner = given == 0.f ? 1.0f : fabsf(given);
  const float sc = capped ? a.cap_out_log2 : inner;  // of S, or of tanh(inner * S)
  int lo_r[NQ], hi_r[NQ];
  Frag qf[NQ][KS];
  const int D = p.D;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = row0 + wave * (16 * NQ) + n * 16 + rl;
    const bool ok = row < rows;
    const int tok = (ok ? row : row0) / G, head = kvh * G + (ok ? row : row0) % G;
    row_bounds(a, q_len, k_len, tok, lo_r[n], hi_r[n]);
    const T* q = (const T*)p.q + (int64_t)(q_bos + tok) * p.q_row_stride + (int64_t)head * p.q_head_stride;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = s * 32 + g * 8;
      const u32x4 v = *reinterpret_cast<const u32x4*>(q + (d < D ? d : 0));
      qf[n][s] = __builtin_bit_cast(Frag, (v & (ok && d < D ? q_keep : 0u)) ^ q_flip);
    }
  }
  f32x4 acc[NQ][DT];
  float m_run[NQ], l_run[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m_run[n] = -INFINITY, l_run[n] = 0.f;
#pragma unroll
    for (int j = 0; j < DT; ++j) acc[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // ---- staging: thread -> (row of a pass, 16 bytes of it) -------------------------------------------------------------------
  const int srow = tid / TPR, sat = tid % TPR;   // row in the pass, piece of the row
  const bool piece = sat * EPL < D;              // the piece lies inside the head dim
  const char* const kbase = (const char*)p.k_cache + ((int64_t)kvh * p.k_head_stride + (piece ? sat * EPL : 0)) * EB;
  const char* const vbase = (const char*)p.v_cache + ((int64_t)kvh * p.v_head_stride + (piece ? sat * EPL : 0)) * EB;
  const int32_t* const table = p.block_table + (int64_t)b * p.block_table_stride;
  // Offsets are counted in 16 bytes: 32 bits inside a page, one 32 x 32 -> 64 product for the page.  K and V of one shape,
  // as caches are made, share them.
  const uint32_t kpage = (uint32_t)(p.k_page_stride * EB >> 4), krow = (uint32_t)(p.k_row_stride * EB >> 4);
  const uint32_t vpage = (uint32_t)(p.v_page_stride * EB >> 4), vrow = (uint32_t)(p.v_row_stride * EB >> 4);
  const bool alike = kpage == vpage && krow == vrow;
  u32x4 sk[NP], sv[NP];
  int page[NP];
  auto any_sees = [&](int key) { return (key < seen.hi) & ((key >= seen.lo) | (key < seen.sinks)); };
  auto number = [&](int key) { return POW2 ? key >> a.page_bits : page_of(a, key); };
  auto slot_of = [&](int key) { return POW2 ? key & (p.page_size - 1) : key - page_of(a, key) * p.page_size; };
  // Pages of the thread's keys.  Where no row sees the key the entry of one that is seen is read: its page exists.
  auto look_up = [&](int t) {
    const int key0 = tile_key<kTileKeys>(seen, t);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int key = key0 + i * RPP + srow;
      page[i] = table[number(any_sees(key) ? key : seen.hi - 1)];
    }
  };
  auto request = [&](int t) {
    const int key0 = tile_key<kTileKeys>(seen, t);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const uint32_t slot = (uint32_t)slot_of(key0 + i * RPP + srow);
      const bool known = (uint32_t)page[i] < (uint32_t)a.p.num_pages;
      bad |= !known;
      const uint32_t pg = known ? (uint32_t)page[i] : 0u;
      const uint64_t ko = (uint64_t)pg * kpage + slot * krow;
      const uint64_t vo = alike ? ko : (uint64_t)pg * vpage + slot * vrow;
      sk[i] = *reinterpret_cast<const u32x4*>(kbase + (ko << 4));
      sv[i] = *reinterpret_cast<const u32x4*>(vbase + (vo << 4));
    }
  };
  // K: row `key` of a fragment is MFMA row ((key >> 3) & 3) * 4 + (key & 3)
  auto k_swz = [](int key) { return CPR == 16 ? ((key >> 3) & 3) * 4 + (key & 3) : ((key >> 3) & 3) * 2 + ((key & 3) >> 1); };
  auto v_swz = [](int key) { return CPR == 16 ? (key & 3) * 2 + ((key >> 3) & 1) * 8 : (key & 2) + ((key >> 3) & 1) * 4; };
  auto store = [&](int t, int buf) {
    const int key0 = tile_key<kTileKeys>(seen, t);
    const bool inside = key0 + kTileKeys <= seen.hi && key0 >= seen.lo && D == DP;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = i * RPP + srow;
      u32x4 kv = sk[i], vv = sv[i];
      if (!inside) {                             // keys that no row sees, elements past the head dim: zero
        const bool ok = piece && any_sees(key0 + r);
        if (!ok) kv = vv = u32x4{0u, 0u, 0u, 0u};
      }
      char* const kd = lds[buf][0] + r * RB;
      char* const vd = lds[buf][1] + r * RB;
      if constexpr (WIDE) {
        *reinterpret_cast<u32x4*>(kd + ((sat ^ k_swz(r)) * 16)) = kv;
        *reinterpret_cast<u32x4*>(vd + ((sat ^ v_swz(r)) * 16)) = vv;
      } else {
#pragma unroll
        for (int c = 0; c < CW; ++c) {
          const u32x4 kw = {Widen<T, FMT>::template two<false>(kv[2 * c]), Widen<T, FMT>::template two<true>(kv[2 * c]),
                            Widen<T, FMT>::template two<false>(kv[2 * c + 1]), Widen<T, FMT>::template two<true>(kv[2 * c + 1])};
          const u32x4 vw = {Widen<T, FMT>::template two<false>(vv[2 * c]), Widen<T, FMT>::template two<true>(vv[2 * c]),
                            Widen<T, FMT>::template two<false>(vv[2 * c + 1]), Widen<T, FMT>::template two<true>(vv[2 * c + 1])};
          *reinterpret_cast<u32x4*>(kd + (((sat * 2 + c) ^ k_swz(r)) * 16)) = kw;
          *reinterpret_cast<u32x4*>(vd + (((sat * 2 + c) ^ v_swz(r)) * 16)) = vw;
        }
      }
    }
  };

  // ---- fragment places ------------------------------------------------------------------------------------------------------
  const int kr = (rl >> 2) * 8 + (rl & 3);       // key of the lane's MFMA row in half tile 0 of a 32-key part
  const int vk = g * 8 + (rl >> 2);              // key of the lane's address in a transposing read (and + 4)

  if (t_begin < t_end) {
    look_up(t_begin);
    request(t_begin);
    if (t_begin + 1 < t_end) look_up(t_begin + 1);
    store(t_begin, 0);
  }
  __syncthreads();
  for (int t = t_begin; t < t_end; ++t) {
    const int buf = (t - t_begin) & 1, key0 = tile_key<kTileKeys>(seen, t);
    const bool more = t + 1 < t_end;
    if (more) request(t + 1);
    if (t + 2 < t_end) look_up(t + 2);
    const char* const kt = lds[buf][0];
    const char* const vt = lds[buf][1];
    bool full = true;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
      full = full & (key0 + kTileKeys <= hi_r[n]) & ((key0 >= lo_r[n]) | (key0 + kTileKeys <= seen.sinks));
    full = __builtin_amdgcn_ballot_w64(full) == ~0ull;
    // ---- scores: s[n][u * 2 + t] element e is key u * 32 + g * 8 + t * 4 + e -----------------------------------------------
    f32x4 s[NQ][4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int row = (h >> 1) * 32 + (h & 1) * 4 + kr;
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[n][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(kt + row * RB + (((st * 4 + g) ^ k_swz(row)) * 16));
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][h] = Mma16<T>::mma(__builtin_bit_cast(Frag, w), qf[n][st], s[n][h]);
      }
    }
    // ---- softmax --------------------------------------------------------------------------------------------------------------
    float top[NQ];
    bool moves = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      if (capped) {
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][h][e] = tanh_of(s[n][h][e] * inner);
      }
      if (!full) {
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + (h >> 1) * 32 + g * 8 + (h & 1) * 4 + e;
            const bool sees = (key < hi_r[n]) & ((key >= lo_r[n]) | (key < seen.sinks));
            s[n][h][e] = sees ? s[n][h][e] : -INFINITY;
          }
      }
      top[n] = -INFINITY;
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) top[n] = fmaxf(top[n], s[n][h][e]);
      top[n] *= sc;
      moves = moves | (top[n] > m_run[n] + 8.0f);
    }
    if (__builtin_amdgcn_ballot_w64(moves) != 0) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float m = fmaxf(top[n], __shfl_xor(top[n], 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        m = m > m_run[n] + 8.0f ? m : m_run[n];
        const float alpha = m == m_run[n] ? 1.0f : __builtin_amdgcn_exp2f(m_run[n] - m);
        m_run[n] = m;
        l_run[n] *= alpha;
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][j][e] *= alpha;
      }
    }
    Frag pf[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float m_use = m_run[n] == -INFINITY ? 0.f : m_run[n];
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        T pr[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = __builtin_amdgcn_exp2f(fmaf(s[n][u * 2 + (e >> 2)][e & 3], sc, -m_use));
          sum += v;
          pr[e] = (T)v;
        }
        pf[n][u] = *reinterpret_cast<Frag*>(pr);
      }
      l_run[n] += sum;
    }
    // ---- output: sub-tile j is elements 16 j + (MFMA row) -----------------------------------------------------------------------
#pragma unroll
    for (int j = 0; j < DT; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r0 = u * 32 + vk, r1 = r0 + 4;
        const int c = 2 * j + ((rl >> 1) & 1), at = (rl & 1) * 8;
        const u32x2 w0 = read_tr(vt + r0 * RB + ((c ^ v_swz(r0)) * 16) + at);
        const u32x2 w1 = read_tr(vt + r1 * RB + ((c ^ v_swz(r1)) * 16) + at);
        const u32x4 w = {w0[0], w0[1], w1[0], w1[1]};
#pragma unroll
        for (int n = 0; n < NQ; ++n) acc[n][j] = Mma16<T>::mma(__builtin_bit_cast(Frag, w), pf[n][u], acc[n][j]);
      }
    if (more) store(t + 1, buf ^ 1);
    __syncthreads();
  }

  // ---- epilogue: lane (row, g) holds elements 16 j + 4 g + e ---------------------------------------------------------------------
  const bool broken = __syncthreads_or(bad) != 0;
  const float v_scale = seq.v_scale;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float l = l_run[n];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (broken) l = NAN;
    const int row = row0 + wave * (16 * NQ) + n * 16 + rl;
    if (row >= rows) continue;
    const int tok = row / G, head = kvh * G + row % G;
    if (a.splits > 1) {
      const int64_t at = part_row(a, split, b, q_bos, tok) * p.Hq + head;
#pragma unroll
      for (int j = 0; j < DT; ++j) *reinterpret_cast<f32x4*>(a.part_o + at * DP + j * 16 + g * 4) = acc[n][j];
      if (g == 0) a.part_ml[at * 2] = m_run[n], a.part_ml[at * 2 + 1] = l;
      continue;
    }
    const bool empty = l == 0.f;
    const float f = empty ? 0.f : v_scale / l;
    T* const o = (T*)p.out + (int64_t)(q_bos + tok) * p.o_row_stride + (int64_t)head * p.o_head_stride;
#pragma unroll
    for (int j = 0; j < DT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = j * 16 + g * 4 + e;
        if (d < D) o[d] = (T)(empty ? 0.f : acc[n][j][e] * f);
      }
    if (g == 0 && p.lse != nullptr)
      p.lse[(int64_t)head * p.total_q + q_bos + tok] =
          empty ? INFINITY : (m_run[n] == -INFINITY ? 0.f : m_run[n]) * 0.6931471805599453f + logf(l);
  }
}

// Workgroups of a launch for `batch` sequences with up to max_q new tokens.
inline int64_t tile_blocks(const FgFlashParams& p, int64_t max_q, int nq, int splits, int64_t batch) {
  return fg_cdiv(max_q * (p.Hq / p.Hk), 64 * nq) * splits * 8 * fg_cdiv(batch * p.Hk, 8);
}

template <typename T, int FMT, int DP, int NQ>
int launch_tile(const CacheAttnArgs& a, hipStream_t st) {
  const FgFlashParams& p = a.p.base;
  const int64_t blocks = tile_blocks(p, a.max_q, NQ, a.splits, p.batch);
  FG_REQUIRE(blocks < kMostBlocks, FG_ERR_UNSUPPORTED, "cache_attn_fwd: too many query rows for one launch");
  if (a.page_bits >= 0)
    hipLaunchKernelGGL((attn_tile_kernel<T, FMT, DP, true, NQ>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((attn_tile_kernel<T, FMT, DP, false, NQ>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  if (a.splits > 1) return launch_merge<T, DP, kTileKeys, 64 * NQ, 1>(a, st);
  return fg_check_launch("cache_attn_fwd");
}
