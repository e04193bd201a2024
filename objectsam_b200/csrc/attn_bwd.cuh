// Attention backward (see attn.cuh): one kernel in two forms.  Each CTA keeps 128 rows of one side in shared memory
// and streams 64-row tiles of the other:
//   DKV: 128 keys of a key head stay (K, V), the queries of every head of the group stream (Q, dO):
//        dV += Pᵀ·dO, dK += dSᵀ·Q — the sum over a shared key head's query heads is this accumulation
//   DQ : 128 queries of one head stay (Q, dO), the keys stream (K, V):  dQ += dS·K
// Two passes compute S and dP twice (7 products instead of 5) but every sum is taken in one order: no atomics, results that
// do not depend on scheduling.  One CTA takes it whole, without an fp32 copy; or, with few tiles (`parts`), up to eight share
// the streamed side and k_attn_sum adds their fp32 parts in order.
//
// Per tile, rows = the stationary side (TMEM lanes), columns = the streamed side:
//   X = stat1·strm1ᵀ (scores), Y = stat2·strm2ᵀ (dP), both fp32 in TMEM
//   two threads per row (32 columns each): p = 2^(x − lse), ds = p·(dp − δ)·(1 − t²), back to TMEM in 16 bits over
//   X and Y
//   acc2 += P·strm2 (DKV), acc1 += dS·strm1, P and dS as TMEM operands
// fp16 keeps its precision over long rows and gradients of any size by powers of two: P is held times 2^8 and dS times
// 2^8·F, both taken back in fp32 at the end; bf16 needs neither.  F comes from a bound: with dP_ij = dO_i·v_j and
// δ_i = Σ_k p_ik dP_ik, |dS_ij| = p_ij·|dP_ij − δ_i| ≤ 2·p_ij·(1 − p_ij)·max_k |dP_ik| ≤ ½·‖dO_i‖·max‖v‖.  F = 2^(7−e), e the
// exponent of max‖dO‖·max‖v‖ (of the key head and its group for DKV, of the row's block and its key head for DQ),
// keeps dS within 2^15 and leaves 2^29 below that to normal numbers.
// Warps: 8 per buffer of (X, Y) for the element-wise part (warps w and w + 4 share rows), then the TMA producer and the
// MMA issuer.  Up to 64 head dims one buffer and 256 TMEM columns, two CTAs per SM; above, two buffers in one CTA
// with all 512 columns: the tensor cores work on one while the other is in the element-wise part.
#pragma once
#include <algorithm>
#include <type_traits>

#include "attn.cuh"

namespace osam {

template <int DP>
struct AbCfg {
  static constexpr int PANELS = DP / 64;
  static constexpr int NB = DP == 64 ? 1 : 2;   // (X, Y) buffers, each with eight warps
  static constexpr int CTAS = DP == 64 ? 2 : 1; // per SM
  static constexpr int STAGES = 4;
  static constexpr int STAT = PANELS * kAbRows * 128;  // bytes of one stationary operand
  static constexpr int STRM = PANELS * kAbCols * 128;  // bytes of one streamed operand
  static constexpr int ROWS = kAbCols * 8;             // (lse, δ) of a query tile
  static constexpr int SMEM = 1024 + 2 * STAT + STAGES * (2 * STRM + ROWS);
  static constexpr int TMEM = DP == 64 ? 256 : 512;
  static constexpr int COL_ACC1 = 128 * NB, COL_ACC2 = COL_ACC1 + DP;
  static constexpr int SOFT = 256 * NB;  // element-wise threads
  static constexpr int THREADS = SOFT + 64;
};

// Visits (head of the group, tile) pairs, heads outermost.
struct AbIter {
  int g, t;
  __device__ __forceinline__ void start(const AtTiles& T) {
    g = 0;
    t = T.first();
  }
  __device__ __forceinline__ bool more(const AtTiles& T, int heads) const { return g < heads && t < T.end; }
  __device__ __forceinline__ void step(const AtTiles& T) {
    t = T.next(t);
    if (t >= T.end) {
      g++;
      t = T.first();
    }
  }
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <typename T, int DP, bool DKV, int CAP, int BIAS>
__global__ void __launch_bounds__(AbCfg<DP>::THREADS, AbCfg<DP>::CTAS)
    k_attn_bwd(const __grid_constant__ AttnBwdLaunch P) {
  using Cfg = AbCfg<DP>;
  constexpr bool BF16 = Half16<T>::kBf16;
  constexpr int NB = Cfg::NB;
  extern __shared__ uint8_t ab_raw[];
  __shared__ __align__(8) uint64_t stat_full, full[Cfg::STAGES], empty[Cfg::STAGES], xy_full[NB], ds_full[NB], acc_done;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t live[kAtDocWords], mix[kAtDocWords], pad[kAtDocWords];
  __shared__ __align__(16) int col_doc[NB][2][kAbCols];
  __shared__ __align__(16) float col_y[NB][BIAS == 2 ? 2 : 1][kAbCols], col_x[NB][BIAS == 2 ? 2 : 1][kAbCols];

  if (!P.late) grid_dep_wait();
  const AttnDev& A = P.d;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  uint8_t* smem = ab_raw + ((1024 - (smem_u32(ab_raw) & 1023)) & 1023);
  uint8_t* strm = smem + 2 * Cfg::STAT;
  uint8_t* srows = strm + Cfg::STAGES * 2 * Cfg::STRM;

  // ---- which tile (with a causal bound the longest first)
  const int heads = DKV ? A.Hk : A.Hq, nt = ((DKV ? A.Lk : A.Lq) + kAbRows - 1) / kAbRows;
  int rt, rest;
  at_order(blockIdx.x, nt, A.B * heads * P.parts, P.group, rt, rest);
  if (!DKV && A.mask != OSAM_ATTN_NONE) rt = nt - 1 - rt;
  const int part = rest % P.parts;
  rest /= P.parts;
  const int hd = rest % heads, b = rest / heads;
  const int row0 = rt * kAbRows;
  const int n = at_keys(A, b), off = n - A.Lq;
  const int prefix = A.mask == OSAM_ATTN_PREFIX ? A.prefix[b] : 0;
  const int nq64 = (A.Lq + kAbCols - 1) / kAbCols, nk64 = (A.Lk + kAbCols - 1) / kAbCols;
  const bool causal = A.mask != OSAM_ATTN_NONE;
  const int streams = DKV ? A.G : 1;  // query heads that stream past
  AtTiles tiles;
  int lim_min = 0;  // DQ: bound of the tile's first query
  if (DKV) {  // queries from the first that sees key row0
    tiles.begin = causal && prefix <= row0 ? max(0, row0 - off) / kAbCols : 0;
    tiles.end = row0 < n ? nq64 : tiles.begin;
    tiles.begin = min(tiles.begin, tiles.end);
  } else {
    const int last = min(row0 + kAbRows, A.Lq) - 1;
    tiles.begin = 0;
    tiles.end = (at_limit(A, n, prefix, off + last) + kAbCols - 1) / kAbCols;
    lim_min = at_limit(A, n, prefix, off + row0);
  }
  if (P.parts > 1) {
    const int first = tiles.begin;
    const long long len = max(0, tiles.end - first);
    tiles.begin = first + int(len * part / P.parts);
    tiles.end = first + int(len * (part + 1) / P.parts);
  }
  tiles.from = tiles.begin - 1;  // the order does not matter here: upwards
  const bool docs = A.doc_q != nullptr;
  tiles.live = docs ? live : nullptr;

  // the producer warp sets the barriers up and, where no document summaries have to be looked through first, starts
  // loading at once, under the rest of the prologue
  AbIter made;
  made.start(tiles);
  int n_made = 0;
  auto load_stat = [&]() {
    mbar_arrive_expect_tx(&stat_full, 2 * Cfg::STAT);
    for (int p = 0; p < Cfg::PANELS; p++) {
      tma_load_4d(smem + p * kAbRows * 128, &P.stat1, &stat_full, p * 64, row0, hd, b);
      tma_load_4d(smem + Cfg::STAT + p * kAbRows * 128, &P.stat2, &stat_full, p * 64, row0, hd, b);
    }
  };
  auto load_strm = [&](int it, const AbIter& x) {
    const int s = it % Cfg::STAGES, h = DKV ? hd * A.G + x.g : hd / A.G;
    uint8_t* d = strm + s * 2 * Cfg::STRM;
    mbar_arrive_expect_tx(&full[s], 2 * Cfg::STRM + (DKV ? Cfg::ROWS : 0));
    for (int p = 0; p < Cfg::PANELS; p++) {
      tma_load_4d(d + p * kAbCols * 128, &P.strm1, &full[s], p * 64, x.t * kAbCols, h, b);
      tma_load_4d(d + Cfg::STRM + p * kAbCols * 128, &P.strm2, &full[s], p * 64, x.t * kAbCols, h, b);
    }
    if (DKV)
      bulk_load(srows + s * Cfg::ROWS, P.rows + (((long long)b * A.Hq + h) * nq64 + x.t) * 2 * kAbCols, Cfg::ROWS, &full[s]);
  };
  if (warp == 8 * NB && lane == 0) {
    mbar_init(&stat_full, 1);
    for (int i = 0; i < Cfg::STAGES; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < NB; i++) {
      mbar_init(&xy_full[i], 1);
      mbar_init(&ds_full[i], 8);
    }
    mbar_init(&acc_done, 1);
    fence_barrier_init();
    if (!docs && made.more(tiles, streams)) {
      load_stat();
      for (; n_made < Cfg::STAGES && made.more(tiles, streams); made.step(tiles), n_made++) load_strm(n_made, made);
    }
  }
  if (warp == 8 * NB + 1) {
    tmem_alloc(&tmem_slot, Cfg::TMEM);
    tmem_relinquish();
    // the CTA's one signal, given once TMEM is its own: the next kernel's CTAs may take columns and then wait for this one
    grid_dep_launch();
  }
  if (docs) {
    const AtDocs* sq = A.sum_q + (long long)b * nq64;
    const AtDocs* sk = A.sum_k + (long long)b * nk64;
    const AtDocs own = at_docs(DKV ? sk : sq, rt * 2, 2, DKV ? nk64 : nq64);
    at_doc_bits(own, DKV ? sq : sk, DKV ? nq64 : nk64, 1, tiles.begin, tiles.end, warp, Cfg::THREADS / 32, live, mix, pad);
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 8 * NB) {
    if (lane == 0) {
      if (docs) {
        made.start(tiles);
        if (made.more(tiles, streams)) load_stat();
      }
      int it = n_made;
      for (; made.more(tiles, streams); made.step(tiles), it++) {
        if (it >= Cfg::STAGES && !at_wait(&empty[it % Cfg::STAGES], ((it / Cfg::STAGES) & 1) ^ 1, A.err)) break;
        load_strm(it, made);
      }
      // no copy of this CTA may be in flight when it ends
      if (it > 0) at_wait(&stat_full, 0, A.err);
      for (int i = max(0, it - Cfg::STAGES); i < it; i++) at_wait(&full[i % Cfg::STAGES], (i / Cfg::STAGES) & 1, A.err);
    }
    __syncwarp();
  } else if (warp == 8 * NB + 1) {
    const uint32_t leader = elect_leader();
    const int ks = (A.D + 15) / 16;
    const uint32_t id_x = at_idesc(BF16, 128, kAbCols, false), id_g = at_idesc(BF16, 128, 16 * ks, true);
    const uint32_t a1 = smem_u32(smem), sb = smem_u32(strm);
    const uint64_t da1 = smem_desc_kmajor(a1, 128), da2 = smem_desc_kmajor(a1 + Cfg::STAT, 128);
    const uint64_t db = smem_desc_kmajor(sb, 128), dg = at_desc_mn(sb, kAbCols * 128);  // offsets: bytes / 16
    const int count = __shfl_sync(0xffffffffu, tiles.count(), 0) * streams;
    // X and Y of streamed tile `it`
    auto scores = [&](int it) {
      const uint64_t b1 = db + ((it % Cfg::STAGES) * 2 * Cfg::STRM >> 4), b2 = b1 + (Cfg::STRM >> 4);
      const uint32_t d = tmem + (it % NB) * 128;
#pragma unroll
      for (int k = 0; k < DP / 16; k++)
        if (k < ks)
          mma_ss(leader, d, da1 + (((k / 4) * kAbRows * 128 + (k % 4) * 32) >> 4),
                 b1 + (((k / 4) * kAbCols * 128 + (k % 4) * 32) >> 4), id_x, k > 0);
#pragma unroll
      for (int k = 0; k < DP / 16; k++)
        if (k < ks)
          mma_ss(leader, d + 64, da2 + (((k / 4) * kAbRows * 128 + (k % 4) * 32) >> 4),
                 b2 + (((k / 4) * kAbCols * 128 + (k % 4) * 32) >> 4), id_x, k > 0);
      mma_commit(leader, &xy_full[it % NB]);
    };
    bool ok = count == 0 || at_wait_warp(&stat_full, 0, A.err);
    for (int it = 0; ok && it < NB && it < count; it++) {
      if (!(ok = at_wait_warp(&full[it % Cfg::STAGES], (it / Cfg::STAGES) & 1, A.err))) break;
      tc_fence_after();
      scores(it);
    }
    for (int it = 0; ok && it < count; it++) {
      const int s = it % Cfg::STAGES, buf = it % NB, ia = it + NB;
      if (!(ok = at_wait_warp(&ds_full[buf], (it / NB) & 1, A.err))) break;
      tc_fence_after();
      const uint64_t g1 = dg + (s * 2 * Cfg::STRM >> 4), g2 = g1 + (Cfg::STRM >> 4);
      const uint32_t d = tmem + buf * 128;
      if (DKV) {
#pragma unroll
        for (int k = 0; k < kAbCols / 16; k++)
          mma_ts(leader, tmem + Cfg::COL_ACC2, d + k / 2 * 32 + k % 2 * 8, g2 + (k * 16 * 128 >> 4), id_g, (it | k) != 0);
      }
#pragma unroll
      for (int k = 0; k < kAbCols / 16; k++)
        mma_ts(leader, tmem + Cfg::COL_ACC1, d + 64 + k / 2 * 32 + k % 2 * 8, g1 + (k * 16 * 128 >> 4), id_g, (it | k) != 0);
      mma_commit(leader, &empty[s]);
      if (ia < count) {
        if (!(ok = at_wait_warp(&full[ia % Cfg::STAGES], (ia / Cfg::STAGES) & 1, A.err))) break;
        tc_fence_after();
        scores(ia);
      }
    }
    mma_commit(leader, &acc_done);
    if (!ok) at_wait_warp(&acc_done, 0, A.err);  // the issued MMAs finish before TMEM is freed
  } else {
    const int buf = warp / 8, half = warp / 4 % 2, r = tid % 128;
    const uint32_t lane_base = uint32_t((warp % 4) * 32) << 16;
    const int row = row0 + r;
    const bool valid = row < (DKV ? A.Lk : A.Lq);
    // ---- what this thread's row is: a key (DKV) or a query (DQ)
    const int pos = DKV ? row : off + row;
    int my_doc = -2;
    if (docs && valid) {
      my_doc = (DKV ? A.doc_k : A.doc_q)[(long long)b * (DKV ? A.Lk : A.Lq) + row];
      if (my_doc < 0) my_doc = -2;
    }
    // DKV: queries from `from` on see the key; DQ: keys below `lim` are seen
    const int from = row >= n ? INT_MAX : (!causal || prefix > row ? 0 : row - off);
    const int lim = !DKV && valid ? at_limit(A, n, prefix, pos) : 0;
    float F = 1.f;
    if (!BF16) {
      float peak = 0.f, vpeak = 0.f;
      const float* vk = P.vpeak + ((long long)b * A.Hk + (DKV ? hd : hd / A.G)) * nk64;
      for (int i = lane; i < nk64; i += 32) vpeak = fmaxf(vpeak, vk[i]);
      if (DKV) {
        const float* pk = P.peak + ((long long)b * A.Hq + hd * A.G) * nq64;
        for (int i = lane; i < A.G * nq64; i += 32) peak = fmaxf(peak, pk[i]);
      } else if (valid) {
        peak = P.peak[((long long)b * A.Hq + hd) * nq64 + row / kAbCols];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        vpeak = fmaxf(vpeak, __shfl_xor_sync(0xffffffffu, vpeak, o));
        if (DKV) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, o));
      }
      peak *= vpeak;  // at most 2^40: rows of 128 fp16 numbers
      const int e = (__float_as_int(peak) >> 23) & 255;
      if (peak > 0.f) F = __int_as_float(min(227, max(27, 127 + 7 + 127 - e)) << 23);  // at most 2^±100
    }
    float row_lse = 0.f, row_delta = 0.f;
    if (!DKV) {
      const float* v = P.rows + (((long long)b * A.Hq + hd) * nq64 + row / kAbCols) * 2 * kAbCols + row % kAbCols;
      row_lse = valid ? v[0] : -INFINITY;
      row_delta = valid ? v[kAbCols] * F : 0.f;
    }
    AtBias bias;
    bias.mul = CAP ? 2.f * A.scale * kAtLog2e / A.cap : A.scale * kAtLog2e;
    bias.cap2 = A.cap * kAtLog2e;
    bias.lin = A.scale * kAtLog2e;
    bias.arg = A.scale / A.cap;
    bias.slope = bias.away = bias.y = bias.x = 0.f;
    int slope_of = -1;
    AbIter x;
    x.start(tiles);
    bool ok = true;
    int it = 0, tile = 0;
    auto run = [&](auto minus) {
    for (; x.more(tiles, streams); x.step(tiles), it++) {
      if (NB > 1 && it % NB != buf) continue;
      const int c0 = x.t * kAbCols, h0 = half * 32;  // first column: query (DKV) or key (DQ); this thread's first
      const int h = DKV ? hd * A.G + x.g : hd;
      if (BIAS && slope_of != h) {
        bias.slope = A.slopes[h] * kAtLog2e;
        bias.away = copysignf(1.f, -bias.slope);
        slope_of = h;
        if (BIAS == 2) {
          const float2 cell = at_cell(A, pos);
          bias.y = cell.x * bias.slope;
          bias.x = cell.y * bias.slope;
        }
      }
      const bool by_doc = docs && at_bit(mix, x.t - tiles.begin);
      const bool has_pad = docs && at_bit(pad, x.t - tiles.begin);
      const bool by_lim = DKV ? row0 + kAbRows > n || (causal && prefix < row0 + kAbRows && c0 < row0 + kAbRows - 1 - off)
                              : c0 + kAbCols > lim_min;
      const int slot = tile & 1;
      if (by_doc || BIAS == 2) {
        if (half == 0 && r < kAbCols) {
          if (docs) {
            const int c = c0 + r, L = DKV ? A.Lq : n;
            const int id = c < L ? (DKV ? A.doc_q : A.doc_k)[(long long)b * (DKV ? A.Lq : A.Lk) + c] : -1;
            col_doc[buf][slot][r] = id < 0 ? -1 : id;
          }
          if (BIAS == 2) {
            const float2 cell = at_cell(A, DKV ? off + c0 + r : c0 + r);
            col_y[buf][slot][r] = cell.x;
            col_x[buf][slot][r] = cell.y;
          }
        }
        named_bar_sync(1 + buf, 256);
      }
      // DKV: full counts the rows' bulk copy
      ok = ok && at_wait_warp(&xy_full[buf], (it / NB) & 1, A.err) &&
           (!DKV || at_wait_warp(&full[it % Cfg::STAGES], (it / Cfg::STAGES) & 1, A.err));
      tc_fence_after();
      const int s = it % Cfg::STAGES;
      const float* rows = reinterpret_cast<const float*>(srows + s * Cfg::ROWS) + h0;
      if (BIAS == 1) bias.y = float(pos - (DKV ? off + c0 : c0) - h0) * bias.slope;
      const uint32_t xcol = tmem + lane_base + buf * 128;
      float sv[32], dp[32];
      at_ld32x2(xcol + h0, sv, xcol + 64 + h0, dp);
      uint32_t vis = 0xffffffffu;
      if (by_lim || by_doc) {  // hidden: p = 0 and ds = 0 whatever the operands hold
        vis = DKV ? (from == INT_MAX ? 0u : ~at_low_bits(from - c0 - h0)) : at_low_bits(lim - c0 - h0);
        if (by_doc) vis &= at_same_doc<32>(&col_doc[buf][slot][h0], my_doc);
        at_mask(sv, vis, CAP ? 0.f : -INFINITY);
        at_mask(dp, vis, 0.f);
      }
      AtLine line;
      if (BIAS == 1) line.start(bias);
      uint32_t pp[16], dd[16];
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        float2 v[2] = {make_float2(sv[c], sv[c + 1]), make_float2(sv[c + 2], sv[c + 3])}, sig[2];
        float2 add[2], del[2];  // −lse (with P's factor) and −δ
        if (DKV) {
          const float4 ql = *reinterpret_cast<const float4*>(rows + c), qd = *reinterpret_cast<const float4*>(rows + kAbCols + c);
          add[0] = make_float2(ql.x, ql.y);
          add[1] = make_float2(ql.z, ql.w);
          del[0] = make_float2(qd.x, qd.y);
          del[1] = make_float2(qd.z, qd.w);
        } else {
          add[0] = add[1] = make_float2(row_lse, row_lse);
          del[0] = del[1] = make_float2(row_delta, row_delta);
        }
        if (CAP && (by_lim || by_doc)) {
          add[0] = make_float2((vis >> c) & 1 ? add[0].x : -INFINITY, (vis >> (c + 1)) & 1 ? add[0].y : -INFINITY);
          add[1] = make_float2((vis >> (c + 2)) & 1 ? add[1].x : -INFINITY, (vis >> (c + 3)) & 1 ? add[1].y : -INFINITY);
        }
        float4 ky = {}, kx = {};
        if (BIAS == 2) {
          ky = *reinterpret_cast<const float4*>(&col_y[buf][slot][h0 + c]);
          kx = *reinterpret_cast<const float4*>(&col_x[buf][slot][h0 + c]);
        }
        at_scores4<CAP, BIAS, true, minus.value>(bias, v, add, line, ky, kx, sig);
#pragma unroll
        for (int i = 0; i < 2; i++) {
          float2 p = make_float2(at_ex2(v[i].x), at_ex2(v[i].y));
          // (dP − δ)·F: for DQ in one step, δ being the row's; for DKV with P's factor below
          float2 d = make_float2(dp[c + 2 * i], dp[c + 2 * i + 1]);
          d = BF16 || DKV ? add2(d, del[i]) : fma2(d, make_float2(F, F), del[i]);
          if (CAP) {  // 1 − t² = 4·sig·(1 − sig)
            const float2 g = fma2(sig[i], make_float2(-4.f, -4.f), make_float2(4.f, 4.f));
            d = mul2(d, mul2(g, sig[i]));
          }
          d = mul2(d, BF16 || !DKV ? p : mul2(p, make_float2(F, F)));
          if (DKV) pp[c / 2 + i] = Half16<T>::pack(p.x, p.y);
          dd[c / 2 + i] = Half16<T>::pack_sat(d.x, d.y);
        }
      }
      if (DKV) tmem_st16(xcol + h0, pp);  // over the scores that this thread has read
      tmem_st16(xcol + 64 + h0, dd);
      // streamed rows that nothing sees hold anything, NaN included: 0·NaN must not enter the sums
      if (has_pad || (DKV ? causal && c0 < -off : n < A.Lk && c0 + kAbCols > n)) {
        const int c = c0 + r % kAbCols, panel = half;
        const bool dead = DKV ? rows[r % kAbCols - h0] == -INFINITY : c >= n || (docs && A.doc_k[(long long)b * A.Lk + c] < 0);
        if (ok && dead && panel < Cfg::PANELS) {
          uint8_t* d = strm + s * 2 * Cfg::STRM + (r / kAbCols) * Cfg::STRM + panel * kAbCols * 128 + (r % kAbCols) * 128;
#pragma unroll
          for (int k = 0; k < 8; k++) *reinterpret_cast<uint4*>(d + k * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && ok) at_arrive(smem_u32(&ds_full[buf]));
      tile++;
    }
    };
    // along the line twice in the code: where no slope is negative its sign is free (2 × 4096 causal tokens, 8/2 × 64: 293 us,
    // in one loop 301); on the map that gains nothing (8 × 1600 tokens, 4 × 64: 178 and 174)
    bool plus = BIAS == 1;
    if (BIAS == 1)
      for (int g = 0; g < streams; g++) plus &= !(A.slopes[(DKV ? hd * A.G : hd) + g] < 0.f);
    if (BIAS == 0 || (BIAS == 1 && plus))
      run(std::false_type());
    else
      run(std::true_type());
    const bool any = it > 0;
    ok = ok && at_wait_warp(&acc_done, 0, A.err);
    if (ok) {
      tc_fence_after();
      const float down = BF16 ? 1.f : 1.f / 256.f;
      // four warpgroups (two where NB = 1) share the outputs: by accumulator where there are two, then by columns
      const int wgs = 2 * NB, me = warp / 4, outs = DKV ? 2 : 1, parts = wgs / outs;
      const int which = me / parts;
      {
        const AtView& v = which == 0 ? P.out1 : P.out2;
        const float f = which == 0 ? A.scale * down / F : down;
        const uint32_t acc = tmem + lane_base + (which == 0 ? Cfg::COL_ACC1 : Cfg::COL_ACC2);
        T* o = static_cast<T*>(v.p) + b * v.sb + row * v.st + hd * v.sh;
        const int lo = me % parts * (DP / parts), hi = lo + DP / parts;
        for (int c = lo; c < hi && c < A.D; c += 16) {
          float a[16];
          if (any) at_ld16(acc + c, a);
#pragma unroll
          for (int i = 0; i < 16; i++) a[i] = any ? a[i] * f : 0.f;
          if (!valid) continue;
          if (P.parts > 1) {
            float* f32 = P.part + ((((long long)part * outs + which) * A.B + b) * heads + hd) * ((long long)(DKV ? A.Lk : A.Lq) * A.D) +
                         (long long)row * A.D + c;
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              if (c + i < A.D) *reinterpret_cast<float4*>(f32 + i) = make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]);
            continue;
          }
          const float lo8[8] = {a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7]};
          const float hi8[8] = {a[8], a[9], a[10], a[11], a[12], a[13], a[14], a[15]};
          *reinterpret_cast<uint4*>(o + c) = pack8<T>(lo8);
          if (c + 8 < A.D) *reinterpret_cast<uint4*>(o + c + 8) = pack8<T>(hi8);
        }
      }
    }
  }
  if (P.late) grid_dep_wait();  // what waits for this kernel's end then waits for the one in front too
  tc_fence_before();
  __syncthreads();
  if (warp == 8 * NB + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM);
  }
}

// Shared memory of which an SM has room for one CTA only.  The passes run side by side, and where the GPU holds both at once,
// dQ's CTAs were at times put on the SMs of dK's and dV's all the same, beside idle ones (297 tokens, 4 heads × 64: the
// backward in 26.9 us, so 21.0; 2 × 605 tokens, 16/4 × 64: 66.6 and 64.5).
constexpr int kAbAlone = 116 * 1024;

template <typename T, int DP, bool DKV, int CAP, int BIAS>
cudaError_t attn_bwd_one(const AttnBwdLaunch& L, int grid, cudaStream_t st) {
  static bool set[64] = {};  // per device; a race only repeats the call
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  auto* k = k_attn_bwd<T, DP, DKV, CAP, BIAS>;
  if (dev >= 64 || !set[dev]) {
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, std::max(AbCfg<DP>::SMEM, kAbAlone));
    if (e != cudaSuccess) return e;
    if (dev < 64) set[dev] = true;
  }
  return launch_dependent(k, grid, AbCfg<DP>::THREADS, L.alone ? std::max(AbCfg<DP>::SMEM, kAbAlone) : AbCfg<DP>::SMEM, st, L);
}

template <typename T, int DP, bool DKV, int CAP>
cudaError_t attn_bwd_cap(const AttnBwdLaunch& L, int grid, cudaStream_t st) {
  const int bias = !L.d.slopes ? 0 : L.d.grid_w > 0 ? 2 : 1;
  return bias == 0   ? attn_bwd_one<T, DP, DKV, CAP, 0>(L, grid, st)
         : bias == 1 ? attn_bwd_one<T, DP, DKV, CAP, 1>(L, grid, st)
                     : attn_bwd_one<T, DP, DKV, CAP, 2>(L, grid, st);
}

template <typename T, int DP, bool DKV>
cudaError_t attn_bwd_dp(const AttnBwdLaunch& L, int grid, cudaStream_t st) {
  return L.d.cap == 0.f          ? attn_bwd_cap<T, DP, DKV, 0>(L, grid, st)
         : L.d.cap <= kAtCapLarge ? attn_bwd_cap<T, DP, DKV, 1>(L, grid, st)
                                  : attn_bwd_cap<T, DP, DKV, 2>(L, grid, st);
}

template <typename T, bool DKV>
cudaError_t launch_attn_bwd(const AttnBwdLaunch& L, cudaStream_t st) {
  const int nt = ((DKV ? L.d.Lk : L.d.Lq) + kAbRows - 1) / kAbRows;
  const int grid = nt * L.d.B * (DKV ? L.d.Hk : L.d.Hq) * L.parts;
  if (grid == 0) return cudaSuccess;
  return L.d.D <= 64 ? attn_bwd_dp<T, 64, DKV>(L, grid, st) : attn_bwd_dp<T, 128, DKV>(L, grid, st);
}

}  // namespace osam
