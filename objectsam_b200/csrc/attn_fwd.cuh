// Attention forward (see attn.cuh for the mathematics).  One CTA per 128 query rows of one key head: the rows are
// (token, head of the group) pairs, token-major, so shared key heads read K and V once for the whole group and a
// single token of many heads still fills rows.  Long caches with few rows are split over the keys: each split
// writes its unnormalised output with its maximum and sum, and k_attn_join (attn.cu) adds them.
//
// Per 64-key tile:  S = Q·Kᵀ (tcgen05, fp32 in TMEM) → two threads per row read 32 scores each into registers, apply cap,
// bias and masks, take p = 2^(x − m) against the row's reference maximum m and write P in 16 bits back to TMEM → O +=
// P·V with P as the TMEM operand.  A row is a TMEM lane: its maximum and sum need no shuffles.  m follows the maximum
// only when a tile exceeds it by more than 2^8 (P, fp16's held times 2^7, stays in range, the sum is fp32):
// then the row's two threads agree on it and O, which stays in TMEM, is rescaled; otherwise one flag barrier of the
// two warps tells that nothing is to do.  Tiles are visited from the CTA's own positions outwards, so that with a
// distance bias the largest scores come first and this stays rare.
// Up to 32 rows (single tokens): a warp's instructions cost the same for one row as for 32, and all rows would lie in the
// lanes of two warps, on one of the SM's four schedulers.  So the rows are repeated in the four 32-lane groups, and
// group g takes columns 8g … 8g+7 of each half alone, with a maximum and a sum of its own; P of the other columns stays
// zero, and the groups' outputs are joined in shared memory at the end (16 sequences over caches of 8192–32768 keys: 282
// us without this, 250 with it).
// Warps 0–7: softmax (warps w and w + 4 share rows), warp 8: TMA producer, warp 9: TMEM owner and MMA issuer.  The
// softmax is a chain of latencies (barriers, TMEM loads, the exponentials' unit) that four warps a scheduler hide:
// two CTAs per SM, 256 TMEM columns each: S, which the next tile's Q·Kᵀ overwrites as soon as it is in registers,
// two buffers of P, and O.
#pragma once
#include <type_traits>

#include "attn.cuh"

namespace osam {

constexpr int kAfSoft = 256;    // softmax threads
constexpr int kAfThreads = kAfSoft + 64;
constexpr float kAfGrow = 8.f;  // log2 growth over a row's reference maximum that forces a rescale
constexpr float kAfUp = 7.f;    // fp16: P is held times 2^7 (at most 2^15), so weights down to 2^-31 of the reference enter O

template <int DP>
struct AfCfg {
  static constexpr int PANELS = DP / 64;
  static constexpr int STAGES = DP == 64 ? 4 : 2;
  static constexpr int COL_S = 0, COL_P = 64, COL_O = 128;  // P buffer i at COL_P + 32·i
  static constexpr int QPANEL = kAfRows * 128, KPANEL = kAfKeys * 128;  // bytes of a 64-dim panel
  static constexpr int QTILE = PANELS * QPANEL, TILE = PANELS * KPANEL;
  static constexpr int SMEM = 1024 + QTILE + 2 * STAGES * TILE;
};

// The chunk (at_best_chunk) for the lengths that `lens` has.
__device__ __forceinline__ int at_chunk(const AttnDev& A, int per, int min_tiles, int lane) {
  int total = 0;
  for (int b = lane; b < A.B; b += 32) total += at_seq_tiles(A, b);
  total = __reduce_add_sync(0xffffffffu, total);
  return at_best_chunk(A.B, per, min_tiles, (A.Lk + kAfKeys - 1) / kAfKeys, total, [&](int chunk) {
    int n = 0;
    const float inv = 1.f / float(chunk);
    for (int b = lane; b < A.B; b += 32) {
      const int t = at_seq_tiles(A, b) + chunk - 1;
      int s = int(float(t) * inv);  // within one of t / chunk
      s += (s + 1) * chunk <= t;
      s -= s * chunk > t;
      n += max(1, s);
    }
    return __reduce_add_sync(0xffffffffu, n);
  });
}
// What CTA `cta` of a split call works on: sequence, number of its splits (0: more CTAs than these lengths need), index
// among the sequence's CTAs.
struct AtSplitCta {
  int seq, splits, i, chunk;
};
static __device__ __noinline__ AtSplitCta at_split_cta(const AttnFwdLaunch& P, int per, int lane, int cta) {
  const AttnDev& A = P.d;
  AtSplitCta r{0, 0, 0, A.lens ? at_chunk(A, per, P.min_tiles, lane) : P.chunk_all};
  int base = 0;
  for (int b0 = 0; b0 < A.B; b0 += 32) {
    const int s = b0 + lane < A.B ? at_seq_splits(A, b0 + lane, r.chunk) : 0;
    int end = s * per;
#pragma unroll
    for (int k = 1; k < 32; k *= 2) {
      const int left = __shfl_up_sync(0xffffffffu, end, k);
      if (lane >= k) end += left;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, cta < base + end);
    if (past) {
      const int f = __ffs(past) - 1;
      r.seq = b0 + f;
      r.splits = __shfl_sync(0xffffffffu, s, f);
      r.i = cta - base - __shfl_sync(0xffffffffu, end, f) + r.splits * per;
      break;
    }
    base += __shfl_sync(0xffffffffu, end, 31);
  }
  return r;
}

template <typename T, int DP, int CAP, int BIAS, bool SPREAD>
__global__ void __launch_bounds__(kAfThreads, 2) k_attn_fwd(const __grid_constant__ AttnFwdLaunch P) {
  using Cfg = AfCfg<DP>;
  constexpr bool BF16 = Half16<T>::kBf16;
  constexpr int KEYS = kAfKeys, N = SPREAD ? 8 : 32;  // N: columns of a thread
  constexpr float up = BF16 ? 0.f : kAfUp;
  extern __shared__ uint8_t af_raw[];
  __shared__ __align__(8) uint64_t k_full[Cfg::STAGES], k_empty[Cfg::STAGES], v_full[Cfg::STAGES], v_empty[Cfg::STAGES];
  __shared__ __align__(8) uint64_t s_full, s_free, p_full[2], pv_done, o_done;
  __shared__ uint32_t tmem_slot;
  __shared__ float pair_top[2][kAfRows], pair_sum[2][kAfRows];  // what the two threads of a row tell each other
  __shared__ float pair_low[2][SPREAD ? kAfRows : 1];
  __shared__ uint32_t live[kAtDocWords], mix[kAtDocWords], pad[kAtDocWords];
  __shared__ AtDocs own_docs[4];
  __shared__ __align__(16) int col_doc[2][KEYS];
  __shared__ __align__(16) float col_y[BIAS == 2 ? 2 : 1][KEYS], col_x[BIAS == 2 ? 2 : 1][KEYS];

  grid_dep_wait();
  const AttnDev& A = P.d;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  uint8_t* smem = af_raw + ((1024 - (smem_u32(af_raw) & 1023)) & 1023);
  const uint32_t sq = smem_u32(smem), sk = sq + Cfg::QTILE, sv = sk + Cfg::STAGES * Cfg::TILE;

  // ---- which tile: with a causal bound the longest rows first; or which split
  const int rows = A.Lq * A.G, nq = (rows + kAfRows - 1) / kAfRows;
  int qt, rest, split = 0, splits = 1, first_tile = 0, own_tiles = 1 << 26;
  if (P.splits == 1) {
    at_order(blockIdx.x, nq, A.B * A.Hk, P.group, qt, rest);
    if (A.mask != OSAM_ATTN_NONE) qt = nq - 1 - qt;
  } else {
    const AtSplitCta c = at_split_cta(P, nq * A.Hk, lane, blockIdx.x);
    if (blockIdx.x == 0 && tid == 0) *P.chunk = c.chunk;  // for the join
    if (c.splits == 0) return;
    split = c.i % c.splits;
    qt = c.i / c.splits / A.Hk;
    rest = c.seq * A.Hk + c.i / c.splits % A.Hk;
    splits = c.splits;
    own_tiles = (at_seq_tiles(A, c.seq) + splits - 1) / splits;
    first_tile = split * own_tiles;
  }
  const int hk = rest % A.Hk, b = rest / A.Hk;
  const int r0 = qt * kAfRows, r_last = min(r0 + kAfRows, rows) - 1;
  const int n = at_keys(A, b), off = n - A.Lq;
  const int prefix = A.mask == OSAM_ATTN_PREFIX ? A.prefix[b] : 0;
  const int lim_max = at_limit(A, n, prefix, off + A.f_g.quo(r_last)), lim_min = at_limit(A, n, prefix, off + A.f_g.quo(r0));
  AtTiles tiles;
  tiles.begin = first_tile;
  tiles.end = max(tiles.begin, min((lim_max + KEYS - 1) / KEYS, tiles.begin + own_tiles));
  tiles.from = min(max((off + A.f_g.quo(r_last)) / KEYS, tiles.begin), tiles.end - 1);
  const bool docs = A.doc_q != nullptr;
  tiles.live = docs ? live : nullptr;

  // ---- this thread's row
  const int r = r0 + (SPREAD ? lane : tid % kAfRows);
  const bool valid = warp < 8 && r < rows;
  const int qi = valid ? A.f_g.quo(r) : 0, head = hk * A.G + (valid ? r - qi * A.G : 0);
  int my_doc = -2;
  if (valid && docs) {
    my_doc = A.doc_q[(long long)b * A.Lq + qi];
    if (my_doc < 0) my_doc = -2;
  }

  // the producer warp sets the barriers up and, where no document summaries have to be looked through first, starts
  // loading at once, under the rest of the prologue
  int made = 0, next_tile = tiles.end;
  auto load = [&](int it, int t, bool v) {
    const int s = it % Cfg::STAGES;
    uint64_t* bar = v ? &v_full[s] : &k_full[s];
    mbar_arrive_expect_tx(bar, Cfg::TILE);
    for (int p = 0; p < Cfg::PANELS; p++)
      tma_load_4d(smem + Cfg::QTILE + ((v ? Cfg::STAGES : 0) + s) * Cfg::TILE + p * Cfg::KPANEL, v ? &P.tv : &P.tk, bar,
                  p * 64, t * KEYS, hk, b);
  };
  if (warp == 8 && lane == 0) {
    for (int i = 0; i < Cfg::STAGES; i++) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(&s_full, 1);
    mbar_init(&s_free, 8);
    mbar_init(&p_full[0], 8);  // two: a warp may be a tile ahead of another
    mbar_init(&p_full[1], 8);
    mbar_init(&pv_done, 1);
    mbar_init(&o_done, 1);
    fence_barrier_init();
    if (!docs)
      for (next_tile = tiles.first(); made < Cfg::STAGES && next_tile < tiles.end; next_tile = tiles.next(next_tile), made++) {
        load(made, next_tile, false);
        load(made, next_tile, true);
      }
  }
  if (warp == 9) {
    tmem_alloc(&tmem_slot, 256);
    tmem_relinquish();
    // the CTA's one signal, given once TMEM is its own: the next kernel's CTAs may take columns and then wait for this one
    grid_dep_launch();
  }
  if (warp < 8) {
    // Q rows into the K-major swizzled panels; rows past the end and dims past D are zero
    constexpr int CH = DP / 8;
    const T* q = static_cast<const T*>(P.q.p) + b * P.q.sb;
#pragma unroll 8
    for (int c = tid; c < kAfRows * CH; c += kAfSoft) {
      const int row = c / CH, ch = c % CH, rr = r0 + (SPREAD ? row % 32 : row);
      uint4 u = make_uint4(0, 0, 0, 0);
      if (rr < rows && ch * 8 < A.D) {
        const int i = A.f_g.quo(rr), h = hk * A.G + rr - i * A.G;
        u = *reinterpret_cast<const uint4*>(q + i * P.q.st + h * P.q.sh + ch * 8);
      }
      *reinterpret_cast<uint4*>(smem + (ch / 8) * Cfg::QPANEL + at_sw128(row, ch % 8)) = u;
    }
    fence_proxy_async_smem();
    if (docs && warp < 4) {
      AtDocs d{my_doc >= 0 ? my_doc : INT_MAX, my_doc, valid && my_doc < 0, 0};
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        d.lo = min(d.lo, __shfl_xor_sync(0xffffffffu, d.lo, o));
        d.hi = max(d.hi, __shfl_xor_sync(0xffffffffu, d.hi, o));
        d.pad |= __shfl_xor_sync(0xffffffffu, d.pad, o);
      }
      if (lane == 0) own_docs[warp] = d;
    }
  }
  __syncthreads();
  if (docs) {
    AtDocs own = own_docs[0];
    for (int w = 1; w < 4; w++) {
      own.lo = min(own.lo, own_docs[w].lo);
      own.hi = max(own.hi, own_docs[w].hi);
      own.pad |= own_docs[w].pad;
    }
    const int nb = (A.Lk + kAtDocBlock - 1) / kAtDocBlock;
    at_doc_bits(own, A.sum_k + (long long)b * nb, nb, KEYS / kAtDocBlock, tiles.begin, tiles.end, warp,
                kAfThreads / 32, live, mix, pad);
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 8) {
    if (lane == 0) {
      if (docs) next_tile = tiles.first();
      int it = made;
      for (int t = next_tile; t < tiles.end; t = tiles.next(t), it++) {
        const int s = it % Cfg::STAGES;
        const uint32_t ph = ((it / Cfg::STAGES) & 1) ^ 1;
        if (it >= Cfg::STAGES && !at_wait(&k_empty[s], ph, A.err)) break;
        load(it, t, false);
        if (it >= Cfg::STAGES && !at_wait(&v_empty[s], ph, A.err)) {
          at_wait(&k_full[s], (it / Cfg::STAGES) & 1, A.err);
          break;
        }
        load(it, t, true);
      }
      // no copy of this CTA may be in flight when it ends
      for (int i = max(0, it - Cfg::STAGES); i < it; i++) {
        at_wait(&k_full[i % Cfg::STAGES], (i / Cfg::STAGES) & 1, A.err);
        at_wait(&v_full[i % Cfg::STAGES], (i / Cfg::STAGES) & 1, A.err);
      }
    }
    __syncwarp();
  } else if (warp == 9) {
    const uint32_t leader = elect_leader();
    const int ks = (A.D + 15) / 16;  // K steps of Q·Kᵀ; N of P·V is 16·ks
    const uint32_t id_s = at_idesc(BF16, 128, KEYS, false), id_o = at_idesc(BF16, 128, 16 * ks, true);
    const uint64_t dq = smem_desc_kmajor(sq, 128), dk = smem_desc_kmajor(sk, 128), dv = at_desc_mn(sv, Cfg::KPANEL);
    const int count = __shfl_sync(0xffffffffu, tiles.count(), 0);
    auto qk = [&](int it) {  // offsets in a descriptor: bytes / 16
      const uint64_t kb = dk + ((it % Cfg::STAGES) * Cfg::TILE >> 4);
#pragma unroll
      for (int k = 0; k < DP / 16; k++)
        if (k < ks)
          mma_ss(leader, tmem + Cfg::COL_S, dq + (((k / 4) * Cfg::QPANEL + (k % 4) * 32) >> 4),
                 kb + (((k / 4) * Cfg::KPANEL + (k % 4) * 32) >> 4), id_s, k > 0);
      mma_commit(leader, &s_full);
      mma_commit(leader, &k_empty[it % Cfg::STAGES]);
    };
    bool ok = true;
    if (count > 0 && (ok = at_wait_warp(&k_full[0], 0, A.err))) {
      tc_fence_after();
      qk(0);
    }
    for (int it = 0; ok && it < count; it++) {
      const int s = it % Cfg::STAGES, s1 = (it + 1) % Cfg::STAGES;
      if (it + 1 < count) {
        if (!(ok = at_wait_warp(&k_full[s1], ((it + 1) / Cfg::STAGES) & 1, A.err))) break;
        if (!(ok = at_wait_warp(&s_free, it & 1, A.err))) break;
        tc_fence_after();
        qk(it + 1);
      }
      if (!(ok = at_wait_warp(&v_full[s], (it / Cfg::STAGES) & 1, A.err))) break;
      if (!(ok = at_wait_warp(&p_full[it & 1], (it >> 1) & 1, A.err))) break;
      tc_fence_after();
      const uint64_t vb = dv + (s * Cfg::TILE >> 4);
#pragma unroll
      for (int k = 0; k < KEYS / 16; k++)
        mma_ts(leader, tmem + Cfg::COL_O, tmem + Cfg::COL_P + (it & 1) * 32 + k * 8,
               vb + (k * 16 * 128 >> 4), id_o, (it | k) != 0);
      mma_commit(leader, &v_empty[s]);
      mma_commit(leader, &pv_done);
    }
    mma_commit(leader, &o_done);
    if (!ok) at_wait_warp(&o_done, 0, A.err);  // the issued MMAs finish before TMEM is freed
  } else {
    const int half = warp / 4, row_of = tid % kAfRows, h0 = half * 32, pair_bar = 2 + warp % 4;
    const uint32_t lane_base = uint32_t((warp % 4) * 32) << 16;
    const bool idle = !SPREAD && r0 + (warp % 4) * 32 >= rows;  // no row of this warp exists: it only keeps step
    const int pos = off + qi;
    const int lim = valid ? at_limit(A, n, prefix, pos) : 0;
    // without cap and bias the scale is applied with the exponent's FMA: x·cmul are scores in log2 units
    const float cmul = CAP || BIAS ? 1.f : A.scale * kAtLog2e;
    AtBias bias;
    bias.mul = CAP ? 2.f * A.scale * kAtLog2e / A.cap : A.scale * kAtLog2e;
    bias.cap2 = A.cap * kAtLog2e;
    bias.lin = A.scale * kAtLog2e;
    bias.arg = A.scale / A.cap;
    bias.slope = BIAS && valid ? A.slopes[head] * kAtLog2e : 0.f;
    bias.y = bias.x = 0.f;
    if (BIAS == 2) {
      const float2 cell = at_cell(A, pos);
      bias.y = cell.x * bias.slope;
      bias.x = cell.y * bias.slope;
    }
    float m = -INFINITY;  // the row's reference maximum, log2 units (−∞: nothing seen yet)
    float neg = 0.f;      // up − m, or 0 while there is none
    float l = 0.f;        // this thread's part of its sum (of P as it is held)
    float l16 = 0.f;      // SPREAD: the same of P as the tensor cores read it, rounded to 16 bits
    const uint32_t bar_s = smem_u32(&s_full), bar_free = smem_u32(&s_free), bar_p = smem_u32(&p_full[0]);
    const int c1 = h0 + (SPREAD ? 8 * (warp % 4) : 0);  // first column of this thread
    const uint32_t s_addr = tmem + lane_base + Cfg::COL_S + c1, p_addr = tmem + lane_base + Cfg::COL_P + c1 / 2;
    if (SPREAD) {  // what a group never writes of P
      const uint32_t zero[16] = {};
      tmem_st16(tmem + lane_base + Cfg::COL_P + h0 / 2, zero);
      tmem_st16(tmem + lane_base + Cfg::COL_P + 32 + h0 / 2, zero);
    }
    bias.away = copysignf(1.f, -bias.slope);
    const int tail = n < A.Lk ? n : INT_MAX;  // keys from here on hold anything
    bool ok = true, lead = lane == 0;  // lead: arrives for the warp, until a wait of its own or its partner's has run out
    int it = 0, fills = 0;
    auto run = [&](auto minus) {
    for (int t = tiles.first(); t < tiles.end; it++) {
      const int j0 = t * KEYS;
      bool by_doc = false, dirty = j0 + KEYS > tail;
      if (docs) {
        by_doc = at_bit(mix, t - tiles.begin);
        dirty |= at_bit(pad, t - tiles.begin);
      }
      const bool masked = by_doc || j0 + KEYS > lim_min;
      // Per-key data of the tile, one key a thread.  The buffer goes by the fills, not by the tiles: the barrier of the fill
      // in between tells that all warps have read what this one overwrites (tiles without a fill have no barrier).
      const int slot = fills & 1;
      if (by_doc || BIAS == 2) {
        fills++;
        if (tid < KEYS) {
          const int j = j0 + tid;
          if (docs) {
            const int id = j < n ? A.doc_k[(long long)b * A.Lk + j] : -1;
            col_doc[slot][tid] = id < 0 ? -1 : id;
          }
          if (BIAS == 2) {
            const float2 cell = at_cell(A, j);
            col_y[slot][tid] = cell.x;
            col_x[slot][tid] = cell.y;
          }
        }
        named_bar_sync(1, kAfSoft);
      }
      if (ok) ok = at_wait(bar_s, it & 1, A.err);
      tc_fence_after();
      float top = -INFINITY;
      float x[N];
      if constexpr (!SPREAD)
        at_ld32(s_addr, x);
      else
        at_ld8(s_addr, x);
      tc_fence_before();
      __syncwarp();
      if (lead) at_arrive(bar_free);
      t = tiles.next(t);
      if (!idle) {
        uint32_t vis = 0xffffffffu;
        if (masked) {
          vis = at_low_bits(lim - j0 - c1);
          if (by_doc) vis &= at_same_doc<N>(&col_doc[slot][c1], my_doc);
          if (CAP) at_mask(x, vis, 0.f);
        }
        if (CAP || BIAS) {
          AtLine line;
          if (BIAS == 1) {
            bias.y = float(pos - j0 - c1) * bias.slope;
            line.start(bias);
          }
          const float2 none[2] = {};
#pragma unroll
          for (int c = 0; c < N; c += 4) {
            float2 s2[2] = {make_float2(x[c], x[c + 1]), make_float2(x[c + 2], x[c + 3])}, sig[2];
            float4 ky = {}, kx = {};
            if (BIAS == 2) {
              ky = *reinterpret_cast<const float4*>(&col_y[slot][c1 + c]);
              kx = *reinterpret_cast<const float4*>(&col_x[slot][c1 + c]);
            }
            at_scores4<CAP, BIAS, false, minus.value>(bias, s2, none, line, ky, kx, sig);
            x[c] = s2[0].x;
            x[c + 1] = s2[0].y;
            x[c + 2] = s2[1].x;
            x[c + 3] = s2[1].y;
          }
        }
        if (masked) at_mask(x, vis, -INFINITY);
        float top1 = fmaxf(x[2], x[3]);
        top = fmaxf(x[0], x[1]);
#pragma unroll
        for (int c = 4; c < N; c += 4) {
          top = fmaxf(fmaxf(top, x[c]), x[c + 1]);
          top1 = fmaxf(fmaxf(top1, x[c + 2]), x[c + 3]);
        }
        top = fmaxf(top, top1) * cmul;
      }
      if (at_pair_any(pair_bar, top > m + kAfGrow || !ok)) {  // also the first score that a row sees: −∞ + 8 = −∞
        ok = !at_pair_any(pair_bar, !ok);
        pair_top[half][row_of] = top;
        named_bar_sync(pair_bar, 64);
        top = fmaxf(top, pair_top[half ^ 1][row_of]);
        float f = 1.f;
        if (top > m + kAfGrow) {
          f = m == -INFINITY ? 0.f : at_ex2(m - top);
          m = top;
          neg = up - m;
          l *= f;
          l16 *= f;
        }
        if (ok && it > 0) ok = at_wait_warp(&pv_done, (it - 1) & 1, A.err);  // the previous P·V is in O
        lead &= ok;
        tc_fence_after();
#pragma unroll 1
        for (int c = half * (DP / 2); it > 0 && c < (half + 1) * (DP / 2); c += 16) {
          float o[16];
          at_ld16(tmem + lane_base + Cfg::COL_O + c, o);
#pragma unroll
          for (int i = 0; i < 16; i++) o[i] = f == 0.f ? 0.f : o[i] * f;
          tmem_st16(tmem + lane_base + Cfg::COL_O + c, reinterpret_cast<const uint32_t*>(o));
        }
      }
      if (!idle) {
        const float2 mul = make_float2(cmul, cmul), add = make_float2(neg, neg);
        float2 sum[2] = {make_float2(l, 0.f), make_float2(0.f, 0.f)}, low = make_float2(l16, 0.f);
        uint32_t p[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
          float2 e = make_float2(x[2 * i], x[2 * i + 1]);
          e = CAP || BIAS ? add2(e, add) : fma2(e, mul, add);
          e.x = at_ex2(e.x);
          e.y = at_ex2(e.y);
          sum[i & 1] = add2(sum[i & 1], e);
          p[i] = Half16<T>::pack(e.x, e.y);
          if (SPREAD) low = add2(low, Half16<T>::unpack(p[i]));
        }
        if (SPREAD) l16 = low.x + low.y;
        // this buffer of P is free: S tells that the P·V before last is done
        if constexpr (!SPREAD)
          tmem_st16(p_addr + (it & 1) * 32, p);
        else
          tmem_st4(p_addr + (it & 1) * 32, p);
        const float2 s = add2(sum[0], sum[1]);
        l = s.x + s.y;
      }
      if (dirty) {  // V rows of keys that no query sees hold anything, NaN included: 0·NaN must not enter O
        if (ok) lead &= ok = at_wait_warp(&v_full[it % Cfg::STAGES], (it / Cfg::STAGES) & 1, A.err);
        const int key = tid % KEYS, j = j0 + key, panel = tid / KEYS;  // a thread per row and panel
        if (ok && panel < Cfg::PANELS && (j >= n || (docs && A.doc_k[(long long)b * A.Lk + j] < 0))) {
          uint8_t* v = smem + Cfg::QTILE + (Cfg::STAGES + it % Cfg::STAGES) * Cfg::TILE + panel * Cfg::KPANEL + key * 128;
#pragma unroll
          for (int c = 0; c < 8; c++) *reinterpret_cast<uint4*>(v + c * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lead) at_arrive(bar_p + (it & 1) * 8);
    }
    };
    // twice in the code: with slopes of one sign in the warp, as nearly always, the sign costs nothing (8191 tokens with a bias
    // along the line 166 us, with both signs in one loop 173)
    if (BIAS && __any_sync(0xffffffffu, bias.slope < 0.f))
      run(std::integral_constant<bool, BIAS != 0>());
    else
      run(std::false_type());
    ok = ok && at_wait_warp(&o_done, 0, A.err);
    tc_fence_after();
    pair_sum[half][row_of] = l;
    if (SPREAD) {
      pair_low[half][row_of] = l16;
      if (half == 0) pair_top[0][row_of] = m;
      ok = !at_any(1, !ok, kAfSoft);
    } else {
      ok = !at_pair_any(pair_bar, !ok);
    }
    l += pair_sum[half ^ 1][row_of];
    // few or nearly equal weights share their rounding to 16 bits; against the sum of the rounded weights it cancels (two
    // tokens over 10860 keys, bf16: error 1.7e-3 instead of 1.9e-3, o's own rounding being 1.6e-3); lse keeps the exact sum
    float fix = 1.f;
    float w4[4] = {1.f, 0.f, 0.f, 0.f};  // the groups' weights
    const int g = warp % 4;
    if (SPREAD) {
      l16 += pair_low[half ^ 1][row_of];
      if (l16 > 0.f) fix = l / l16;
      float M = -INFINITY;
#pragma unroll
      for (int k = 0; k < 4; k++) M = fmaxf(M, pair_top[0][k * 32 + lane]);
      l = 0.f;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float mk = pair_top[0][k * 32 + lane];
        w4[k] = mk == -INFINITY ? 0.f : at_ex2(mk - M);
        l = fmaf(w4[k], pair_sum[0][k * 32 + lane] + pair_sum[1][k * 32 + lane], l);
      }
      m = M;
    }
    if (ok) {
      m -= up;  // from here on l's reference
      const long long row = ((long long)b * A.Hq + head) * A.Lq + qi;
      const long long part_row = (long long)split * A.B * A.Hq * A.Lq + row;
      T* o_ptr = static_cast<T*>(P.o.p) + b * P.o.sb + qi * P.o.st + head * P.o.sh;
      // eight dims of the row against m, l: to o, or for a split as they are
      auto put = [&](int c, const float (&v)[8], float inv) {
        if (P.splits == 1) {
          float w[8];
#pragma unroll
          for (int k = 0; k < 8; k++) w[k] = v[k] * inv;
          *reinterpret_cast<uint4*>(o_ptr + c) = pack8<T>(w);
        } else {
          float4* d = reinterpret_cast<float4*>(P.part + part_row * A.D + c);
          d[0] = make_float4(v[0], v[1], v[2], v[3]);
          d[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
      };
      float* joined = reinterpret_cast<float*>(smem);  // [group][row][DP + 4]: the operands' room is free by now
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // a NaN sum stays one
#pragma unroll
      for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 16) {
        if (c >= A.D) break;
        float o[16];
        if (it > 0) at_ld16(tmem + lane_base + Cfg::COL_O + c, o);
#pragma unroll
        for (int i = 0; i < 16; i++) o[i] = it > 0 && l != 0.f ? (SPREAD ? o[i] * fix : o[i]) : 0.f;
        if (!valid) continue;
        const float lo[8] = {o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7]};
        const float hi[8] = {o[8], o[9], o[10], o[11], o[12], o[13], o[14], o[15]};
        if (SPREAD) {
          float4* d = reinterpret_cast<float4*>(joined + (g * 32 + lane) * (DP + 4) + c);
          d[0] = make_float4(lo[0], lo[1], lo[2], lo[3]);
          d[1] = make_float4(lo[4], lo[5], lo[6], lo[7]);
          d[2] = make_float4(hi[0], hi[1], hi[2], hi[3]);
          d[3] = make_float4(hi[4], hi[5], hi[6], hi[7]);
          continue;
        }
        put(c, lo, inv);
        if (c + 8 < A.D) put(c + 8, hi, inv);
      }
      if (SPREAD) {  // group g joins every fourth of the row's 8-dim pieces of its half
        named_bar_sync(1, kAfSoft);
        for (int c = half * (DP / 2) + g * 8; valid && c < (half + 1) * (DP / 2) && c < A.D; c += 32) {
          float v[8] = {};
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const float4* d = reinterpret_cast<const float4*>(joined + (k * 32 + lane) * (DP + 4) + c);
            const float4 a = d[0], e = d[1];
            if (w4[k] == 0.f) continue;  // a group that saw nothing
            v[0] = fmaf(w4[k], a.x, v[0]);
            v[1] = fmaf(w4[k], a.y, v[1]);
            v[2] = fmaf(w4[k], a.z, v[2]);
            v[3] = fmaf(w4[k], a.w, v[3]);
            v[4] = fmaf(w4[k], e.x, v[4]);
            v[5] = fmaf(w4[k], e.y, v[5]);
            v[6] = fmaf(w4[k], e.z, v[6]);
            v[7] = fmaf(w4[k], e.w, v[7]);
          }
          put(c, v, inv);
        }
      }
      if (valid && half == 0 && (!SPREAD || g == 0)) {
        if (P.splits > 1)
          P.stats[part_row] = make_float2(m, l);
        else if (P.lse)
          P.lse[row] = l == 0.f ? -INFINITY : (m + at_lg2(l)) * kAtLn2;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

template <typename T, int DP, int CAP, int BIAS, bool SPREAD>
cudaError_t attn_fwd_one(const AttnFwdLaunch& L, cudaStream_t st) {
  static bool set[64] = {};  // per device; a race only repeats the call
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  auto* k = k_attn_fwd<T, DP, CAP, BIAS, SPREAD>;
  if (dev >= 64 || !set[dev]) {
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, AfCfg<DP>::SMEM);
    if (e != cudaSuccess) return e;
    if (dev < 64) set[dev] = true;
  }
  return launch_dependent(k, L.grid, kAfThreads, AfCfg<DP>::SMEM, st, L);
}

template <typename T, int DP, int CAP, bool SPREAD>
cudaError_t attn_fwd_cap(const AttnFwdLaunch& L, cudaStream_t st) {
  const int bias = !L.d.slopes ? 0 : L.d.grid_w > 0 ? 2 : 1;
  return bias == 0   ? attn_fwd_one<T, DP, CAP, 0, SPREAD>(L, st)
         : bias == 1 ? attn_fwd_one<T, DP, CAP, 1, SPREAD>(L, st)
                     : attn_fwd_one<T, DP, CAP, 2, SPREAD>(L, st);
}

template <typename T, int DP, bool SPREAD>
cudaError_t attn_fwd_dp(const AttnFwdLaunch& L, cudaStream_t st) {
  return L.d.cap == 0.f          ? attn_fwd_cap<T, DP, 0, SPREAD>(L, st)
         : L.d.cap <= kAtCapLarge ? attn_fwd_cap<T, DP, 1, SPREAD>(L, st)
                                  : attn_fwd_cap<T, DP, 2, SPREAD>(L, st);
}

template <typename T>
cudaError_t launch_attn_fwd(const AttnFwdLaunch& L, cudaStream_t st) {
  if (L.d.Lq * L.d.G <= 32)  // one row a lane of a 32-lane group
    return L.d.D <= 64 ? attn_fwd_dp<T, 64, true>(L, st) : attn_fwd_dp<T, 128, true>(L, st);
  return L.d.D <= 64 ? attn_fwd_dp<T, 64, false>(L, st) : attn_fwd_dp<T, 128, false>(L, st);
}

}  // namespace osam
