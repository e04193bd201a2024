// Attention forward (see attn.cuh for the mathematics).  One CTA per 128 query rows of one key head: the rows are
// (token, head of the group) pairs, token-major, so shared key heads read K and V once for the whole group and a
// single token of many heads still fills rows.  Long caches with few rows are split over the keys: each split
// writes its unnormalised output with its maximum and sum, and k_attn_join (attn.cu) adds them.
//
// Per 128-key tile:  S = Q·Kᵀ (tcgen05, fp32 in TMEM) → one thread per row reads its 128 scores from TMEM, applies
// cap, bias and masks, keeps the running maximum and sum (no shuffles: a row is a lane) and writes P in 16 bits
// back to TMEM → O += P·V with P as the TMEM operand.  O stays in TMEM; it is rescaled only when a row's maximum
// grew by more than 2^8 (P ≤ 2^8 keeps its relative precision in 16 bits, the sum is fp32), which after the first
// tiles is rare.
// Warps 0–3: softmax (thread = row = TMEM lane), warp 4: TMA producer, warp 5: TMEM owner and MMA issuer.
// TMEM, 256 columns a CTA (two CTAs per SM, whose softmax and MMA phases overlap): up to 64 head dims S | O | P with S
// released as soon as it is in registers, so the next Q·Kᵀ runs under the softmax; above, S | O with P written over S.
#pragma once
#include "attn.cuh"

namespace osam {

constexpr int kAfRows = 128, kAfKeys = 128;
constexpr int kAfThreads = 192;
constexpr int kAfPanel = kAfRows * 128;  // bytes of a 64-dim panel of 128 rows
constexpr float kAfGrow = 8.f;           // log2 growth of a row's maximum that forces a rescale

template <int DP>
struct AfCfg {
  static constexpr int PANELS = DP / 64;
  static constexpr int STAGES = DP == 64 ? 2 : 1;
  static constexpr bool EARLY = DP == 64;  // P beside S
  static constexpr int COL_S = 0, COL_O = 128, COL_P = EARLY ? 192 : 0;
  static constexpr int TILE = PANELS * kAfPanel;
  static constexpr int SMEM = 1024 + TILE * (1 + 2 * STAGES);
};

template <typename T, int DP, bool CAP, int BIAS>
__global__ void __launch_bounds__(kAfThreads, 2) k_attn_fwd(const __grid_constant__ AttnFwdLaunch P) {
  using Cfg = AfCfg<DP>;
  constexpr bool BF16 = Half16<T>::kBf16;
  extern __shared__ uint8_t af_raw[];
  __shared__ __align__(8) uint64_t k_full[Cfg::STAGES], k_empty[Cfg::STAGES], v_full[Cfg::STAGES], v_empty[Cfg::STAGES];
  __shared__ __align__(8) uint64_t s_full, s_free, p_full, pv_done, drain;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t live[kAtDocWords], mix[kAtDocWords], pad[kAtDocWords];
  __shared__ AtDocs own_docs[4];
  __shared__ __align__(16) int col_doc[2][kAfKeys];
  __shared__ __align__(16) float2 col_cell[BIAS == 2 ? 2 : 1][kAfKeys];

  const AttnDev& A = P.d;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  uint8_t* smem = af_raw + ((1024 - (smem_u32(af_raw) & 1023)) & 1023);
  const uint32_t sq = smem_u32(smem), sk = sq + Cfg::TILE, sv = sk + Cfg::STAGES * Cfg::TILE;

  // ---- which tile: with a causal bound the longest rows first
  const int rows = A.Lq * A.G, nq = (rows + kAfRows - 1) / kAfRows;
  const int per_q = A.B * A.Hk * P.splits;
  const int qt = A.mask == OSAM_ATTN_NONE ? int(blockIdx.x) % nq : nq - 1 - int(blockIdx.x) / per_q;
  int rest = A.mask == OSAM_ATTN_NONE ? int(blockIdx.x) / nq : int(blockIdx.x) % per_q;
  const int split = rest % P.splits;
  rest /= P.splits;
  const int hk = rest % A.Hk, b = rest / A.Hk;
  const int r0 = qt * kAfRows, r_last = min(r0 + kAfRows, rows) - 1;
  const int n = at_keys(A, b), off = n - A.Lq;
  const int prefix = A.mask == OSAM_ATTN_PREFIX ? A.prefix[b] : 0;
  const int lim_max = at_limit(A, n, prefix, off + r_last / A.G), lim_min = at_limit(A, n, prefix, off + r0 / A.G);
  AtTiles tiles;
  tiles.begin = split * P.tiles_per_split;
  tiles.end = max(tiles.begin, min((lim_max + kAfKeys - 1) / kAfKeys, tiles.begin + P.tiles_per_split));
  const bool docs = A.doc_q != nullptr;
  tiles.live = docs ? live : nullptr;

  // ---- this thread's row
  const int r = r0 + tid;
  const bool valid = warp < 4 && r < rows;
  const int qi = valid ? r / A.G : 0, head = hk * A.G + (valid ? r - qi * A.G : 0);
  int my_doc = -2;
  if (valid && docs) {
    my_doc = A.doc_q[(long long)b * A.Lq + qi];
    if (my_doc < 0) my_doc = -2;
  }

  if (tid == 0) {
    for (int i = 0; i < Cfg::STAGES; i++) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(&s_full, 1);
    mbar_init(&s_free, 4);
    mbar_init(&p_full, 4);
    mbar_init(&pv_done, 1);
    mbar_init(&drain, 1);
    fence_barrier_init();
    tma_prefetch_desc(&P.tk);
    tma_prefetch_desc(&P.tv);
  }
  if (warp == 5) {
    tmem_alloc(&tmem_slot, 256);
    tmem_relinquish();
  }
  if (warp < 4) {
    // Q rows into the K-major swizzled panels; rows past the end and dims past D are zero
    constexpr int CH = DP / 8;
    const T* q = static_cast<const T*>(P.q.p) + b * P.q.sb;
#pragma unroll 8
    for (int c = tid; c < kAfRows * CH; c += 128) {
      const int row = c / CH, ch = c % CH, rr = r0 + row;
      uint4 u = make_uint4(0, 0, 0, 0);
      if (rr < rows && ch * 8 < A.D) {
        const int i = rr / A.G, h = hk * A.G + rr - i * A.G;
        u = *reinterpret_cast<const uint4*>(q + i * P.q.st + h * P.q.sh + ch * 8);
      }
      *reinterpret_cast<uint4*>(smem + (ch / 8) * kAfPanel + at_sw128(row, ch % 8)) = u;
    }
    fence_proxy_async_smem();
    if (docs) {
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
    at_doc_bits(own, A.sum_k + (long long)b * nb, nb, kAfKeys / kAtDocBlock, tiles.begin, tiles.end, warp,
                kAfThreads / 32, live, mix, pad);
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 4) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int t = tiles.first(); t < tiles.end; t = tiles.next(t + 1), it++) {
        const int s = it % Cfg::STAGES;
        const uint32_t ph = ((it / Cfg::STAGES) & 1) ^ 1;
        if (it >= Cfg::STAGES && !(ok = mbar_wait(&k_empty[s], ph, A.err))) break;
        mbar_arrive_expect_tx(&k_full[s], Cfg::TILE);
        for (int p = 0; p < Cfg::PANELS; p++)
          tma_load_4d(smem + (1 + s) * Cfg::TILE + p * kAfPanel, &P.tk, &k_full[s], p * 64, t * kAfKeys, hk, b);
        if (it >= Cfg::STAGES && !(ok = mbar_wait(&v_empty[s], ph, A.err))) {
          mbar_wait(&k_full[s], (it / Cfg::STAGES) & 1, A.err);
          break;
        }
        mbar_arrive_expect_tx(&v_full[s], Cfg::TILE);
        for (int p = 0; p < Cfg::PANELS; p++)
          tma_load_4d(smem + (1 + Cfg::STAGES + s) * Cfg::TILE + p * kAfPanel, &P.tv, &v_full[s], p * 64, t * kAfKeys,
                      hk, b);
      }
      // no copy of this CTA may be in flight when it ends
      for (int i = max(0, it - Cfg::STAGES); i < it; i++) {
        mbar_wait(&k_full[i % Cfg::STAGES], (i / Cfg::STAGES) & 1, A.err);
        mbar_wait(&v_full[i % Cfg::STAGES], (i / Cfg::STAGES) & 1, A.err);
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    if (lane == 0) {
      const int ks = (A.D + 15) / 16;  // K steps of Q·Kᵀ; N of P·V is 16·ks
      const uint32_t id_s = at_idesc(BF16, 128, kAfKeys, false), id_o = at_idesc(BF16, 128, 16 * ks, true);
      auto qk = [&](int it) {
        const uint32_t kb = sk + (it % Cfg::STAGES) * Cfg::TILE;
        for (int k = 0; k < ks; k++) {
          const uint32_t o = (k / 4) * kAfPanel + (k % 4) * 32;
          umma_f16(tmem + Cfg::COL_S, smem_desc_kmajor(sq + o, 128), smem_desc_kmajor(kb + o, 128), id_s, k > 0);
        }
        umma_commit(&k_empty[it % Cfg::STAGES]);
        umma_commit(&s_full);
      };
      int it = 0, t = tiles.first();
      bool ok = true;
      if (t < tiles.end && (ok = mbar_wait(&k_full[0], 0, A.err))) {
        tc_fence_after();
        qk(0);
      }
      while (ok && t < tiles.end) {
        const int tn = tiles.next(t + 1), s = it % Cfg::STAGES, s1 = (it + 1) % Cfg::STAGES;
        const uint32_t ph = (it / Cfg::STAGES) & 1, ph1 = ((it + 1) / Cfg::STAGES) & 1;
        if (Cfg::EARLY && tn < tiles.end) {
          if (!(ok = mbar_wait(&k_full[s1], ph1, A.err) && mbar_wait(&s_free, it & 1, A.err))) break;
          tc_fence_after();
          qk(it + 1);
        }
        if (!(ok = mbar_wait(&v_full[s], ph, A.err) && mbar_wait(&p_full, it & 1, A.err))) break;
        tc_fence_after();
        const uint32_t vb = sv + s * Cfg::TILE;
#pragma unroll
        for (int k = 0; k < kAfKeys / 16; k++)
          umma_f16_ts(tmem + Cfg::COL_O, tmem + Cfg::COL_P + k * 8, at_desc_mn(vb + k * 16 * 128, kAfPanel), id_o,
                      (it | k) != 0);
        umma_commit(&v_empty[s]);
        umma_commit(&pv_done);
        if (!Cfg::EARLY && tn < tiles.end) {
          if (!(ok = mbar_wait(&k_full[s1], ph1, A.err))) break;
          tc_fence_after();
          qk(it + 1);
        }
        t = tn;
        it++;
      }
      if (!ok) {  // let the issued MMAs finish before TMEM is freed
        umma_commit(&drain);
        mbar_wait(&drain, 0, A.err);
      }
    }
    __syncwarp();
  } else {
    const uint32_t lane_base = uint32_t(warp * 32) << 16;
    const bool idle = r0 + warp * 32 >= rows;  // no row of this warp exists: it only keeps step
    const int pos = off + qi;
    const int lim = valid ? at_limit(A, n, prefix, pos) : 0;
    // scores in log2 units are x·cmul: the scale is applied with the exponent's FMA when nothing else needs it
    const float cmul = CAP || BIAS ? 1.f : A.scale * kAtLog2e;
    const float cap2 = A.cap * kAtLog2e, cap_in = CAP ? 2.f * A.scale * kAtLog2e / A.cap : 0.f;
    const float slope = BIAS && valid ? A.slopes[head] * kAtLog2e : 0.f;
    const float2 cell = BIAS == 2 ? at_cell(A, pos) : make_float2(0.f, 0.f);
    float m = -INFINITY, l = 0.f;  // reference maximum (log2 units) and sum
    int it = 0;
    bool ok = true;
    for (int t = tiles.first(); t < tiles.end; t = tiles.next(t + 1), it++) {
      const int j0 = t * kAfKeys;
      const bool by_doc = docs && at_bit(mix, t - tiles.begin);
      const bool dirty = (n < A.Lk && j0 + kAfKeys > n) || (docs && at_bit(pad, t - tiles.begin));
      int key_doc = 0;
      if (by_doc || BIAS == 2) {  // per-key data of the tile, one key a thread
        if (docs) {
          key_doc = j0 + tid < n ? A.doc_k[(long long)b * A.Lk + j0 + tid] : -1;
          col_doc[it & 1][tid] = key_doc < 0 ? -1 : key_doc;
        }
        if (BIAS == 2) col_cell[it & 1][tid] = at_cell(A, j0 + tid);
        named_bar_sync(1, 128);
      }
      if (!(ok = at_wait_warp(&s_full, it & 1, A.err))) break;
      tc_fence_after();
      float x[kAfKeys];
#pragma unroll
      for (int c = 0; c < kAfKeys; c += 32) tmem_ld32_nowait(tmem + lane_base + Cfg::COL_S + c, x + c);
      tmem_wait_ld();
      if (Cfg::EARLY) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free);
      }
      if (!idle) {
        if (CAP) {
#pragma unroll
          for (int c = 0; c < kAfKeys; c++)
            x[c] = fmaf(-2.f * cap2, at_rcp(1.f + at_ex2(x[c] * cap_in)), cap2);
        } else if (BIAS) {
#pragma unroll
          for (int c = 0; c < kAfKeys; c++) x[c] *= A.scale * kAtLog2e;
        }
        if (BIAS == 1) {
          const float rel = float(pos - j0);
#pragma unroll
          for (int c = 0; c < kAfKeys; c++) x[c] = fmaf(-slope, fabsf(rel - float(c)), x[c]);
        }
        if (BIAS == 2) {
          const float4* cells = reinterpret_cast<const float4*>(col_cell[it & 1]);
#pragma unroll
          for (int c = 0; c < kAfKeys; c += 2) {
            const float4 k2 = cells[c / 2];
            x[c] = fmaf(-slope, fabsf(cell.x - k2.x) + fabsf(cell.y - k2.y), x[c]);
            x[c + 1] = fmaf(-slope, fabsf(cell.x - k2.z) + fabsf(cell.y - k2.w), x[c + 1]);
          }
        }
        if (j0 + kAfKeys > lim_min) {
          const int e = lim - j0;
#pragma unroll
          for (int c = 0; c < kAfKeys; c++) x[c] = c < e ? x[c] : -INFINITY;
        }
        if (by_doc) {
          const int4* kd = reinterpret_cast<const int4*>(col_doc[it & 1]);
#pragma unroll
          for (int c = 0; c < kAfKeys; c += 4) {
            const int4 d = kd[c / 4];
            x[c] = d.x == my_doc ? x[c] : -INFINITY;
            x[c + 1] = d.y == my_doc ? x[c + 1] : -INFINITY;
            x[c + 2] = d.z == my_doc ? x[c + 2] : -INFINITY;
            x[c + 3] = d.w == my_doc ? x[c + 3] : -INFINITY;
          }
        }
      }
      float factor = 1.f;
      if (!idle) {
        float top4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int c = 4; c < kAfKeys; c++) top4[c % 4] = fmaxf(top4[c % 4], x[c]);
        const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * cmul;
        if (top > m + kAfGrow || (m == -INFINITY && top > -INFINITY)) {
          factor = m == -INFINITY ? 0.f : at_ex2(m - top);
          m = top;
          l *= factor;
        }
      }
      // O and P are free once the previous P·V is done
      if (it > 0) {
        if (!(ok = at_wait_warp(&pv_done, (it - 1) & 1, A.err))) break;
        tc_fence_after();
        if (__any_sync(0xffffffffu, factor != 1.f)) {
#pragma unroll
          for (int c = 0; c < DP; c += 16) {
            float o[16];
            tmem_ld16(tmem + lane_base + Cfg::COL_O + c, o);
#pragma unroll
            for (int i = 0; i < 16; i++) o[i] = factor == 0.f ? 0.f : o[i] * factor;
            tmem_st16(tmem + lane_base + Cfg::COL_O + c, reinterpret_cast<const uint32_t*>(o));
          }
        }
      }
      if (!idle) {
        const float neg = m == -INFINITY ? 0.f : -m;
        const float2 mul = make_float2(cmul, cmul), add = make_float2(neg, neg);
        float2 sum[2] = {make_float2(l, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < kAfKeys; c += 64) {
          uint32_t p[32];
#pragma unroll
          for (int i = 0; i < 32; i++) {
            float2 e = make_float2(x[c + 2 * i], x[c + 2 * i + 1]);
            e = CAP || BIAS ? add2(e, add) : fma2(e, mul, add);
            e.x = at_ex2(e.x);
            e.y = at_ex2(e.y);
            sum[i & 1] = add2(sum[i & 1], e);
            p[i] = Half16<T>::pack(e.x, e.y);
          }
          tmem_st32(tmem + lane_base + Cfg::COL_P + c / 2, p);
        }
        const float2 s = add2(sum[0], sum[1]);
        l = s.x + s.y;
      }
      if (dirty) {  // V rows of keys that no query sees hold anything, NaN included: 0·NaN must not enter O
        if (!(ok = at_wait_warp(&v_full[it % Cfg::STAGES], (it / Cfg::STAGES) & 1, A.err))) break;
        const int j = j0 + tid;
        if (j >= n || (docs && A.doc_k[(long long)b * A.Lk + j] < 0)) {
          uint8_t* v = smem + (1 + Cfg::STAGES + it % Cfg::STAGES) * Cfg::TILE + tid * 128;
          for (int p = 0; p < Cfg::PANELS; p++)
#pragma unroll
            for (int c = 0; c < 8; c++) *reinterpret_cast<uint4*>(v + p * kAfPanel + c * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full);
    }
    if (ok && it > 0) ok = at_wait_warp(&pv_done, (it - 1) & 1, A.err);
    if (ok) {
      tc_fence_after();
      const long long row = ((long long)b * A.Hq + head) * A.Lq + qi;
      const long long part_row = (long long)split * A.B * A.Hq * A.Lq + row;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // a NaN sum stays one
      T* o_ptr = static_cast<T*>(P.o.p) + b * P.o.sb + qi * P.o.st + head * P.o.sh;
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        if (c >= A.D) break;
        float o[32];
        if (it > 0) {
          tmem_ld32_nowait(tmem + lane_base + Cfg::COL_O + c, o);
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 32; i++) o[i] = it > 0 && l != 0.f ? o[i] : 0.f;
        if (!valid) continue;
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          if (c + i >= A.D) break;
          float v8[8];
#pragma unroll
          for (int k = 0; k < 8; k++) v8[k] = o[i + k];
          if (P.splits == 1) {
#pragma unroll
            for (int k = 0; k < 8; k++) v8[k] *= inv;
            *reinterpret_cast<uint4*>(o_ptr + c + i) = pack8<T>(v8);
          } else {
            float4* d = reinterpret_cast<float4*>(P.part + part_row * A.D + c + i);
            d[0] = make_float4(v8[0], v8[1], v8[2], v8[3]);
            d[1] = make_float4(v8[4], v8[5], v8[6], v8[7]);
          }
        }
      }
      if (valid) {
        if (P.splits > 1)
          P.stats[part_row] = make_float2(m, l);
        else if (P.lse)
          P.lse[row] = l == 0.f ? -INFINITY : (m + at_lg2(l)) * kAtLn2;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

template <typename T, int DP, bool CAP, int BIAS>
cudaError_t attn_fwd_one(const AttnFwdLaunch& L, int grid, cudaStream_t st) {
  static bool set[64] = {};  // per device; a race only repeats the call
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  auto* k = k_attn_fwd<T, DP, CAP, BIAS>;
  if (dev >= 64 || !set[dev]) {
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, AfCfg<DP>::SMEM);
    if (e != cudaSuccess) return e;
    if (dev < 64) set[dev] = true;
  }
  k<<<grid, kAfThreads, AfCfg<DP>::SMEM, st>>>(L);
  return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t attn_fwd_dp(const AttnFwdLaunch& L, int grid, cudaStream_t st) {
  const int bias = !L.d.slopes ? 0 : L.d.grid_w > 0 ? 2 : 1;
  if (L.d.cap > 0.f)
    return bias == 0   ? attn_fwd_one<T, DP, true, 0>(L, grid, st)
           : bias == 1 ? attn_fwd_one<T, DP, true, 1>(L, grid, st)
                       : attn_fwd_one<T, DP, true, 2>(L, grid, st);
  return bias == 0   ? attn_fwd_one<T, DP, false, 0>(L, grid, st)
         : bias == 1 ? attn_fwd_one<T, DP, false, 1>(L, grid, st)
                     : attn_fwd_one<T, DP, false, 2>(L, grid, st);
}

template <typename T>
cudaError_t launch_attn_fwd(const AttnFwdLaunch& L, cudaStream_t st) {
  const int nq = (L.d.Lq * L.d.G + kAfRows - 1) / kAfRows;
  const int grid = nq * L.d.B * L.d.Hk * L.splits;
  return L.d.D <= 64 ? attn_fwd_dp<T, 64>(L, grid, st) : attn_fwd_dp<T, 128>(L, grid, st);
}

}  // namespace osam
