// Shared parts of the attention kernels (attn_fwd.cuh, attn_bwd.cuh, attn.cu): the device description of a call,
// the visibility rules, and the tcgen05 forms these kernels add to sm100.cuh.
//
//   s_ij = cap·tanh(scale·q_i·k_j/cap)  (cap > 0)   or   scale·q_i·k_j
//   x_ij = s_ij − slope_h·dist(i, j)
//   o_i  = Σ_j p_ij v_j,  p_ij = exp(x_ij − lse_i) over the keys j that i sees
// Query i stands at position i + n_b − len_q (n_b: keys in use of sequence b), key j at position j.  dist is
// |pos_i − j|, or on a map `grid_w` wide |y_i − y_j| + |x_i − x_j|.  i sees j when j < lim_i and, with documents,
// doc_q[i] = doc_k[j] ≥ 0;  lim_i = n_b (no mask), min(n_b, pos_i + 1) (causal) or min(n_b, max(pos_i + 1,
// prefix_b)): every mask but the documents is one bound per query, which grows with i.
#pragma once
#include <limits.h>

#include "conv_internal.h"
#include "half16.cuh"
#include "launch.cuh"
#include "pair_math.cuh"
#include "sm100.cuh"

namespace osam {

constexpr float kAtLog2e = 1.4426950408889634f, kAtLn2 = 0.6931471805599453f;
constexpr int kAtDocBlock = 64;      // tokens per document summary
constexpr int kAtDocWords = 512;     // 32-bit words of a CTA's key-tile bitmaps: 16384 tiles of 64 keys
constexpr int kAtSms = 148;
constexpr int kAfRows = 128, kAfKeys = 64;  // a forward CTA's query rows, and the keys of a tile
constexpr int kAfPlaces = 2 * kAtSms, kAfRounds = 2;  // forward CTAs at a time, and rounds of them that splits may fill

// A [batch][token][head][dim] tensor: element strides, dim contiguous.
struct AtView {
  void* p;
  long long sb, st, sh;
};

// Documents of 64 tokens: the smallest and largest id ≥ 0 (lo > hi: none) and whether a token has none (id < 0) or, for the
// backward's queries, sees nothing.
struct AtDocs {
  int lo, hi, pad, unused;
};

struct AttnDev {
  int B, Lq, Lk, Hq, Hk, G, D;
  int mask;  // OSAM_ATTN_*
  float scale, cap;
  int grid_w;
  FastDiv f_g;  // ÷ G
  FastDiv f_w;  // ÷ grid_w (positions are not negative there or clamped, see at_cell)
  const int* lens;
  const int* prefix;
  const int* doc_q;
  const int* doc_k;
  const AtDocs* sum_q;  // [B][⌈Lq/64⌉]
  const AtDocs* sum_k;  // [B][⌈Lk/64⌉]
  const float* slopes;
  int* err;
};

// Keys in use of sequence b.
__device__ __forceinline__ int at_keys(const AttnDev& A, int b) {
  return A.lens ? max(0, min(A.lens[b], A.Lk)) : A.Lk;
}
// Key tiles of a sequence, and its splits of up to `chunk` tiles (one at least: it writes the output's zeros).
__device__ __forceinline__ int at_seq_tiles(const AttnDev& A, int b) { return (at_keys(A, b) + kAfKeys - 1) / kAfKeys; }
__device__ __forceinline__ int at_seq_splits(const AttnDev& A, int b, int chunk) {
  return max(1, (at_seq_tiles(A, b) + chunk - 1) / chunk);
}
// Tiles of a split at most, `count(chunk)` being the splits of all B sequences: the smallest chunk with which they fit
// one or two rounds of the GPU's places, `per` CTAs each, whichever takes less (a CTA's start and end cost about five
// tiles).  So sequences of any lengths take their share of the CTAs (back to back, 16 caches of 8192–32768 keys:
// 233 us, with one number of splits for all 255; 16 caches of 8192 keys: 88 and 108).
template <typename Count>
__host__ __device__ __forceinline__ int at_best_chunk(int B, int per, int min_tiles, int max_tiles, int total, Count count) {
  int best = 0, least = INT_MAX;
  for (int k = 1; k <= kAfRounds; k++) {
    const int room = k * kAfPlaces / per;  // at least B
    int lo = (total + room - 1) / room;    // nothing smaller can fit; rounding up adds less than a split a sequence
    lo = lo > min_tiles ? lo : min_tiles;
    int hi = room > B ? (total + room - B - 1) / (room - B) : max_tiles;
    if (hi < lo || count(lo) <= room) hi = lo;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (count(mid) <= room)
        hi = mid;
      else
        lo = mid + 1;
    }
    if (k * (lo + 5) < least) {
      least = k * (lo + 5);
      best = lo;
    }
  }
  return best;
}
// Order of the CTAs: `tile` of `unit` (a head, a part of one) for CTA i.  Units go in groups; in a group all units' first
// tiles come first.  With a causal bound the tiles are ordered longest first, so groups keep a tail of short ones, but all
// that a group streams stays in L2 over its tiles (at_group has what that measured).
__device__ __forceinline__ void at_order(int i, int tiles, int units, int group, int& tile, int& unit) {
  const int first = i / (group * tiles) * group, here = min(group, units - first);
  i -= first * tiles;
  tile = i / here;
  unit = first + i - tile * here;
}
// lim_i of the query at position pos.
__device__ __forceinline__ int at_limit(const AttnDev& A, int n, int prefix, int pos) {
  if (A.mask == OSAM_ATTN_NONE) return n;
  return max(0, min(n, max(pos + 1, prefix)));
}
// (y, x) of a position on the map; rows continue above the map for negative positions.
__device__ __forceinline__ float2 at_cell(const AttnDev& A, int pos) {
  const int y = pos >= 0 ? A.f_w.quo(pos) : -A.f_w.quo(A.grid_w - 1 - pos);
  return make_float2(float(y), float(pos - y * A.grid_w));
}

__device__ __forceinline__ float at_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float at_lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float at_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// min that keeps a NaN.
__device__ __forceinline__ float at_min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// The first n of 32 bits (n may lie outside 0 … 32).
__device__ __forceinline__ uint32_t at_low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
// x where bit i of `vis` is set, `other` elsewhere, over N columns.
template <int N>
__device__ __forceinline__ void at_mask(float (&x)[N], uint32_t vis, float other) {
#pragma unroll
  for (int c = 0; c < N; c++) x[c] = (vis >> c) & 1 ? x[c] : other;
}
// Which of N columns have document `doc`.
template <int N>
__device__ __forceinline__ uint32_t at_same_doc(const int* cols, int doc) {
  uint32_t v = 0;
#pragma unroll
  for (int c = 0; c < N; c += 4) {
    const int4 d = *reinterpret_cast<const int4*>(cols + c);
    v |= (uint32_t(d.x == doc) << c) | (uint32_t(d.y == doc) << (c + 1)) | (uint32_t(d.z == doc) << (c + 2)) |
         (uint32_t(d.w == doc) << (c + 3));
  }
  return v;
}

// 1 / (1 + 2^u) of four values with one reciprocal: 1/a = (1/abcd)·bcd.  u is held to 30, where 1 − tanh is below
// fp32's resolution, so the product of four stays finite.  A NaN spreads to all four: hidden scores are replaced before.
__device__ __forceinline__ void at_sigmoid4(float2 (&u)[2]) {
  float2 a[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    a[i].x = at_ex2(at_min_nan(u[i].x, 30.f));
    a[i].y = at_ex2(at_min_nan(u[i].y, 30.f));
    a[i] = add2(a[i], make_float2(1.f, 1.f));
  }
  const float2 pr = mul2(make_float2(a[0].x, a[1].x), make_float2(a[0].y, a[1].y));
  const float r = at_rcp(pr.x * pr.y);
  const float2 half = mul2(make_float2(r, r), make_float2(pr.y, pr.x));  // 1 / (product of each pair)
  u[0] = mul2(make_float2(half.x, half.x), make_float2(a[0].y, a[0].x));
  u[1] = mul2(make_float2(half.y, half.y), make_float2(a[1].y, a[1].x));
}

// Scores in log2 units: s ← cap·tanh(scale·s/cap)·log2 e (CAP) or s·scale·log2 e, minus slope·dist.  tanh y is taken as
// 1 − 2/(1 + e^2y), which is off by 2^-23 whatever y is: cap·tanh by 2e-7·cap, 2.6e-5 at kAtCapLarge, a tenth of fp16's
// rounding of P.  Above it (CAP = 2) small y, |y| < ½, go by tanh's series to y^13, off by 9e-8 of the score (the other form by
// 4e-7 beyond), at a price: 2 × 4096 causal tokens, 16/4 heads × 128, forward 255 → 347 us, backward 659 → 871.
constexpr float kAtCapLarge = 128.f;
struct AtBias {
  float mul;        // scale·log2 e, or with a cap 2·scale·log2 e / cap
  float cap2;       // cap·log2 e
  float lin, arg;   // CAP = 2: scale·log2 e and scale / cap
  float slope;      // of the row's head, ·log2 e
  float away;       // −1, or 1 where the slope is negative
  float y, x;       // the row's position on the map times the slope; line: y only, relative to the chunk's first column
};
// tanh(y)/y from z = y² < ¼: its Taylor series.
__device__ __forceinline__ float2 at_tanh_ratio(float2 z) {
  constexpr float c[7] = {1.f, -1.f / 3, 2.f / 15, -17.f / 315, 62.f / 2835, -1382.f / 155925, 21844.f / 6081075};
  float2 r = make_float2(c[6], c[6]);
#pragma unroll
  for (int i = 5; i >= 0; i--) r = fma2(r, z, make_float2(c[i], c[i]));
  return r;
}
// Distances along the line of four consecutive columns, carried from one group of four to the next.
struct AtLine {
  float2 d[2], step;
  __device__ __forceinline__ void start(const AtBias& P) {
    d[0] = make_float2(P.y, P.y - P.slope);
    d[1] = make_float2(P.y - 2.f * P.slope, P.y - 3.f * P.slope);
    step = make_float2(-4.f * P.slope, -4.f * P.slope);
  }
  __device__ __forceinline__ void next() {
    d[0] = add2(d[0], step);
    d[1] = add2(d[1], step);
  }
};
// Distances (times the slope's size) of four consecutive columns: `line` holds them signed, ky / kx the columns' cells (grid).
template <int BIAS>
__device__ __forceinline__ void at_far4(const AtBias& P, AtLine& line, const float4& ky, const float4& kx, float2 (&t)[2]) {
  if (BIAS == 1) {
    t[0] = make_float2(fabsf(line.d[0].x), fabsf(line.d[0].y));
    t[1] = make_float2(fabsf(line.d[1].x), fabsf(line.d[1].y));
    line.next();
  }
  if (BIAS == 2) {
    const float2 ns = make_float2(-P.slope, -P.slope), y = make_float2(P.y, P.y), x = make_float2(P.x, P.x);
    const float2 y0 = fma2(ns, make_float2(ky.x, ky.y), y), y1 = fma2(ns, make_float2(ky.z, ky.w), y);
    const float2 x0 = fma2(ns, make_float2(kx.x, kx.y), x), x1 = fma2(ns, make_float2(kx.z, kx.w), x);
    t[0] = make_float2(fabsf(y0.x) + fabsf(x0.x), fabsf(y0.y) + fabsf(x0.y));
    t[1] = make_float2(fabsf(y1.x) + fabsf(x1.x), fabsf(y1.y) + fabsf(x1.y));
  }
}
// Four consecutive columns; out: the scores plus `add` (ADD); with CAP, sig = 1/(1 + 2^u), from which 1 − tanh² =
// 4·sig·(1 − sig).  NEG: slopes may be negative; without, the sign rides on the operand.
template <int CAP, int BIAS, bool ADD, bool NEG>
__device__ __forceinline__ void at_scores4(const AtBias& P, float2 (&s)[2], const float2 (&add)[2], AtLine& line,
                                           const float4& ky, const float4& kx, float2 (&sig)[2]) {
  const float2 mul = make_float2(P.mul, P.mul);
  float2 b[2] = {add[0], add[1]};
  if (BIAS) {
    float2 t[2];
    at_far4<BIAS>(P, line, ky, kx, t);
    const float2 away = make_float2(P.away, P.away);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const float2 a = NEG ? mul2(t[i], away) : make_float2(-t[i].x, -t[i].y);
      b[i] = !ADD ? a : NEG ? fma2(t[i], away, b[i]) : add2(b[i], a);
    }
  }
  if (CAP) {
    sig[0] = mul2(s[0], mul);
    sig[1] = mul2(s[1], mul);
    at_sigmoid4(sig);
    const float2 m2 = make_float2(-2.f * P.cap2, -2.f * P.cap2), c2 = make_float2(P.cap2, P.cap2);
    if (CAP == 2) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float2 y = mul2(s[i], make_float2(P.arg, P.arg)), lin = mul2(s[i], make_float2(P.lin, P.lin)),
                     far = fma2(m2, sig[i], c2), r = mul2(lin, at_tanh_ratio(mul2(y, y)));
        s[i] = make_float2(fabsf(y.x) < 0.5f ? r.x : far.x, fabsf(y.y) < 0.5f ? r.y : far.y);
        if (ADD || BIAS) s[i] = add2(s[i], b[i]);
      }
      return;
    }
    s[0] = fma2(m2, sig[0], ADD || BIAS ? add2(c2, b[0]) : c2);
    s[1] = fma2(m2, sig[1], ADD || BIAS ? add2(c2, b[1]) : c2);
  } else if (ADD || BIAS) {
    s[0] = fma2(s[0], mul, b[0]);
    s[1] = fma2(s[1], mul, b[1]);
  } else {
    s[0] = mul2(s[0], mul);
    s[1] = mul2(s[1], mul);
  }
}

// Barrier of `threads` threads with the OR of a flag.  A named barrier has no bound of its own: a warp whose bounded wait
// ran out stays in step with the others through all of them, without arriving anywhere else and without writing results.
__device__ __forceinline__ bool at_any(int id, bool flag, int threads) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(uint32_t(flag)), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}
// Of the two warps that share rows.
__device__ __forceinline__ bool at_pair_any(int id, bool flag) { return at_any(id, flag, 64); }

// The MMA warp runs its loop with all lanes and issues from one, `leader`, by predicate: with warp-uniform control flow
// the descriptors stay in uniform registers, where the instruction reads them (issued from inside a one-lane branch,
// every MMA first moved its operands over, about 100 cycles each: more than these small MMAs take).
__device__ __forceinline__ uint32_t elect_leader() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}\n" : "=r"(e));
  return e;
}
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
// A's 128 rows are TMEM lanes, two 16-bit values of K per 32-bit column.
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}
// kind::f16 instruction descriptor, fp32 D, K-major A; bf16 or fp16 operands; b_mn: MN-major B.
__host__ __device__ constexpr uint32_t at_idesc(bool bf16, int M, int N, bool b_mn) {
  return (1u << 4) | (uint32_t(bf16) << 7) | (uint32_t(bf16) << 10) | (uint32_t(b_mn) << 16) |
         (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}
// MN-major operand in 128-byte swizzled rows of 64 elements: `panel` = bytes between 64-element column panels.
__device__ __forceinline__ uint64_t at_desc_mn(uint32_t saddr, uint32_t panel) {
  uint64_t d = (saddr & 0x3FFFFu) >> 4;
  d |= uint64_t((panel >> 4) & 0x3FFFu) << 16;
  d |= uint64_t(1024 >> 4) << 32;  // next 8 rows
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}
__device__ __forceinline__ uint32_t at_sw128(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// TMEM → registers: 32 lanes × consecutive 32-bit columns, a lane a thread.  Load and completion wait are one
// statement: between two, the compiler may place a use of the registers, which nothing ties to the wait.
__device__ __forceinline__ void at_ld16(uint32_t taddr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), 
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void at_ld8(uint32_t taddr, float (&v)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void at_ld32(uint32_t taddr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
      "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), 
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), 
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), 
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void at_ld32x2(uint32_t ta, float (&v)[32], uint32_t tb, float (&w)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
      "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, "
      "%52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), 
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), 
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), 
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]), 
        "=f"(w[0]), "=f"(w[1]), "=f"(w[2]), "=f"(w[3]), "=f"(w[4]), "=f"(w[5]), "=f"(w[6]), "=f"(w[7]), 
        "=f"(w[8]), "=f"(w[9]), "=f"(w[10]), "=f"(w[11]), "=f"(w[12]), "=f"(w[13]), "=f"(w[14]), "=f"(w[15]), 
        "=f"(w[16]), "=f"(w[17]), "=f"(w[18]), "=f"(w[19]), "=f"(w[20]), "=f"(w[21]), "=f"(w[22]), "=f"(w[23]), 
        "=f"(w[24]), "=f"(w[25]), "=f"(w[26]), "=f"(w[27]), "=f"(w[28]), "=f"(w[29]), "=f"(w[30]), "=f"(w[31])
      : "r"(ta), "r"(tb)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bounded wait (as mbar_wait) without the suspend-time hint, with which the test sleeps in steps of a microsecond and
// more (about a tile's time); the clock is read every 1024 tests, which keeps the loop to a few instructions.
__device__ __forceinline__ bool at_wait(uint32_t bar, uint32_t parity, int* err) {
  unsigned long long t0 = 0;
  for (uint32_t n = 1;; n++) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if (n % 1024 == 0) {
      const unsigned long long t = globaltimer();
      if (t0 == 0) t0 = t;
      if (t - t0 > kWaitBudgetNs) break;
    }
  }
  record_error(err, kDevErrTimeout);
  return false;
}
__device__ __forceinline__ bool at_wait(uint64_t* bar, uint32_t parity, int* err) {
  return at_wait(smem_u32(bar), parity, err);
}
// A wait that a whole warp takes together: every lane learns whether any lane's budget ran out.
__device__ __forceinline__ bool at_wait_warp(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, at_wait(bar, parity, err));
}
__device__ __forceinline__ void at_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Which tiles of the streamed side a CTA visits: of [begin, end) all, or with documents those whose bit is set (built
// by at_doc_bits).  The order is from `from` down to `begin`, then from + 1 up to end − 1: with `from` the tile of
// the CTA's own positions, the keys nearest in distance come first, and with them a row's largest scores.
struct AtTiles {
  int begin, end, from;
  const uint32_t* live;  // nullptr: all
  __device__ __forceinline__ int up(int t) const {  // first live tile ≥ t (end: none)
    if (!live || t >= end) return t;
    uint32_t w = live[(t - begin) >> 5] >> ((t - begin) & 31);
    while (!w) {
      t = begin + (((t - begin) >> 5) + 1) * 32;
      if (t >= end) return end;
      w = live[(t - begin) >> 5];
    }
    return min(end, t + __ffs(w) - 1);
  }
  __device__ __forceinline__ int down(int t) const {  // last live tile ≤ t (begin − 1: none)
    if (!live || t < begin) return t;
    uint32_t w = live[(t - begin) >> 5] << (31 - ((t - begin) & 31));
    while (!w) {
      t = begin + ((t - begin) >> 5) * 32 - 1;
      if (t < begin) return begin - 1;
      w = live[(t - begin) >> 5];
    }
    return t - __clz(w);
  }
  __device__ __forceinline__ int count() const {
    if (!live) return max(0, end - begin);
    int n = 0;
    for (int w = 0; w * 32 < end - begin; w++) n += __popc(live[w]);
    return n;
  }
  // `end` says that there is none (any more)
  __device__ __forceinline__ int first() const {
    const int t = down(from);
    return t >= begin ? t : up(from + 1);
  }
  __device__ __forceinline__ int next(int t) const {
    if (!live) return t > from ? t + 1 : t == begin ? from + 1 : t - 1;
    if (t > from) return up(t + 1);
    t = down(t - 1);
    return t >= begin ? t : up(from + 1);
  }
};
__device__ __forceinline__ bool at_bit(const uint32_t* w, int i) { return (w[i >> 5] >> (i & 31)) & 1; }

// Summary of `n64` consecutive 64-token blocks.
__device__ __forceinline__ AtDocs at_docs(const AtDocs* s, int first, int n64, int total) {
  AtDocs d{INT_MAX, -1, 0, 0};
  for (int i = first; i < min(first + n64, total); i++) {
    const AtDocs e = s[i];
    d.lo = min(d.lo, e.lo);
    d.hi = max(d.hi, e.hi);
    d.pad |= e.pad;
  }
  return d;
}
// Bitmaps over the tiles [begin, end) of the streamed side against the stationary tile's summary `own`: `live` =
// some id in common is possible, `mix` = ids must be compared, `pad` = a token without a document is inside.
// Called by whole warps: warp w of nw fills words w, w + nw, …
__device__ __forceinline__ void at_doc_bits(const AtDocs& own, const AtDocs* s, int total64, int tile64, int begin,
                                            int end, int w, int nw, uint32_t* live, uint32_t* mix, uint32_t* pad) {
  const int lane = threadIdx.x % 32;
  for (int word = w; word * 32 < end - begin; word += nw) {
    const int t = begin + word * 32 + lane;
    AtDocs d{INT_MAX, -1, 0, 0};
    if (t < end) d = at_docs(s, t * tile64, tile64, total64);
    const bool on = t < end && d.lo <= own.hi && own.lo <= d.hi;
    const bool same = d.lo == d.hi && own.lo == own.hi && !d.pad && !own.pad;
    const uint32_t a = __ballot_sync(0xffffffffu, on), m = __ballot_sync(0xffffffffu, !same),
                   p = __ballot_sync(0xffffffffu, d.pad != 0);
    if (lane == 0) {
      live[word] = a;
      mix[word] = m;
      pad[word] = p;
    }
  }
}

// ---- host side (attn.cu): one call's launches
struct AttnFwdLaunch {
  AttnDev d;
  CUtensorMap tk, tv;
  AtView q, o;
  float* lse;
  int grid;
  int group;      // at_order
  int splits;     // of a sequence's keys at most; 1: not split
  int min_tiles;  // of a split at least
  int chunk_all;  // tiles of a split where all sequences have len_k keys, and for the join what the kernel took
  int* chunk;
  float* part;    // [split][B][Hq][Lq][D] unnormalised outputs
  float2* stats;  // [split][B][Hq][Lq] (reference maximum in log2 units, sum)
};
template <typename T>
cudaError_t launch_attn_fwd(const AttnFwdLaunch& L, cudaStream_t st);

constexpr int kAbRows = 128, kAbCols = 64;
constexpr float kAbUp = 8.f;  // fp16: P is held times 2^8

struct AttnBwdLaunch {
  AttnDev d;
  CUtensorMap stat1, stat2, strm1, strm2;
  AtView out1, out2;      // dK, dV (DKV); dQ (DQ)
  const float* rows;      // [B][Hq][⌈Lq/64⌉][2][64]: log2 of P's factor − lse·log2 e (−∞ where the query is empty), −δ
  const float* peak;      // fp16: [B][Hq][⌈Lq/64⌉] max ‖dO_i‖ of the block
  const float* vpeak;     // fp16: [B][Hk][⌈Lk/64⌉] max ‖v_j‖ of the block
  int alone;              // has its SMs to itself, one CTA each
  int late;               // DQ behind DKV, which it does not depend on: waits for that kernel's end only at its own end
  int group;              // at_order
  int parts;              // CTAs that share a tile's streamed side (few tiles: to fill the GPU); above 1 they write
  float* part;            // [parts][outputs][B][heads][L][D] fp32, which k_attn_sum adds in order
};
template <typename T, bool DKV>
cudaError_t launch_attn_bwd(const AttnBwdLaunch& L, cudaStream_t st);

}  // namespace osam
