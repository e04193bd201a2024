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
#include "sm100.cuh"

namespace osam {

constexpr float kAtLog2e = 1.4426950408889634f, kAtLn2 = 0.6931471805599453f;
constexpr int kAtDocBlock = 64;      // tokens per document summary
constexpr int kAtDocWords = 512;     // 32-bit words of a CTA's key-tile bitmaps: 16384 tiles of 64 keys
constexpr int kAtSms = 148;

// A [batch][token][head][dim] tensor: element strides, dim contiguous.
struct AtView {
  void* p;
  long long sb, st, sh;
};

// Documents of 64 tokens: the smallest and largest id ≥ 0 (lo > hi: none) and whether a token has none (id < 0).
struct AtDocs {
  int lo, hi, pad, unused;
};

struct AttnDev {
  int B, Lq, Lk, Hq, Hk, G, D;
  int mask;  // OSAM_ATTN_*
  float scale, cap;
  int grid_w;
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

// Two fp32 operations per instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)),
        "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}

// D[tmem] (+)= A[tmem] · B[smem]: A's 128 rows are TMEM lanes, two 16-bit values of K per 32-bit column.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
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

// 32 lanes × 32 consecutive 32-bit columns, without the completion wait (tmem_wait_ld).
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
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
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A wait that a whole warp takes together: every lane learns whether any lane's budget ran out.
__device__ __forceinline__ bool at_wait_warp(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err));
}

// Which tiles of the streamed side a CTA visits.  Without documents every tile of [begin, end); with them, the
// tiles whose bit is set (built by at_doc_bits).
struct AtTiles {
  int begin, end;
  const uint32_t* live;  // nullptr: all
  __device__ __forceinline__ int next(int t) const {  // first visited tile ≥ t (end: none)
    if (!live || t >= end) return t;
    uint32_t w = live[(t - begin) >> 5] >> ((t - begin) & 31);
    while (!w) {
      t = begin + (((t - begin) >> 5) + 1) * 32;
      if (t >= end) return end;
      w = live[(t - begin) >> 5];
    }
    return min(end, t + __ffs(w) - 1);
  }
  __device__ __forceinline__ int first() const { return next(begin); }
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
  int splits, tiles_per_split;
  float* part;    // [split][B][Hq][Lq][D] unnormalised outputs
  float2* stats;  // [split][B][Hq][Lq] (reference maximum in log2 units, sum)
};
template <typename T>
cudaError_t launch_attn_fwd(const AttnFwdLaunch& L, cudaStream_t st);

}  // namespace osam
