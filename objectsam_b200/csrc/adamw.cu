// AdamW over many tensors in one launch, with the moments in 32 bits or in 8 bits with a scale per 256 elements,
// and an optional clip by the global norm of the gradients.
//
//   g' = g·mul;  m = β1·m + (1−β1)·g';  v = β2·v + (1−β2)·g'²
//   p = p·(1 − lr·wd) − lr/(1−β1ᵗ)·m / (√v/√(1−β2ᵗ) + eps)          (wd = 0 for tensors marked so)
// 8-bit states, per block of 256 elements: m = e4m3·s_m with s_m = max|m|/448, and the ROOT of v likewise
// (√v = e4m3·s_v; the scales by a product with 1/448, values by 448·(1/max), each within a rounding of the quotient): the root halves the exponent range, so e4m3's 2^18 covers 2^36 in v.  A v above zero is never
// stored as zero (it takes the smallest e4m3 value): a moment that survives beside a vanished v would make its
// step m/eps.  The step uses the new moments before they are rounded.
//
// Bound by HBM: 28 bytes an element with 32-bit states (16 + 1/16 with 8 bits and 32-bit gradients) and 2 more for a
// 16-bit weight copy; with 8-bit states the arithmetic (one IEEE square root an element, e4m3 both ways) is close
// behind, so it runs on pairs (two fp32 operations an instruction, rounded as the single ones are).  A table in
// device memory, written once, has a record for every chunk of 2048 elements with all that the chunk needs, so
// small and large tensors share one launch with no search and one dependent load before the data.  One CTA per chunk:
// many small CTAs hide each other's latencies better than persistent ones that load ahead (measured: 56 against 69
// us on 11.8M parameters with 32-bit states).  A warp owns 256 consecutive
// elements — one quantisation block, whose maximum is five shuffles.  Lanes hold 8 consecutive elements (16-byte
// accesses) where the chunk's pointers allow it, else every 32nd element, so that unaligned tensors (slices of a
// packed gradient arena) stay coalesced too.
// The norm pass reads the gradients once more: fixed chunks per CTA, the last CTA to arrive adds the partial sums
// in a fixed order in fp64 and writes the norm and the multiplier; a norm that is not finite makes the step leave
// parameters and states alone.
// Measured: 11.8M parameters with 32-bit states, fp16 copies and the clip in 69 us (under the profiler, cold: norm pass
// 14, step 57); 278M with 8-bit states, bf16 gradients and copies and the clip in 894 us (5 TB/s).
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "conv_internal.h"
#include "half16.cuh"
#include "launch.cuh"
#include "pair_math.cuh"
#include "sm100.cuh"

namespace osam {
namespace {

constexpr int kAdThreads = 256;
constexpr int kAdChunk = kAdThreads * 8;  // elements per CTA
constexpr int kAdBlock = 256;             // elements per quantisation scale (one warp)
constexpr long long kAdMaxElems = 0x7fffffffLL * kAdChunk;  // of a grid's CTAs; below, the layouts' sums stay in range
constexpr int kAdNormCtas = 148 * 8;
constexpr float kE4m3Max = 448.f;
constexpr float kTiny = 1e-30f;           // a block whose maximum is below this is stored as zeros

enum : int { kAdVec = 1, kAdDecay = 2 };  // 16-byte accesses; weight decay
struct __align__(16) AdChunk {  // of one tensor, pointers at its first element
  float* p;
  const void* g;
  void* copy;
  long long state;    // offset of its states (elements)
  int n, flags;
  int gtype, ctype;   // OSAM_F32 / F16 / BF16; ctype −1: no copy
};

struct AdState {
  void* m;
  void* v;
  float* ms;
  float* vs;
};
struct AdHyper {
  float b1, b2, c1, c2, step, inv_root, eps, keep;  // c = 1 − β; step = lr/(1−β1ᵗ); inv_root = 1/√(1−β2ᵗ); keep = 1 − lr·wd
};
struct AdNorm {  // in the table's buffer
  float mul, pad;
  unsigned arrivals, pad2;
  float part[kAdNormCtas];
};

// 16 bytes of global memory (pointers out of the table carry no address space).
__device__ __forceinline__ uint4 ldg16(const void* p) {
  uint4 r;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ void stg16(void* p, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.global.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void stg16(void* p, float2 a, float2 b) {
  stg16(p, __float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
}
__device__ __forceinline__ AdChunk ad_chunk(const AdChunk* c) {
  AdChunk r;
  const uint4* s = reinterpret_cast<const uint4*>(c);
  uint4* d = reinterpret_cast<uint4*>(&r);
#pragma unroll
  for (int i = 0; i < 3; i++) d[i] = __ldg(s + i);  // the table does not change
  return r;
}
__device__ __forceinline__ float load_g(const void* g, int type, int i) {
  if (type == OSAM_F32) return static_cast<const float*>(g)[i];
  if (type == OSAM_F16) return __half2float(static_cast<const __half*>(g)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(g)[i]);
}
// Eight consecutive gradients as they lie (16 or 32 bytes), and as floats.
struct AdGrad8 {
  uint4 a, b;
};
__device__ __forceinline__ AdGrad8 load_g8(const void* g, int type, int i) {
  AdGrad8 r;
  if (type == OSAM_F32) {
    r.a = ldg16(static_cast<const float*>(g) + i);
    r.b = ldg16(static_cast<const float*>(g) + i + 4);
  } else {
    r.a = ldg16(static_cast<const uint16_t*>(g) + i);
    r.b = make_uint4(0, 0, 0, 0);
  }
  return r;
}
__device__ __forceinline__ void unpack_g8(const AdGrad8& r, int type, float2 (&o)[4]) {
  if (type == OSAM_F32) {
    o[0] = make_float2(__uint_as_float(r.a.x), __uint_as_float(r.a.y));
    o[1] = make_float2(__uint_as_float(r.a.z), __uint_as_float(r.a.w));
    o[2] = make_float2(__uint_as_float(r.b.x), __uint_as_float(r.b.y));
    o[3] = make_float2(__uint_as_float(r.b.z), __uint_as_float(r.b.w));
  } else if (type == OSAM_F16) {
    o[0] = Half16<__half>::unpack(r.a.x);
    o[1] = Half16<__half>::unpack(r.a.y);
    o[2] = Half16<__half>::unpack(r.a.z);
    o[3] = Half16<__half>::unpack(r.a.w);
  } else {
    o[0] = Half16<__nv_bfloat16>::unpack(r.a.x);
    o[1] = Half16<__nv_bfloat16>::unpack(r.a.y);
    o[2] = Half16<__nv_bfloat16>::unpack(r.a.z);
    o[3] = Half16<__nv_bfloat16>::unpack(r.a.w);
  }
}

__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t q) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)q, __NV_E4M3)));
}
__device__ __forceinline__ uint32_t float2_to_e4m3x2(float2 f) {
  return __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
}

// Σ g² of the gradients: CTA b walks chunks b, b + gridDim, …, many warps in flight
// rather than many loads of one (30 against 35 us on 128 MB); the last CTA adds the CTAs' sums in order.
__global__ void __launch_bounds__(kAdThreads, 8) k_adamw_norm(const AdChunk* chunks, int nchunks, AdNorm* st, float scale,
                                                           float max_norm, float* norm) {
  __shared__ double red[kAdThreads / 32];
  __shared__ bool last;
  grid_dep_wait();
  grid_dep_launch();
  float s = 0.f;
  AdChunk next;
  if ((int)blockIdx.x < nchunks) next = ad_chunk(chunks + blockIdx.x);
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
    const AdChunk T = next;
    const int i = threadIdx.x * 8;
    if ((T.flags & kAdVec) && i + 8 <= T.n) {
      const AdGrad8 g = load_g8(T.g, T.gtype, i);
      if (c + (int)gridDim.x < nchunks) next = ad_chunk(chunks + c + gridDim.x);
      float2 f[4];
      unpack_g8(g, T.gtype, f);
#pragma unroll
      for (int e = 0; e < 4; e++) s = fmaf(f[e].y, f[e].y, fmaf(f[e].x, f[e].x, s));
      continue;
    }
    if (c + (int)gridDim.x < nchunks) next = ad_chunk(chunks + c + gridDim.x);
    const int j0 = T.flags & kAdVec ? i : (int)threadIdx.x, step = T.flags & kAdVec ? 1 : kAdThreads;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int j = j0 + e * step;
      const float v = j < T.n ? load_g(T.g, T.gtype, j) : 0.f;
      s = fmaf(v, v, s);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double d = red[0];
#pragma unroll
    for (int i = 1; i < kAdThreads / 32; i++) d += red[i];
    st->part[blockIdx.x] = float(d);
    __threadfence();
    last = atomicAdd(&st->arrivals, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double d = 0;
  for (int i = threadIdx.x; i < gridDim.x; i += kAdThreads) d += *reinterpret_cast<volatile float*>(&st->part[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = d;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < kAdThreads / 32; i++) d += red[i];
    const float n = __fsqrt_rn(float(d)) * scale;
    *norm = n;
    st->mul = isfinite(n) ? scale * fminf(1.f, __frcp_rn(n + 1e-6f) * max_norm) : n;
    st->arrivals = 0;
  }
}

// What a lane loads of a chunk: 8 elements.
template <bool Q8>
struct AdData {
  float2 p[4];
  AdGrad8 g;
  float2 m[Q8 ? 1 : 4], v[Q8 ? 1 : 4];
  uint2 mq, vq;
  float sm, sv;
};

template <bool Q8>
__device__ __forceinline__ void ad_load(const AdChunk& T, const AdState& S, AdData<Q8>& d) {
  const int lane = threadIdx.x % 32, blk0 = threadIdx.x / 32 * kAdBlock;  // the warp's elements
  if (blk0 >= T.n) return;
  const bool vec = T.flags & kAdVec;
  const long long sb = (T.state + blk0) / kAdBlock;
  if (Q8) {
    d.sm = S.ms[sb];
    d.sv = S.vs[sb];
  }
  if (vec && blk0 + kAdBlock <= T.n) {
    const int i = blk0 + lane * 8;
    const long long s = T.state + i;  // states start at a multiple of their block: aligned
    const uint4 a = ldg16(T.p + i), b = ldg16(T.p + i + 4);
    d.p[0] = make_float2(__uint_as_float(a.x), __uint_as_float(a.y));
    d.p[1] = make_float2(__uint_as_float(a.z), __uint_as_float(a.w));
    d.p[2] = make_float2(__uint_as_float(b.x), __uint_as_float(b.y));
    d.p[3] = make_float2(__uint_as_float(b.z), __uint_as_float(b.w));
    d.g = load_g8(T.g, T.gtype, i);
    if (Q8) {
      d.mq = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(S.m) + s);
      d.vq = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(S.v) + s);
    } else {
      const float4* mp = reinterpret_cast<const float4*>(static_cast<const float*>(S.m) + s);
      const float4* vp = reinterpret_cast<const float4*>(static_cast<const float*>(S.v) + s);
      const float4 m0 = mp[0], m1 = mp[1], v0 = vp[0], v1 = vp[1];
      d.m[0] = make_float2(m0.x, m0.y);
      d.m[1 % (Q8 ? 1 : 4)] = make_float2(m0.z, m0.w);
      d.m[2 % (Q8 ? 1 : 4)] = make_float2(m1.x, m1.y);
      d.m[3 % (Q8 ? 1 : 4)] = make_float2(m1.z, m1.w);
      d.v[0] = make_float2(v0.x, v0.y);
      d.v[1 % (Q8 ? 1 : 4)] = make_float2(v0.z, v0.w);
      d.v[2 % (Q8 ? 1 : 4)] = make_float2(v1.x, v1.y);
      d.v[3 % (Q8 ? 1 : 4)] = make_float2(v1.z, v1.w);
    }
    return;
  }
  // element k of the lane: consecutive with `vec`, else every 32nd
  const int i0 = blk0 + (vec ? lane * 8 : lane), step = vec ? 1 : 32;
  float p[8], g[8], m[8] = {}, v[8] = {};
  uint32_t mq[2] = {}, vq[2] = {};
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const int i = i0 + k * step;
    const bool in = i < T.n;
    const long long s = T.state + i;
    p[k] = in ? T.p[i] : 0.f;
    g[k] = in ? load_g(T.g, T.gtype, i) : 0.f;
    if (Q8) {
      mq[k / 4] |= uint32_t(in ? static_cast<const uint8_t*>(S.m)[s] : 0) << (8 * (k % 4));
      vq[k / 4] |= uint32_t(in ? static_cast<const uint8_t*>(S.v)[s] : 0) << (8 * (k % 4));
    } else {
      m[k] = in ? static_cast<const float*>(S.m)[s] : 0.f;
      v[k] = in ? static_cast<const float*>(S.v)[s] : 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < 4; k++) {
    d.p[k] = make_float2(p[2 * k], p[2 * k + 1]);
    if (!Q8) {
      d.m[k % (Q8 ? 1 : 4)] = make_float2(m[2 * k], m[2 * k + 1]);
      d.v[k % (Q8 ? 1 : 4)] = make_float2(v[2 * k], v[2 * k + 1]);
    }
  }
  // as fp32 bits, whatever their type
  d.g.a = make_uint4(__float_as_uint(g[0]), __float_as_uint(g[1]), __float_as_uint(g[2]), __float_as_uint(g[3]));
  d.g.b = make_uint4(__float_as_uint(g[4]), __float_as_uint(g[5]), __float_as_uint(g[6]), __float_as_uint(g[7]));
  d.mq = make_uint2(mq[0], mq[1]);
  d.vq = make_uint2(vq[0], vq[1]);
}

template <bool Q8>
__device__ __forceinline__ void ad_update(const AdChunk& T, const AdState& S, const AdHyper& H, float mul, AdData<Q8>& d) {
  const int lane = threadIdx.x % 32, blk0 = threadIdx.x / 32 * kAdBlock;
  if (blk0 >= T.n) return;
  const bool vec = T.flags & kAdVec, full = vec && blk0 + kAdBlock <= T.n;
  float2 g[4], m[4], root[4];
  unpack_g8(d.g, full ? T.gtype : OSAM_F32, g);
  const float keep1 = T.flags & kAdDecay ? H.keep : 1.f;
  const float2 keep = make_float2(keep1, keep1), b1 = make_float2(H.b1, H.b1), b2 = make_float2(H.b2, H.b2),
               c1 = make_float2(H.c1, H.c1), c2 = make_float2(H.c2, H.c2), mu = make_float2(mul, mul),
               st = make_float2(H.step, H.step), ir = make_float2(H.inv_root, H.inv_root), ep = make_float2(H.eps, H.eps);
  float mtop = 0.f, vtop = 0.f;
  float2 v[4];
#pragma unroll
  for (int k = 0; k < 4; k++) {  // one rounding a step, in the order of the formula
    if (Q8) {
      const uint32_t mw = k < 2 ? d.mq.x : d.mq.y, vw = k < 2 ? d.vq.x : d.vq.y;
      m[k] = mul2(e4m3x2_to_float2((mw >> (16 * (k % 2))) & 0xffff), make_float2(d.sm, d.sm));
      const float2 r = mul2(e4m3x2_to_float2((vw >> (16 * (k % 2))) & 0xffff), make_float2(d.sv, d.sv));
      v[k] = mul2(r, r);
    } else {
      m[k] = d.m[k % (Q8 ? 1 : 4)];
      v[k] = d.v[k % (Q8 ? 1 : 4)];
    }
    g[k] = mul2(g[k], mu);
    m[k] = add2(mul2(b1, m[k]), mul2(c1, g[k]));
    v[k] = add2(mul2(b2, v[k]), mul2(c2, mul2(g[k], g[k])));
    root[k] = make_float2(__fsqrt_rn(v[k].x), __fsqrt_rn(v[k].y));
    const float2 num = mul2(st, m[k]), den = add2(mul2(root[k], ir), ep);
    const float2 q = make_float2(-__fdividef(num.x, den.x), -__fdividef(num.y, den.y));
    d.p[k] = add2(mul2(d.p[k], keep), q);
    mtop = fmaxf(mtop, fmaxf(fabsf(m[k].x), fabsf(m[k].y)));
    vtop = fmaxf(vtop, fmaxf(root[k].x, root[k].y));
  }
  uint32_t mq[2] = {0, 0}, vq[2] = {0, 0};
  if (Q8) {
    // both maxima are not negative: their order is that of their bits, which one warp instruction takes
    mtop = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mtop)));
    vtop = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(vtop)));
    const bool mlive = mtop >= kTiny, vlive = vtop >= kTiny;
    const float mi = mlive ? kE4m3Max * __frcp_rn(mtop) : 0.f, vi = vlive ? kE4m3Max * __frcp_rn(vtop) : 0.f,
                vleast = vlive ? 1.f / 512.f : 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t a = float2_to_e4m3x2(mul2(m[k], make_float2(mi, mi)));
      float2 r = mul2(root[k], make_float2(vi, vi));  // what is above zero stays above zero: the smallest e4m3 value
      r.x = root[k].x > 0.f ? fmaxf(r.x, vleast) : root[k].x;
      r.y = root[k].y > 0.f ? fmaxf(r.y, vleast) : root[k].y;
      const uint32_t b = float2_to_e4m3x2(r);
      mq[k / 2] |= a << (16 * (k % 2));
      vq[k / 2] |= b << (16 * (k % 2));
    }
    if (lane == 0) {
      const long long sb = (T.state + blk0) / kAdBlock;
      S.ms[sb] = mlive ? mtop * (1.f / kE4m3Max) : 0.f;
      S.vs[sb] = vlive ? vtop * (1.f / kE4m3Max) : 0.f;
    }
  }
  if (full) {
    const int i = blk0 + lane * 8;
    const long long s = T.state + i;
    stg16(T.p + i, d.p[0], d.p[1]);
    stg16(T.p + i + 4, d.p[2], d.p[3]);
    if (T.ctype == OSAM_F16)
      stg16(static_cast<__half*>(T.copy) + i, Half16<__half>::pack(d.p[0].x, d.p[0].y), Half16<__half>::pack(d.p[1].x, d.p[1].y),
                     Half16<__half>::pack(d.p[2].x, d.p[2].y), Half16<__half>::pack(d.p[3].x, d.p[3].y));
    if (T.ctype == OSAM_BF16)
      stg16(static_cast<__nv_bfloat16*>(T.copy) + i, Half16<__nv_bfloat16>::pack(d.p[0].x, d.p[0].y), Half16<__nv_bfloat16>::pack(d.p[1].x, d.p[1].y),
          Half16<__nv_bfloat16>::pack(d.p[2].x, d.p[2].y), Half16<__nv_bfloat16>::pack(d.p[3].x, d.p[3].y));
    if (Q8) {
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(S.m) + s) = make_uint2(mq[0], mq[1]);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(S.v) + s) = make_uint2(vq[0], vq[1]);
    } else {
      float4* mp = reinterpret_cast<float4*>(static_cast<float*>(S.m) + s);
      float4* vp = reinterpret_cast<float4*>(static_cast<float*>(S.v) + s);
      mp[0] = make_float4(m[0].x, m[0].y, m[1].x, m[1].y);
      mp[1] = make_float4(m[2].x, m[2].y, m[3].x, m[3].y);
      vp[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
      vp[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    }
    return;
  }
  const int i0 = blk0 + (vec ? lane * 8 : lane), step = vec ? 1 : 32;
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const int i = i0 + k * step;
    if (i >= T.n) continue;
    const long long s = T.state + i;
    const float p = k % 2 ? d.p[k / 2].y : d.p[k / 2].x;
    T.p[i] = p;
    if (T.ctype == OSAM_F16) static_cast<__half*>(T.copy)[i] = __float2half_rn(p);
    if (T.ctype == OSAM_BF16) static_cast<__nv_bfloat16*>(T.copy)[i] = __float2bfloat16_rn(p);
    if (Q8) {
      static_cast<uint8_t*>(S.m)[s] = uint8_t(mq[k / 4] >> (8 * (k % 4)));
      static_cast<uint8_t*>(S.v)[s] = uint8_t(vq[k / 4] >> (8 * (k % 4)));
    } else {
      static_cast<float*>(S.m)[s] = k % 2 ? m[k / 2].y : m[k / 2].x;
      static_cast<float*>(S.v)[s] = k % 2 ? v[k / 2].y : v[k / 2].x;
    }
  }
}

template <bool Q8>
__global__ void __launch_bounds__(kAdThreads, 4) k_adamw(const AdChunk* chunks, const AdState S, const AdHyper H,
                                                         const AdNorm* norm, float scale) {
  const AdChunk T = ad_chunk(chunks + blockIdx.x);  // of the table, which no kernel writes
  grid_dep_wait();
  grid_dep_launch();
  AdData<Q8> d;
  ad_load<Q8>(T, S, d);
  float mul = scale;
  if (norm) {
    mul = norm->mul;
    if (!isfinite(mul)) return;  // some gradient is not finite: no step
  }
  ad_update<Q8>(T, S, H, mul, d);
}

int ad_fail(int code, const char* what) {
  set_last_error("%s", what);
  return code;
}

constexpr int ad_unit(int bits) { return bits == 8 ? kAdBlock : 64; }

// Layout of the device table: AdNorm | AdChunk[chunks].
struct AdLayout {
  long long chunks = 0, state = 0;
  size_t chunks_at = 0, bytes = 0;
};
AdLayout ad_layout(const osam_adamw_tensor* t, int n, int bits) {
  AdLayout L;
  for (int i = 0; i < n; i++) {
    L.chunks += (t[i].n + kAdChunk - 1) / kAdChunk;
    L.state += (t[i].n + ad_unit(bits) - 1) / ad_unit(bits) * ad_unit(bits);
  }
  L.chunks_at = (sizeof(AdNorm) + 255) / 256 * 256;
  L.bytes = L.chunks_at + sizeof(AdChunk) * (size_t)L.chunks;
  return L;
}
int ad_check(const osam_adamw_tensor* t, int n, int bits) {
  if (bits != 8 && bits != 32) return ad_fail(OSAM_ERR_INVALID, "adamw: states have 8 or 32 bits");
  if (n < 0 || (n > 0 && !t)) return ad_fail(OSAM_ERR_INVALID, "adamw: no tensors");
  long long chunks = 0;
  for (int i = 0; i < n; i++) {
    if (t[i].n > kAdMaxElems) return ad_fail(OSAM_ERR_INVALID, "adamw: too many elements");
    if (t[i].n < 0 || (t[i].n > 0 && (!t[i].p || !t[i].g)))
      return ad_fail(OSAM_ERR_INVALID, "adamw: null parameter or gradient");
    if (t[i].grad_type != OSAM_F32 && t[i].grad_type != OSAM_F16 && t[i].grad_type != OSAM_BF16)
      return ad_fail(OSAM_ERR_INVALID, "adamw: gradients are OSAM_F32, OSAM_F16 or OSAM_BF16");
    if (t[i].copy && t[i].copy_type != OSAM_F16 && t[i].copy_type != OSAM_BF16)
      return ad_fail(OSAM_ERR_INVALID, "adamw: weight copies are OSAM_F16 or OSAM_BF16");
    const size_t ga = t[i].grad_type == OSAM_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(t[i].p) & 3) || (reinterpret_cast<uintptr_t>(t[i].g) & ga) ||
        (reinterpret_cast<uintptr_t>(t[i].copy) & 1))
      return ad_fail(OSAM_ERR_INVALID, "adamw: pointer not aligned to its type");
    chunks += (t[i].n + kAdChunk - 1) / kAdChunk;
  }
  if (chunks > 0x7fffffffLL) return ad_fail(OSAM_ERR_INVALID, "adamw: too many elements");
  return OSAM_OK;
}

}  // namespace
}  // namespace osam

struct osam_adamw {
  int bits, n;
  long long chunks, state;
  char* table;
  size_t chunks_at;
};

using namespace osam;

extern "C" {

int osam_adamw_sizes(const osam_adamw_tensor* tensors, int n, int bits, size_t* table_bytes, int64_t* state_elems) {
  if (!table_bytes || !state_elems) return ad_fail(OSAM_ERR_INVALID, "adamw: null argument");
  const int rc = ad_check(tensors, n, bits);
  if (rc != OSAM_OK) return rc;
  const AdLayout L = ad_layout(tensors, n, bits);
  *table_bytes = L.bytes;
  *state_elems = L.state;
  return OSAM_OK;
}

int osam_adamw_create(const osam_adamw_tensor* tensors, int n, int bits, void* table, size_t table_bytes,
                      osam_stream_t stream, osam_adamw** out) {
  if (!out) return ad_fail(OSAM_ERR_INVALID, "adamw: null argument");
  *out = nullptr;
  const int rc = ad_check(tensors, n, bits);
  if (rc != OSAM_OK) return rc;
  const AdLayout L = ad_layout(tensors, n, bits);
  if (!table || table_bytes < L.bytes || (reinterpret_cast<uintptr_t>(table) & 255))
    return ad_fail(OSAM_ERR_INVALID, "adamw: table (osam_adamw_sizes, 256-byte aligned)");
  osam_adamw* a = nullptr;
  try {
    std::vector<char> host(L.bytes, 0);
    AdChunk* C = reinterpret_cast<AdChunk*>(host.data() + L.chunks_at);
    long long state = 0;
    for (int i = 0; i < n; i++) {
      const osam_adamw_tensor& t = tensors[i];
      const uintptr_t all = reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g) |
                            reinterpret_cast<uintptr_t>(t.copy);
      const int flags = ((all & 15) == 0 ? kAdVec : 0) | (t.decay ? kAdDecay : 0), gsize = t.grad_type == OSAM_F32 ? 4 : 2;
      for (long long at = 0; at < t.n; at += kAdChunk, C++)
        *C = AdChunk{t.p + at, static_cast<const char*>(t.g) + at * gsize,
                     t.copy ? static_cast<char*>(t.copy) + at * 2 : nullptr, state + at,
                     (int)std::min<long long>(t.n - at, kAdChunk), flags, t.grad_type, t.copy ? t.copy_type : -1};
      state += (t.n + ad_unit(bits) - 1) / ad_unit(bits) * ad_unit(bits);
    }
    a = new osam_adamw{bits, n, L.chunks, L.state, static_cast<char*>(table), L.chunks_at};
    // pageable source: the copy has left `host` when the call returns
    const cudaError_t e = cudaMemcpyAsync(table, host.data(), L.bytes, cudaMemcpyHostToDevice,
                                          reinterpret_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) {
      delete a;
      set_last_error("adamw: table copy: %s", cudaGetErrorString(e));
      return OSAM_ERR_CUDA;
    }
  } catch (const std::bad_alloc&) {
    return ad_fail(OSAM_ERR_NOMEM, "adamw: out of host memory");
  }
  *out = a;
  return OSAM_OK;
}

int osam_adamw_destroy(osam_adamw* a) {
  delete a;
  return OSAM_OK;
}

int osam_adamw_step(const osam_adamw* a, void* m, void* v, float* m_scale, float* v_scale, int64_t t, double lr,
                    double beta1, double beta2, double eps, double weight_decay, double grad_scale, double max_norm,
                    float* norm, osam_stream_t stream) {
  if (!a) return ad_fail(OSAM_ERR_INVALID, "adamw: null plan");
  if (t < 1 || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) ||
      !std::isfinite(lr) || !std::isfinite(weight_decay) || !std::isfinite(grad_scale) || std::isnan(max_norm))
    return ad_fail(OSAM_ERR_INVALID, "adamw: step counts from 1, betas in [0, 1), eps ≥ 0, finite factors");
  const bool clip = max_norm > 0;
  if (clip && !norm) return ad_fail(OSAM_ERR_INVALID, "adamw: clipping writes the norm: null norm");
  if (a->chunks == 0) {
    if (clip && cudaMemsetAsync(norm, 0, sizeof(float), reinterpret_cast<cudaStream_t>(stream)) != cudaSuccess)
      return ad_fail(OSAM_ERR_CUDA, "adamw: memset");
    return OSAM_OK;
  }
  if (!m || !v || (a->bits == 8 && (!m_scale || !v_scale)) ||
      ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 15) ||
      ((reinterpret_cast<uintptr_t>(m_scale) | reinterpret_cast<uintptr_t>(v_scale) | reinterpret_cast<uintptr_t>(norm)) & 3))
    return ad_fail(OSAM_ERR_INVALID, "adamw: null or misaligned (16 bytes, scales and norm 4) states");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const AdChunk* chunks = reinterpret_cast<const AdChunk*>(a->table + a->chunks_at);
  AdNorm* ns = reinterpret_cast<AdNorm*>(a->table);
  const AdState S{m, v, m_scale, v_scale};
  AdHyper H;
  H.b1 = (float)beta1;
  H.b2 = (float)beta2;
  H.c1 = (float)(1.0 - beta1);
  H.c2 = (float)(1.0 - beta2);
  H.step = (float)(lr / (1.0 - std::pow(beta1, (double)t)));
  H.inv_root = 1.f / (float)std::sqrt(1.0 - std::pow(beta2, (double)t));
  H.eps = (float)eps;
  H.keep = (float)(1.0 - lr * weight_decay);
  const float gs = (float)grad_scale;
  cudaError_t e = cudaSuccess;
  if (clip) {
    const unsigned grid = (unsigned)std::min<long long>(a->chunks, kAdNormCtas);
    e = launch_dependent(k_adamw_norm, grid, kAdThreads, 0, st, chunks, (int)a->chunks, ns, gs, (float)max_norm, norm);
  }
  if (e == cudaSuccess)
    e = launch_dependent(a->bits == 8 ? k_adamw<true> : k_adamw<false>, (unsigned)a->chunks, kAdThreads, 0, st, chunks, S, H,
                         (const AdNorm*)(clip ? ns : nullptr), gs);
  if (e != cudaSuccess) {
    set_last_error("osam_adamw_step launch: %s", cudaGetErrorString(e));
    return OSAM_ERR_CUDA;
  }
  return OSAM_OK;
}

}  // extern "C"
