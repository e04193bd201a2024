// AdamW over many tensors in one launch, with the moments in 32 bits or in 8 bits with a scale per 256 elements,
// and an optional clip by the global norm of the gradients.
//
//   g' = g·mul;  m = β1·m + (1−β1)·g';  v = β2·v + (1−β2)·g'²
//   p = p·(1 − lr·wd) − lr/(1−β1ᵗ)·m / (√v/√(1−β2ᵗ) + eps)          (wd = 0 for tensors marked so)
// 8-bit states, per block of 256 elements: m = e4m3·s_m with s_m = max|m|/448, and the ROOT of v likewise
// (√v = e4m3·s_v): the root halves the exponent range, so e4m3's 2^18 covers 2^36 in v.  A v above zero is never
// stored as zero (it takes the smallest e4m3 value): a moment that survives beside a vanished v would make its
// step m/eps.  The step uses the new moments before they are rounded.
//
// Bound by HBM: 28 bytes an element with 32-bit states (14 + 1/32 with 8 bits) and 2 more for a 16-bit weight
// copy.  A table in device memory, written once, names each tensor's arrays, and a second one the tensor and
// offset of every 2048-element chunk: one CTA per chunk, so small and large tensors share one launch with no
// search.  A warp owns 256 consecutive elements — one quantisation block, whose maximum is five shuffles.  Lanes
// hold 8 consecutive elements (16-byte accesses) where the tensor's pointers allow it, else every 32nd element,
// so that unaligned tensors (slices of a packed gradient arena) stay coalesced too.
// The norm pass reads the gradients once more: fixed chunks per CTA, the last CTA to arrive adds the partial sums
// in a fixed order in fp64 and writes the norm and the multiplier; a norm that is not finite makes the step leave
// parameters and states alone.
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "conv_internal.h"
#include "half16.cuh"
#include "sm100.cuh"

namespace osam {
namespace {

constexpr int kAdThreads = 256;
constexpr int kAdChunk = kAdThreads * 8;  // elements per CTA
constexpr int kAdBlock = 256;             // elements per quantisation scale (one warp)
constexpr int kAdNormCtas = 148 * 4;
constexpr float kE4m3Max = 448.f;
constexpr float kTiny = 1e-30f;           // a block whose maximum is below this is stored as zeros

struct AdTensor {  // device table entry
  float* p;
  const void* g;
  void* copy;
  long long n, state;  // elements; offset of its states (elements)
  int gtype, ctype;    // OSAM_F32 / F16 / BF16; ctype −1: no copy
  int decay, vec;      // vec: 16-byte accesses allowed
};
struct AdChunk {
  int tensor, index;  // chunk `index` of the tensor
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

__device__ __forceinline__ float load_g(const void* g, int type, long long i) {
  if (type == OSAM_F32) return static_cast<const float*>(g)[i];
  if (type == OSAM_F16) return __half2float(static_cast<const __half*>(g)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(g)[i]);
}
__device__ __forceinline__ void load_g8(const void* g, int type, long long i, float (&o)[8]) {
  if (type == OSAM_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(g) + i);
    const float4 a = p[0], b = p[1];
    o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w;
    o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
    return;
  }
  const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(g) + i);
  if (type == OSAM_F16)
    unpack8<__half>(u, o);
  else
    unpack8<__nv_bfloat16>(u, o);
}
__device__ __forceinline__ void load8f(const float* p, float (&o)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w;
  o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
}
__device__ __forceinline__ void store8f(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

__device__ __forceinline__ float e4m3_to_float(uint8_t q) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(q, __NV_E4M3)));
}
__device__ __forceinline__ uint8_t float_to_e4m3(float f) { return __nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3); }

// Σ g² of the gradients: CTA b walks chunks b, b + gridDim, …; the last CTA adds the CTAs' sums in order.
__global__ void __launch_bounds__(kAdThreads) k_adamw_norm(const AdTensor* tab, const AdChunk* chunks, int nchunks,
                                                           AdNorm* st, float scale, float max_norm, float* norm) {
  __shared__ float red[kAdThreads / 32];
  __shared__ bool last;
  float s = 0.f;
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
    const AdChunk ck = chunks[c];
    const AdTensor T = tab[ck.tensor];
    const long long i0 = (long long)ck.index * kAdChunk;
    const long long i = i0 + threadIdx.x * 8;
    if (T.vec && i + 8 <= T.n) {
      float g[8];
      load_g8(T.g, T.gtype, i, g);
#pragma unroll
      for (int k = 0; k < 8; k++) s = fmaf(g[k], g[k], s);
    } else if (T.vec) {
      for (long long j = i; j < T.n && j < i + 8; j++) {
        const float g = load_g(T.g, T.gtype, j);
        s = fmaf(g, g, s);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const long long j = i0 + k * kAdThreads + threadIdx.x;
        const float g = j < T.n ? load_g(T.g, T.gtype, j) : 0.f;
        s = fmaf(g, g, s);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < kAdThreads / 32; i++) s += red[i];
    st->part[blockIdx.x] = s;
    __threadfence();
    last = atomicAdd(&st->arrivals, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last || threadIdx.x >= 32) return;
  __threadfence();
  double d = 0;
  for (int i = threadIdx.x; i < gridDim.x; i += 32) d += *reinterpret_cast<volatile float*>(&st->part[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  if (threadIdx.x == 0) {
    const float n = __fsqrt_rn(float(d)) * scale;
    *norm = n;
    st->mul = isfinite(n) ? scale * fminf(1.f, __frcp_rn(n + 1e-6f) * max_norm) : n;
    st->arrivals = 0;
  }
}

// New moments and parameter of one element; every step is one rounding, in the order of the formula.
__device__ __forceinline__ void adamw_one(const AdHyper& H, float keep, float g, float& p, float& m, float& v,
                                          float& root) {
  m = __fadd_rn(__fmul_rn(H.b1, m), __fmul_rn(H.c1, g));
  v = __fadd_rn(__fmul_rn(H.b2, v), __fmul_rn(H.c2, __fmul_rn(g, g)));
  root = __fsqrt_rn(v);
  p = __fsub_rn(__fmul_rn(p, keep), __fdiv_rn(__fmul_rn(H.step, m), __fadd_rn(__fmul_rn(root, H.inv_root), H.eps)));
}

template <bool Q8>
__global__ void __launch_bounds__(kAdThreads) k_adamw(const AdTensor* tab, const AdChunk* chunks, const AdState S,
                                                      const AdHyper H, const AdNorm* norm, float scale) {
  grid_dep_wait();
  const AdChunk ck = chunks[blockIdx.x];
  const AdTensor T = tab[ck.tensor];
  float mul = scale;
  if (norm) {
    mul = norm->mul;
    if (!isfinite(mul)) return;  // some gradient is not finite: no step
  }
  const int lane = threadIdx.x % 32;
  const long long blk0 = (long long)ck.index * kAdChunk + (threadIdx.x / 32) * kAdBlock;  // the warp's elements
  if (blk0 >= T.n) return;
  const float keep = T.decay ? H.keep : 1.f;
  // element k of this lane: consecutive with `vec`, else every 32nd; full: no bounds checks
  const bool vec = T.vec;
  const long long i0 = blk0 + (vec ? lane * 8 : lane);
  const int step = vec ? 1 : 32;
  const bool full = blk0 + kAdBlock <= T.n;
  float p[8], g[8], m[8], v[8], root[8];
  const long long s0 = T.state + i0;  // states start at a multiple of their block: aligned
  long long sb = 0;
  float sm = 0.f, sv = 0.f;
  if (Q8) {
    sb = (T.state + blk0) / kAdBlock;
    sm = S.ms[sb];
    sv = S.vs[sb];
  }
  if (vec && full) {
    load8f(T.p + i0, p);
    load_g8(T.g, T.gtype, i0, g);
    if (Q8) {
      const uint2 mu = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(S.m) + s0);
      const uint2 vu = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(S.v) + s0);
#pragma unroll
      for (int k = 0; k < 8; k++) {
        m[k] = e4m3_to_float(uint8_t((k < 4 ? mu.x : mu.y) >> (8 * (k % 4))));
        v[k] = e4m3_to_float(uint8_t((k < 4 ? vu.x : vu.y) >> (8 * (k % 4))));
      }
    } else {
      load8f(static_cast<const float*>(S.m) + s0, m);
      load8f(static_cast<const float*>(S.v) + s0, v);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const bool in = i0 + k * step < T.n;
      const long long i = i0 + k * step, s = s0 + k * step;
      p[k] = in ? T.p[i] : 0.f;
      g[k] = in ? load_g(T.g, T.gtype, i) : 0.f;
      if (Q8) {
        m[k] = in ? e4m3_to_float(static_cast<const uint8_t*>(S.m)[s]) : 0.f;
        v[k] = in ? e4m3_to_float(static_cast<const uint8_t*>(S.v)[s]) : 0.f;
      } else {
        m[k] = in ? static_cast<const float*>(S.m)[s] : 0.f;
        v[k] = in ? static_cast<const float*>(S.v)[s] : 0.f;
      }
    }
  }
  float mtop = 0.f, vtop = 0.f;
#pragma unroll
  for (int k = 0; k < 8; k++) {
    if (Q8) {
      m[k] = __fmul_rn(m[k], sm);
      v[k] = __fmul_rn(v[k], sv);
      v[k] = __fmul_rn(v[k], v[k]);
    }
    adamw_one(H, keep, __fmul_rn(g[k], mul), p[k], m[k], v[k], root[k]);
    mtop = fmaxf(mtop, fabsf(m[k]));
    vtop = fmaxf(vtop, root[k]);
  }
  uint32_t mq[2] = {0, 0}, vq[2] = {0, 0};
  if (Q8) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mtop = fmaxf(mtop, __shfl_xor_sync(0xffffffffu, mtop, o));
      vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, o));
    }
    const bool mlive = mtop >= kTiny, vlive = vtop >= kTiny;
    const float mi = mlive ? kE4m3Max * __frcp_rn(mtop) : 0.f, vi = vlive ? kE4m3Max * __frcp_rn(vtop) : 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const uint32_t a = float_to_e4m3(m[k] * mi);
      uint32_t b = float_to_e4m3(root[k] * vi);
      if (b == 0 && vlive && root[k] > 0.f) b = 1;  // the smallest e4m3 value
      mq[k / 4] |= a << (8 * (k % 4));
      vq[k / 4] |= b << (8 * (k % 4));
    }
    if (lane == 0) {
      S.ms[sb] = mlive ? mtop * (1.f / kE4m3Max) : 0.f;
      S.vs[sb] = vlive ? vtop * (1.f / kE4m3Max) : 0.f;
    }
  }
  if (vec && full) {
    store8f(T.p + i0, p);
    if (T.ctype == OSAM_F16) *reinterpret_cast<uint4*>(static_cast<__half*>(T.copy) + i0) = pack8<__half>(p);
    if (T.ctype == OSAM_BF16)
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(T.copy) + i0) = pack8<__nv_bfloat16>(p);
    if (Q8) {
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(S.m) + s0) = make_uint2(mq[0], mq[1]);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(S.v) + s0) = make_uint2(vq[0], vq[1]);
    } else {
      store8f(static_cast<float*>(S.m) + s0, m);
      store8f(static_cast<float*>(S.v) + s0, v);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const long long i = i0 + k * step, s = s0 + k * step;
    if (i >= T.n) continue;
    T.p[i] = p[k];
    if (T.ctype == OSAM_F16) static_cast<__half*>(T.copy)[i] = __float2half_rn(p[k]);
    if (T.ctype == OSAM_BF16) static_cast<__nv_bfloat16*>(T.copy)[i] = __float2bfloat16_rn(p[k]);
    if (Q8) {
      static_cast<uint8_t*>(S.m)[s] = uint8_t(mq[k / 4] >> (8 * (k % 4)));
      static_cast<uint8_t*>(S.v)[s] = uint8_t(vq[k / 4] >> (8 * (k % 4)));
    } else {
      static_cast<float*>(S.m)[s] = m[k];
      static_cast<float*>(S.v)[s] = v[k];
    }
  }
}

int ad_fail(int code, const char* what) {
  set_last_error("%s", what);
  return code;
}

constexpr int ad_unit(int bits) { return bits == 8 ? kAdBlock : 64; }

// Layout of the device table: AdNorm | AdTensor[n] | AdChunk[chunks].
struct AdLayout {
  long long chunks = 0, state = 0;
  size_t tensors_at = 0, chunks_at = 0, bytes = 0;
};
AdLayout ad_layout(const osam_adamw_tensor* t, int n, int bits) {
  AdLayout L;
  for (int i = 0; i < n; i++) {
    L.chunks += (t[i].n + kAdChunk - 1) / kAdChunk;
    L.state += (t[i].n + ad_unit(bits) - 1) / ad_unit(bits) * ad_unit(bits);
  }
  L.tensors_at = (sizeof(AdNorm) + 255) / 256 * 256;
  L.chunks_at = L.tensors_at + (sizeof(AdTensor) * (size_t)n + 255) / 256 * 256;
  L.bytes = L.chunks_at + sizeof(AdChunk) * (size_t)L.chunks;
  return L;
}
int ad_check(const osam_adamw_tensor* t, int n, int bits) {
  if (bits != 8 && bits != 32) return ad_fail(OSAM_ERR_INVALID, "adamw: states have 8 or 32 bits");
  if (n < 0 || (n > 0 && !t)) return ad_fail(OSAM_ERR_INVALID, "adamw: no tensors");
  long long chunks = 0;
  for (int i = 0; i < n; i++) {
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
  size_t tensors_at, chunks_at;
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
    AdTensor* T = reinterpret_cast<AdTensor*>(host.data() + L.tensors_at);
    AdChunk* C = reinterpret_cast<AdChunk*>(host.data() + L.chunks_at);
    long long state = 0, c = 0;
    for (int i = 0; i < n; i++) {
      const osam_adamw_tensor& t = tensors[i];
      const uintptr_t all = reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g) |
                            reinterpret_cast<uintptr_t>(t.copy);
      T[i] = AdTensor{t.p, t.g, t.copy, t.n, state, t.grad_type, t.copy ? t.copy_type : -1, t.decay != 0,
                      (all & 15) == 0};
      state += (t.n + ad_unit(bits) - 1) / ad_unit(bits) * ad_unit(bits);
      for (long long k = 0; k * kAdChunk < t.n; k++) C[c++] = AdChunk{i, (int)k};
    }
    a = new osam_adamw{bits, n, L.chunks, L.state, static_cast<char*>(table), L.tensors_at, L.chunks_at};
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
      ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 15))
    return ad_fail(OSAM_ERR_INVALID, "adamw: null or misaligned (16 bytes) states");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const AdTensor* tab = reinterpret_cast<const AdTensor*>(a->table + a->tensors_at);
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
  if (clip) {
    const int grid = (int)std::min<long long>(a->chunks, kAdNormCtas);
    k_adamw_norm<<<grid, kAdThreads, 0, st>>>(tab, chunks, (int)a->chunks, ns, gs, (float)max_norm, norm);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)a->chunks);
  cfg.blockDim = dim3(kAdThreads);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = clip ? 1 : 0;
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess)
    e = a->bits == 8 ? cudaLaunchKernelEx(&cfg, k_adamw<true>, tab, chunks, S, H, (const AdNorm*)(clip ? ns : nullptr), gs)
                     : cudaLaunchKernelEx(&cfg, k_adamw<false>, tab, chunks, S, H, (const AdNorm*)(clip ? ns : nullptr), gs);
  if (e != cudaSuccess) {
    set_last_error("osam_adamw_step launch: %s", cudaGetErrorString(e));
    return OSAM_ERR_CUDA;
  }
  return OSAM_OK;
}

}  // extern "C"
