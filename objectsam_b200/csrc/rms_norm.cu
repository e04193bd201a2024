// RMS norm over the channels of each row with the residual's addition in front (output in 16 bits or in e4m3
// with a scale per 128 channels), and its backward pass.
//
//   h = x + r                      (fp32; stored rounded to 16 bits as the new residual stream)
//   y = h·rstd·w,   rstd = 1/√(Σ h²/C + eps)
//   q = e4m3(y·448/amax), qscale = amax/448, amax = max |y| over a group of 128 channels
//   dh = rstd·(w·dy − ĥ·Σ(w·dy·ĥ)/C) (+ dsum),  dw = Σ_rows dy·ĥ,   ĥ = h·rstd
//
// Bound by HBM: each tensor is read or written once, so a row stays in registers between the reduction and the
// use of its result.  A row belongs to TPR consecutive threads, each holding NV vectors of eight channels (16
// bytes): 4–32 threads while a row fits one warp (up to 1024 channels: the reduction is a few shuffles and a warp
// carries several short rows), 256 threads with a shared-memory reduction for longer rows.  Grids are persistent, so
// w is read once per thread and dw accumulates in registers over the rows a thread walks; the CTAs' partial dw rows
// go to the workspace and a second small kernel adds them in a fixed order (no atomics: the result does not depend on
// scheduling).
// Measured: 16397 rows of 4096 channels with a residual into e4m3 in 81 us (5.8 TB/s of a copy's 6.6); 25600 rows of
// 256 channels forward and backward in 25 us, of which 16 are bytes and the rest three launches' starts and ends.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "conv_internal.h"
#include "half16.cuh"
#include "launch.cuh"
#include "sm100.cuh"

namespace osam {
namespace {

constexpr int kRmsThreads = 256;
constexpr int kRmsMaxC = 8192;
constexpr int kRmsGroup = 128;       // channels per e4m3 scale
constexpr float kE4m3Max = 448.f;
constexpr int kRmsSms = 148;
constexpr int kRmsBwdCtas = 4 * kRmsSms;  // at most this many partial dw rows (rows above 1024 channels)

struct RmsFwd {
  const void* x;
  const void* r;
  const float* w;
  void* sum;
  void* y;
  float* qscale;
  float* rstd;
  long long ldx, ldr, lds, ldy, rows;
  int C, groups;
  float eps, inv_c;
};

struct RmsBwd {
  const void* dy;
  const void* h;
  const void* dsum;
  const float* w;
  const float* rstd;
  void* dx;
  float* part;  // [gridDim.x][C]
  long long lddy, ldh, ldds, lddx, rows;
  int C;
  float inv_c;
};

// Sum over the TPR threads of a row (TPR ≤ 32: lanes of one warp; else the whole CTA row group in shared memory).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (TPR > 32) {
    constexpr int W = TPR / 32;
    const int group = threadIdx.x / TPR, wr = (threadIdx.x % TPR) / 32;
    __syncthreads();  // the previous row's sums have been read
    if (threadIdx.x % 32 == 0) red[group * W + wr] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < W; i++) v += red[group * W + i];
  }
  return v;
}

template <typename T, int TPR, int NV, bool Q8>
__global__ void __launch_bounds__(kRmsThreads) k_rms_fwd(const RmsFwd P) {
  __shared__ float red[kRmsThreads / 32];
  constexpr int RPC = kRmsThreads / TPR;  // rows per CTA
  grid_dep_wait();
  grid_dep_launch();
  const int t = threadIdx.x % TPR, C8 = P.C / 8;
  float w[NV][8];
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const int v = t + k * TPR;
#pragma unroll
    for (int i = 0; i < 8; i++) w[k][i] = v < C8 ? P.w[v * 8 + i] : 0.f;
  }
  // every thread of the CTA takes the same number of turns (the row reduction has CTA barriers)
  for (long long row0 = (long long)blockIdx.x * RPC; row0 < P.rows; row0 += (long long)gridDim.x * RPC) {
    const long long row = row0 + threadIdx.x / TPR;
    const bool live = row < P.rows;
    uint4 xu[NV], ru[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int v = t + k * TPR;
      xu[k] = make_uint4(0, 0, 0, 0);
      ru[k] = make_uint4(0, 0, 0, 0);
      if (live && v < C8) {
        xu[k] = *reinterpret_cast<const uint4*>(static_cast<const T*>(P.x) + row * P.ldx + v * 8);
        if (P.r) ru[k] = *reinterpret_cast<const uint4*>(static_cast<const T*>(P.r) + row * P.ldr + v * 8);
      }
    }
    float h[NV][8], ss = 0.f;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      unpack8<T>(xu[k], h[k]);
      if (P.r) {
        float r[8];
        unpack8<T>(ru[k], r);
#pragma unroll
        for (int i = 0; i < 8; i++) h[k][i] += r[i];
      }
#pragma unroll
      for (int i = 0; i < 8; i++) ss = fmaf(h[k][i], h[k][i], ss);
      const int v = t + k * TPR;
      if (P.sum && live && v < C8)
        *reinterpret_cast<uint4*>(static_cast<T*>(P.sum) + row * P.lds + v * 8) = pack8<T>(h[k]);
    }
    const float rstd = rsqrtf(fmaf(row_sum<TPR>(ss, red), P.inv_c, P.eps));
    if (live && t == 0 && P.rstd) P.rstd[row] = rstd;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int v = t + k * TPR;
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; i++) y[i] = h[k][i] * rstd * w[k][i];
      if (!Q8) {
        if (live && v < C8) *reinterpret_cast<uint4*>(static_cast<T*>(P.y) + row * P.ldy + v * 8) = pack8<T>(y);
        continue;
      }
      // 16 consecutive vectors share a scale: with TPR a power of two they are 16 (or all TPR) adjacent lanes
      float top = 0.f;
      bool bad = false;  // a NaN, which fmaxf drops
#pragma unroll
      for (int i = 0; i < 8; i++) {
        top = fmaxf(top, fabsf(y[i]));
        bad |= y[i] != y[i];
      }
      if (bad) top = __int_as_float(0x7fffffff);
#pragma unroll
      for (int o = (TPR < 16 ? TPR : 16) / 2; o > 0; o >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, top, o);
        top = (top != top || other != other) ? __int_as_float(0x7fffffff) : fmaxf(top, other);
      }
      // 448/top is not finite below 2^-119: such a group is brought up by a power of two first, its scale left as it is
      const float scale = top / kE4m3Max;
      if (top < 0x1p-100f) {
        top *= 0x1p100f;
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] *= 0x1p100f;
      }
      const float inv = top > 0.f ? kE4m3Max / top : (top == 0.f ? 0.f : top);
      if (live && v < C8) {
        uint2 u;
        __nv_fp8x2_storage_t* q = reinterpret_cast<__nv_fp8x2_storage_t*>(&u);
#pragma unroll
        for (int i = 0; i < 4; i++)
          q[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i] * inv, y[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(P.y) + row * P.ldy + v * 8) = u;
        if (v % 16 == 0) P.qscale[row * P.groups + v / 16] = scale;
      }
    }
  }
}

// Rows within a warp: one CTA of 32 warps per SM (16 where a thread holds 32 channels), so that few partial dw rows
// are left to add; wider rows: as the forward.
template <int TPR, int NV>
constexpr int rms_bwd_threads() {
  return TPR > 32 ? kRmsThreads : NV == 4 ? 512 : 1024;
}
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(rms_bwd_threads<TPR, NV>()) k_rms_bwd(const RmsBwd P) {
  constexpr int THREADS = rms_bwd_threads<TPR, NV>();
  __shared__ float red[THREADS / 32];
  __shared__ float part[TPR <= 32 ? THREADS * 8 : 1];
  constexpr int RPC = THREADS / TPR;
  grid_dep_wait();
  grid_dep_launch();
  const int t = threadIdx.x % TPR, C8 = P.C / 8;
  float w[NV][8], dw[NV][8];
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const int v = t + k * TPR;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      w[k][i] = v < C8 ? P.w[v * 8 + i] : 0.f;
      dw[k][i] = 0.f;
    }
  }
  for (long long row0 = (long long)blockIdx.x * RPC; row0 < P.rows; row0 += (long long)gridDim.x * RPC) {
    const long long row = row0 + threadIdx.x / TPR;
    const bool live = row < P.rows;
    uint4 hu[NV], gu[NV], su[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int v = t + k * TPR;
      hu[k] = gu[k] = su[k] = make_uint4(0, 0, 0, 0);
      if (live && v < C8) {
        hu[k] = *reinterpret_cast<const uint4*>(static_cast<const T*>(P.h) + row * P.ldh + v * 8);
        gu[k] = *reinterpret_cast<const uint4*>(static_cast<const T*>(P.dy) + row * P.lddy + v * 8);
        if (P.dsum) su[k] = *reinterpret_cast<const uint4*>(static_cast<const T*>(P.dsum) + row * P.ldds + v * 8);
      }
    }
    const float rstd = live ? P.rstd[row] : 0.f;
    float dot = 0.f;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      float h[8], g[8];
      unpack8<T>(hu[k], h);
      unpack8<T>(gu[k], g);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float n = h[i] * rstd;
        dw[k][i] = fmaf(g[i], n, dw[k][i]);
        dot = fmaf(g[i] * w[k][i], n, dot);
      }
    }
    dot = row_sum<TPR>(dot, red) * P.inv_c;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int v = t + k * TPR;
      float h[8], g[8], s[8], o[8];
      unpack8<T>(hu[k], h);
      unpack8<T>(gu[k], g);
      unpack8<T>(su[k], s);
#pragma unroll
      for (int i = 0; i < 8; i++) o[i] = fmaf(rstd, fmaf(-dot, h[i] * rstd, g[i] * w[k][i]), s[i]);
      if (live && v < C8) *reinterpret_cast<uint4*>(static_cast<T*>(P.dx) + row * P.lddx + v * 8) = pack8<T>(o);
    }
  }
  // dw of the CTA: the row groups' sums added in group order, one slice of 8·TPR channels at a time
  float* out = P.part + (long long)blockIdx.x * P.C;
#pragma unroll
  for (int k = 0; k < NV; k++) {
    if (RPC == 1) {
      const int v = t + k * TPR;
      if (v < C8)
#pragma unroll
        for (int i = 0; i < 8; i++) out[v * 8 + i] = dw[k][i];
      continue;
    }
    if (TPR <= 32) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; i++) part[(threadIdx.x / TPR) * TPR * 8 + t * 8 + i] = dw[k][i];
      __syncthreads();
      for (int c = threadIdx.x; c < TPR * 8; c += THREADS) {
        float s = 0.f;
#pragma unroll 8
        for (int g = 0; g < RPC; g++) s += part[g * TPR * 8 + c];
        if (k * TPR * 8 + c < P.C) out[k * TPR * 8 + c] = s;
      }
    }
  }
}

// dw[c] = Σ over the CTAs' partial rows, in a fixed order: 32 channels per CTA, 32 threads per channel, four loads of
// each in flight (a chain of single loads took 10 us over 592 rows, as long as the backward pass itself).
__global__ void __launch_bounds__(1024) k_rms_dw(const float* part, int n, int C, float* dw) {
  __shared__ float s[32][33];
  grid_dep_wait();
  grid_dep_launch();
  const int c = blockIdx.x * 32 + threadIdx.x % 32, l = threadIdx.x / 32;
  float a[4] = {};
  if (c < C)
    for (int i = l; i < n; i += 128) {
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (i + 32 * k < n) a[k] += part[(long long)(i + 32 * k) * C + c];
    }
  s[l][threadIdx.x % 32] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  float v = s[threadIdx.x % 32][l];  // warp l adds channel l's 32 sums
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int out = blockIdx.x * 32 + l;
  if (threadIdx.x % 32 == 0 && out < C) dw[out] = v;
}

int rms_fail(int code, const char* what) {
  set_last_error("%s", what);
  return code;
}
int rms_cuda(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return OSAM_OK;
  set_last_error("%s: %s", what, cudaGetErrorString(e));
  return OSAM_ERR_CUDA;
}
bool rms_view(const void* p, long long ld, int C, int bytes_per_8) {  // 8-channel vectors are aligned
  return p && ld >= C && ld % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & (bytes_per_8 - 1)) == 0;
}

bool rms_f32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// Calls f(TPR, NV) as compile-time constants for a row of C channels.
template <typename F>
void rms_shape(int C, F f) {
  using std::integral_constant;
  const int v = C / 8;
#define OSAM_RMS_SHAPE(limit, tpr, nv) \
  if (v <= limit) return f(integral_constant<int, tpr>(), integral_constant<int, nv>())
  OSAM_RMS_SHAPE(4, 4, 1);
  OSAM_RMS_SHAPE(8, 8, 1);
  OSAM_RMS_SHAPE(16, 16, 1);
  OSAM_RMS_SHAPE(32, 32, 1);
  OSAM_RMS_SHAPE(64, 32, 2);
  OSAM_RMS_SHAPE(128, 32, 4);
  OSAM_RMS_SHAPE(256, 256, 1);
  OSAM_RMS_SHAPE(512, 256, 2);
  OSAM_RMS_SHAPE(1024, 256, 4);
#undef OSAM_RMS_SHAPE
}

template <typename T, bool Q8>
cudaError_t launch_rms_fwd(const RmsFwd& P, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  rms_shape(P.C, [&](auto tpr, auto nv) {
    constexpr int RPC = kRmsThreads / tpr.value;
    const long long need = (P.rows + RPC - 1) / RPC;
    const int grid = (int)std::min<long long>(need, kRmsSms * 8);
    e = launch_dependent(k_rms_fwd<T, tpr.value, nv.value, Q8>, grid, kRmsThreads, 0, st, P);
  });
  return e;
}

int rms_fwd(int dtype, RmsFwd P, bool q8, cudaStream_t st, const char* name) {
  if (dtype != OSAM_F16 && dtype != OSAM_BF16) return rms_fail(OSAM_ERR_INVALID, "rms: dtype is OSAM_F16 or OSAM_BF16");
  if (P.rows < 0 || P.C < 8 || P.C % 8 || P.C > kRmsMaxC)
    return rms_fail(OSAM_ERR_INVALID, "rms: channels are a multiple of 8, at most 8192");
  if (P.rows == 0) return OSAM_OK;
  if (!P.w || !rms_view(P.x, P.ldx, P.C, 16) || !rms_view(P.y, P.ldy, P.C, q8 ? 8 : 16) ||
      (P.r && !rms_view(P.r, P.ldr, P.C, 16)) || (P.sum && !rms_view(P.sum, P.lds, P.C, 16)) || (q8 && !P.qscale))
    return rms_fail(OSAM_ERR_INVALID, "rms: null, misaligned (16 bytes; 8 for e4m3) or overlapping rows");
  if (!rms_f32(P.w) || !rms_f32(P.rstd) || !rms_f32(P.qscale))
    return rms_fail(OSAM_ERR_INVALID, "rms: w, rstd and scales are 4-byte aligned");
  P.inv_c = 1.f / P.C;
  P.groups = (P.C + kRmsGroup - 1) / kRmsGroup;
  const cudaError_t e =
      dtype == OSAM_F16 ? (q8 ? launch_rms_fwd<__half, true>(P, st) : launch_rms_fwd<__half, false>(P, st))
                        : (q8 ? launch_rms_fwd<__nv_bfloat16, true>(P, st) : launch_rms_fwd<__nv_bfloat16, false>(P, st));
  return rms_cuda(e, name);
}

template <typename T>
int launch_rms_bwd(const RmsBwd& P, float* dw, cudaStream_t st) {
  int grid = 0;
  cudaError_t e = cudaSuccess;
  rms_shape(P.C, [&](auto tpr, auto nv) {
    constexpr int threads = rms_bwd_threads<tpr.value, nv.value>(), RPC = threads / tpr.value;
    const int most = tpr.value > 32 ? kRmsBwdCtas : threads == 512 ? 2 * kRmsSms : kRmsSms;
    grid = (int)std::min<long long>((P.rows + RPC - 1) / RPC, most);
    e = launch_dependent(k_rms_bwd<T, tpr.value, nv.value>, grid, threads, 0, st, P);
  });
  if (e == cudaSuccess)
    e = launch_dependent(k_rms_dw, (P.C + 31) / 32, 1024, 0, st, (const float*)P.part, grid, P.C, dw);
  return rms_cuda(e, "osam_rms_bwd launch");
}

}  // namespace
}  // namespace osam

using namespace osam;

extern "C" {

int osam_rms_fwd(int dtype, const void* x, int64_t ldx, const void* res, int64_t ldres, const float* w, int64_t rows,
                 int C, float eps, void* sum, int64_t ldsum, void* y, int64_t ldy, float* rstd, osam_stream_t stream) {
  RmsFwd P{};
  P.x = x; P.ldx = ldx;
  P.r = res; P.ldr = ldres;
  P.w = w;
  P.sum = sum; P.lds = ldsum;
  P.y = y; P.ldy = ldy;
  P.rstd = rstd;
  P.rows = rows; P.C = C; P.eps = eps;
  return rms_fwd(dtype, P, false, reinterpret_cast<cudaStream_t>(stream), "osam_rms_fwd launch");
}

int osam_rms_fwd_q8(int dtype, const void* x, int64_t ldx, const void* res, int64_t ldres, const float* w,
                    int64_t rows, int C, float eps, void* sum, int64_t ldsum, void* q, int64_t ldq, float* qscale,
                    float* rstd, osam_stream_t stream) {
  RmsFwd P{};
  P.x = x; P.ldx = ldx;
  P.r = res; P.ldr = ldres;
  P.w = w;
  P.sum = sum; P.lds = ldsum;
  P.y = q; P.ldy = ldq;
  P.qscale = qscale;
  P.rstd = rstd;
  P.rows = rows; P.C = C; P.eps = eps;
  return rms_fwd(dtype, P, true, reinterpret_cast<cudaStream_t>(stream), "osam_rms_fwd_q8 launch");
}

size_t osam_rms_bwd_workspace_size(int C) {
  return C >= 8 && C <= kRmsMaxC ? (size_t)kRmsBwdCtas * C * sizeof(float) : 0;
}

int osam_rms_bwd(int dtype, const void* dy, int64_t lddy, const void* h, int64_t ldh, const float* w,
                 const float* rstd, const void* dsum, int64_t lddsum, int64_t rows, int C, void* dx, int64_t lddx,
                 float* dw, void* ws, size_t ws_bytes, osam_stream_t stream) {
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype != OSAM_F16 && dtype != OSAM_BF16) return rms_fail(OSAM_ERR_INVALID, "rms: dtype is OSAM_F16 or OSAM_BF16");
  if (rows < 0 || C < 8 || C % 8 || C > kRmsMaxC)
    return rms_fail(OSAM_ERR_INVALID, "rms: channels are a multiple of 8, at most 8192");
  if (!dw || !rms_f32(dw)) return rms_fail(OSAM_ERR_INVALID, "rms: null or misaligned dw");
  if (rows == 0) return rms_cuda(cudaMemsetAsync(dw, 0, (size_t)C * sizeof(float), st), "osam_rms_bwd memset");
  if (!w || !rstd || !rms_view(dy, lddy, C, 16) || !rms_view(h, ldh, C, 16) || !rms_view(dx, lddx, C, 16) ||
      (dsum && !rms_view(dsum, lddsum, C, 16)))
    return rms_fail(OSAM_ERR_INVALID, "rms: null, misaligned (16 bytes) or overlapping rows");
  if (!rms_f32(w) || !rms_f32(rstd)) return rms_fail(OSAM_ERR_INVALID, "rms: w and rstd are 4-byte aligned");
  if (!ws || ws_bytes < osam_rms_bwd_workspace_size(C) || (reinterpret_cast<uintptr_t>(ws) & 15))
    return rms_fail(OSAM_ERR_INVALID, "rms: workspace (osam_rms_bwd_workspace_size, 16-byte aligned)");
  RmsBwd P{};
  P.dy = dy; P.lddy = lddy;
  P.h = h; P.ldh = ldh;
  P.w = w; P.rstd = rstd;
  P.dsum = dsum; P.ldds = lddsum;
  P.dx = dx; P.lddx = lddx;
  P.part = static_cast<float*>(ws);
  P.rows = rows; P.C = C; P.inv_c = 1.f / C;
  return dtype == OSAM_F16 ? launch_rms_bwd<__half>(P, dw, st) : launch_rms_bwd<__nv_bfloat16>(P, dw, st);
}

}  // extern "C"
