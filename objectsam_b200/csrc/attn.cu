// Attention: the C entry points, argument checks and workspace layout, and the small kernels around the two main
// ones (attn_fwd.cuh, attn_bwd.cuh): document summaries, the join of split keys, the backward's row terms.
#include <float.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "attn.cuh"

namespace osam {
namespace {

// Per 64-token block: smallest and largest document id, and whether a token has none.  One warp per block; the
// query blocks first, then the key blocks (`both`: the same array serves as both).
__global__ void __launch_bounds__(256) k_attn_docs(const int* doc_q, const int* doc_k, int B, int Lq, int Lk, AtDocs* sq,
                                                   AtDocs* sk) {
  const int nq = (Lq + kAtDocBlock - 1) / kAtDocBlock, nk = (Lk + kAtDocBlock - 1) / kAtDocBlock;
  const int w = (blockIdx.x * 256 + threadIdx.x) / 32, lane = threadIdx.x % 32;
  grid_dep_wait();
  grid_dep_launch();
  const bool is_q = w < B * nq;
  const int i = is_q ? w : w - B * nq, nb = is_q ? nq : nk, L = is_q ? Lq : Lk;
  if (i >= B * nb) return;
  const int b = i / nb, t0 = (i - b * nb) * kAtDocBlock;
  const int* d = (is_q ? doc_q : doc_k) + (long long)b * L;
  AtDocs s{INT_MAX, -1, 0, 0};
#pragma unroll
  for (int k = 0; k < kAtDocBlock; k += 32) {
    const int t = t0 + k + lane;
    if (t >= L) continue;
    const int id = d[t];
    if (id < 0) {
      s.pad = 1;
    } else {
      s.lo = min(s.lo, id);
      s.hi = max(s.hi, id);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s.lo = min(s.lo, __shfl_xor_sync(0xffffffffu, s.lo, o));
    s.hi = max(s.hi, __shfl_xor_sync(0xffffffffu, s.hi, o));
    s.pad |= __shfl_xor_sync(0xffffffffu, s.pad, o);
  }
  if (lane == 0) (is_q ? sq : sk)[i] = s;
}

// Joins the key splits: o = Σ 2^(m_s − M) o_s / Σ 2^(m_s − M) l_s over the splits.  `W` warps share a row and take
// every W-th split each, four loads in flight; their sums are added in warp order.  (One warp a row took as long for
// 64 splits as the attention in front of it.)
template <typename T>
__global__ void __launch_bounds__(256) k_attn_join(const float* part, const float2* stats, const __grid_constant__ AttnDev A,
                                                   const int* chunk, int W, long long nrows, AtView o, float* lse) {
  __shared__ float4 acc_of[8][32];
  __shared__ float l_of[8];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, w = warp % W;
  const long long row = (long long)blockIdx.x * (8 / W) + warp / W;
  const bool live = row < nrows;
  const int D = A.D;
  const long long bh = row / A.Lq, b = bh / A.Hq;
  grid_dep_wait();
  grid_dep_launch();
  const int splits = live ? at_seq_splits(A, int(b), *chunk) : 0;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f, M = -INFINITY;
  if (live) {
    for (int s = lane; s < splits; s += 32) M = fmaxf(M, stats[s * nrows + row].x);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
    for (int s0 = w; s0 < splits; s0 += 4 * W) {
      float2 st[4];
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int s = s0 + k * W;
        st[k] = s < splits ? stats[s * nrows + row] : make_float2(0.f, 0.f);
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (s < splits && lane * 4 < D) v[k] = *reinterpret_cast<const float4*>(part + (s * nrows + row) * D + lane * 4);
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if (st[k].y == 0.f) continue;  // no key in this split
        const float f = at_ex2(st[k].x - M);
        l = fmaf(f, st[k].y, l);
        acc.x = fmaf(f, v[k].x, acc.x);
        acc.y = fmaf(f, v[k].y, acc.y);
        acc.z = fmaf(f, v[k].z, acc.z);
        acc.w = fmaf(f, v[k].w, acc.w);
      }
    }
  }
  if (W > 1) {
    acc_of[warp][lane] = acc;
    if (lane == 0) l_of[warp] = l;
    __syncthreads();
    if (w != 0) return;
    for (int i = 1; i < W; i++) {
      const float4 a = acc_of[warp + i][lane];
      acc.x += a.x;
      acc.y += a.y;
      acc.z += a.z;
      acc.w += a.w;
      l += l_of[warp + i];
    }
  }
  if (!live) return;
  const int i = int(row - bh * A.Lq), h = int(bh % A.Hq);
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  if (lane * 4 < D) {
    T* p = static_cast<T*>(o.p) + b * o.sb + i * o.st + h * o.sh + lane * 4;
    *reinterpret_cast<uint2*>(p) =
        make_uint2(Half16<T>::pack(acc.x * inv, acc.y * inv), Half16<T>::pack(acc.z * inv, acc.w * inv));
  }
  if (lane == 0 && lse) lse[row] = l == 0.f ? -INFINITY : (M + at_lg2(l)) * kAtLn2;
}

// Adds the parts of one gradient in part order and rounds: a thread per 8 dims of a (batch, head, token) row.
template <typename T>
__global__ void __launch_bounds__(256) k_attn_sum(const float* part, int parts, long long stride, int heads, int L, int D,
                                                  long long n8, AtView out) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  grid_dep_wait();
  grid_dep_launch();
  if (i >= n8) return;
  float v[8] = {};
  for (int p = 0; p < parts; p++) {
    const float4* s = reinterpret_cast<const float4*>(part + p * stride + i * 8);
    const float4 a = s[0], b = s[1];
    v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
    v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
  }
  const int c8 = D / 8;
  const long long row = i / c8, bh = row / L;
  const int c = int(i - row * c8) * 8, t = int(row - bh * L), h = int(bh % heads);
  *reinterpret_cast<uint4*>(static_cast<T*>(out.p) + bh / heads * out.sb + t * out.st + h * out.sh + c) = pack8<T>(v);
}

// Row terms of the backward pass, per 64-query block (padded to whole blocks): (u − lse·log2 e, −δ), δ = do·o, u = log2
// of the factor that the backward holds P times — (−∞, 0) for queries that see nothing and for the padding, whose P is
// then 0 — and for fp16 the block's largest ‖dO_i‖ and, in CTAs behind the query blocks', the largest ‖v_j‖ of each
// 64-key block, over rows that are finite (another one's gradients are not finite whatever dS is held times) and keys in
// use.  One CTA per block, 16 lanes per row (a 16-byte vector each); eight CTAs an SM at 32 registers, a few spilled (2 × 4096
// tokens, 16 heads × 128: 17 us, with 38 registers 20; 8 × 1600, 4 × 64, fp16: 12 and 14).
template <typename T>
__global__ void __launch_bounds__(256, 8) k_attn_rows(const __grid_constant__ AttnDev A, const AtView o, const AtView dout,
                                                   const AtView v, const float* lse, float* rows, float* peak, float* vpeak,
                                                   AtDocs* sum_q) {
  __shared__ float top[8];
  constexpr bool BF16 = Half16<T>::kBf16;
  constexpr float up = BF16 ? 0.f : kAbUp;
  const int nq = (A.Lq + kAbCols - 1) / kAbCols, nk = (A.Lk + kAbCols - 1) / kAbCols;
  const int c = threadIdx.x % 16, D = A.D;
  const bool keys = !BF16 && (int)blockIdx.x >= nq * A.Hq * A.B;
  const int at = keys ? blockIdx.x - nq * A.Hq * A.B : blockIdx.x, nb = keys ? nk : nq, heads = keys ? A.Hk : A.Hq;
  const int blk = at % nb, h = (at / nb) % heads, b = at / nb / heads;
  const long long bh = (long long)b * heads + h;
  grid_dep_wait();
  grid_dep_launch();
  float big = 0.f;     // largest ‖·‖²
  bool blind = false;  // a query that sees nothing: the same in all heads
  auto norm2 = [](const float (&g)[8]) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) s = fmaf(g[e], g[e], s);
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    return s <= FLT_MAX ? s : 0.f;  // neither infinite nor NaN
  };
  if (keys) {
    const int n = at_keys(A, b);
    int id[kAbCols / 16];
    uint4 u[kAbCols / 16];
#pragma unroll
    for (int k = 0; k < kAbCols / 16; k++) {  // all loads first
      const int i = blk * kAbCols + k * 16 + threadIdx.x / 16;
      id[k] = i < n ? (A.doc_k ? A.doc_k[(long long)b * A.Lk + i] : 0) : -1;
      u[k] = make_uint4(0, 0, 0, 0);
      if (i < n && c * 8 < D) u[k] = *reinterpret_cast<const uint4*>(static_cast<const T*>(v.p) + b * v.sb + i * v.st + h * v.sh + c * 8);
    }
#pragma unroll
    for (int k = 0; k < kAbCols / 16; k++) {
      float g[8];
      unpack8<T>(u[k], g);
      const float s = norm2(g);
      if (id[k] >= 0) big = fmaxf(big, s);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kAbCols; k += 16) {
      const int r = k + threadIdx.x / 16, i = blk * kAbCols + r;
      const float L = i < A.Lq ? lse[bh * A.Lq + i] : -INFINITY;
      const bool live = L != -INFINITY;
      blind |= i < A.Lq && !live;
      float a[8] = {}, g[8] = {};
      if (live && c * 8 < D) {
        unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(o.p) + b * o.sb + i * o.st + h * o.sh + c * 8), a);
        unpack8<T>(
            *reinterpret_cast<const uint4*>(static_cast<const T*>(dout.p) + b * dout.sb + i * dout.st + h * dout.sh + c * 8), g);
      }
      float d = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) d = fmaf(a[e], g[e], d);
#pragma unroll
      for (int s = 8; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
      if (!BF16) big = fmaxf(big, norm2(g));
      if (c == 0) {
        float* out = rows + (bh * nb + blk) * 2 * kAbCols + r;
        out[0] = live ? up - L * kAtLog2e : -INFINITY;
        out[kAbCols] = live ? -d : 0.f;
      }
    }
  }
  if (sum_q && h == 0 && blind && c == 0) sum_q[(long long)b * nq + blk].pad = 1;
  if (BF16) return;
  big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 16));
  if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = big;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; w++) big = fmaxf(big, top[w]);
    (keys ? vpeak : peak)[bh * nb + blk] = sqrtf(big);
  }
}

int at_fail(int code, const char* what) {
  set_last_error("attention: %s", what);
  return code;
}
int at_cuda(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return OSAM_OK;
  set_last_error("attention: %s: %s", what, cudaGetErrorString(e));
  return OSAM_ERR_CUDA;
}

bool at_misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) & 3; }

int at_check(const osam_attn_desc* a) {
  if (!a) return at_fail(OSAM_ERR_INVALID, "null description");
  if (a->dtype != OSAM_F16 && a->dtype != OSAM_BF16) return at_fail(OSAM_ERR_INVALID, "dtype is OSAM_F16 or OSAM_BF16");
  if (a->batch < 0 || a->len_q < 0 || a->len_k < 0 || a->heads_q < 1 || a->heads_k < 1 || a->heads_q % a->heads_k)
    return at_fail(OSAM_ERR_INVALID, "lengths ≥ 0 and heads_q a multiple of heads_k");
  if (a->dim < 8 || a->dim > 128 || a->dim % 8) return at_fail(OSAM_ERR_INVALID, "dim is a multiple of 8 up to 128");
  if (!(a->scale > 0.f) || std::isinf(a->scale)) return at_fail(OSAM_ERR_INVALID, "scale is positive and finite");
  if (!(a->cap >= 0.f) || std::isinf(a->cap)) return at_fail(OSAM_ERR_INVALID, "cap is 0 or positive and finite");
  if (a->cap > 0.f && std::isinf(2.f * a->scale * kAtLog2e / a->cap))  // a score of 0 would be 0·∞
    return at_fail(OSAM_ERR_INVALID, "cap is too small beside the scale");
  if (a->mask != OSAM_ATTN_NONE && a->mask != OSAM_ATTN_CAUSAL && a->mask != OSAM_ATTN_PREFIX)
    return at_fail(OSAM_ERR_INVALID, "unknown mask");
  if (a->mask == OSAM_ATTN_PREFIX && !a->prefix) return at_fail(OSAM_ERR_INVALID, "a prefix mask needs prefix lengths");
  if ((a->doc_q == nullptr) != (a->doc_k == nullptr)) return at_fail(OSAM_ERR_INVALID, "doc_q and doc_k come together");
  if (at_misaligned(a->slopes) || at_misaligned(a->lens) || at_misaligned(a->prefix) || at_misaligned(a->doc_q) ||
      at_misaligned(a->doc_k))
    return at_fail(OSAM_ERR_INVALID, "slopes, lens, prefix and documents are 4-byte aligned");
  if (a->grid_w < 0) return at_fail(OSAM_ERR_INVALID, "grid_w is not negative");
  // in doubles: exact up to here, and products of any descriptions stay in range
  const double most = 1 << 30, B = a->batch, q64 = std::ceil(a->len_q / 64.), k64 = std::ceil(a->len_k / 64.);
  if ((double)a->len_q * (a->heads_q / a->heads_k) > most || a->len_k > most || B * a->heads_q * q64 > most ||
      B * a->heads_k * k64 > most)
    return at_fail(OSAM_ERR_INVALID, "too many tokens");
  if (a->grid_w > most) return at_fail(OSAM_ERR_INVALID, "grid_w is at most 2^30");
  if (a->doc_q && (a->len_q > 1048576 || a->len_k > 1048576))
    return at_fail(OSAM_ERR_INVALID, "with documents at most 1048576 tokens");
  return OSAM_OK;
}

int at_view_check(const osam_view& v, int batch, int len, int heads, const char* name) {
  if (!v.p || (reinterpret_cast<uintptr_t>(v.p) & 15)) {
    set_last_error("attention: %s is null or not 16-byte aligned", name);
    return OSAM_ERR_INVALID;
  }
  const int64_t s[3] = {v.sb, v.st, v.sh};
  const int n[3] = {batch, len, heads};
  for (int i = 0; i < 3; i++)
    if (n[i] > 1 && (s[i] <= 0 || s[i] % 8 || s[i] >= (1LL << 38))) {
      set_last_error("attention: %s has a stride that is not a positive multiple of 8 elements", name);
      return OSAM_ERR_INVALID;
    }
  return OSAM_OK;
}

AtView at_view(const osam_view& v) { return AtView{v.p, v.sb, v.st, v.sh}; }

// (dim, token, head, batch) map with boxes of 64 dims × `rows` tokens.
int at_map(CUtensorMap* tm, const osam_view& v, int batch, int len, int heads, int dim, int rows, bool bf16) {
  const uint64_t dims[4] = {(uint64_t)dim, (uint64_t)len, (uint64_t)heads, (uint64_t)batch};
  const uint64_t st[3] = {len > 1 ? (uint64_t)v.st * 2 : 16, heads > 1 ? (uint64_t)v.sh * 2 : 16,
                          batch > 1 ? (uint64_t)v.sb * 2 : 16};
  const uint32_t box[4] = {64, (uint32_t)rows, 1, 1};
  return make_map(tm, v.p, 4, dims, st, box, 128, bf16);
}

// How the keys are split.  Nothing is gained once the query tiles fill the GPU's places; below, the kernel takes the
// splits' size from the sequences' lengths (at_best_chunk) and only their bounds are set here: 256 keys at least, 512 over
// long caches (one sequence, 4 heads, 32768 keys: 16 us, with 256 keys 21), and the CTAs that fill kAfRounds rounds.
// The join costs a launch: a cache of 517 keys takes 11 us whole and 15 in two, one of 860 keys 21 and 15.
struct AtSplit {
  int splits, min_tiles, grid, usual;  // at most, …, CTAs, splits of a sequence with all CTAs in use
  int chunk;  // where every sequence has len_k keys
};
AtSplit at_split(const osam_attn_desc& a) {
  const int tiles = (a.len_k + kAfKeys - 1) / kAfKeys;
  const long long per = ((long long)a.len_q * (a.heads_q / a.heads_k) + kAfRows - 1) / kAfRows * a.heads_k;
  const long long ctas = per * a.batch;
  AtSplit s{1, std::max(tiles, 1), (int)ctas, 1, tiles};
  if (ctas == 0 || a.len_k < 768 || ctas >= kAfPlaces) return s;
  s.min_tiles = a.len_k <= 2048 ? 4 : 8;
  const int most = (tiles + s.min_tiles - 1) / s.min_tiles;
  s.splits = std::min(most, (int)(kAfRounds * kAfPlaces / per) - (a.batch - 1));
  s.grid = (int)std::min<long long>(kAfRounds * kAfPlaces / per * per, ctas * most);
  s.usual = (s.grid + (int)ctas - 1) / (int)ctas;
  s.chunk = at_best_chunk(a.batch, (int)per, s.min_tiles, tiles, a.batch * tiles,
                          [&](int chunk) { return a.batch * ((tiles + chunk - 1) / chunk); });
  return s;
}

// Units of a group (at_order), `bytes` being what one streams: without a bound one; with it all while that stays near
// L2's size (the last group's longest tiles start late: 64 heads of 4096 × 64 in two groups 308 us instead of 277);
// beyond, half of L2 (512 heads of 4096 × 64: 2016 us, with a quarter 2097), but three rounds of the GPU's places at
// least.  512 heads of 4096 × 128: forward 3189 us in one group, 2418 in groups, backward 9121 and 7684.
int at_group(const osam_attn_desc& a, long long tiles, long long units, double bytes) {
  if (a.mask == OSAM_ATTN_NONE) return 1;
  if (bytes * units <= 192e6) return (int)std::max(units, 1LL);
  return (int)std::min(units, std::max((long long)(64e6 / bytes), 3 * kAfPlaces / std::max(tiles, 1LL) + 1));
}

// Into how many parts the backward splits the streamed side of a tile: by a model of its time in units of a streamed
// tile (0.7 us measured): rounds of CTAs over the GPU × (tiles of a part + 5 for a CTA's start and end), and for the
// parts' sum 8 and its traffic.  One part where the tiles fill the GPU (16 heads of 4096 tokens); with 2 key heads of
// 8192 tokens (128 tiles for 296 places) two parts took the whole backward from 907 to 675 us.
int at_parts(const osam_attn_desc& a, bool dkv) {
  const int slots = kAtSms * (a.dim <= 64 ? 2 : 1), own = dkv ? a.len_k : a.len_q, other = dkv ? a.len_q : a.len_k;
  const int heads = dkv ? a.heads_k : a.heads_q;
  const double ctas = (double)((own + 127) / 128) * a.batch * heads;
  const double tiles = (double)((other + 63) / 64) * (dkv ? a.heads_q / a.heads_k : 1) * (a.mask == OSAM_ATTN_NONE ? 1 : 0.5);
  const double out_us = (double)own * a.batch * heads * a.dim * (dkv ? 2 : 1) * 8 / 4e6;
  int best = 1;
  double least = 1e30;
  for (int p = 1; p <= 8 && (p == 1 || (other + 63) / 64 >= 4 * p); p++) {
    const double t = std::ceil(ctas * p / slots) * (tiles / p + 5) + (p > 1 ? 8 + p * out_us / 0.7 : 0);
    if (t < least) {
      least = t;
      best = p;
    }
  }
  return best;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Workspace: document summaries | split outputs and statistics (forward) or row terms (backward).
struct AtLayout {
  size_t sum_q = 0, sum_k = 0, part = 0, stats = 0, chunk = 0, rows = 0, peak = 0, vpeak = 0, grad = 0, bytes = 0;
};
AtLayout at_layout(const osam_attn_desc& a) {
  AtLayout L;
  size_t at = 0;
  if (a.doc_q) {
    L.sum_q = at;
    at += up256((size_t)a.batch * ((a.len_q + 63) / 64) * sizeof(AtDocs));
    L.sum_k = at;
    at += up256((size_t)a.batch * ((a.len_k + 63) / 64) * sizeof(AtDocs));
  }
  const size_t rows = (size_t)a.batch * a.heads_q * a.len_q;
  const AtSplit s = at_split(a);
  L.part = L.rows = at;
  size_t fwd = at;
  if (s.splits > 1) {
    fwd += up256(rows * s.splits * a.dim * sizeof(float));
    L.stats = fwd;
    fwd += up256(rows * s.splits * sizeof(float2));
    L.chunk = fwd;
    fwd += 256;
  }
  const size_t blocks = (size_t)a.batch * a.heads_q * ((a.len_q + kAbCols - 1) / kAbCols);
  L.peak = at + up256(blocks * 2 * kAbCols * sizeof(float));
  L.vpeak = L.peak + up256(blocks * sizeof(float));
  L.grad = L.vpeak + up256((size_t)a.batch * a.heads_k * ((a.len_k + kAbCols - 1) / kAbCols) * sizeof(float));
  const int pk = at_parts(a, true), pq = at_parts(a, false);
  const size_t nk = (size_t)a.batch * a.heads_k * a.len_k * a.dim, nq = rows * a.dim;
  const size_t grad = std::max(pk > 1 ? pk * 2 * nk : 0, pq > 1 ? pq * nq : 0) * sizeof(float);
  L.bytes = std::max(fwd, L.grad + up256(grad));
  return L;
}

int at_dev(const osam_attn_desc& a, const AtLayout& W, char* ws, AttnDev* A, cudaStream_t st) {
  A->B = a.batch; A->Lq = a.len_q; A->Lk = a.len_k; A->Hq = a.heads_q; A->Hk = a.heads_k;
  A->G = a.heads_q / a.heads_k; A->D = a.dim;
  A->mask = a.mask; A->scale = a.scale; A->cap = a.cap;
  A->grid_w = a.grid_w;
  A->f_g.set(A->G);
  A->f_w.set(a.grid_w);
  A->lens = a.lens; A->prefix = a.prefix; A->doc_q = a.doc_q; A->doc_k = a.doc_k; A->slopes = a.slopes;
  A->err = device_error_word();
  if (!A->err) return at_fail(OSAM_ERR_CUDA, "no device error word");
  if (a.doc_q) {
    AtDocs* sq = reinterpret_cast<AtDocs*>(ws + W.sum_q);
    AtDocs* sk = reinterpret_cast<AtDocs*>(ws + W.sum_k);
    A->sum_q = sq;
    A->sum_k = sk;
    const long long warps = (long long)a.batch * ((a.len_q + 63) / 64 + (a.len_k + 63) / 64);
    return at_cuda(launch_dependent(k_attn_docs, (unsigned)((warps + 7) / 8), 256, 0, st, a.doc_q, a.doc_k, a.batch, a.len_q,
                                    a.len_k, sq, sk),
                   "document summaries");
  }
  return OSAM_OK;
}

}  // namespace
}  // namespace osam

using namespace osam;

extern "C" {

size_t osam_attn_workspace_size(const osam_attn_desc* a) { return at_check(a) == OSAM_OK ? at_layout(*a).bytes : 0; }

int osam_attn_fwd(const osam_attn_desc* a, osam_view q, osam_view k, osam_view v, osam_view o, float* lse, void* ws,
                  size_t ws_bytes, osam_stream_t stream) {
  int rc = at_check(a);
  if (rc != OSAM_OK) return rc;
  if (a->batch == 0 || a->len_q == 0) return OSAM_OK;
  if ((rc = at_view_check(q, a->batch, a->len_q, a->heads_q, "q")) != OSAM_OK ||
      (rc = at_view_check(o, a->batch, a->len_q, a->heads_q, "o")) != OSAM_OK)
    return rc;
  if (at_misaligned(lse)) return at_fail(OSAM_ERR_INVALID, "lse is 4-byte aligned");
  if (a->len_k > 0 && ((rc = at_view_check(k, a->batch, a->len_k, a->heads_k, "k")) != OSAM_OK ||
                       (rc = at_view_check(v, a->batch, a->len_k, a->heads_k, "v")) != OSAM_OK))
    return rc;
  const AtLayout W = at_layout(*a);
  if (W.bytes && (!ws || ws_bytes < W.bytes || (reinterpret_cast<uintptr_t>(ws) & 255)))
    return at_fail(OSAM_ERR_INVALID, "workspace (osam_attn_workspace_size, 256-byte aligned)");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  char* w = static_cast<char*>(ws);
  const AtSplit s = at_split(*a);
  AttnFwdLaunch L{};
  if ((rc = at_dev(*a, W, w, &L.d, st)) != OSAM_OK) return rc;
  const bool bf16 = a->dtype == OSAM_BF16;
  // without keys every query is empty: no tile is visited, so the maps only have to be valid
  const osam_view& kk = a->len_k > 0 ? k : q;
  const osam_view& vv = a->len_k > 0 ? v : q;
  if ((rc = at_map(&L.tk, kk, a->batch, std::max(a->len_k, 1), a->heads_k, a->dim, kAfKeys, bf16)) != OSAM_OK ||
      (rc = at_map(&L.tv, vv, a->batch, std::max(a->len_k, 1), a->heads_k, a->dim, kAfKeys, bf16)) != OSAM_OK)
    return rc;
  L.q = at_view(q);
  L.o = at_view(o);
  L.lse = lse;
  L.splits = s.splits;
  L.min_tiles = s.min_tiles;
  L.grid = s.grid;
  const int g = a->heads_q / a->heads_k;
  L.group = at_group(*a, ((long long)a->len_q * g + kAfRows - 1) / kAfRows, (long long)a->batch * a->heads_k, 4.0 * a->len_k * a->dim);
  L.chunk_all = s.chunk;
  L.chunk = reinterpret_cast<int*>(w + W.chunk);
  L.part = reinterpret_cast<float*>(w + W.part);
  L.stats = reinterpret_cast<float2*>(w + W.stats);
  cudaError_t e = bf16 ? launch_attn_fwd<__nv_bfloat16>(L, st) : launch_attn_fwd<__half>(L, st);
  if (e != cudaSuccess || s.splits == 1) return at_cuda(e, "forward launch");
  const long long nrows = (long long)a->batch * a->heads_q * a->len_q;
  const int warps = s.usual <= 4 ? 1 : s.usual <= 16 ? 4 : 8;
  const unsigned grid = (unsigned)((nrows + 8 / warps - 1) / (8 / warps));
  e = launch_dependent(bf16 ? k_attn_join<__nv_bfloat16> : k_attn_join<__half>, grid, 256, 0, st, (const float*)L.part,
                       (const float2*)L.stats, L.d, (const int*)L.chunk, warps, nrows, L.o, lse);
  return at_cuda(e, "join launch");
}

int osam_attn_bwd(const osam_attn_desc* a, osam_view q, osam_view k, osam_view v, osam_view o, const float* lse,
                  osam_view dout, osam_view dq, osam_view dk, osam_view dv, void* ws, size_t ws_bytes,
                  osam_stream_t stream) {
  int rc = at_check(a);
  if (rc != OSAM_OK) return rc;
  if (a->batch == 0 || (a->len_q == 0 && a->len_k == 0)) return OSAM_OK;
  if (a->len_q > 0) {
    const osam_view* t[] = {&q, &o, &dout, &dq};
    const char* name[] = {"q", "o", "dout", "dq"};
    for (int i = 0; i < 4; i++)
      if ((rc = at_view_check(*t[i], a->batch, a->len_q, a->heads_q, name[i])) != OSAM_OK) return rc;
    if (!lse || at_misaligned(lse)) return at_fail(OSAM_ERR_INVALID, "the backward pass needs the forward's lse, 4-byte aligned");
  }
  if (a->len_k > 0) {
    const osam_view* t[] = {&k, &v, &dk, &dv};
    const char* name[] = {"k", "v", "dk", "dv"};
    for (int i = 0; i < 4; i++)
      if ((rc = at_view_check(*t[i], a->batch, a->len_k, a->heads_k, name[i])) != OSAM_OK) return rc;
  }
  const AtLayout W = at_layout(*a);
  if (W.bytes && (!ws || ws_bytes < W.bytes || (reinterpret_cast<uintptr_t>(ws) & 255)))
    return at_fail(OSAM_ERR_INVALID, "workspace (osam_attn_workspace_size, 256-byte aligned)");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  char* w = static_cast<char*>(ws);
  const bool bf16 = a->dtype == OSAM_BF16;
  AttnBwdLaunch L{};
  if ((rc = at_dev(*a, W, w, &L.d, st)) != OSAM_OK) return rc;
  float* rows = reinterpret_cast<float*>(w + W.rows);
  float* peak = reinterpret_cast<float*>(w + W.peak);
  float* vpeak = reinterpret_cast<float*>(w + W.vpeak);
  const int blocks = a->batch * a->heads_q * ((a->len_q + kAbCols - 1) / kAbCols);
  if (blocks > 0) {
    const unsigned grid = blocks + (bf16 ? 0u : (unsigned)a->batch * a->heads_k * ((a->len_k + kAbCols - 1) / kAbCols));
    if ((rc = at_cuda(launch_dependent(bf16 ? k_attn_rows<__nv_bfloat16> : k_attn_rows<__half>, grid, 256, 0, st, L.d, at_view(o),
                                       at_view(dout), at_view(v), lse, rows, peak, vpeak,
                                       a->doc_q ? reinterpret_cast<AtDocs*>(w + W.sum_q) : (AtDocs*)nullptr),
                      "row terms")) != OSAM_OK)
      return rc;
  }
  L.rows = rows;
  L.peak = peak;
  L.vpeak = vpeak;
  // a side of length 0 is never visited: its maps only have to be valid
  const bool eq = a->len_q == 0, ek = a->len_k == 0;
  const osam_view &vq = eq ? k : q, &vdo = eq ? k : dout, &vk = ek ? q : k, &vv = ek ? q : v;
  const int lq = eq ? 1 : a->len_q, lk = ek ? 1 : a->len_k, hq = eq ? a->heads_k : a->heads_q;
  auto map = [&](CUtensorMap* m, const osam_view& t, bool query, int box) {
    return at_map(m, t, a->batch, query ? lq : lk, query ? hq : a->heads_k, a->dim, box, bf16);
  };
  L.part = reinterpret_cast<float*>(w + W.grad);
  auto sum = [&](const osam_view& out, int which, int outs, int heads, int len) {
    const long long n8 = (long long)a->batch * heads * len * (a->dim / 8);
    return at_cuda(launch_dependent(bf16 ? k_attn_sum<__nv_bfloat16> : k_attn_sum<__half>, (unsigned)((n8 + 255) / 256), 256, 0,
                                    st, (const float*)(L.part + which * n8 * 8), L.parts, n8 * 8 * outs, heads, len, a->dim, n8,
                                    at_view(out)),
                   "sum launch");
  };
  const int g = a->heads_q / a->heads_k;
  const auto ctas = [&](bool dkv) {
    return (double)(((dkv ? a->len_k : a->len_q) + kAbRows - 1) / kAbRows) * a->batch * (dkv ? a->heads_k : a->heads_q) *
           at_parts(*a, dkv);
  };
  const double nkv = ctas(true), nq = ctas(false);
  if (!ek) {
    L.alone = nkv + std::ceil(nq / 2) <= kAtSms;  // the longer pass; dQ's CTAs then have the other SMs, two each
    L.parts = at_parts(*a, true);
    L.group = at_group(*a, (a->len_k + kAbRows - 1) / kAbRows, (long long)a->batch * a->heads_k * L.parts,
                       4.0 * a->len_q * a->dim * g / L.parts);
    if ((rc = map(&L.stat1, vk, false, kAbRows)) != OSAM_OK || (rc = map(&L.stat2, vv, false, kAbRows)) != OSAM_OK ||
        (rc = map(&L.strm1, vq, true, kAbCols)) != OSAM_OK || (rc = map(&L.strm2, vdo, true, kAbCols)) != OSAM_OK)
      return rc;
    L.out1 = at_view(dk);
    L.out2 = at_view(dv);
    const cudaError_t e = bf16 ? launch_attn_bwd<__nv_bfloat16, true>(L, st) : launch_attn_bwd<__half, true>(L, st);
    if (e != cudaSuccess) return at_cuda(e, "backward launch (dK, dV)");
    if (L.parts > 1 && ((rc = sum(dk, 0, 2, a->heads_k, a->len_k)) != OSAM_OK || (rc = sum(dv, 1, 2, a->heads_k, a->len_k)) != OSAM_OK))
      return rc;
  }
  if (!eq) {
    L.alone = nkv + nq <= kAtSms;
    L.parts = at_parts(*a, false);
    L.group = at_group(*a, (a->len_q + kAbRows - 1) / kAbRows, (long long)a->batch * a->heads_q * L.parts,
                       4.0 * a->len_k * a->dim / g / L.parts);
    L.late = !ek && L.parts == 1;  // its own parts would go over those that a sum in front still reads
    if ((rc = map(&L.stat1, vq, true, kAbRows)) != OSAM_OK || (rc = map(&L.stat2, vdo, true, kAbRows)) != OSAM_OK ||
        (rc = map(&L.strm1, vk, false, kAbCols)) != OSAM_OK || (rc = map(&L.strm2, vv, false, kAbCols)) != OSAM_OK)
      return rc;
    L.out1 = at_view(dq);
    const cudaError_t e = bf16 ? launch_attn_bwd<__nv_bfloat16, false>(L, st) : launch_attn_bwd<__half, false>(L, st);
    if (e != cudaSuccess) return at_cuda(e, "backward launch (dQ)");
    if (L.parts > 1) return sum(dq, 0, 1, a->heads_q, a->len_q);
  }
  return OSAM_OK;
}

}  // extern "C"
