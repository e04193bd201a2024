// 16-bit storage types of the token operators: conversions of eight values at a time (one 16-byte vector) and
// pairwise packing, for fp16 and bf16.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace osam {

template <typename T>
struct Half16;

template <>
struct Half16<__half> {
  static constexpr bool kBf16 = false;
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  // as pack, with what lies outside fp16's range at its ends (a NaN stays one)
  static __device__ __forceinline__ uint32_t pack_sat(float a, float b) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
};

template <>
struct Half16<__nv_bfloat16> {
  static constexpr bool kBf16 = true;
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t pack_sat(float a, float b) { return pack(a, b); }
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&o)[8]) {
  const float2 a = Half16<T>::unpack(u.x), b = Half16<T>::unpack(u.y), c = Half16<T>::unpack(u.z),
               d = Half16<T>::unpack(u.w);
  o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
  o[4] = c.x; o[5] = c.y; o[6] = d.x; o[7] = d.y;
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(Half16<T>::pack(v[0], v[1]), Half16<T>::pack(v[2], v[3]), Half16<T>::pack(v[4], v[5]),
                    Half16<T>::pack(v[6], v[7]));
}

}  // namespace osam
