// 16-byte vectors of fp32, bf16 or fp16 as pairs of floats, and the packed two-float arithmetic of sm_100.
#pragma once

#include <type_traits>

#include "dtype.cuh"

namespace b200 {

__device__ __forceinline__ float2 splat2(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

// 2^v; results below 2^-126 are 0.
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// max that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
struct Vec16 {
  static constexpr int kElems = 16 / int(sizeof(T));
  static constexpr int kPairs = kElems / 2;
};

__device__ __forceinline__ float2 pair_of(uint32_t u, __nv_bfloat16) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ float2 pair_of(uint32_t u, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
__device__ __forceinline__ uint32_t word_of(float2 f, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t word_of(float2 f, __half) {
  const __half2 p = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&p);
}

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& v, float2 (&f)[Vec16<T>::kPairs]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    f[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  } else {
    f[0] = pair_of(v.x, T{});
    f[1] = pair_of(v.y, T{});
    f[2] = pair_of(v.z, T{});
    f[3] = pair_of(v.w, T{});
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float2 (&f)[Vec16<T>::kPairs]) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x),
                      __float_as_uint(f[1].y));
  else
    return make_uint4(word_of(f[0], T{}), word_of(f[1], T{}), word_of(f[2], T{}), word_of(f[3], T{}));
}

// The largest element of a vector (NaN elements do not count).
template <typename T>
__device__ __forceinline__ float max16(const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else {
    using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const P* p = reinterpret_cast<const P*>(&v);
    const P m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    const float2 f = pair_of(*reinterpret_cast<const uint32_t*>(&m), T{});
    return fmaxf(f.x, f.y);
  }
}

// 16 bytes, read once, from memory that this kernel may write later (not through the read-only path).
__device__ __forceinline__ uint4 ld_once_u4(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ void st_stream_u4(void* p, uint4 v) {
  asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

}  // namespace b200
