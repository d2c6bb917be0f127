// Element types of the tensors that come from a model (fp32, bf16 or fp16), loaded into and rounded
// from fp32, in which all arithmetic is done.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "b200_common.cuh"

namespace b200 {

enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };  // B200_F32, B200_BF16, B200_F16

inline bool dtype_ok(int d) { return d == kF32 || d == kBF16 || d == kF16; }
inline int dtype_size(int d) { return d == kF32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// One rounding, to nearest even.
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Calls f(T{}) with the C++ type of a dtype code.
template <typename F>
inline int with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case kF32: return f(float{});
    case kBF16: return f(__nv_bfloat16{});
    case kF16: return f(__half{});
    default: return kInvalidArgument;
  }
}

}  // namespace b200
