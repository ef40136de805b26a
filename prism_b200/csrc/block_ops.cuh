// Element types and reductions shared by the norm, rotary and clipping kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "prism_common.cuh"

namespace prism {

template <typename T> struct Elem;
template <> struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Elem<__half> {
  static __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
};
template <> struct Elem<float> {
  static __device__ __forceinline__ float to_f(float v) { return v; }
  static __device__ __forceinline__ float from_f(float v) { return v; }
};

// A 16-byte vector of elements as fp32 values, and back (round to nearest even).
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[16 / sizeof(T)]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(u[i]);
    } else if constexpr (std::is_same_v<T, __half>) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    } else {
      f[2 * i] = __uint_as_float(u[i] << 16), f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&f)[16 / sizeof(T)]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      u[i] = __float_as_uint(f[i]);
    } else if constexpr (std::is_same_v<T, __half>) {
      const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&p);
    } else {
      const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ bool is_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Calls fn with a null pointer of the element type that `dtype` names; false if none does.
template <typename F>
inline bool dispatch_dtype(int dtype, F&& fn) {
  switch (dtype) {
    case PRISM_BF16: fn(static_cast<__nv_bfloat16*>(nullptr)); return true;
    case PRISM_FP16: fn(static_cast<__half*>(nullptr)); return true;
    case PRISM_FP32: fn(static_cast<float*>(nullptr)); return true;
    default: return false;
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace prism
