// Rotary positions: the factor of a pair, and the rotation of vectors of a head's elements.
#pragma once
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "block_ops.cuh"

namespace prism {
namespace rotary {

__device__ __forceinline__ float2 cos_sin(double pos, double freq, float scale, float sign) {
  constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
  double t = pos * (freq * kTurn);
  t -= rint(t);
  float s, c;
  sincospif(2.0f * (float)t, &s, &c);
  return make_float2(c * scale, s * scale * sign);
}

// kVec elements of T as one load, and as fp32.
template <typename T, int kVec>
struct Vec {
  static constexpr int kBytes = kVec * (int)sizeof(T);
  using Raw = std::conditional_t<kBytes == 16, uint4,
                                 std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 4, uint32_t, uint16_t>>>;
  static __device__ __forceinline__ void word(uint32_t u, float* f) {
    if constexpr (sizeof(T) == 4) {
      f[0] = __uint_as_float(u);
    } else if constexpr (std::is_same_v<T, __half>) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u));
      f[0] = p.x, f[1] = p.y;
    } else {
      f[0] = __uint_as_float(u << 16), f[1] = __uint_as_float(u & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint32_t word(const float* f) {
    if constexpr (sizeof(T) == 4) {
      return __float_as_uint(f[0]);
    } else if constexpr (std::is_same_v<T, __half>) {
      const __half2 p = __floats2half2_rn(f[0], f[1]);
      return *reinterpret_cast<const uint32_t*>(&p);
    } else {
      const __nv_bfloat162 p = __floats2bfloat162_rn(f[0], f[1]);
      return *reinterpret_cast<const uint32_t*>(&p);
    }
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[kVec]) {
    constexpr int kStep = 4 / (int)sizeof(T);
    if constexpr (kBytes == 16) {
      word(r.x, f), word(r.y, f + kStep), word(r.z, f + 2 * kStep), word(r.w, f + 3 * kStep);
    } else if constexpr (kBytes == 8) {
      word(r.x, f), word(r.y, f + kStep);
    } else if constexpr (kBytes == 4) {
      word(r, f);
    } else {
      f[0] = Elem<T>::to_f(*reinterpret_cast<const T*>(&r));
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[kVec]) {
    constexpr int kStep = 4 / (int)sizeof(T);
    if constexpr (kBytes == 16) {
      return make_uint4(word(f), word(f + kStep), word(f + 2 * kStep), word(f + 3 * kStep));
    } else if constexpr (kBytes == 8) {
      return make_uint2(word(f), word(f + kStep));
    } else if constexpr (kBytes == 4) {
      return word(f);
    } else {
      const T v = Elem<T>::from_f(f[0]);
      return *reinterpret_cast<const Raw*>(&v);
    }
  }
};

// One unit: the pairs' factors are at f.
template <typename T, int kVec, bool kAdjacent>
struct Unit {
  using V = Vec<T, kVec>;
  using Raw = typename V::Raw;
  static constexpr int kPairs = kAdjacent ? kVec / 2 : kVec;
  Raw lo, hi;
  __device__ __forceinline__ void load(const T* p, bool turn, int apart) {
    lo = *reinterpret_cast<const Raw*>(p);
    if constexpr (!kAdjacent) {
      if (turn) hi = *reinterpret_cast<const Raw*>(p + apart);
    }
  }
  __device__ __forceinline__ void copy(T* p) const { *reinterpret_cast<Raw*>(p) = lo; }
  __device__ __forceinline__ void turn(T* p, int apart, const float2* f) const {
    if constexpr (kAdjacent) {
      float x[kVec];
      V::unpack(lo, x);
#pragma unroll
      for (int e = 0; e < kVec; e += 2) {
        const float2 cs = f[e / 2];
        const float a = x[e], d = x[e + 1];
        x[e] = a * cs.x - d * cs.y;
        x[e + 1] = a * cs.y + d * cs.x;
      }
      *reinterpret_cast<Raw*>(p) = V::pack(x);
    } else {
      float x[kVec], y[kVec];
      V::unpack(lo, x);
      V::unpack(hi, y);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float2 cs = f[e];
        const float a = x[e];
        x[e] = a * cs.x - y[e] * cs.y;
        y[e] = a * cs.y + y[e] * cs.x;
      }
      *reinterpret_cast<Raw*>(p) = V::pack(x);
      *reinterpret_cast<Raw*>(p + apart) = V::pack(y);
    }
  }
};

}  // namespace rotary
}  // namespace prism
