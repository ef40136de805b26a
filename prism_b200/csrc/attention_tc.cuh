// Pieces that the tensor-core attention kernels share: rows of scores between TMEM and
// registers, their maximum, and the rescaling of accumulators in TMEM.
#pragma once
#include <stdint.h>

#include "sm100.cuh"

namespace prism {
namespace tc {

using namespace sm100;

__device__ __forceinline__ uint8_t* align1024(uint8_t* p) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~(uintptr_t)1023);
}

__device__ __forceinline__ float u2f(uint32_t x) { return __uint_as_float(x); }

// 32 * N consecutive TMEM columns of this warp's 32 lanes -> registers (waited).
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t taddr, float (&out)[32 * N]) {
  uint32_t raw[N][32];
#pragma unroll
  for (int c = 0; c < N; ++c) tmem_ld32(taddr + c * 32, raw[c]);
#pragma unroll
  for (int c = 0; c < N; ++c) tmem_wait_ld_dep(raw[c]);
#pragma unroll
  for (int c = 0; c < N; ++c)
#pragma unroll
    for (int i = 0; i < 32; ++i) out[c * 32 + i] = u2f(raw[c][i]);
}

__device__ __forceinline__ float tile_max(const float (&s)[64]) {
  float m0 = s[0], m1 = s[1], m2 = s[2], m3 = s[3];
#pragma unroll
  for (int c = 4; c < 64; c += 4) {
    m0 = fmaxf(m0, s[c]);
    m1 = fmaxf(m1, s[c + 1]);
    m2 = fmaxf(m2, s[c + 2]);
    m3 = fmaxf(m3, s[c + 3]);
  }
  return fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
}

// Rows of this warp's TMEM lanes, columns [0, 32 * NC) of taddr, times alpha.
template <int NC>
__device__ __forceinline__ void scale_tmem_rows(uint32_t taddr, float alpha) {
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    uint32_t raw[32];
    tmem_ld32(taddr + c * 32, raw);
    tmem_wait_ld_dep(raw);
#pragma unroll
    for (int i = 0; i < 32; ++i) raw[i] = __float_as_uint(u2f(raw[i]) * alpha);
    tmem_st32(taddr + c * 32, raw);
  }
}

__device__ __forceinline__ void tmem_ld_16x256b_x8(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_16x128b_x8(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}

}  // namespace tc
}  // namespace prism
