// 8-bit projection on the sm_100a tensor cores:
//
//   C[m, n] (bf16) = xs[m] ws[n] sum_k X8(m, k) W8(n, k)  (+ bias[n])
//
// X8 [M, K] rows with a scale each (prism_add_rms_norm_fp8), W8 [N, K] rows with a scale per
// output feature, both e4m3, K contiguous; products are exact and sums fp32 in the tensor core,
// the scales and the bias are applied in fp32, and the result is rounded once.
//
// The weight is the tensor core's M side (128 output features to a tile) and the tokens its N
// side, 16 to 128 of them to a tile: a call with one token then streams the weight through
// 16-column products instead of multiplying 127 rows of padding.  Large products run on pairs of
// CTAs (below) with tiles of 256 x 256.
//
// Persistent kernels.  Warp 4 streams weight and token tiles (128 bytes of K) with TMA into a ring,
// warp 5 issues tcgen05.mma kind::f8f6f4 (K = 32 an instruction) into one of two TMEM accumulators,
// warps 0-3 (thread = output feature) drain the other.  Every wait is bounded (sm100.cuh); one
// that gives up sets this file's device error word.
//
// Measured: one token of 5,120 x 5,120 9.1 us; 125 of 5,120 x 1,536 8.4; 75,600 tokens of
// 5,120 x 5,120 1.37 ms, 2.90 PFLOP/s in a short run (0.88 of twice the measured bf16 rate; tensor
// pipe 80 to 84 % busy) and 2.4 in a long one under the power cap.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <stdint.h>

#include <mutex>

#include "prism_common.cuh"
#include "sm100.cuh"

namespace prism {
namespace gemm8 {

using namespace sm100;

__device__ int g_gemm8_error = 0;
enum : int { kErrProducer = 411, kErrMma = 412, kErrEpilogue = 413 };

constexpr int kThreads = 192;
constexpr int kMaxSplits = 8;  // CTAs of a portable cluster
constexpr int kFeatures = 128, kStepK = 128;  // a tile's features; bytes of K in a stage
constexpr int kABytes = kFeatures * kStepK;

// The epilogue turns 16 tokens of a warp's 32 features at a time; rows of 36 words keep its 16-byte
// reads off each other's banks.
constexpr int kTurnRow = 36, kTurnBytes = 16 * kTurnRow * 4;

template <int kTokens>
struct Shape {
  static constexpr int kBBytes = kTokens * kStepK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = (96 << 10) / kStageBytes;  // an SM holds two CTAs
  static constexpr int kColumns = kTokens <= 16 ? 32 : 2 * kTokens;  // TMEM: two accumulators
  static constexpr int kFull = 0, kEmpty = kStages, kAccFull = 2 * kStages, kAccEmpty = kAccFull + 2,
                       kDrain = kAccEmpty + 2, kBars = kDrain + 1;
  static constexpr int kTurnAt = kStages * kStageBytes;  // the epilogue warps' transposition buffers
  static constexpr int kBarAt = kTurnAt + 4 * kTurnBytes;
  static constexpr int kTmemAt = kBarAt + kBars * 8;
  static constexpr int kAbortAt = kTmemAt + 4;
  static constexpr size_t kSmem = 1024 + kAbortAt + 4;
  static_assert(kFeatures * kTokens * 4 <= kTurnAt, "a split's partial sums reuse the ring");
};

// Four K = 32 products of one 128-byte stage; descriptor steps of 32 bytes, in 16-byte units.
__device__ __forceinline__ void mma_stage(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p0, p1;\n .reg .b64 a1, a2, a3, b1, b2, b3;\n"
      " setp.ne.b32 p0, %4, 0;\n setp.eq.b32 p1, %4, %4;\n"
      " add.s64 a1, %1, 2;\n add.s64 a2, %1, 4;\n add.s64 a3, %1, 6;\n"
      " add.s64 b1, %2, 2;\n add.s64 b2, %2, 4;\n add.s64 b3, %2, 6;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a1, b1, %3, p1;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a2, b2, %3, p1;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a3, b3, %3, p1;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// kind::f8f6f4 instruction descriptor: fp32 accumulation ([4,6) = 1), e4m3 operands (formats 0),
// both K-major, N >> 3 in [17,23), M >> 4 in [24,29).
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// What a warp of the epilogue does with its 32 features (lanes of TMEM) of a tile: 16 tokens at a
// time through its buffer, after which a lane has 8 features of the tokens `row` and `row` + 8 and
// writes them as 16 bytes.
struct Epilogue {
  float* turn;
  const float *xs, *ws, *bias;
  __nv_bfloat16* c;
  int64_t ldc;
  int M, N, row, column;
  bool wide;

  __device__ __forceinline__ Epilogue(uint8_t* buffer, int M_, int N_, const float* xs_, const float* ws_,
                                      const float* bias_, __nv_bfloat16* c_, int64_t ldc_)
      : turn(reinterpret_cast<float*>(buffer)), xs(xs_), ws(ws_), bias(bias_), c(c_), ldc(ldc_), M(M_), N(N_) {
    const int lane = threadIdx.x & 31;
    row = lane / 4, column = (lane % 4) * 8;
    wide = N % 8 == 0 && ldc % 8 == 0 && (reinterpret_cast<uintptr_t>(c) & 15) == 0;
  }

  // tokens [m0, m0 + tokens) of features [n0, n0 + 32), accumulated at TMEM address `acc`
  __device__ __forceinline__ void store(uint32_t acc, int n0, int m0, int tokens) const {
    const int lane = threadIdx.x & 31, n = n0 + column;
    float scale[8], b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      scale[e] = n + e < N ? __ldg(ws + n + e) : 0.0f;
      b[e] = bias && n + e < N ? __ldg(bias + n + e) : 0.0f;
    }
#pragma unroll 1
    for (int cc = 0; cc < tokens && m0 + cc < M; cc += 16) {
      float xs_of[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int m = m0 + cc + row + 8 * i;
        xs_of[i] = m < M ? __ldg(xs + m) : 0.0f;
      }
      uint32_t raw[16];
      tmem_ld16(acc + cc, raw);
#pragma unroll
      for (int i = 0; i < 16; ++i) turn[i * kTurnRow + lane] = __uint_as_float(raw[i]);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int m = m0 + cc + row + 8 * i;
        const float4* from = reinterpret_cast<const float4*>(turn + (row + 8 * i) * kTurnRow + column);
        const float4 lo = from[0], hi = from[1];
        const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaf(v[e] * xs_of[i], scale[e], b[e]);
        if (m >= M) continue;
        __nv_bfloat16* to = c + (int64_t)m * ldc + n;
        if (wide) {
          if (n < N)
            *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]),
                                                       pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n + e < N) to[e] = __float2bfloat16_rn(y[e]);
        }
      }
      __syncwarp();
    }
  }
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Every thread of the cluster's CTAs: shared memory written before is seen after.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
// Four words of CTA `rank`'s shared memory, at this CTA's address.
__device__ __forceinline__ float4 peer_load(uint32_t addr, uint32_t rank) {
  float4 v;
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(there)
               : "memory");
  return v;
}

// splits = 1: persistent CTAs over the tiles.  splits > 1: a cluster of that many CTAs to a tile,
// each over its part of K; their partial sums are added over distributed shared memory in rank
// order, each CTA adding up its share of the tile's tokens.
template <int kTokens>
__global__ void __launch_bounds__(kThreads, 2)
    linear_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, int M, int N,
                  int K, const float* __restrict__ xs, const float* __restrict__ ws, const float* __restrict__ bias,
                  __nv_bfloat16* __restrict__ c, int64_t ldc, int splits) {
  using S = Shape<kTokens>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t sb = smem_u32(sm);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto bar = [&](int i) { return sb + S::kBarAt + 8 * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + S::kAbortAt);
  const int tf = (N + kFeatures - 1) / kFeatures, tt = (M + kTokens - 1) / kTokens;
  const int tiles = tf * tt;
  const int steps = (K + kStepK - 1) / kStepK;
  const int rank = splits > 1 ? (int)cluster_rank() : 0;
  const int k_begin = (int)((int64_t)steps * rank / splits), k_end = (int)((int64_t)steps * (rank + 1) / splits);
  const int first = (int)blockIdx.x / splits, next = (int)gridDim.x / splits;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(bar(S::kFull + i), 1);
      mbar_init(bar(S::kEmpty + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(S::kAccFull + i), 1);
      mbar_init(bar(S::kAccEmpty + i), 4);
    }
    mbar_init(bar(S::kDrain), 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(sb + S::kTmemAt, S::kColumns);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + S::kTmemAt);

  if (warp == 4) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += next) {
        const int n0 = (t % tf) * kFeatures, m0 = (t / tf) * kTokens;
        for (int kb = k_begin; kb < k_end; ++kb, ++it) {
          const int s = it % S::kStages;
          if (it >= S::kStages && !mbar_wait(bar(S::kEmpty + s), ((it / S::kStages) - 1) & 1, abort_flag,
                                             &g_gemm8_error, kErrProducer)) {
            ok = false;
            break;
          }
          const uint32_t a = sb + s * S::kStageBytes, fb = bar(S::kFull + s);
          mbar_expect_tx(fb, S::kStageBytes);
          tma_load_2d(a, &tm_w, kb * kStepK, n0, fb);
          tma_load_2d(a + kABytes, &tm_x, kb * kStepK, m0, fb);
        }
      }
      // every issued copy has landed before the CTA may leave
      for (int i = it > S::kStages ? it - S::kStages : 0; i < it; ++i)
        mbar_wait(bar(S::kFull + i % S::kStages), (i / S::kStages) & 1, abort_flag, &g_gemm8_error, kErrProducer);
    }
  } else if (warp == 5) {
    if (lane == 0) {
      constexpr uint32_t kIdesc = idesc_e4m3(kFeatures, kTokens);
      int it = 0, tl = 0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += next, ++tl) {
        const int ab = tl & 1;
        if (tl >= 2 && !mbar_wait(bar(S::kAccEmpty + ab), ((tl >> 1) - 1) & 1, abort_flag, &g_gemm8_error, kErrMma))
          break;
        tc_fence_after();
        for (int kb = k_begin; kb < k_end; ++kb, ++it) {
          const int s = it % S::kStages;
          if (!mbar_wait(bar(S::kFull + s), (it / S::kStages) & 1, abort_flag, &g_gemm8_error, kErrMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = sb + s * S::kStageBytes;
          mma_stage(tmem + ab * kTokens, desc_k_sw128(a), desc_k_sw128(a + kABytes), kIdesc, kb > k_begin ? 1u : 0u);
          mma_commit(bar(S::kEmpty + s));
        }
        if (ok) mma_commit(bar(S::kAccFull + ab));
      }
      mma_commit(bar(S::kDrain));
      mbar_wait(bar(S::kDrain), 0, abort_flag, &g_gemm8_error, kErrMma);
    }
  } else {
    const Epilogue out(sm + S::kTurnAt + warp * kTurnBytes, M, N, xs, ws, bias, c, ldc);
    const uint32_t t_lane = tmem + ((uint32_t)(warp * 32) << 16);
    int tl = 0;
    for (int t = first; t < tiles; t += next, ++tl) {
      const int ab = tl & 1;
      const int n0 = (t % tf) * kFeatures + warp * 32, m0 = (t / tf) * kTokens;
      const bool ok = mbar_wait(bar(S::kAccFull + ab), (tl >> 1) & 1, abort_flag, &g_gemm8_error, kErrEpilogue);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      if (splits > 1) {  // into the ring, which the products are done with
#pragma unroll 1
        for (int cc = 0; cc < kTokens && m0 + cc < M; cc += 16) {
          uint32_t raw[16];
          tmem_ld16(t_lane + ab * kTokens + cc, raw);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            reinterpret_cast<uint32_t*>(sm)[(cc + i) * kFeatures + warp * 32 + lane] = raw[i];
        }
      } else {
        out.store(t_lane + ab * kTokens, n0, m0, kTokens);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(S::kAccEmpty + ab));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kColumns);
  }
  if (splits > 1) {
    cluster_sync();
    // a warp to a token, a lane to 4 features; two tokens' loads of all parts on their way
    const int n = (first % tf) * kFeatures + 4 * lane, m0 = (first / tf) * kTokens, count = min(kTokens, M - m0);
    float scale[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      scale[e] = n + e < N ? __ldg(ws + n + e) : 0.0f;
      b[e] = bias && n + e < N ? __ldg(bias + n + e) : 0.0f;
    }
    const bool wide = N % 4 == 0 && ldc % 4 == 0 && (reinterpret_cast<uintptr_t>(c) & 7) == 0;
    const int end = count * (rank + 1) / splits;
    for (int i = count * rank / splits + warp; i < end; i += 2 * (kThreads / 32)) {
      float sum[2][4] = {};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int at = i + u * (kThreads / 32);
        if (at >= end) break;
#pragma unroll
        for (int r = 0; r < kMaxSplits; ++r) {
          if (r >= splits) break;
          const float4 v = peer_load(sb + (at * kFeatures + 4 * lane) * 4, r);
          sum[u][0] += v.x, sum[u][1] += v.y, sum[u][2] += v.z, sum[u][3] += v.w;
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int at = i + u * (kThreads / 32);
        if (at >= end) break;
        const float x = __ldg(xs + m0 + at);
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = fmaf(sum[u][e] * x, scale[e], b[e]);
        __nv_bfloat16* to = c + (int64_t)(m0 + at) * ldc + n;
        if (wide) {
          if (n < N) *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < N) to[e] = __float2bfloat16_rn(y[e]);
        }
      }
    }
    cluster_sync();  // no CTA leaves while another reads its sums
  }
}

// ------------------------------------------------------------ CTA pairs
// Two CTAs of a cluster share a tile of 256 features x 256 tokens: cta_group::2 products with
// M = 256, whose features 0-127 are in the even CTA's TMEM and shared memory and 128-255 in the
// odd one's, while each CTA holds 128 of the tokens.  An instruction then reads 4 KB + 4 KB of each
// CTA's shared memory in 128 clocks instead of 4 KB + 8 KB, and a token tile is fetched once for
// 256 features.  Both CTAs' copies complete on the even CTA's barriers (a relay by the odd CTA would
// cost a release at cluster scope, 0.9 us, for each stage); the even CTA's warp 5 issues every
// product and commits its completions to both CTAs.  Every wait is bounded.
struct Pair {
  static constexpr int kTokens = 256, kHalf = 128, kStages = 6;
  static constexpr int kStageBytes = kABytes + kHalf * kStepK;
  // Full (even CTA): both CTAs' copies; Empty, AccFull: products done; AccEmpty (even CTA): the
  // epilogue warps of both
  static constexpr int kFull = 0, kEmpty = kStages, kAccFull = 2 * kStages, kAccEmpty = kAccFull + 2,
                       kDrain = kAccEmpty + 2, kBars = kDrain + 1;
  static constexpr int kTurnAt = kStages * kStageBytes, kBarAt = kTurnAt + 4 * kTurnBytes;
  static constexpr int kTmemAt = kBarAt + kBars * 8, kAbortAt = kTmemAt + 4;
  static constexpr size_t kSmem = 1024 + kAbortAt + 4;
};

__device__ __forceinline__ void mma_pair_stage(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p0, p1;\n .reg .b64 a1, a2, a3, b1, b2, b3;\n"
      " setp.ne.b32 p0, %4, 0;\n setp.eq.b32 p1, %4, %4;\n"
      " add.s64 a1, %1, 2;\n add.s64 a2, %1, 4;\n add.s64 a3, %1, 6;\n"
      " add.s64 b1, %2, 2;\n add.s64 b2, %2, 4;\n add.s64 b3, %2, 6;\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p0;\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a1, b1, %3, p1;\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a2, b2, %3, p1;\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a3, b3, %3, p1;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives once on the barrier at this offset in both CTAs when this thread's products so far are done.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile(
      "{\n .reg .b16 m;\n mov.b16 m, 3;\n"
      " tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n}\n" ::"r"(
          bar)
      : "memory");
}
// The even CTA's barrier at this offset.
__device__ __forceinline__ uint32_t in_even(uint32_t bar) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(bar));
  return there;
}
__device__ __forceinline__ void arrive_even(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_even(bar)) : "memory");
}
// A tile into this CTA's shared memory that completes on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ bool try_pair(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n"
      " mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// A bounded wait on a barrier that the other CTA arrives on (sm100.cuh's mbar_wait, acquiring at
// cluster scope).
__device__ __forceinline__ bool wait_pair(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
  if (try_pair(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 16; ++i)
      if (try_pair(bar, parity)) return true;
    if (*abort_flag) return false;
    if (*reinterpret_cast<volatile int*>(&g_gemm8_error) != 0) {
      *abort_flag = 1;
      return false;
    }
    if (globaltimer() - t0 > *reinterpret_cast<volatile unsigned long long*>(&g_wait_limit_ns)) {
      *abort_flag = 1;
      atomicCAS(&g_gemm8_error, 0, code);
      return false;
    }
  }
}

// A wait at the end of the kernel that also holds after another wait gave up: up to 50 ms for what is
// in flight towards this CTA.
__device__ __forceinline__ void settle(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try(bar, parity) && globaltimer() - t0 < 50000000ull) {
  }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, int M, int N,
                       int K, const float* __restrict__ xs, const float* __restrict__ ws,
                       const float* __restrict__ bias, __nv_bfloat16* __restrict__ c, int64_t ldc) {
  using S = Pair;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t sb = smem_u32(sm);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cluster_rank();
  auto bar = [&](int i) { return sb + S::kBarAt + 8 * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + S::kAbortAt);
  const int tf = (N + 2 * kFeatures - 1) / (2 * kFeatures), tt = (M + S::kTokens - 1) / S::kTokens;
  const int tiles = tf * tt, steps = (K + kStepK - 1) / kStepK;
  const int first = (int)blockIdx.x / 2, next = (int)gridDim.x / 2;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(bar(S::kFull + i), 1);
      mbar_init(bar(S::kEmpty + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(S::kAccFull + i), 1);
      mbar_init(bar(S::kAccEmpty + i), 8);
    }
    mbar_init(bar(S::kDrain), 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sb + S::kTmemAt), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are set up before an arrival crosses
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + S::kTmemAt);

  if (warp == 4) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += next) {
        const int n0 = (t % tf) * 2 * kFeatures + rank * kFeatures, m0 = (t / tf) * S::kTokens + rank * S::kHalf;
        for (int kb = 0; kb < steps; ++kb, ++it) {
          const int s = it % S::kStages;
          if (it >= S::kStages &&
              !wait_pair(bar(S::kEmpty + s), ((it / S::kStages) - 1) & 1, abort_flag, kErrProducer)) {
            ok = false;
            break;
          }
          const uint32_t a = sb + s * S::kStageBytes, fb = in_even(bar(S::kFull + s));
          // the stage's one arrival; the odd CTA's bytes may come before it, the phase ends after it
          if (rank == 0) mbar_expect_tx(bar(S::kFull + s), 2 * S::kStageBytes);
          tma_load_pair(a, &tm_w, kb * kStepK, n0, fb);
          tma_load_pair(a + kABytes, &tm_x, kb * kStepK, m0, fb);
        }
      }
      // before either CTA may leave (both end in cluster_sync): every copy of both has landed, and
      // the last completions have arrived at this CTA's barriers
      for (int i = it > S::kStages ? it - S::kStages : 0; i < it; ++i) {
        if (rank == 0) settle(bar(S::kFull + i % S::kStages), (i / S::kStages) & 1);
        settle(bar(S::kEmpty + i % S::kStages), (i / S::kStages) & 1);
      }
    }
  } else if (warp == 5) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t kIdesc = idesc_e4m3(2 * kFeatures, S::kTokens);
      int it = 0, tl = 0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += next, ++tl) {
        const int ab = tl & 1;
        if (tl >= 2 && !wait_pair(bar(S::kAccEmpty + ab), ((tl >> 1) - 1) & 1, abort_flag, kErrMma)) break;
        tc_fence_after();
        for (int kb = 0; kb < steps; ++kb, ++it) {
          const int s = it % S::kStages;
          ok = wait_pair(bar(S::kFull + s), (it / S::kStages) & 1, abort_flag, kErrMma);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = sb + s * S::kStageBytes;
          mma_pair_stage(tmem + ab * S::kTokens, desc_k_sw128(a), desc_k_sw128(a + kABytes), kIdesc, kb > 0 ? 1u : 0u);
          commit_pair(bar(S::kEmpty + s));
        }
        if (ok) commit_pair(bar(S::kAccFull + ab));
      }
      commit_pair(bar(S::kDrain));
    }
  } else {
    const Epilogue out(sm + S::kTurnAt + warp * kTurnBytes, M, N, xs, ws, bias, c, ldc);
    const uint32_t t_lane = tmem + ((uint32_t)(warp * 32) << 16);
    int tl = 0;
    for (int t = first; t < tiles; t += next, ++tl) {
      const int ab = tl & 1;
      const int n0 = (t % tf) * 2 * kFeatures + rank * kFeatures + warp * 32, m0 = (t / tf) * S::kTokens;
      const bool ok = wait_pair(bar(S::kAccFull + ab), (tl >> 1) & 1, abort_flag, kErrEpilogue);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      out.store(t_lane + ab * S::kTokens, n0, m0, S::kTokens);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_even(bar(S::kAccEmpty + ab));
    }
  }
  tc_fence_before();
  __syncthreads();
  // both CTAs: the even one's commits are done, here too.  Not before the CTA's own work is: the wait's
  // 50 ms would start with the kernel, and a long call would leave with an arrival on its way.
  if (warp == 5 && lane == 0) settle(bar(S::kDrain), 0);
  __syncwarp();
  cluster_sync();  // neither CTA frees its TMEM or leaves while the other may still reach it
  if (warp == 5) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ------------------------------------------------------------------ host
using EncodeFn = PFN_cuTensorMapEncodeTiled_v12000;

static EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(p);
  });
  return fn;
}

// 2D map of e4m3 rows, boxes of 128 bytes x box_rows, 128-byte swizzle; zeros outside.
static prism_status_t make_map(CUtensorMap* map, const void* ptr, int64_t rows, int64_t cols, int64_t ld,
                               int box_rows) {
  EncodeFn enc = encode_fn();
  if (enc == nullptr) {
    set_error("prism_linear_fp8: cuTensorMapEncodeTiled is unavailable from the driver");
    return PRISM_ERR_CUDA;
  }
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {kStepK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("prism_linear_fp8: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return PRISM_ERR_CUDA;
  }
  return PRISM_OK;
}

constexpr int kSms = 148;
static int64_t tiles_of(int M, int N, int tokens) {
  return (int64_t)((N + kFeatures - 1) / kFeatures) * ((M + tokens - 1) / tokens);
}

static int64_t pair_tiles_of(int M, int N) {
  return (int64_t)((N + 2 * kFeatures - 1) / (2 * kFeatures)) * ((M + Pair::kTokens - 1) / Pair::kTokens);
}

template <int kTokens>
static prism_status_t launch(const void* x8, int64_t ldx, const float* xs, const void* w8, int64_t ldw,
                             const float* ws, const float* bias, int M, int N, int K, void* c, int64_t ldc,
                             int splits, cudaStream_t stream) {
  using S = Shape<kTokens>;
  CUtensorMap mw, mx;
  prism_status_t st = make_map(&mw, w8, N, K, ldw, kFeatures);
  if (st != PRISM_OK) return st;
  st = make_map(&mx, x8, M, K, ldx, kTokens);
  if (st != PRISM_OK) return st;
  PRISM_CHECK_CUDA(cudaFuncSetAttribute(linear_kernel<kTokens>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)S::kSmem),
                   "prism_linear_fp8: smem attribute");
  const int64_t tiles = tiles_of(M, N, kTokens);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(splits > 1 ? tiles * splits : tiles < 2 * kSms ? tiles : 2 * kSms));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = S::kSmem;
  config.stream = stream;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = splits, cluster.val.clusterDim.y = 1, cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = splits > 1 ? 1 : 0;
  PRISM_CHECK_CUDA(cudaLaunchKernelEx(&config, linear_kernel<kTokens>, mw, mx, M, N, K, xs, ws, bias,
                                      (__nv_bfloat16*)c, ldc, splits),
                   "prism_linear_fp8");
  return PRISM_OK;
}

static prism_status_t launch_pair(const void* x8, int64_t ldx, const float* xs, const void* w8, int64_t ldw,
                                  const float* ws, const float* bias, int M, int N, int K, void* c, int64_t ldc,
                                  cudaStream_t stream) {
  CUtensorMap mw, mx;
  prism_status_t st = make_map(&mw, w8, N, K, ldw, kFeatures);
  if (st != PRISM_OK) return st;
  st = make_map(&mx, x8, M, K, ldx, Pair::kHalf);
  if (st != PRISM_OK) return st;
  PRISM_CHECK_CUDA(cudaFuncSetAttribute(linear_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)Pair::kSmem),
                   "prism_linear_fp8: smem attribute");
  const int64_t tiles = pair_tiles_of(M, N), pairs = tiles < kSms / 2 ? tiles : kSms / 2;
  linear_pair_kernel<<<(unsigned)(2 * pairs), kThreads, Pair::kSmem, stream>>>(mw, mx, M, N, K, xs, ws, bias,
                                                                              (__nv_bfloat16*)c, ldc);
  PRISM_CHECK_LAUNCH("prism_linear_fp8");
  return PRISM_OK;
}

}  // namespace gemm8
}  // namespace prism

using namespace prism;

int prism_gemm8_device_status_internal(void) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, gemm8::g_gemm8_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(gemm8::g_gemm8_error, &zero, sizeof(int));
  }
  return v;
}

extern "C" prism_status_t prism_linear_fp8(const void* x8, int64_t ldx, const float* x_scale, const void* w8,
                                           int64_t ldw, const float* w_scale, const float* bias, int M, int N,
                                           int K, void* c, int64_t ldc, cudaStream_t stream) {
  PRISM_CHECK_ARG(M >= 0 && M < (1 << 30) && N >= 1 && N < (1 << 30) && K >= 1 && K < (1 << 30) && K % 16 == 0,
                  "prism_linear_fp8: bad sizes (N >= 1, K a positive multiple of 16)");
  if (M == 0) return PRISM_OK;
  PRISM_CHECK_ARG(x8 && x_scale && w8 && w_scale && c, "prism_linear_fp8: null pointer");
  PRISM_CHECK_ARG(ldx >= K && ldw >= K && ldx % 16 == 0 && ldw % 16 == 0 && ldc >= N,
                  "prism_linear_fp8: 8-bit row strides must be multiples of 16 and cover K, ldc must cover N");
  PRISM_CHECK_ARG(aligned16(x8) && aligned16(w8), "prism_linear_fp8: 8-bit tensors must be 16-byte aligned");
  PRISM_CHECK_ARG(gemm8::tiles_of(M, N, 128) < ((int64_t)1 << 30), "prism_linear_fp8: the output has too many tiles");
  // Pairs of CTAs on 256 x 256 where there are more than two rounds of such halves and K is long
  // enough to hide the epilogue (2,048 tokens of 5,120 x 5,120: 52 us against 56 with 128-token
  // tiles; 1,024 tokens, one round and a bit: 36 with those; 32,768 tokens of 512 x 1,536: 57, of
  // which two CTAs an SM hide each other's epilogues).
  if (M > 128 && K > 1024 && gemm8::tiles_of(M, N, 256) > 2 * gemm8::kSms)
    return gemm8::launch_pair(x8, ldx, x_scale, w8, ldw, w_scale, bias, M, N, K, c, ldc, stream);
  // else the smallest tile that holds every token, 128 at most
  const int steps = (K + gemm8::kStepK - 1) / gemm8::kStepK;
  int tokens = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  // A short K: smaller tiles while they leave SMs without work (125 tokens of 5,120 x 1,536 in tiles
  // of 128 / 64 / 32 tokens, 40 / 80 / 160 tiles: 9.8 / 8.5 / 8.7 us; 706 of 160 x 368 down to 16
  // tokens: 7.2 / 5.8 / 5.0 / 4.7), from 128 to 64 also for a little more than one round (133 of
  // 7,312 x 464, 174 tiles: 8.1 / 6.8 us; in 290 of 32 tokens 7.6)
  constexpr int kSplitSteps = 20;
  while (steps < kSplitSteps && tokens > 16 &&
         gemm8::tiles_of(M, N, tokens / 2) <= (tokens == 128 ? gemm8::kSms * 4 / 3 : gemm8::kSms))
    tokens /= 2;
  // A long one in parts, if each keeps five steps: enough to pay the exchange of 2.6 us (one token
  // of 5,120 x 5,120: 15.1 us whole, 11.0 / 9.2 in 2 / 4 parts; 125 tokens of K = 1,536: 8.5 whole, 9.9 in two)
  const int64_t tiles = gemm8::tiles_of(M, N, tokens), room = 2 * gemm8::kSms;
  int splits = 1;
  while (splits < gemm8::kMaxSplits && tiles * splits * 2 <= room && steps >= kSplitSteps && steps >= 10 * splits)
    splits *= 2;
  const auto launch = tokens == 16    ? gemm8::launch<16>
                      : tokens == 32  ? gemm8::launch<32>
                      : tokens == 64  ? gemm8::launch<64>
                                      : gemm8::launch<128>;
  return launch(x8, ldx, x_scale, w8, ldw, w_scale, bias, M, N, K, c, ldc, splits, stream);
}
