// Residual addition + RMS norm of rows, forward (16-, 32- and 8-bit outputs) and backward.
//
//   h   = x + r, rounded to the rows' type (the residual stream as the next layer reads it)
//   u   = (mean_j h_j^2 + eps)^(-1/2)
//   y_j = w_j h_j u
// 8-bit rows: s = max(max_j |y_j| / 448, 2^-100), y8_j = e4m3(y_j / s).  u cancels in y_j / s,
// so one reduction gives both sum h^2 and max |w h|.  A row that holds a NaN or an infinity has
// scale NaN.
// Backward, with gy = dL/dy and gh = dL/dh:
//   dL/dh_j = u (w_j gy_j) - h_j u^3 / C * sum_i w_i gy_i h_i + gh_j   (also dL/dx and dL/dr)
//   dL/dw_j = sum over rows of gy_j h_j u
// Sums, u and the gradient of w are held in fp32.  Where the squares of finite values leave it
// (rows above some 1e19), the row is summed again times 2^-80: a branch that ordinary rows do not
// take.  The backward forms h u, of order one, before any product with h.
//
// Bound by memory: each tensor is read or written once.  A row stays with one group of threads --
// a power of two of lanes for narrow rows, a CTA for wide ones -- which holds it in registers
// between the row's reduction and its outputs, 8 or 16 elements a thread.  Groups are persistent
// (they hold their columns of w, and sum their columns of dL/dw, in registers over all their
// rows) and fetch the next rows with cp.async into slots of shared memory that only the fetching
// thread reads: no barrier but the reduction's, and the loads of the next row or two are on their
// way while one is reduced.  Measured at 75,600 x 5,120 bf16 with a residual: forward 484 us
// (6.4 TB/s, half of it writes), backward 456 us (6.8); 9,450 rows to 8 bits 54 us (6.3).
#include <cuda_fp8.h>
#include <math.h>

#include "block_ops.cuh"

namespace prism {
namespace norm {

constexpr float kFp8Max = 448.0f;                      // largest finite e4m3 value
constexpr float kScaleFloor = 7.8886090522101181e-31f;  // 2^-100: 1 / scale stays finite
constexpr float kFloatMax = 3.402823466e38f;
// Takes every finite row's squares into fp32, 16,384 of up to 2^96, and leaves those that make up a sum of
// 2^128 and more above 2^-32.
constexpr float kDown = 8.2718061255302767e-25f;  // 2^-80
constexpr int kThreads = 256;   // of the kernels whose groups are smaller than a CTA
constexpr int kSms = 148;

struct SumMax {
  float sum, max;
};

// The larger one, a NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// The largest magnitude, a NaN if any is.
__device__ __forceinline__ float max_abs_nan(float a, float b, float c) {
  float m;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

// Sum where kSum, maximum where kMax, over aligned runs of `lanes` lanes, a power of two; every
// lane gets them.
template <bool kSum, bool kMax>
__device__ __forceinline__ SumMax lane_reduce(SumMax v, int lanes) {
  for (int o = lanes / 2; o >= 1; o >>= 1) {
    if constexpr (kSum) v.sum += __shfl_xor_sync(0xffffffffu, v.sum, o);
    if constexpr (kMax) v.max = max_nan(v.max, __shfl_xor_sync(0xffffffffu, v.max, o));
  }
  return v;
}

// The same over a whole warp: the maximum in one instruction.
template <bool kSum, bool kMax>
__device__ __forceinline__ SumMax warp_reduce(SumMax v) {
  if constexpr (kMax) asm volatile("redux.sync.max.NaN.f32 %0, %0, 0xffffffff;" : "+f"(v.max));
  if constexpr (kSum) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v.sum += __shfl_xor_sync(0xffffffffu, v.sum, o);
  }
  return v;
}

// The same over the group of lanes, or over the CTA.  `red` alternates between two rows, so that
// one barrier a reduction is enough.
template <bool kCta, bool kSum, bool kMax>
__device__ __forceinline__ SumMax group_reduce(SumMax v, int group, SumMax (*red)[32], int turn) {
  if constexpr (kCta) {
    v = warp_reduce<kSum, kMax>(v);
    SumMax* row = red[turn & 1];
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) row[threadIdx.x >> 5] = v;
    __syncthreads();
    // every warp adds up the warps' values in the same tree
    v = lane < warps ? row[lane] : SumMax{0.0f, 0.0f};
    return warp_reduce<kSum, kMax>(v);
  } else {
    return lane_reduce<kSum, kMax>(v, group);
  }
}

// scale of an 8-bit row and the factor that takes w h to its 8-bit values.
struct Quant {
  float scale, factor;
};
__device__ __forceinline__ Quant quantizer(const SumMax& t, float u) {
  Quant q;
  q.scale = fmaxf(t.max * u * (1.0f / kFp8Max), kScaleFloor);
  if (!(t.max <= kFloatMax)) q.scale = NAN;
  q.factor = __fdividef(u, q.scale);  // two units off at most; the scale is below 2^120
  return q;
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// Where a thread works: its group's rows and its columns of a row.  With kShift the rows are not
// 16-byte aligned, all tensors' in the same way: `lead` single elements, vectors, single elements;
// a thread has at most one single element.  The rows of a group are all shifted alike (the groups'
// row step is a multiple of the period of the shifts).
template <typename T, int kPer, bool kCta, bool kShift>
struct Place {
  static constexpr int kWidth = 16 / sizeof(T), kVecs = kPer / kWidth;
  int group, lane, lead, vecs, single;  // single: column of the single element, or -1
  int64_t first, warp_first, step;      // the group's first row, that of the warp's first group

  __device__ __forceinline__ Place(const T* base, int64_t ld, int cols, int group_) {
    group = kCta ? (int)blockDim.x : group_;
    lane = kCta ? (int)threadIdx.x : (int)(threadIdx.x & (group - 1));
    const int per_cta = kCta ? 1 : (int)blockDim.x / group;
    const int64_t at = (int64_t)blockIdx.x * per_cta;
    first = kCta ? at : at + threadIdx.x / group;
    warp_first = kCta ? at : at + (threadIdx.x & ~31u) / group;
    step = (int64_t)gridDim.x * per_cta;
    lead = 0, single = -1;
    if (kShift) {
      const unsigned off = (unsigned)(reinterpret_cast<uintptr_t>(base) + (uint64_t)(first * ld) * sizeof(T)) & 15u;
      lead = min(cols, (int)((16u - off) & 15u) / (int)sizeof(T));
    }
    vecs = (cols - lead) / kWidth;
    if (kShift) {
      const int tail = cols - lead - vecs * kWidth;
      if (lane < lead) single = lane;
      else if (lane - lead < tail) single = cols - tail + lane - lead;
    }
  }
  // column of the thread's v-th vector, or -1
  __device__ __forceinline__ int column(int v) const {
    const int i = lane + v * group;
    return i < vecs ? lead + i * kWidth : -1;
  }
};

// Thread-private slots: kStages rows of kTensors tensors.
template <int kTensors, int kVecs, int kStages>
struct Ring {
  uint4* slots;
  __device__ __forceinline__ explicit Ring(uint4* smem) : slots(smem + threadIdx.x) {}
  __device__ __forceinline__ uint4* at(int stage, int tensor, int v) const {
    return slots + ((stage * kTensors + tensor) * kVecs + v) * (int)blockDim.x;
  }
  static __device__ __forceinline__ void load(uint4* slot, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(slot)), "l"(src)
                 : "memory");
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  // The oldest of the `depth` rows on their way has arrived.
  static __device__ __forceinline__ void wait(int depth = kStages) {
    if (depth == kStages)
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    else
      asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  static __device__ __forceinline__ void drain() { asm volatile("cp.async.wait_all;" ::: "memory"); }
};

// A thread's columns of w (1 without a weight) as registers; one more for the single element.
template <int kPer, typename P>
__device__ __forceinline__ void load_weight(const P& p, const float* w, float (&wv)[kPer], float& ws) {
#pragma unroll
  for (int v = 0; v < P::kVecs; ++v) {
    const int c = p.column(v);
#pragma unroll
    for (int e = 0; e < P::kWidth; ++e) wv[v * P::kWidth + e] = w && c >= 0 ? __ldg(w + c + e) : 1.0f;
  }
  ws = w && p.single >= 0 ? __ldg(w + p.single) : 1.0f;
}

// Rows of a group on their way, at most.  fp32 rows at 16 elements a thread (64 bytes) have to do with one:
// 220 KB hold no more of 1,024 threads' slots.
constexpr int stages(int bytes) { return bytes <= 32 ? 2 : 1; }

// A row of a group that met one whose squares leave fp32: from h as it is kept, summed and, if it is such a
// row, normalised times kDown, element by element.  count: its columns, or 0 for a group that only takes
// part in its warp's shuffles.  After the rows' loop, which it would take registers from; looking for such
// rows costs the loop 2 % (forward of 75,600 x 5,120 bf16 474 -> 484 us).
template <typename T, bool kCta, bool kQuant>
__device__ __forceinline__ void large_row(const T* h, const float* w, float eps, int count, int64_t row, int cols, int lane,
                                       int group, SumMax (*red)[32], int turn, void* y, float* aux) {
  if constexpr (!kCta) __syncwarp();  // the group's other threads wrote h
  SumMax t = {0.0f, 0.0f};
#pragma unroll 1
  for (int c = lane; c < count; c += group) {
    const float f = Elem<T>::to_f(h[c]) * kDown;
    t.sum += f * f;
    if (kQuant) t.max = max_nan(t.max, fabsf(w ? f * w[c] : f));
  }
  t = group_reduce<kCta, true, kQuant>(t, group, red, turn);
  // half of fp32's range, whose sums both ways have: the loop added them up in another order
  if (!(t.sum > 0.5f * kFloatMax * kDown * kDown)) return;
  const float u = rsqrtf(t.sum / (float)cols + eps * kDown * kDown);
  Quant q = {};
  if constexpr (kQuant) q = quantizer(t, u);
#pragma unroll 1
  for (int c = lane; c < count; c += group) {
    float f = Elem<T>::to_f(h[c]) * kDown;
    if (w) f *= w[c];
    if constexpr (kQuant) static_cast<uint8_t*>(y)[row * cols + c] = (uint8_t)e4m3x2(f * q.factor, 0.0f);
    else static_cast<T*>(y)[row * cols + c] = Elem<T>::from_f(f * u);
  }
  if (lane == 0 && count > 0) {
    if constexpr (kQuant) aux[row] = q.scale;
    else if (aux) aux[row] = u * kDown;
  }
}

// kQuant: 8-bit rows.  Without kNorm the rows themselves (u = 1, no sum: 60,000 x 5,120 bf16 to 8
// bits 160 us, with a sum that nothing reads 191).  depth: rows of a group on their way, one or
// kStages.
template <typename T, int kPer, bool kCta, bool kShift, bool kQuant, bool kNorm>
__global__ void __launch_bounds__(kCta ? 1024 : kThreads, kCta ? 1 : 4)
    fwd_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ r, int64_t ldr,
               const float* __restrict__ w, float eps, int64_t rows, int cols, int group, int depth,
               void* __restrict__ y, T* __restrict__ h, float* __restrict__ aux) {
  using P = Place<T, kPer, kCta, kShift>;
  constexpr int kWidth = P::kWidth, kVecs = P::kVecs;
  extern __shared__ uint4 smem[];
  __shared__ SumMax red[2][32];
  const P p(x, ldx, cols, group);
  constexpr int kStages = stages(kPer * sizeof(T));
  constexpr bool kResum = kNorm && !std::is_same_v<T, __half>;  // fp16 squares always fit
  const Ring<2, kVecs, kStages> ring(smem);
  const auto fetch = [&](int64_t row, int stage) {
    if (row < rows) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const int c = p.column(v);
        if (c >= 0) {
          ring.load(ring.at(stage, 0, v), x + row * ldx + c);
          if (r) ring.load(ring.at(stage, 1, v), r + row * ldr + c);
        }
      }
    }
    ring.commit();
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s)
    if (s < depth) fetch(p.first + s * p.step, s);
  float wv[kPer], ws;
  load_weight(p, w, wv, ws);
  const bool has_single = kShift && p.single >= 0;
  float xs = 0.0f, rs = 0.0f;
  const auto fetch_single = [&](int64_t row) {
    if (has_single && row < rows) {
      xs = Elem<T>::to_f(x[row * ldx + p.single]);
      if (r) rs = Elem<T>::to_f(r[row * ldr + p.single]);
    }
  };
  if (kShift) fetch_single(p.first);

  const float inv_cols = 1.0f / (float)cols;
  int stage = 0, turn = 0;
  bool large = false;  // one of the group's rows is to be summed again
  for (int64_t row = p.first, warp_row = p.warp_first; warp_row < rows; row += p.step, warp_row += p.step, ++turn) {
    ring.wait(depth);
    const bool live = kCta || row < rows;
    float hv[kPer], hs = xs;  // w h for 8-bit rows
    SumMax t = {0.0f, 0.0f};
    const auto take = [&](float& f, float wf) {
      if (kNorm) t.sum += f * f;
      if (kQuant && (kNorm || w)) f *= wf;
    };
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const int c = p.column(v);
      float f[kWidth] = {};
      if (live && c >= 0) {
        unpack<T>(*ring.at(stage, 0, v), f);
        if (r) {
          float g[kWidth];
          unpack<T>(*ring.at(stage, 1, v), g);
#pragma unroll
          for (int e = 0; e < kWidth; ++e) f[e] += g[e];
          const uint4 packed = pack<T>(f);
          *reinterpret_cast<uint4*>(h + row * cols + c) = packed;
          unpack<T>(packed, f);
        }
      }
#pragma unroll
      for (int e = 0; e < kWidth; ++e) {
        take(f[e], wv[v * kWidth + e]);
        hv[v * kWidth + e] = f[e];
      }
      if (kQuant) {
#pragma unroll
        for (int e = 0; e < kWidth; e += 2) t.max = max_abs_nan(t.max, f[e], f[e + 1]);
      }
    }
    if (has_single && live) {
      if (r) {
        const T v = Elem<T>::from_f(xs + rs);
        h[row * cols + p.single] = v;
        hs = Elem<T>::to_f(v);
      }
      take(hs, ws);
      if (kQuant) t.max = max_abs_nan(t.max, hs, hs);
    }
    fetch(row + depth * p.step, stage);
    if (kShift) fetch_single(row + p.step);
    stage = stage + 1 == depth ? 0 : stage + 1;
    t = group_reduce<kCta, kNorm, kQuant>(t, p.group, red, turn);
    if (kResum) large = large || t.sum > kFloatMax;
    const float u = kNorm ? rsqrtf(t.sum * inv_cols + eps) : 1.0f;
    if (!live) continue;
    if constexpr (kQuant) {
      const Quant q = quantizer(t, u);
      uint8_t* out = static_cast<uint8_t*>(y) + row * cols;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const int c = p.column(v);
        if (c < 0) continue;
        uint32_t b[kWidth / 4];
#pragma unroll
        for (int e = 0; e < kWidth; e += 4) {
          const int i = v * kWidth + e;
          b[e / 4] = e4m3x2(hv[i] * q.factor, hv[i + 1] * q.factor) |
                     e4m3x2(hv[i + 2] * q.factor, hv[i + 3] * q.factor) << 16;
        }
        if constexpr (kShift) {  // the bytes' alignment is not the elements'
          if (reinterpret_cast<uintptr_t>(out + c) % 4 == 0) {
#pragma unroll
            for (int e = 0; e < kWidth; e += 4) *reinterpret_cast<uint32_t*>(out + c + e) = b[e / 4];
          } else {
#pragma unroll
            for (int e = 0; e < kWidth; ++e) out[c + e] = (uint8_t)(b[e / 4] >> (8 * (e % 4)));
          }
        } else if constexpr (kWidth == 8) {
          *reinterpret_cast<uint2*>(out + c) = make_uint2(b[0], b[1]);
        } else {
          *reinterpret_cast<uint32_t*>(out + c) = b[0];
        }
      }
      if (has_single) out[p.single] = (uint8_t)e4m3x2(hs * q.factor, 0.0f);
      if (p.lane == 0) aux[row] = q.scale;
    } else {
      T* out = static_cast<T*>(y) + row * cols;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const int c = p.column(v);
        if (c < 0) continue;
        float f[kWidth];
#pragma unroll
        for (int e = 0; e < kWidth; ++e) f[e] = hv[v * kWidth + e] * u * wv[v * kWidth + e];
        *reinterpret_cast<uint4*>(out + c) = pack<T>(f);
      }
      if (has_single) out[p.single] = Elem<T>::from_f(hs * u * ws);
      if (p.lane == 0 && aux) aux[row] = u;
    }
  }
  ring.drain();
  if constexpr (kResum) {
    if (kCta ? large : __any_sync(0xffffffffu, large)) {
      for (int64_t row = p.first, warp_row = p.warp_first; warp_row < rows; row += p.step, warp_row += p.step, ++turn)
        large_row<T, kCta, kQuant>(r ? h + row * cols : x + row * ldx, w, eps, large && row < rows ? cols : 0, row, cols,
                                   p.lane, p.group, red, turn, y, aux);
    }
  }
}

// dL/dh of the rows, and each CTA's sum of dL/dw -> part[CTA][cols] (part NULL: not wanted).
template <typename T, int kPer, bool kCta, bool kShift>
__global__ void __launch_bounds__(kCta ? 1024 : kThreads, kCta ? 1 : 4)
    bwd_kernel(const T* __restrict__ gy, int64_t ldgy, const T* __restrict__ h, int64_t ldh,
               const T* __restrict__ gh, int64_t ldgh, const float* __restrict__ w,
               const float* __restrict__ rstd, int64_t rows, int cols, int group, T* __restrict__ dx,
               float* __restrict__ part) {
  using P = Place<T, kPer, kCta, kShift>;
  constexpr int kWidth = P::kWidth, kVecs = P::kVecs;
  extern __shared__ uint4 smem[];
  __shared__ SumMax red[2][32];
  const P p(gy, ldgy, cols, group);
  constexpr int kStages = stages(kPer * sizeof(T));
  const Ring<3, kVecs, kStages> ring(smem);
  const auto fetch = [&](int64_t row, int stage) {
    if (row < rows) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const int c = p.column(v);
        if (c >= 0) {
          ring.load(ring.at(stage, 0, v), gy + row * ldgy + c);
          ring.load(ring.at(stage, 1, v), h + row * ldh + c);
          if (gh) ring.load(ring.at(stage, 2, v), gh + row * ldgh + c);
        }
      }
    }
    ring.commit();
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) fetch(p.first + s * p.step, s);
  float wv[kPer], ws, dw[kPer] = {}, dws = 0.0f;
  load_weight(p, w, wv, ws);
  const bool has_single = kShift && p.single >= 0;
  float gs = 0.0f, hs = 0.0f, ghs = 0.0f, u_next = 0.0f;
  const auto fetch_single = [&](int64_t row) {
    if (row < rows) {
      u_next = __ldg(rstd + row);
      if (has_single) {
        gs = Elem<T>::to_f(gy[row * ldgy + p.single]);
        hs = Elem<T>::to_f(h[row * ldh + p.single]);
        if (gh) ghs = Elem<T>::to_f(gh[row * ldgh + p.single]);
      }
    }
  };
  fetch_single(p.first);

  const float inv_cols = 1.0f / (float)cols;
  int stage = 0, turn = 0;
  for (int64_t row = p.first, warp_row = p.warp_first; warp_row < rows; row += p.step, warp_row += p.step, ++turn) {
    ring.wait();
    const bool live = kCta || row < rows;
    const float u = u_next, gs0 = gs, hs0 = hs, ghs0 = ghs;
    SumMax t = {0.0f, 0.0f};
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      if (!live || p.column(v) < 0) continue;
      float g[kWidth], hf[kWidth];
      unpack<T>(*ring.at(stage, 0, v), g);
      unpack<T>(*ring.at(stage, 1, v), hf);
#pragma unroll
      for (int e = 0; e < kWidth; ++e) {
        const float d = g[e] * (hf[e] * u);
        t.sum += d * wv[v * kWidth + e];
        dw[v * kWidth + e] += d;
      }
    }
    if (has_single && live) {
      const float d = gs0 * (hs0 * u);
      t.sum += d * ws;
      dws += d;
    }
    fetch_single(row + p.step);
    t = group_reduce<kCta, true, false>(t, p.group, red, turn);
    const float k = t.sum * inv_cols * u;
    // the row is read a second time from its slots: held in registers it would spill
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const int c = p.column(v);
      if (!live || c < 0) continue;
      float g[kWidth], hf[kWidth], add[kWidth] = {};
      unpack<T>(*ring.at(stage, 0, v), g);
      unpack<T>(*ring.at(stage, 1, v), hf);
      if (gh) unpack<T>(*ring.at(stage, 2, v), add);
#pragma unroll
      for (int e = 0; e < kWidth; ++e) add[e] += (g[e] * wv[v * kWidth + e] - hf[e] * k) * u;
      *reinterpret_cast<uint4*>(dx + row * cols + c) = pack<T>(add);
    }
    if (has_single && live) dx[row * cols + p.single] = Elem<T>::from_f((gs0 * ws - hs0 * k) * u + ghs0);
    fetch(row + kStages * p.step, stage);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  ring.drain();
  if (part == nullptr) return;
  float* out = part + (int64_t)blockIdx.x * cols;
  float* mine = out;
  float* sums = reinterpret_cast<float*>(smem);  // [groups of the CTA][cols], the ring is done
  if (!kCta) {
    __syncthreads();
    mine = sums + (int)(threadIdx.x / p.group) * cols;
  }
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    const int c = p.column(v);
    if (c < 0) continue;
#pragma unroll
    for (int e = 0; e < kWidth; ++e) mine[c + e] = dw[v * kWidth + e];
  }
  if (has_single) mine[p.single] = dws;
  if (!kCta) {
    __syncthreads();
    const int groups = blockDim.x / p.group;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      float s = 0.0f;
      for (int i = 0; i < groups; ++i) s += sums[i * cols + c];
      out[c] = s;
    }
  }
}

// dL/dw = sum of the partial sums: 32 columns a CTA, 32 threads a column, in a fixed order.
__global__ void __launch_bounds__(1024)
    weight_sum_kernel(const float* __restrict__ part, int parts, int cols, float* __restrict__ dw) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < cols)
    for (int i = group; i < parts; i += 32) s += part[(int64_t)i * cols + c];
  red[group][lane] = s;
  __syncthreads();
  s = warp_sum(red[lane][group]);
  if (lane == 0 && blockIdx.x * 32 + group < cols) dw[blockIdx.x * 32 + group] = s;
}

// ------------------------------------------- rows of any width, alignment and stride
// One CTA per row, element by element: rows of more than 16,384 columns, and rows whose tensors start
// differently in 16 bytes.  The row is read again for its outputs, by the backward's weight gradient a third time.  4,000
// rows of 16,392 bf16 columns: forward 131 us, 8-bit rows 125, backward 382 in three kernels; of
// 16,384 columns in the kernels above 86, 79 and 99.
template <typename T, bool kQuant>
__global__ void __launch_bounds__(kThreads)
    fwd_any_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ r, int64_t ldr,
                   const float* __restrict__ w, float eps, int normalize, int cols, void* __restrict__ y,
                   T* h, float* __restrict__ aux) {
  __shared__ SumMax red[2][32];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  const T* rr = r ? r + row * ldr : nullptr;
  T* hr = h ? h + row * cols : nullptr;
  SumMax t = {0.0f, 0.0f};
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    T v = xr[c];
    if (rr) {
      v = Elem<T>::from_f(Elem<T>::to_f(v) + Elem<T>::to_f(rr[c]));
      hr[c] = v;
    }
    const float f = Elem<T>::to_f(v);
    t.sum += f * f;
    if (kQuant) t.max = max_nan(t.max, fabsf(w ? f * w[c] : f));
  }
  t = group_reduce<true, true, kQuant>(t, kThreads, red, 0);
  const T* src = rr ? hr : xr;  // each thread reads back what it wrote
  float down = 1.0f;
  if (normalize && t.sum > kFloatMax) {
    down = kDown;
    t = {0.0f, 0.0f};
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      const float f = Elem<T>::to_f(src[c]) * down;
      t.sum += f * f;
      if (kQuant) t.max = max_nan(t.max, fabsf(w ? f * w[c] : f));
    }
    t = group_reduce<true, true, kQuant>(t, kThreads, red, 1);
  }
  const float u = normalize ? rsqrtf(t.sum / (float)cols + eps * down * down) : 1.0f;  // of the row times `down`
  if constexpr (kQuant) {
    const Quant q = quantizer(t, u);
    uint8_t* out = static_cast<uint8_t*>(y) + row * cols;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      const float f = Elem<T>::to_f(src[c]) * down;
      out[c] = (uint8_t)e4m3x2((w ? f * w[c] : f) * q.factor, 0.0f);
    }
    if (threadIdx.x == 0) aux[row] = q.scale;
  } else {
    T* out = static_cast<T*>(y) + row * cols;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      const float f = Elem<T>::to_f(src[c]) * down * u;
      out[c] = Elem<T>::from_f(w ? f * w[c] : f);
    }
    if (threadIdx.x == 0 && aux) aux[row] = u * down;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    bwd_any_kernel(const T* __restrict__ gy, int64_t ldgy, const T* __restrict__ h, int64_t ldh,
                   const T* __restrict__ gh, int64_t ldgh, const float* __restrict__ w,
                   const float* __restrict__ rstd, int cols, T* __restrict__ dx) {
  __shared__ SumMax red[2][32];
  const int64_t row = blockIdx.x;
  const T* gr = gy + row * ldgy;
  const T* hr = h + row * ldh;
  SumMax t = {0.0f, 0.0f};
  const float u = rstd[row];
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    const float g = Elem<T>::to_f(gr[c]);
    t.sum += (w ? g * w[c] : g) * (Elem<T>::to_f(hr[c]) * u);
  }
  t = group_reduce<true, true, false>(t, kThreads, red, 0);
  const float k = t.sum / (float)cols * u;
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    const float g = Elem<T>::to_f(gr[c]);
    float d = ((w ? g * w[c] : g) - Elem<T>::to_f(hr[c]) * k) * u;
    if (gh) d += Elem<T>::to_f(gh[row * ldgh + c]);
    dx[row * cols + c] = Elem<T>::from_f(d);
  }
}

// Partial sums of dL/dw over slabs of `per` rows (blockIdx.y), one thread per column.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    weight_any_kernel(const T* __restrict__ gy, int64_t ldgy, const T* __restrict__ h, int64_t ldh,
                      const float* __restrict__ rstd, int64_t rows, int cols, int64_t per,
                      float* __restrict__ part) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= cols) return;
  const int64_t r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
  float s = 0.0f;
  for (int64_t i = r0; i < r1; ++i)
    s += Elem<T>::to_f(gy[i * ldgy + c]) * (Elem<T>::to_f(h[i * ldh + c]) * rstd[i]);
  part[(int64_t)blockIdx.y * cols + c] = s;
}

// ------------------------------------------------------------------ host
struct Operand {
  const void* ptr;  // NULL: absent
  int64_t ld;
};

// How a call runs: by whole vectors, by vectors between single elements, or element by element.
struct Plan {
  bool any = true, shift = false, cta = false;
  int per = 8, group = 32, threads = kThreads, per_cta = 1, align = 1, depth = 1, grid = 0;
  size_t ring = 0, smem = 0;
};

constexpr int kMaxPerSm = 16, kMaxParts = kMaxPerSm * kSms + 8;  // CTAs of a persistent launch, at most

// `tensors`: the row tensors of one element size, the first `loaded` of them inputs.  Vectors need rows that
// start alike in 16 bytes: all aligned (with whole vectors to a row), or all shifted alike.
//
// A thread takes 8 elements of a row, or 16 where 8 would need more than `wide` threads: fewer
// warps to a barrier and more CTAs to an SM, against more rows on their way and fewer idle lanes in
// narrow rows.  Measured at 1,024 / 2,048 / 4,096 columns (us, 8 against 16 a thread):
//   bf16, 120 M elements: forward 165 / 157 / 165 against 147 / 148 / 146,
//     8-bit 141 / 135 / 130 against 132 / 129 / 128, backward 145 / 146 / 149 against 150 / 147 / 153
//   fp32, 60 M elements: forward 156 / 158 / 163 against 150 / 151 / 158,
//     8-bit 130 / 127 / 118 against 117 / 118 / 117, backward 155 / 153 / 143 against 141 / 139 / 144
// and at 768 columns (8 M bf16 elements) forward 11.6 against 13.7, 8-bit 12.4 against 13.6; bf16
// backward at 5,120: 173 against 149.  Hence 96, for the bf16 backward 512.  It is not best everywhere: at
// 5,120 columns 8 a thread takes 146 us against 153 in the bf16 forward, 142 against 154 in the fp32 backward.
// A row of up to 32 threads' elements, 8 each, goes to a power-of-two group of lanes.
template <size_t kSize>
Plan plan_rows(const Operand* tensors, int count, int64_t rows, int cols, int loaded, int wide) {
  constexpr int kWidth = 16 / (int)kSize;
  Plan p;
  const auto off = [](const void* q) { return (unsigned)(reinterpret_cast<uintptr_t>(q) & 15); };
  bool aligned = cols % kWidth == 0, alike = true;
  for (int i = 0; i < count; ++i) {
    if (tensors[i].ptr == nullptr) continue;
    aligned = aligned && off(tensors[i].ptr) == 0 && (rows == 1 || tensors[i].ld % kWidth == 0);
    alike = alike && off(tensors[i].ptr) == off(tensors[0].ptr) && off(tensors[i].ptr) % kSize == 0 &&
            (rows == 1 || tensors[i].ld % kWidth == tensors[0].ld % kWidth);
  }
  if (!aligned && !alike) return p;
  p.shift = !aligned;
  const int need = (cols + 7) / 8;
  // Shifted rows: 16 a thread helps the bf16 backward too (1,535 columns 313 -> 183 us), but not the
  // fp32 one, which then has one row on its way (18 -> 22 us at 4,095 x 1,535).
  if (p.shift) wide = kSize == 4 && loaded == 3 ? 256 : 128;
  p.per = need > wide ? 16 : 8;
  const int lanes = (cols + p.per - 1) / p.per;  // threads that a row keeps busy
  if (lanes > 1024) return p;
  p.any = false;
  if (lanes <= 32) {
    // the single elements (fewer than two vectors) need a lane each
    p.group = p.shift ? 2 * kWidth : 1;
    while (p.group < lanes) p.group *= 2;
  } else {
    p.cta = true;
    p.threads = (lanes + 31) / 32 * 32;
  }
  const int per_cta = p.cta ? 1 : p.threads / p.group;
  // the ring, and room for a sum of dL/dw from each group
  const int bytes = p.per * (int)kSize;
  p.depth = stages(bytes);
  p.smem = (size_t)loaded * p.depth * bytes * p.threads;
  const size_t sums = p.cta ? 0 : (size_t)per_cta * cols * sizeof(float);
  int present = 0;
  for (int i = 0; i < loaded; ++i) present += tensors[i].ptr != nullptr;
  p.ring = p.smem / loaded * present;
  if (p.smem < sums) p.smem = sums;
  p.per_cta = per_cta;
  p.align = p.shift ? kWidth : 1;
  return p;
}

// The persistent grid: as many CTAs an SM as keep `budget` bytes of rows on their way, and two
// (one computes while the other waits at its barrier) if that is at most 80 KB.  More bytes are
// worse where the kernel also writes much: 120 M bf16 elements in 2,048 columns forward (half of
// the traffic writes) took 148 us with 48 KB an SM and 174 us with 96 KB; 8-bit rows in 4,096
// columns 128 us with 64 KB and 148 us with 96 KB; the backward (a quarter writes) wants all that
// fit.  So the forward has one row of a group on its way where a second one would leave the budget
// to a single CTA: 5,120 columns 153 against 173 us, 8-bit rows 130 against 135 us.
void size_grid(Plan& p, int64_t rows, int budget, int regs, bool forward) {
  if (p.shift) budget = 180 << 10;  // their single elements are loaded a row ahead only
  if (forward && p.cta && p.depth == 2 && (int)p.ring < budget && 2 * (int)p.ring > budget) {
    p.depth = 1;
    p.ring /= 2;
    p.smem /= 2;
  }
  const int fit[] = {65536 / (((regs + 7) / 8 * 8) * p.threads), 2048 / p.threads, (int)((220 << 10) / (p.smem + 1024)),
                     kMaxPerSm};
  int per_sm = budget / (int)p.ring;
  if (per_sm < 2) per_sm = p.ring <= 40 << 10 ? 2 : 1;
  for (int f : fit) per_sm = per_sm < f ? per_sm : f;
  if (per_sm < 1) per_sm = 1;
  const int64_t want = (rows + p.per_cta - 1) / p.per_cta;
  p.grid = (int)(want < per_sm * kSms ? want : per_sm * kSms);
  // groups' rows shifted alike: the row step is a multiple of the shifts' period (rounded down where the
  // CTAs that this adds would wait for the others' SMs)
  if (p.grid * p.per_cta % p.align != 0) {
    const int up = (p.grid + p.align - 1) / p.align * p.align;
    p.grid = up <= per_sm * kSms ? up : up - p.align;
  }
}

template <typename K>
int registers_of(K kernel) {
  cudaFuncAttributes a;
  return cudaFuncGetAttributes(&a, kernel) == cudaSuccess ? a.numRegs : 64;
}

// The limit is the kernel's, not the launch's, and calls from other threads set it too: always to `most`,
// what any plan of this kernel asks for at most.
template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes, size_t most) {
  return bytes > (40 << 10)  // 48 KB without asking, static arrays included
             ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most)
             : cudaSuccess;
}
constexpr size_t most_smem(int tensors, int per, int size, bool cta) {
  return (size_t)tensors * stages(per * size) * per * size * (cta ? 1024 : kThreads);
}
static_assert(most_smem(3, 16, 4, true) <= 220 << 10, "a CTA's shared memory");

// Calls fn with the plan's compile-time choices: fn(elements a thread, CTA rows, shifted rows).
template <typename F>
cudaError_t with_plan(const Plan& p, F&& fn) {
  using std::integral_constant;
  const auto shift = [&](auto per, auto cta) {
    return p.shift ? fn(per, cta, integral_constant<bool, true>{}) : fn(per, cta, integral_constant<bool, false>{});
  };
  using std::true_type;
  if (p.per == 16) return shift(integral_constant<int, 16>{}, true_type{});  // wide rows
  return p.cta ? shift(integral_constant<int, 8>{}, true_type{}) : shift(integral_constant<int, 8>{}, std::false_type{});
}

template <typename T, bool kQuant>
cudaError_t forward(const T* x, int64_t ldx, const T* r, int64_t ldr, const float* w, float eps, int normalize,
                    int64_t rows, int cols, void* y, T* h, float* aux, cudaStream_t stream) {
  const Operand tensors[4] = {{x, ldx}, {r, ldr}, {h, cols}, {kQuant ? nullptr : y, cols}};
  Plan p = plan_rows<sizeof(T)>(tensors, 4, rows, cols, 2, 96);
  // whole vectors of bytes: the 8-bit rows start on their own vectors' boundaries
  if (kQuant && !p.any && !p.shift && reinterpret_cast<uintptr_t>(y) % (16 / sizeof(T)) != 0) p.any = true;
  if (p.any) {
    fwd_any_kernel<T, kQuant><<<(unsigned)rows, kThreads, 0, stream>>>(x, ldx, r, ldr, w, eps, normalize, cols, y, h,
                                                                       aux);
    return cudaGetLastError();
  }
  const auto run = [&](auto norm) {
    return with_plan(p, [&](auto per, auto cta, auto shift) {
      const auto kernel = fwd_kernel<T, per(), cta(), shift(), kQuant, norm()>;
      static const int regs = registers_of(kernel);
      size_grid(p, rows, kQuant ? 64 << 10 : 48 << 10, regs, true);
      const cudaError_t e = allow_smem(kernel, p.smem, most_smem(2, per(), sizeof(T), cta()));
      if (e != cudaSuccess) return e;
      kernel<<<p.grid, p.threads, p.smem, stream>>>(x, ldx, r, ldr, w, eps, rows, cols, p.group, p.depth, y, h, aux);
      return cudaGetLastError();
    });
  };
  if constexpr (kQuant)
    if (!normalize) return run(std::false_type{});
  return run(std::true_type{});
}

template <typename T>
cudaError_t backward(const T* gy, int64_t ldgy, const T* h, int64_t ldh, const T* gh, int64_t ldgh, const float* w,
                     const float* rstd, int64_t rows, int cols, T* dx, float* part, float* dw, cudaStream_t stream) {
  const Operand tensors[4] = {{gy, ldgy}, {h, ldh}, {gh, ldgh}, {dx, cols}};
  Plan p = plan_rows<sizeof(T)>(tensors, 4, rows, cols, 3, sizeof(T) == 2 ? 512 : 96);
  int parts = 0;
  if (p.any) {
    bwd_any_kernel<T><<<(unsigned)rows, kThreads, 0, stream>>>(gy, ldgy, h, ldh, gh, ldgh, w, rstd, cols, dx);
    if (dw) {
      const int64_t slabs = rows < kMaxParts ? rows : kMaxParts, per = (rows + slabs - 1) / slabs;
      parts = (int)slabs;
      weight_any_kernel<T><<<dim3((unsigned)((cols + kThreads - 1) / kThreads), (unsigned)slabs), kThreads, 0, stream>>>(
          gy, ldgy, h, ldh, rstd, rows, cols, per, part);
    }
  } else {
    const cudaError_t e = with_plan(p, [&](auto per, auto cta, auto shift) {
      const auto kernel = bwd_kernel<T, per(), cta(), shift()>;
      static const int regs = registers_of(kernel);
      size_grid(p, rows, 180 << 10, regs, false);
      parts = p.grid;
      const cudaError_t a = allow_smem(kernel, p.smem, most_smem(3, per(), sizeof(T), cta()));
      if (a != cudaSuccess) return a;
      kernel<<<p.grid, p.threads, p.smem, stream>>>(gy, ldgy, h, ldh, gh, ldgh, w, rstd, rows, cols, p.group, dx,
                                                    dw ? part : nullptr);
      return cudaGetLastError();
    });
    if (e != cudaSuccess) return e;
  }
  if (dw) weight_sum_kernel<<<(unsigned)((cols + 31) / 32), 1024, 0, stream>>>(part, parts, cols, dw);
  return cudaGetLastError();
}

bool rows_ok(int64_t rows, int cols) {
  return rows >= 0 && rows < ((int64_t)1 << 31) && cols >= 1 && cols < (1 << 30);
}

}  // namespace norm
}  // namespace prism

using namespace prism;

extern "C" {

prism_status_t prism_add_rms_norm(const void* x, int64_t ldx, const void* r, int64_t ldr,
                                  const float* weight, float eps, int64_t rows, int cols, int dtype,
                                  void* y, void* h, float* rstd, cudaStream_t stream) {
  PRISM_CHECK_ARG(norm::rows_ok(rows, cols) && ldx >= 0 && ldr >= 0, "prism_add_rms_norm: bad sizes");
  if (rows == 0) return PRISM_OK;
  PRISM_CHECK_ARG(x && y && (r == nullptr) == (h == nullptr),
                  "prism_add_rms_norm: null pointer (h goes with r)");
  cudaError_t err = cudaSuccess;
  const bool known = dispatch_dtype(dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    err = norm::forward<T, false>((const T*)x, ldx, (const T*)r, ldr, weight, eps, 1, rows, cols, y, (T*)h, rstd,
                                  stream);
  });
  PRISM_CHECK_ARG(known, "prism_add_rms_norm: unknown element type %d", dtype);
  PRISM_CHECK_CUDA(err, "prism_add_rms_norm");
  return PRISM_OK;
}

prism_status_t prism_add_rms_norm_fp8(const void* x, int64_t ldx, const void* r, int64_t ldr,
                                      const float* weight, float eps, int normalize, int64_t rows,
                                      int cols, int dtype, void* y8, float* scale, void* h,
                                      cudaStream_t stream) {
  PRISM_CHECK_ARG(norm::rows_ok(rows, cols) && ldx >= 0 && ldr >= 0, "prism_add_rms_norm_fp8: bad sizes");
  if (rows == 0) return PRISM_OK;
  PRISM_CHECK_ARG(x && y8 && scale && (r == nullptr) == (h == nullptr),
                  "prism_add_rms_norm_fp8: null pointer (h goes with r)");
  cudaError_t err = cudaSuccess;
  const bool known = dispatch_dtype(dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    err = norm::forward<T, true>((const T*)x, ldx, (const T*)r, ldr, weight, eps, normalize, rows, cols, y8, (T*)h,
                                 scale, stream);
  });
  PRISM_CHECK_ARG(known, "prism_add_rms_norm_fp8: unknown element type %d", dtype);
  PRISM_CHECK_CUDA(err, "prism_add_rms_norm_fp8");
  return PRISM_OK;
}

size_t prism_add_rms_norm_bwd_workspace_bytes(int64_t rows, int cols) {
  // a partial sum of dL/dw for each CTA; rows shifted in 16 bytes round the CTAs up to 8
  const int64_t parts = rows + 8 < norm::kMaxParts ? rows + 8 : norm::kMaxParts;
  return rows <= 0 || cols <= 0 ? 0 : (size_t)parts * (size_t)cols * sizeof(float);
}

prism_status_t prism_add_rms_norm_bwd(const void* gy, int64_t ldgy, const void* h, int64_t ldh,
                                      const void* gh, int64_t ldgh, const float* weight,
                                      const float* rstd, int64_t rows, int cols, int dtype, void* dx,
                                      void* workspace, float* dweight, cudaStream_t stream) {
  PRISM_CHECK_ARG(norm::rows_ok(rows, cols) && ldgy >= 0 && ldh >= 0 && ldgh >= 0,
                  "prism_add_rms_norm_bwd: bad sizes");
  PRISM_CHECK_ARG(rows == 0 || (gy && h && rstd && dx && (dweight == nullptr || workspace)),
                  "prism_add_rms_norm_bwd: null pointer");
  if (rows == 0) {
    if (dweight)
      PRISM_CHECK_CUDA(cudaMemsetAsync(dweight, 0, sizeof(float) * cols, stream), "prism_add_rms_norm_bwd");
    return PRISM_OK;
  }
  cudaError_t err = cudaSuccess;
  const bool known = dispatch_dtype(dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    err = norm::backward<T>((const T*)gy, ldgy, (const T*)h, ldh, (const T*)gh, ldgh, weight, rstd, rows, cols,
                            (T*)dx, (float*)workspace, dweight, stream);
  });
  PRISM_CHECK_ARG(known, "prism_add_rms_norm_bwd: unknown element type %d", dtype);
  PRISM_CHECK_CUDA(err, "prism_add_rms_norm_bwd");
  return PRISM_OK;
}

}  // extern "C"
