// Global gradient norm over many tensors, and clipping:
//   norm = sqrt(sum over tensors of sum g^2),  f = min(1, max_norm / (norm + 1e-6)),  g' = f g.
// Sums of squares are held in fp64: fp32 squares lose gradients below 1e-23 and overflow above
// 1.8e19.  Every sum has a fixed order.
//
// The tensors' addresses and sizes travel as a kernel parameter (no device table to fill, keep
// or race on), kTable tensors a launch; each tensor is cut into chunks of kChunk elements.
#include <math.h>

#include "block_ops.cuh"

namespace prism {
namespace clip {

constexpr int kThreads = 256;
constexpr int kTable = 1000;
constexpr int64_t kChunk = 32768;

struct Table {
  const void* in[kTable];
  void* out[kTable];
  int64_t n[kTable];
  int first[kTable + 1];  // first chunk of each tensor
  uint8_t dtype[kTable];
  int count;
};
static_assert(sizeof(Table) + 128 <= 32764, "the table is a kernel parameter");

__device__ __forceinline__ int tensor_of_chunk(const Table& t, int chunk) {
  int lo = 0, hi = t.count;  // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double red[kThreads / 32];
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < kThreads / 32; ++i) s += red[i];
  return s;
}

template <typename T>
__device__ __forceinline__ double sum_squares(const T* g, int64_t n) {
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += kThreads) {
    const double v = (double)Elem<T>::to_f(g[i]);
    s += v * v;
  }
  return s;
}

// One CTA per chunk: its sum of squares.
__global__ void __launch_bounds__(kThreads)
    square_kernel(const __grid_constant__ Table t, double* __restrict__ part) {
  const int k = tensor_of_chunk(t, blockIdx.x);
  const int64_t at = (blockIdx.x - t.first[k]) * kChunk, n = min(kChunk, t.n[k] - at);
  double s;
  if (t.dtype[k] == PRISM_BF16) s = sum_squares((const __nv_bfloat16*)t.in[k] + at, n);
  else if (t.dtype[k] == PRISM_FP16) s = sum_squares((const __half*)t.in[k] + at, n);
  else s = sum_squares((const float*)t.in[k] + at, n);
  s = block_sum(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// norm_factor[0] = norm, [1] = the factor.
__global__ void __launch_bounds__(kThreads)
    norm_kernel(const double* __restrict__ part, int64_t chunks, float max_norm, float* __restrict__ norm,
                float* __restrict__ factor) {
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < chunks; i += kThreads) s += part[i];
  s = block_sum(s);
  if (threadIdx.x == 0) {
    const float v = (float)sqrt(s);
    *norm = v;
    const float f = max_norm / (v + 1e-6f);
    *factor = f > 1.0f ? 1.0f : f;  // a NaN norm stays a NaN factor
  }
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const T* g, T* out, int64_t n, float f) {
  for (int64_t i = threadIdx.x; i < n; i += kThreads) out[i] = Elem<T>::from_f(Elem<T>::to_f(g[i]) * f);
}

__global__ void __launch_bounds__(kThreads)
    scale_kernel(const __grid_constant__ Table t, const float* __restrict__ factor) {
  const int k = tensor_of_chunk(t, blockIdx.x);
  const float f = *factor;
  if (f == 1.0f && t.in[k] == t.out[k]) return;  // in place, nothing to clip
  const int64_t at = (blockIdx.x - t.first[k]) * kChunk, n = min(kChunk, t.n[k] - at);
  if (t.dtype[k] == PRISM_BF16) scale_chunk((const __nv_bfloat16*)t.in[k] + at, (__nv_bfloat16*)t.out[k] + at, n, f);
  else if (t.dtype[k] == PRISM_FP16) scale_chunk((const __half*)t.in[k] + at, (__half*)t.out[k] + at, n, f);
  else scale_chunk((const float*)t.in[k] + at, (float*)t.out[k] + at, n, f);
}

inline int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// Calls fn(table, chunks) for each group of at most kTable non-empty tensors.
template <typename F>
inline void for_tables(const void* const* in, void* const* out, const int64_t* n, const int* dtype, int64_t count,
                       F&& fn) {
  Table t;
  t.count = 0;
  int64_t chunks = 0;
  for (int64_t i = 0; i <= count; ++i) {
    const int64_t c = i < count ? chunks_of(n[i]) : 0;
    if (t.count > 0 && (i == count || t.count == kTable || chunks + c > 0x7fffffff)) {
      t.first[t.count] = (int)chunks;
      fn(t, (int)chunks);
      t.count = 0, chunks = 0;
    }
    if (c == 0) continue;
    t.in[t.count] = in[i], t.out[t.count] = out[i], t.n[t.count] = n[i];
    t.dtype[t.count] = (uint8_t)dtype[i], t.first[t.count] = (int)chunks;
    ++t.count;
    chunks += c;
  }
}

}  // namespace clip
}  // namespace prism

using namespace prism;

extern "C" {

size_t prism_clip_grad_norm_workspace_bytes(const int64_t* sizes, int64_t count) {
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) chunks += clip::chunks_of(sizes[i]);
  return (size_t)chunks * sizeof(double) + 16;
}

prism_status_t prism_clip_grad_norm(const void* const* grads, void* const* outs, const int64_t* sizes,
                                    const int* dtypes, int64_t count, float max_norm, void* workspace,
                                    float* norm, cudaStream_t stream) {
  PRISM_CHECK_ARG(count >= 0 && norm && workspace && (count == 0 || (grads && outs && sizes && dtypes)),
                  "prism_clip_grad_norm: null pointer");
  PRISM_CHECK_ARG(max_norm >= 0.0f, "prism_clip_grad_norm: max_norm must not be negative");
  for (int64_t i = 0; i < count; ++i) {
    PRISM_CHECK_ARG(sizes[i] >= 0 && (sizes[i] == 0 || (grads[i] && outs[i])),
                    "prism_clip_grad_norm: tensor %lld has no data or a negative size", (long long)i);
    PRISM_CHECK_ARG(dtypes[i] >= PRISM_BF16 && dtypes[i] <= PRISM_FP32,
                    "prism_clip_grad_norm: unknown element type %d", dtypes[i]);
  }
  float* factor = (float*)workspace;
  double* part = (double*)((char*)workspace + 16);
  int64_t done = 0;
  clip::for_tables(grads, outs, sizes, dtypes, count, [&](const clip::Table& t, int chunks) {
    clip::square_kernel<<<chunks, clip::kThreads, 0, stream>>>(t, part + done);
    done += chunks;
  });
  clip::norm_kernel<<<1, clip::kThreads, 0, stream>>>(part, done, max_norm, norm, factor);
  clip::for_tables(grads, outs, sizes, dtypes, count, [&](const clip::Table& t, int chunks) {
    clip::scale_kernel<<<chunks, clip::kThreads, 0, stream>>>(t, factor);
  });
  PRISM_CHECK_LAUNCH("prism_clip_grad_norm");
  return PRISM_OK;
}

}  // extern "C"
