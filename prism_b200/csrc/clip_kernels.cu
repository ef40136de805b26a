// Global gradient norm over many tensors, and clipping:
//   norm = sqrt(sum over tensors of sum g^2),  f = min(1, max_norm / (norm + 1e-6)),  g' = f g.
// Squares and sums are held in fp64: fp32 squares lose gradients below 1e-23 and overflow above
// 1.8e19, and the conversions hide under the loads.  Every sum has a fixed order.
//
// Two launches: the sums of squares, a partial sum a CTA, and the scaling, in which every CTA adds
// up the partial sums by itself.  The tensors' addresses and sizes travel as a kernel parameter (no
// device table to fill, keep or race on); each tensor is cut into chunks of kChunk elements, and a
// CTA takes an equal share of consecutive chunks, so that one large tensor, or a thousand small
// ones, spread over all SMs.
//
// Bound by memory: both passes read the gradients (what L2 keeps of a 0.5 GB set between the
// passes is not worth an order: reading backwards took 152 us instead of 154).
#include <math.h>

#include "block_ops.cuh"

namespace prism {
namespace clip {

constexpr int kThreads = 256;
constexpr int kBlocksPerSm = 4;             // 64 registers a thread
constexpr int kBlocks = kBlocksPerSm * 148;  // CTAs of a launch
constexpr int64_t kChunk = 4096;
// 16-byte loads in flight a thread: four for the sums, two where stores share the registers.
constexpr int kSumUnroll = 4, kScaleUnroll = 2;

// Tensors of one launch.  A launch copies its parameters whole, so a short list has its own size.
constexpr int kSmallTable = 100, kTable = 1000;
template <int kMax>
struct Table {
  const void* in[kMax];
  void* out[kMax];
  int64_t n[kMax];
  int first[kMax + 1];  // first chunk of each tensor
  uint8_t dtype[kMax];
  int count;
};
static_assert(sizeof(Table<kTable>) + 128 <= 32764, "the table is a kernel parameter");

template <int kMax>
__device__ __forceinline__ int tensor_of_chunk(const Table<kMax>& t, int chunk) {
  int lo = 0, hi = t.count;  // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The CTA's share of the launch's chunks as runs of consecutive elements of one tensor:
// fn(tensor, offset, elements).
template <int kMax, typename F>
__device__ __forceinline__ void for_runs(const Table<kMax>& t, int chunks, F&& fn) {
  int c = (int)((int64_t)chunks * blockIdx.x / gridDim.x);
  const int last = (int)((int64_t)chunks * (blockIdx.x + 1) / gridDim.x);
  if (c == last) return;
  for (int k = tensor_of_chunk(t, c); c < last;) {
    // 2^16 chunks at most: the element counts below stay 32-bit
    const int end = min(min(last, t.first[k + 1]), c + (1 << 16));
    const int64_t at = (int64_t)(c - t.first[k]) * kChunk;
    fn(k, at, (int)min((int64_t)(end - c) * kChunk, t.n[k] - at));
    c = end;
    if (c == t.first[k + 1]) ++k;
  }
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double red[kThreads / 32];
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < kThreads / 32; ++i) s += red[i];
  return s;
}

// For every index below n that is this thread's, kUnroll at a time: load(i, u) for all of them,
// then use(i, u).
template <int kUnroll, typename Load, typename Use>
__device__ __forceinline__ void strided(int n, Load&& load, Use&& use) {
  for (int i = threadIdx.x; i < n; i += kUnroll * kThreads) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i + u * kThreads < n) load(i + u * kThreads, u);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i + u * kThreads < n) use(i + u * kThreads, u);
  }
}

template <typename T>
__device__ __forceinline__ double sum_squares(const T* g, int n) {
  constexpr int kWidth = 16 / sizeof(T);
  double s = 0.0;
  const auto add = [&](float x) {
    const double v = (double)x;
    s = fma(v, v, s);
  };
  int done = 0;
  if (is_aligned16(g)) {
    const auto* gv = reinterpret_cast<const uint4*>(g);
    uint4 buf[kSumUnroll];
    strided<kSumUnroll>(n / kWidth, [&](int i, int u) { buf[u] = gv[i]; },
                        [&](int, int u) {
                          float f[kWidth];
                          unpack<T>(buf[u], f);
#pragma unroll
                          for (int e = 0; e < kWidth; ++e) add(f[e]);
                        });
    done = n / kWidth * kWidth;
  }
  float buf[kSumUnroll];
  strided<kSumUnroll>(n - done, [&](int i, int u) { buf[u] = Elem<T>::to_f(g[done + i]); },
                      [&](int, int u) { add(buf[u]); });
  return s;
}

template <typename T>
__device__ __forceinline__ void scale_run(const T* g, T* out, int n, float f) {
  constexpr int kWidth = 16 / sizeof(T);
  int done = 0;
  if (is_aligned16(g) && is_aligned16(out)) {
    const auto* gv = reinterpret_cast<const uint4*>(g);
    auto* ov = reinterpret_cast<uint4*>(out);
    uint4 buf[kScaleUnroll];
    strided<kScaleUnroll>(n / kWidth, [&](int i, int u) { buf[u] = gv[i]; },
                          [&](int i, int u) {
                            float v[kWidth];
                            unpack<T>(buf[u], v);
#pragma unroll
                            for (int e = 0; e < kWidth; ++e) v[e] *= f;
                            ov[i] = pack<T>(v);
                          });
    done = n / kWidth * kWidth;
  }
  constexpr int kUnroll = 8;  // single elements
  float buf[kUnroll];
  strided<kUnroll>(n - done, [&](int i, int u) { buf[u] = Elem<T>::to_f(g[done + i]); },
                   [&](int i, int u) { out[done + i] = Elem<T>::from_f(buf[u] * f); });
}

// Sum of squares of each CTA's share -> part[CTA].
template <int kMax>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    square_kernel(const __grid_constant__ Table<kMax> t, int chunks, double* __restrict__ part) {
  double s = 0.0;
  for_runs(t, chunks, [&](int k, int64_t at, int n) {
    if (t.dtype[k] == PRISM_BF16) s += sum_squares((const __nv_bfloat16*)t.in[k] + at, n);
    else if (t.dtype[k] == PRISM_FP16) s += sum_squares((const __half*)t.in[k] + at, n);
    else s += sum_squares((const float*)t.in[k] + at, n);
  });
  s = block_sum(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// Every CTA adds up the partial sums, in the same order, and scales its share.
template <int kMax>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    scale_kernel(const __grid_constant__ Table<kMax> t, int chunks, const double* __restrict__ part, int parts,
                 float max_norm, float* __restrict__ norm) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) s += part[i];
  const float v = (float)sqrt(block_sum(s));
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
  float f = max_norm / (v + 1e-6f);
  f = f > 1.0f || isinf(max_norm) ? 1.0f : f;  // a NaN norm stays a NaN factor
  for_runs(t, chunks, [&](int k, int64_t at, int n) {
    if (f == 1.0f && t.in[k] == t.out[k]) return;  // in place, nothing to clip
    if (t.dtype[k] == PRISM_BF16) scale_run((const __nv_bfloat16*)t.in[k] + at, (__nv_bfloat16*)t.out[k] + at, n, f);
    else if (t.dtype[k] == PRISM_FP16) scale_run((const __half*)t.in[k] + at, (__half*)t.out[k] + at, n, f);
    else scale_run((const float*)t.in[k] + at, (float*)t.out[k] + at, n, f);
  });
}

inline int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// Calls fn(table, chunks) for each group of at most kMax non-empty tensors.
template <int kMax, typename F>
inline void for_tables(const void* const* in, void* const* out, const int64_t* n, const int* dtype, int64_t count,
                       F&& fn) {
  Table<kMax> t;
  t.count = 0;
  int64_t chunks = 0;
  for (int64_t i = 0; i <= count; ++i) {
    const int64_t c = i < count ? chunks_of(n[i]) : 0;
    if (t.count > 0 && (i == count || t.count == kMax)) {
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

template <int kMax>
inline void launch(const void* const* grads, void* const* outs, const int64_t* sizes, const int* dtypes, int64_t count,
                   float max_norm, double* part, float* norm, cudaStream_t stream) {
  int parts = 0;
  for_tables<kMax>(grads, outs, sizes, dtypes, count, [&](const Table<kMax>& t, int chunks) {
    const int grid = chunks < kBlocks ? chunks : kBlocks;
    square_kernel<kMax><<<grid, kThreads, 0, stream>>>(t, chunks, part + parts);
    parts += grid;
  });
  for_tables<kMax>(grads, outs, sizes, dtypes, count, [&](const Table<kMax>& t, int chunks) {
    const int grid = chunks < kBlocks ? chunks : kBlocks;
    scale_kernel<kMax><<<grid, kThreads, 0, stream>>>(t, chunks, part, parts, max_norm, norm);
  });
}

}  // namespace clip
}  // namespace prism

using namespace prism;

extern "C" {

size_t prism_clip_grad_norm_workspace_bytes(int64_t count) {
  // one partial sum a CTA, kTable tensors a launch
  return (size_t)((count > 0 ? count : 1) + clip::kTable - 1) / clip::kTable * clip::kBlocks * sizeof(double);
}

prism_status_t prism_clip_grad_norm(const void* const* grads, void* const* outs, const int64_t* sizes,
                                    const int* dtypes, int64_t count, float max_norm, void* workspace,
                                    float* norm, cudaStream_t stream) {
  PRISM_CHECK_ARG(count >= 0 && norm && workspace && (count == 0 || (grads && outs && sizes && dtypes)),
                  "prism_clip_grad_norm: null pointer");
  PRISM_CHECK_ARG(max_norm >= 0.0f, "prism_clip_grad_norm: max_norm must not be negative");
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    PRISM_CHECK_ARG(sizes[i] >= 0 && (sizes[i] == 0 || (grads[i] && outs[i])),
                    "prism_clip_grad_norm: tensor %lld has no data or a negative size", (long long)i);
    PRISM_CHECK_ARG(dtypes[i] >= PRISM_BF16 && dtypes[i] <= PRISM_FP32,
                    "prism_clip_grad_norm: unknown element type %d", dtypes[i]);
    chunks += clip::chunks_of(sizes[i]);
    PRISM_CHECK_ARG(chunks < ((int64_t)1 << 30), "prism_clip_grad_norm: too many elements");
  }
  if (chunks == 0) {  // no elements at all: the norm is 0
    PRISM_CHECK_CUDA(cudaMemsetAsync(norm, 0, sizeof(float), stream), "prism_clip_grad_norm");
    return PRISM_OK;
  }
  const auto launch = count <= clip::kSmallTable ? clip::launch<clip::kSmallTable> : clip::launch<clip::kTable>;
  launch(grads, outs, sizes, dtypes, count, max_norm, (double*)workspace, norm, stream);
  PRISM_CHECK_LAUNCH("prism_clip_grad_norm");
  return PRISM_OK;
}

}  // extern "C"
