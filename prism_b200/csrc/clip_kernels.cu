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

#include <algorithm>
#include <new>
#include <vector>

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

// What a call reads and writes.  A CTA scales what another may still read, so that memory that is written may
// belong to one entry only.
struct Run {
  uintptr_t begin, end;
};
struct Start {
  uintptr_t begin;
  int64_t tensor;
};
inline int64_t bytes_of(int dtype) { return dtype == PRISM_FP32 ? 4 : 2; }

// By address.  Longer lists as packed words, by 11 of the bits in which addresses differ at a time.
inline void sort_starts(std::vector<Start>& v) {
  const auto before = [](const Start& a, const Start& b) { return a.begin < b.begin; };
  if (std::is_sorted(v.begin(), v.end(), before)) return;
  uintptr_t low = v[0].begin, high = low, differ = 0;
  for (const Start& s : v) low = std::min(low, s.begin), high = std::max(high, s.begin), differ |= s.begin ^ v[0].begin;
  int skip = 0, bits = 0, index_bits = 0;
  while (!(differ >> skip & 1)) ++skip;
  while ((high - low) >> skip >> bits) ++bits;
  while (v.size() >> index_bits) ++index_bits;
  if (v.size() < 48 || bits + index_bits > 64) {
    std::sort(v.begin(), v.end(), before);
    return;
  }
  std::vector<uint64_t> keys(v.size()), other(v.size());
  for (size_t i = 0; i < v.size(); ++i) keys[i] = (uint64_t)((v[i].begin - low) >> skip) << index_bits | i;
  constexpr int kDigit = 11;
  for (int shift = index_bits; shift < index_bits + bits; shift += kDigit) {
    uint32_t at[(1 << kDigit) + 1] = {};
    for (uint64_t k : keys) ++at[(k >> shift & ((1 << kDigit) - 1)) + 1];
    for (int i = 0; i + 1 < 1 << kDigit; ++i) at[i + 1] += at[i];
    for (uint64_t k : keys) other[at[k >> shift & ((1 << kDigit) - 1)]++] = k;
    keys.swap(other);
  }
  std::vector<Start> sorted(v.size());
  for (size_t i = 0; i < v.size(); ++i) sorted[i] = v[keys[i] & ((1ull << index_bits) - 1)];
  v.swap(sorted);
}

// The lists of a call, as its checks see them.
struct Lists {
  const void* const* in;
  void* const* out;
  const int64_t* n;
  const int* dtype;
  int64_t count;
  bool measure;  // an infinite max_norm writes nothing in place

  bool written(int64_t i) const { return n[i] > 0 && !(measure && in[i] == out[i]); }
  bool read_only(int64_t i) const { return n[i] > 0 && (measure || in[i] != out[i]); }
  Run span(const void* p, int64_t i) const {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(p);
    return {begin, begin + n[i] * bytes_of(dtype[i])};
  }
};

// What is written, as a few disjoint runs in order of address: outputs that are slices of flat buffers, or
// short lists.  False where that does not work out.
inline bool few_runs(const Lists& l, std::vector<Run>& runs) {
  constexpr size_t kFew = 8;
  for (int64_t i = 0; i < l.count; ++i) {
    if (!l.written(i)) continue;
    const Run s = l.span(l.out[i], i);
    size_t r = 0;
    while (r < runs.size() && runs[r].end != s.begin) ++r;
    if (r < runs.size()) runs[r].end = s.end;
    else if (r < kFew) runs.push_back(s);
    else return false;
  }
  std::sort(runs.begin(), runs.end(), [](const Run& a, const Run& b) { return a.begin < b.begin; });
  for (size_t r = 1; r < runs.size(); ++r)
    if (runs[r].begin < runs[r - 1].end) return false;
  return true;
}

// Marks the entries that are scaled in place by another entry (repeated; empty where there are none).  Returns the
// index of an entry that shares memory otherwise, or -1.
inline int64_t check_overlap(const Lists& l, std::vector<uint8_t>& repeated) {
  std::vector<Run> runs;
  if (!few_runs(l, runs)) {
    runs.clear();
    std::vector<Start> writes;
    writes.reserve(l.count);
    for (int64_t i = 0; i < l.count; ++i)
      if (l.written(i)) writes.push_back({reinterpret_cast<uintptr_t>(l.out[i]), i});
    sort_starts(writes);
    runs.reserve(writes.size());
    int64_t last = -1;
    for (const Start& s : writes) {
      const int64_t i = s.tensor;
      if (last >= 0 && s.begin < runs.back().end) {
        const bool same = l.out[i] == l.out[last] && l.n[i] == l.n[last] && l.dtype[i] == l.dtype[last];
        if (!same || l.in[i] != l.out[i] || l.in[last] != l.out[last]) return i;
        if (repeated.empty()) repeated.assign(l.count, 0);
        repeated[i] = 1;
        continue;
      }
      last = i;
      runs.push_back(l.span(l.out[i], i));
    }
  }
  for (int64_t i = 0; i < l.count; ++i) {
    if (!l.read_only(i)) continue;
    // the last run that begins before the gradient ends
    const Run g = l.span(l.in[i], i);
    const auto after =
        std::lower_bound(runs.begin(), runs.end(), g.end, [](const Run& r, uintptr_t end) { return r.begin < end; });
    if (after != runs.begin() && (after - 1)->end > g.begin) return i;
  }
  return -1;
}

// Calls fn(table, chunks) for each group of at most kMax non-empty tensors that `skip` (or NULL) does not name.
template <int kMax, typename F>
inline void for_tables(const void* const* in, void* const* out, const int64_t* n, const int* dtype, int64_t count,
                       const uint8_t* skip, F&& fn) {
  Table<kMax> t;
  t.count = 0;
  int64_t chunks = 0;
  for (int64_t i = 0; i <= count; ++i) {
    const int64_t c = i < count && !(skip && skip[i]) ? chunks_of(n[i]) : 0;
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
                   const uint8_t* repeated, float max_norm, double* part, float* norm, cudaStream_t stream) {
  int parts = 0;
  for_tables<kMax>(grads, outs, sizes, dtypes, count, nullptr, [&](const Table<kMax>& t, int chunks) {
    const int grid = chunks < kBlocks ? chunks : kBlocks;
    square_kernel<kMax><<<grid, kThreads, 0, stream>>>(t, chunks, part + parts);
    parts += grid;
  });
  for_tables<kMax>(grads, outs, sizes, dtypes, count, repeated, [&](const Table<kMax>& t, int chunks) {
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
  std::vector<uint8_t> repeated;
  int64_t shared = -1;
  try {
    shared = clip::check_overlap({grads, outs, sizes, dtypes, count, isinf(max_norm) != 0}, repeated);
  } catch (const std::bad_alloc&) {
    set_error("prism_clip_grad_norm: out of host memory");
    return PRISM_ERR_UNSUPPORTED;
  }
  PRISM_CHECK_ARG(shared < 0,
                  "prism_clip_grad_norm: tensor %lld overlaps memory that the call writes (only a whole gradient may "
                  "be its own output, and be given again)",
                  (long long)shared);
  const auto launch = count <= clip::kSmallTable ? clip::launch<clip::kSmallTable> : clip::launch<clip::kTable>;
  launch(grads, outs, sizes, dtypes, count, repeated.empty() ? nullptr : repeated.data(), max_norm, (double*)workspace,
         norm, stream);
  PRISM_CHECK_LAUNCH("prism_clip_grad_norm");
  return PRISM_OK;
}

}  // extern "C"
