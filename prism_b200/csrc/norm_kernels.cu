// Residual addition + RMS norm of rows, forward (16-, 32- and 8-bit outputs) and backward.
//
//   h   = x + r, rounded to the rows' type (the residual stream as the next layer reads it)
//   u   = (mean_j h_j^2 + eps)^(-1/2)
//   y_j = w_j h_j u
// 8-bit rows: s = max(max_j |y_j| / 448, 2^-100), y8_j = e4m3(y_j / s).  u cancels in y_j / s,
// so one reduction gives both sum h^2 and max |w h|.  A row that holds a NaN or an infinity
// has scale NaN.
// Backward, with gy = dL/dy and gh = dL/dh:
//   dL/dh_j = u (w_j gy_j) - h_j u^3 / C * sum_i w_i gy_i h_i + gh_j   (also dL/dx and dL/dr)
//   dL/dw_j = sum over rows of gy_j h_j u
// Sums, u and the gradient of w are held in fp32.
#include <cuda_fp8.h>
#include <math.h>

#include "block_ops.cuh"

namespace prism {
namespace norm {

constexpr float kFp8Max = 448.0f;                      // largest finite e4m3 value
constexpr float kScaleFloor = 7.8886090522101181e-31f;  // 2^-100: 1 / scale stays finite
constexpr int kThreads = 256;

struct SumMax {
  float sum, max;
};

// Block reduction of a sum and a maximum, in a fixed order; every thread gets the result.
__device__ __forceinline__ SumMax block_sum_max(SumMax v, SumMax* red) {
  v.sum = warp_sum(v.sum);
  v.max = warp_max(v.max);
  const int w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) red[w] = v;
  __syncthreads();
  SumMax t = red[0];
  for (int i = 1; i < nw; ++i) {
    t.sum += red[i].sum;
    t.max = fmaxf(t.max, red[i].max);
  }
  return t;
}

// One CTA per row; kQuant: 8-bit rows; normalize = 0: the rows themselves (u = 1).
template <typename T, bool kQuant>
__global__ void __launch_bounds__(kThreads)
    fwd_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ r, int64_t ldr,
               const float* __restrict__ w, float eps, int normalize, int cols, void* __restrict__ y,
               T* h, float* __restrict__ aux) {
  __shared__ SumMax red[32];
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
    if (kQuant) t.max = fmaxf(t.max, fabsf(w ? f * w[c] : f));
  }
  t = block_sum_max(t, red);
  const float u = normalize ? rsqrtf(t.sum / (float)cols + eps) : 1.0f;
  const T* src = rr ? hr : xr;
  if constexpr (kQuant) {
    float scale = fmaxf(t.max * u / kFp8Max, kScaleFloor);
    if (!(t.sum <= 3.402823466e38f)) scale = NAN;
    const float inv = u / scale;
    auto* out = static_cast<__nv_fp8_storage_t*>(y) + row * cols;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      const float f = Elem<T>::to_f(src[c]);
      out[c] = __nv_cvt_float_to_fp8((w ? f * w[c] : f) * inv, __NV_SATFINITE, __NV_E4M3);
    }
    if (threadIdx.x == 0) aux[row] = scale;
  } else {
    T* out = static_cast<T*>(y) + row * cols;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      const float f = Elem<T>::to_f(src[c]) * u;
      out[c] = Elem<T>::from_f(w ? f * w[c] : f);
    }
    if (threadIdx.x == 0 && aux) aux[row] = u;
  }
}

// dL/dh of one row per CTA.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    bwd_row_kernel(const T* __restrict__ gy, int64_t ldgy, const T* __restrict__ h, int64_t ldh,
                   const T* __restrict__ gh, int64_t ldgh, const float* __restrict__ w,
                   const float* __restrict__ rstd, int cols, T* __restrict__ dx) {
  __shared__ SumMax red[32];
  const int64_t row = blockIdx.x;
  const T* gr = gy + row * ldgy;
  const T* hr = h + row * ldh;
  SumMax t = {0.0f, 0.0f};
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    const float g = Elem<T>::to_f(gr[c]);
    t.sum += (w ? g * w[c] : g) * Elem<T>::to_f(hr[c]);
  }
  t = block_sum_max(t, red);
  const float u = rstd[row], k = t.sum * u * u * u / (float)cols;
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    const float g = Elem<T>::to_f(gr[c]);
    float d = (w ? g * w[c] : g) * u - Elem<T>::to_f(hr[c]) * k;
    if (gh) d += Elem<T>::to_f(gh[row * ldgh + c]);
    dx[row * cols + c] = Elem<T>::from_f(d);
  }
}

// Partial sums of dL/dw over slabs of rows (blockIdx.y), one thread per column.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    bwd_weight_kernel(const T* __restrict__ gy, int64_t ldgy, const T* __restrict__ h, int64_t ldh,
                      const float* __restrict__ rstd, int64_t rows, int cols, int64_t per,
                      float* __restrict__ part) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= cols) return;
  const int64_t r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
  float s = 0.0f;
  for (int64_t i = r0; i < r1; ++i)
    s += Elem<T>::to_f(gy[i * ldgy + c]) * Elem<T>::to_f(h[i * ldh + c]) * rstd[i];
  part[(int64_t)blockIdx.y * cols + c] = s;
}

// dL/dw = sum of the slabs' partial sums in slab order.
__global__ void __launch_bounds__(kThreads)
    bwd_weight_sum_kernel(const float* __restrict__ part, int slabs, int cols, float* __restrict__ dw) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= cols) return;
  float s = 0.0f;
  for (int i = 0; i < slabs; ++i) s += part[(int64_t)i * cols + c];
  dw[c] = s;
}

constexpr int kSlabs = 296;

}  // namespace norm
}  // namespace prism

using namespace prism;

namespace {
bool rows_ok(int64_t rows, int cols) { return rows >= 0 && rows < ((int64_t)1 << 31) && cols >= 1; }
}  // namespace

extern "C" {

prism_status_t prism_add_rms_norm(const void* x, int64_t ldx, const void* r, int64_t ldr,
                                  const float* weight, float eps, int64_t rows, int cols, int dtype,
                                  void* y, void* h, float* rstd, cudaStream_t stream) {
  PRISM_CHECK_ARG(rows_ok(rows, cols) && ldx >= 0 && ldr >= 0, "prism_add_rms_norm: bad sizes");
  if (rows == 0) return PRISM_OK;
  PRISM_CHECK_ARG(x && y && (r == nullptr) == (h == nullptr),
                  "prism_add_rms_norm: null pointer (h goes with r)");
  const bool known = dispatch_dtype(dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    norm::fwd_kernel<T, false><<<(unsigned)rows, norm::kThreads, 0, stream>>>(
        (const T*)x, ldx, (const T*)r, ldr, weight, eps, 1, cols, y, (T*)h, rstd);
  });
  PRISM_CHECK_ARG(known, "prism_add_rms_norm: unknown element type %d", dtype);
  PRISM_CHECK_LAUNCH("prism_add_rms_norm");
  return PRISM_OK;
}

prism_status_t prism_add_rms_norm_fp8(const void* x, int64_t ldx, const void* r, int64_t ldr,
                                      const float* weight, float eps, int normalize, int64_t rows,
                                      int cols, int dtype, void* y8, float* scale, void* h,
                                      cudaStream_t stream) {
  PRISM_CHECK_ARG(rows_ok(rows, cols) && ldx >= 0 && ldr >= 0, "prism_add_rms_norm_fp8: bad sizes");
  if (rows == 0) return PRISM_OK;
  PRISM_CHECK_ARG(x && y8 && scale && (r == nullptr) == (h == nullptr),
                  "prism_add_rms_norm_fp8: null pointer (h goes with r)");
  const bool known = dispatch_dtype(dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    norm::fwd_kernel<T, true><<<(unsigned)rows, norm::kThreads, 0, stream>>>(
        (const T*)x, ldx, (const T*)r, ldr, weight, eps, normalize, cols, y8, (T*)h, scale);
  });
  PRISM_CHECK_ARG(known, "prism_add_rms_norm_fp8: unknown element type %d", dtype);
  PRISM_CHECK_LAUNCH("prism_add_rms_norm_fp8");
  return PRISM_OK;
}

size_t prism_add_rms_norm_bwd_workspace_bytes(int64_t rows, int cols) {
  const int64_t slabs = rows < norm::kSlabs ? rows : norm::kSlabs;
  return (size_t)slabs * (size_t)cols * sizeof(float);
}

prism_status_t prism_add_rms_norm_bwd(const void* gy, int64_t ldgy, const void* h, int64_t ldh,
                                      const void* gh, int64_t ldgh, const float* weight,
                                      const float* rstd, int64_t rows, int cols, int dtype, void* dx,
                                      void* workspace, float* dweight, cudaStream_t stream) {
  PRISM_CHECK_ARG(rows_ok(rows, cols) && ldgy >= 0 && ldh >= 0 && ldgh >= 0,
                  "prism_add_rms_norm_bwd: bad sizes");
  PRISM_CHECK_ARG(rows == 0 || (gy && h && rstd && dx && (dweight == nullptr || workspace)),
                  "prism_add_rms_norm_bwd: null pointer");
  if (rows == 0) {
    if (dweight) PRISM_CHECK_CUDA(cudaMemsetAsync(dweight, 0, sizeof(float) * cols, stream), "prism_add_rms_norm_bwd");
    return PRISM_OK;
  }
  const int64_t slabs = rows < norm::kSlabs ? rows : norm::kSlabs, per = (rows + slabs - 1) / slabs;
  const unsigned groups = (unsigned)((cols + norm::kThreads - 1) / norm::kThreads);
  const bool known = dispatch_dtype(dtype, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    norm::bwd_row_kernel<T><<<(unsigned)rows, norm::kThreads, 0, stream>>>(
        (const T*)gy, ldgy, (const T*)h, ldh, (const T*)gh, ldgh, weight, rstd, cols, (T*)dx);
    if (dweight) {
      norm::bwd_weight_kernel<T><<<dim3(groups, (unsigned)slabs), norm::kThreads, 0, stream>>>(
          (const T*)gy, ldgy, (const T*)h, ldh, rstd, rows, cols, per, (float*)workspace);
      norm::bwd_weight_sum_kernel<<<groups, norm::kThreads, 0, stream>>>((const float*)workspace, (int)slabs,
                                                                         cols, dweight);
    }
  });
  PRISM_CHECK_ARG(known, "prism_add_rms_norm_bwd: unknown element type %d", dtype);
  PRISM_CHECK_LAUNCH("prism_add_rms_norm_bwd");
  return PRISM_OK;
}

}  // extern "C"
