// Rotary positions: pair j of a token's head, as a complex number z, becomes
//   scale * z * exp(i p_j f_j),
// f_j radians per position (double), p_j the token's position on the axis that pair j follows.
// Layouts: interleaved pairs (2j, 2j + 1), or halves (j, j + rot/2); columns from rot on are
// copied.  The backward is the same with the conjugate factor.
//
// A product of a long position and a frequency does not fit fp32 (at position 10^6 the last
// place is 0.06 rad), so the angle is formed in turns in fp64, t = p (f / 2 pi), brought to
// [-1/2, 1/2] there and only then rounded to fp32.
#include <math.h>

#include "block_ops.cuh"

namespace prism {
namespace rotary {

constexpr int kThreads = 256;

struct Tensors {
  const void* in[2];   // q, k
  void* out[2];
  int64_t in_b[2], in_s[2], in_h[2], out_b[2], out_s[2], out_h[2];  // strides in elements
  int heads[2];
};

struct Positions {
  const void* ptr;
  int wide;          // 64-bit positions
  int64_t b, s;      // strides
  int end0, end1;    // pairs [0, end0) follow axis 0, [end0, end1) axis 1, the rest axis 2
};

__device__ __forceinline__ double position(const Positions& p, int64_t b, int64_t s, int pair) {
  const int64_t at = b * p.b + s * p.s + (pair >= p.end0) + (pair >= p.end1);
  return p.wide ? (double)static_cast<const long long*>(p.ptr)[at] : (double)static_cast<const int*>(p.ptr)[at];
}

__device__ __forceinline__ float2 cos_sin(double pos, double freq, float scale) {
  constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
  double t = pos * (freq * kTurn);
  t -= rint(t);
  float s, c;
  sincospif(2.0f * (float)t, &s, &c);
  return make_float2(c * scale, s * scale);
}

// One CTA per token; a thread takes a pair (or a copied column) of one head at a time.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    rotary_kernel(const __grid_constant__ Tensors t, const __grid_constant__ Positions pos,
                  const double* __restrict__ freqs, int64_t seq, int dim, int rot, int interleaved, float scale,
                  float sign) {
  const int64_t b = blockIdx.x / seq, s = blockIdx.x - b * seq;
  const int half = rot / 2, units = half + dim - rot;
  for (int i = threadIdx.x; i < (t.heads[0] + t.heads[1]) * units; i += kThreads) {
    int head = i / units;
    const int j = i - head * units, which = head >= t.heads[0];
    head -= which ? t.heads[0] : 0;
    const T* in = static_cast<const T*>(t.in[which]) + b * t.in_b[which] + s * t.in_s[which] + head * t.in_h[which];
    T* out = static_cast<T*>(t.out[which]) + b * t.out_b[which] + s * t.out_s[which] + head * t.out_h[which];
    if (j >= half) {
      out[rot + j - half] = in[rot + j - half];
      continue;
    }
    const float2 cs = cos_sin(position(pos, b, s, j), freqs[j], scale);
    const int c0 = interleaved ? 2 * j : j, c1 = interleaved ? c0 + 1 : j + half;
    const float a = Elem<T>::to_f(in[c0]), d = Elem<T>::to_f(in[c1]), sn = sign * cs.y;
    out[c0] = Elem<T>::from_f(a * cs.x - d * sn);
    out[c1] = Elem<T>::from_f(a * sn + d * cs.x);
  }
}

}  // namespace rotary
}  // namespace prism

using namespace prism;

extern "C" prism_status_t prism_rotary(const void* q, const int64_t* q_strides, int q_heads, const void* k,
                                       const int64_t* k_strides, int k_heads, int64_t batch, int64_t seq,
                                       int dim, int rot, int interleaved, const void* positions,
                                       int positions_64, const int64_t* position_strides,
                                       const int* section_ends, const double* freqs, float scale,
                                       int conjugate, int dtype, void* q_out,
                                       const int64_t* q_out_strides, void* k_out,
                                       const int64_t* k_out_strides, cudaStream_t stream) {
  PRISM_CHECK_ARG(batch >= 0 && seq >= 0 && batch * seq < ((int64_t)1 << 31) && dim >= 1 && rot >= 0 &&
                      rot % 2 == 0 && rot <= dim && q_heads >= 0 && k_heads >= 0,
                  "prism_rotary: bad sizes");
  PRISM_CHECK_ARG((int64_t)(q_heads + (int64_t)k_heads) * dim < ((int64_t)1 << 31), "prism_rotary: too many heads");
  if (batch * seq == 0 || q_heads + k_heads == 0) return PRISM_OK;
  PRISM_CHECK_ARG((q_heads == 0 || (q && q_out && q_strides && q_out_strides)) &&
                      (k_heads == 0 || (k && k_out && k_strides && k_out_strides)) &&
                      (rot == 0 || (positions && position_strides && section_ends && freqs)),
                  "prism_rotary: null pointer");
  rotary::Tensors t = {};
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const int64_t *is[2] = {q_strides, k_strides}, *os[2] = {q_out_strides, k_out_strides};
  const int heads[2] = {q_heads, k_heads};
  for (int i = 0; i < 2; ++i) {
    if (heads[i] == 0) continue;
    t.in[i] = in[i], t.out[i] = out[i], t.heads[i] = heads[i];
    t.in_b[i] = is[i][0], t.in_s[i] = is[i][1], t.in_h[i] = is[i][2];
    t.out_b[i] = os[i][0], t.out_s[i] = os[i][1], t.out_h[i] = os[i][2];
  }
  rotary::Positions p = {};
  if (rot > 0) {
    p = {positions, positions_64, position_strides[0], position_strides[1], section_ends[0], section_ends[1]};
    PRISM_CHECK_ARG(p.end0 >= 0 && p.end1 >= p.end0, "prism_rotary: sections out of order");
  }
  const bool known = dispatch_dtype(dtype, [&](auto* e) {
    using T = std::remove_pointer_t<decltype(e)>;
    rotary::rotary_kernel<T><<<(unsigned)(batch * seq), rotary::kThreads, 0, stream>>>(
        t, p, freqs, seq, dim, rot, interleaved, scale, conjugate ? -1.0f : 1.0f);
  });
  PRISM_CHECK_ARG(known, "prism_rotary: unknown element type %d", dtype);
  PRISM_CHECK_LAUNCH("prism_rotary");
  return PRISM_OK;
}
