// Rotary positions: pair j of a token's head, as a complex number z, becomes
//   scale * z * exp(i p_j f_j),
// f_j radians per position (double), p_j the token's position on the axis that pair j follows.
// Layouts: interleaved pairs (2j, 2j + 1), or halves (j, j + rot/2); columns from rot on are
// copied.  The backward is the same with the conjugate factor.
//
// A product of a long position and a frequency does not fit fp32 (at position 10^6 the last
// place is 0.06 rad), so the angle is formed in turns in fp64, t = p (f / 2 pi), brought to
// [-1/2, 1/2] there and only then rounded to fp32.
//
// Bound by memory: q and k are read and written once, in one launch.  The factors of a token's
// pairs are the same for all its heads: a CTA computes those of its tokens once into shared memory,
// while its first loads are on their way, and each thread keeps those of its columns in registers
// while it goes through the heads of q and k.
#include <math.h>

#include <type_traits>

#include "block_ops.cuh"

namespace prism {
namespace rotary {

constexpr int kThreads = 128;   // a CTA's, where a head is not wider (256: 470 -> 510 us at 80 heads of 128)
constexpr int kSms = 148;
constexpr int kMaxDim = 1024, kMaxThreads = 1024;  // one element a thread, at worst

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

// How a CTA's threads divide its tokens.  A thread keeps one unit (column) of the heads:
// `heads_at_once` threads a unit go through the heads, `tokens_at_once` tokens next to each other.
struct Split {
  int units, heads_at_once, tokens_at_once, cta_tokens;
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

// Units of a head: with kAdjacent (interleaved pairs inside a vector) its dim / kVec vectors; else
// rot / 2 / kVec pairs of vectors that hold the two sides of kVec pairs -- half a rotation apart,
// or, for interleaved pairs at odd addresses, single elements side by side -- and then the
// (dim - rot) / kVec copied vectors.
// kAlongHeads: a thread's batches run along the heads of a token, the token's factors in registers
// (whole tokens are read and written at a time: 80 heads of 128 at 6.7 TB/s, against 6.1 along the
// tokens).  Else, for few heads, along the tokens of a head (9 heads of 64 columns at 4.8 TB/s,
// against 2.7).
// 64 registers, for 1,024 threads an SM: bf16 halves along the heads spill 28 bytes and are still faster
// than with 74 (40,000 tokens of 40 + 8 heads, forward and backward: 342 against 358 us).
template <typename T, int kVec, bool kAdjacent, bool kAlongHeads>
__global__ void __launch_bounds__(kMaxThreads)
    rotary_kernel(const __grid_constant__ Tensors t, const __grid_constant__ Positions pos,
                  const double* __restrict__ freqs, int tokens, int seq, Split split, int rot, int interleaved,
                  float scale, float sign) {
  using U = Unit<T, kVec, kAdjacent>;
  constexpr int kBatch = kAdjacent ? 4 : kAlongHeads ? 2 : 3;  // units of a thread on their way
  constexpr int kPairs = U::kPairs;
  extern __shared__ float2 factors[];        // [token of the CTA][pair]
  const int half = rot / 2, heads = t.heads[0] + t.heads[1];
  const int first = blockIdx.x * split.cta_tokens, count = min(split.cta_tokens, tokens - first);
  const int first_b = first / seq, first_s = first - first_b * seq;

  const int group = threadIdx.x / split.units, unit = threadIdx.x - group * split.units;
  const int token0 = group / split.heads_at_once, head0 = group - token0 * split.heads_at_once;
  // the unit's columns c and c + apart, its pairs from `pair` on; turn = 0: copied
  const int rotated = kAdjacent ? rot / kVec : half / kVec;
  const bool turn = unit < rotated;
  const int c = kAdjacent ? unit * kVec : turn ? (interleaved ? 2 * unit : unit * kVec) : rot + (unit - rotated) * kVec;
  const int apart = interleaved ? 1 : half, pair = unit * kPairs;
  int head = head0, token = token0 < split.tokens_at_once ? token0 : count;
  int b = first_b, s = first_s + token0;
  const auto wrap = [&] {
    for (; s >= seq; s -= seq) ++b;
  };
  wrap();
  U batch[kBatch];

  // along the heads: the token's q and k at this column
  const T* in[2];
  T* out[2];
  const auto at_token = [&] {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      in[i] = static_cast<const T*>(t.in[i]) + (b * t.in_b[i] + s * t.in_s[i]) + c;
      out[i] = static_cast<T*>(t.out[i]) + (b * t.out_b[i] + s * t.out_s[i]) + c;
    }
  };
  const auto load_heads = [&](int from) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = from + i * split.heads_at_once;
      if (h >= heads) break;
      batch[i].load(h >= t.heads[0] ? in[1] + (h - t.heads[0]) * t.in_h[1] : in[0] + h * t.in_h[0], turn, apart);
    }
  };
  // along the tokens: the head's next tokens, up to the end of their sequence
  const T* in_run = nullptr;
  T* out_run = nullptr;
  int64_t in_step = 0, out_step = 0;
  int got = 0;
  const auto at_head = [&] {
    const int which = head >= t.heads[0], h = which ? head - t.heads[0] : head;
    in_run = static_cast<const T*>(t.in[which]) + (b * t.in_b[which] + s * t.in_s[which] + h * t.in_h[which] + c);
    out_run = static_cast<T*>(t.out[which]) + (b * t.out_b[which] + s * t.out_s[which] + h * t.out_h[which] + c);
    in_step = split.tokens_at_once * t.in_s[which], out_step = split.tokens_at_once * t.out_s[which];
  };
  const auto load_tokens = [&] {
    got = 0;
    const int left = min(count - token, seq - s);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (i * split.tokens_at_once < left) {
        batch[i].load(in_run + i * in_step, turn, apart);
        got = i + 1;
      }
    }
  };
  if (token < count && head < heads) {
    if constexpr (kAlongHeads) {
      at_token();
      load_heads(head0);
    } else {
      at_head();
      load_tokens();
    }
  }

  // the factors, a thread's pairs blockDim apart
  if (half > 0) {
    const int step_t = blockDim.x / half, step_j = blockDim.x - step_t * half;
    int ti = threadIdx.x / half, j = threadIdx.x - ti * half;
    for (; ti < count; ti += step_t, j += step_j) {
      if (j >= half) {
        j -= half;
        if (++ti >= count) break;
      }
      int tb = first_b, ts = first_s + ti;
      for (; ts >= seq; ts -= seq) ++tb;
      factors[ti * half + j] = cos_sin(position(pos, tb, ts, j), __ldg(freqs + j), scale, sign);
    }
  }
  __syncthreads();

  if constexpr (kAlongHeads) {
    while (token < count) {
      float2 w[kPairs];
      if (turn) {
#pragma unroll
        for (int e = 0; e < kPairs; ++e) w[e] = factors[token * half + pair + e];
      }
      for (int from = head0; from < heads; from += kBatch * split.heads_at_once) {
        if (from != head0) load_heads(from);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int h = from + i * split.heads_at_once;
          if (h >= heads) break;
          T* p = h >= t.heads[0] ? out[1] + (h - t.heads[0]) * t.out_h[1] : out[0] + h * t.out_h[0];
          if (turn) batch[i].turn(p, apart, w);
          else batch[i].copy(p);
        }
      }
      token += split.tokens_at_once, s += split.tokens_at_once;
      wrap();
      if (token < count) {
        at_token();
        load_heads(head0);
      }
    }
  } else {
    while (got > 0) {
      const float2* f = factors + token * half + pair;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (i >= got) break;
        if (turn) batch[i].turn(out_run + i * out_step, apart, f + i * split.tokens_at_once * half);
        else batch[i].copy(out_run + i * out_step);
      }
      const int done = got * split.tokens_at_once;
      token += done, s += done, in_run += got * in_step, out_run += got * out_step, got = 0;
      if (token >= count) {  // the next head from the first token
        head += split.heads_at_once;
        if (head >= heads) break;
        token = token0, b = first_b, s = first_s + token0;
        wrap();
        at_head();
      } else if (s >= seq) {
        wrap();
        at_head();
      }
      load_tokens();
    }
  }
}

template <typename T, int kVec, bool kAdjacent>
cudaError_t launch(const Tensors& t, const Positions& p, const double* freqs, int tokens, int seq, int dim, int rot,
                   int interleaved, float scale, float sign, cudaStream_t stream) {
  const int heads = t.heads[0] + t.heads[1];
  Split s;
  s.units = kAdjacent ? dim / kVec : rot / 2 / kVec + (dim - rot) / kVec;
  // equal rounds of heads in up to kThreads threads, or, for few tokens, in 512 for the shortest way
  // through (a head wider than that has them all)
  const int limit = tokens <= kSms ? 512 : kThreads;
  const int groups = s.units < limit ? limit / s.units : 1, rounds = (heads + groups - 1) / groups;
  s.heads_at_once = (heads + rounds - 1) / rounds;
  s.tokens_at_once = groups / s.heads_at_once;
  const int threads = (s.units * s.heads_at_once * s.tokens_at_once + 31) / 32 * 32;
  const bool along_heads = rounds >= 4;
  // eight tokens a thread (along the heads: eight items), within 16 KB of factors; few tokens are
  // spread over the SMs
  int per = (along_heads ? (7 + rounds) / rounds : 8) * s.tokens_at_once;
  const int room = rot > 0 ? (16 << 10) / (rot / 2 * (int)sizeof(float2)) : per, spread = (tokens + kSms - 1) / kSms;
  per = per < room ? per : room;
  per = per < spread ? per : spread;
  // whole waves of CTAs (64 registers a thread), where there are few
  const int slots = kSms * (1024 / threads > 0 ? 1024 / threads : 1), waves = (tokens / per + slots - 1) / slots;
  if (waves > 0 && waves < 8) per = (tokens + waves * slots - 1) / (waves * slots);
  s.cta_tokens = per;
  const auto kernel = along_heads ? rotary_kernel<T, kVec, kAdjacent, true> : rotary_kernel<T, kVec, kAdjacent, false>;
  kernel<<<(tokens + per - 1) / per, threads, per * (rot / 2) * sizeof(float2), stream>>>(
      t, p, freqs, tokens, seq, s, rot, interleaved, scale, sign);
  return cudaGetLastError();
}

// The widest vectors, of 16 bytes at most, that every row start, stride and column range allows.
template <typename T>
cudaError_t dispatch(const Tensors& t, const Positions& p, const double* freqs, int64_t batch, int seq, int dim,
                     int rot, int interleaved, float scale, float sign, cudaStream_t stream) {
  uint64_t bits = (uint64_t)dim;  // its low zero bits: the power of two that divides every place
  for (int i = 0; i < 2; ++i) {
    if (t.heads[i] == 0) continue;
    bits |= reinterpret_cast<uintptr_t>(t.in[i]) / sizeof(T) | reinterpret_cast<uintptr_t>(t.out[i]) / sizeof(T);
    if (batch > 1) bits |= (uint64_t)t.in_b[i] | (uint64_t)t.out_b[i];
    if (seq > 1) bits |= (uint64_t)t.in_s[i] | (uint64_t)t.out_s[i];
    if (t.heads[i] > 1) bits |= (uint64_t)t.in_h[i] | (uint64_t)t.out_h[i];
  }
  const int tokens = (int)(batch * seq);
  const auto go = [&](auto vec, auto adjacent) {
    return launch<T, vec(), adjacent()>(t, p, freqs, tokens, seq, dim, rot, interleaved, scale, sign, stream);
  };
  using std::integral_constant;
  const integral_constant<bool, true> inside{};
  const integral_constant<bool, false> apart{};
  if (interleaved) {
    bits |= (uint64_t)rot;  // a vector is rotated or copied whole
    if constexpr (sizeof(T) == 2)
      if (bits % 8 == 0) return go(integral_constant<int, 8>{}, inside);
    if (bits % 4 == 0) return go(integral_constant<int, 4>{}, inside);
    if (bits % 2 == 0) return go(integral_constant<int, 2>{}, inside);
    return go(integral_constant<int, 1>{}, apart);
  }
  bits |= (uint64_t)(rot / 2);
  if constexpr (sizeof(T) == 2)
    if (bits % 8 == 0) return go(integral_constant<int, 8>{}, apart);
  if (bits % 4 == 0) return go(integral_constant<int, 4>{}, apart);
  if (bits % 2 == 0) return go(integral_constant<int, 2>{}, apart);
  return go(integral_constant<int, 1>{}, apart);
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
  PRISM_CHECK_ARG(batch >= 0 && seq >= 0 && batch < ((int64_t)1 << 31) && seq < ((int64_t)1 << 31) &&
                      batch * seq < ((int64_t)1 << 31) - 4096 && dim >= 1 && dim <= rotary::kMaxDim && rot >= 0 &&
                      rot % 2 == 0 && rot <= dim && q_heads >= 0 && k_heads >= 0,
                  "prism_rotary: bad sizes (head dim up to %d, an even part of it rotated)", rotary::kMaxDim);
  PRISM_CHECK_ARG(((int64_t)q_heads + k_heads) * dim < ((int64_t)1 << 30), "prism_rotary: too many heads");
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
  cudaError_t err = cudaSuccess;
  const bool known = dispatch_dtype(dtype, [&](auto* e) {
    using T = std::remove_pointer_t<decltype(e)>;
    err = rotary::dispatch<T>(t, p, freqs, batch, (int)seq, dim, rot, interleaved, scale, conjugate ? -1.0f : 1.0f,
                              stream);
  });
  PRISM_CHECK_ARG(known, "prism_rotary: unknown element type %d", dtype);
  PRISM_CHECK_CUDA(err, "prism_rotary");
  return PRISM_OK;
}
