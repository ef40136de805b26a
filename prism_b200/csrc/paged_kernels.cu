// Keys and values in a paged cache: appending them, with the rotary positions applied on the way, and the
// attention of a few new tokens over them.
//
// A cache is [pages, page_size, Hk, D] for keys and one for values (any strides of page, place and head);
// token j of sequence b is at place j % page_size of page table[b][j / page_size].  lengths[b] counts the
// tokens of sequence b, the new ones (the last n) among them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "block_ops.cuh"
#include "rotary.cuh"

namespace prism {
namespace paged {

constexpr int kSms = 148;

struct Cache {
  void *k, *v;
  int64_t k_page, k_place, k_head, v_page, v_place, v_head;  // strides in elements
  const int* table;
  int64_t table_row;
  int table_width, page_size, pages;
  uint32_t page_inverse;      // floor((2^32 - 1) / page_size)
  const int* lengths;
};

// ======================================================================= append
// One pass: each new token's k (rotated) and v go to its place, its q (rotated) to q_out.  Pair j of a
// head's first `rot` columns, as a complex number, is multiplied by scale * exp(i p f_j), p the token's
// place in its sequence; the angle is formed in fp64 turns (rotary.cuh).
//
// Bound by memory; for one token a sequence by latency: lengths -> table -> place, with the factors
// computed meanwhile.  A CTA takes a few tokens; their places and factors are found once and kept in
// shared memory, and each thread keeps one unit (16 bytes of a head, or the two vectors that a rotation
// of halves needs) and runs along the tokens' heads of q, k and v.
//
// 23,442 tokens of 24 + 8 heads of 128, 96 columns rotated as adjacent pairs: 86 us (5.6 TB/s); one token each
// of 16 sequences: 3.2 us.
struct Append {
  const void* in[3];          // q, k, v
  int64_t in_t[3], in_h[3];   // strides of token and head
  int heads[3];
  void* q_out;                // [tokens, heads, dim]
  const void* offsets;        // NULL: `each` tokens a sequence
  int wide, count, each, tokens;
};

enum Status : int { kThere, kNone, kBad };  // kNone: no place (before the first, or of no sequence): q_out 0

struct TokenPlace {
  int status, position, page, place;
};

__device__ __forceinline__ TokenPlace place_of(const Append& a, const Cache& c, int t) {
  TokenPlace p = {kNone, 0, 0, 0};
  int b, i, n;
  if (a.offsets == nullptr) {
    b = t / a.each, i = t - b * a.each, n = a.each;
  } else {
    const auto at = [&](int j) {
      return a.wide ? static_cast<const long long*>(a.offsets)[j] : (long long)static_cast<const int*>(a.offsets)[j];
    };
    int lo = 0, hi = a.count;  // the last sequence that starts at t or before it
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (at(mid) <= t) lo = mid;
      else hi = mid;
    }
    const long long first = at(lo), end = at(lo + 1);
    if (t < first || t >= end || end - first > a.tokens) return p;
    b = lo, i = (int)(t - first), n = (int)(end - first);
  }
  const int64_t position = (int64_t)c.lengths[b] - n + i;
  if (position < 0) return p;
  p.status = kBad;
  const int64_t entry = position / c.page_size;
  if (entry >= c.table_width) return p;
  p.page = c.table[b * c.table_row + entry];
  if (p.page < 0 || p.page >= c.pages) return p;
  p.status = kThere, p.position = (int)position, p.place = (int)(position - entry * c.page_size);
  return p;
}

constexpr int kAppendThreads = 256;

template <typename T, int kVec, bool kAdjacent>
__global__ void __launch_bounds__(kAppendThreads)
    append_kernel(const __grid_constant__ Append a, const __grid_constant__ Cache c, const double* __restrict__ freqs,
                  int dim, int rot, int interleaved, float scale, int per, int units) {
  using U = rotary::Unit<T, kVec, kAdjacent>;
  using Raw = typename U::Raw;
  constexpr int kBatch = kAdjacent ? 4 : 2;  // units of a thread on their way (halves in 4: 97 -> 105 us)
  extern __shared__ float2 factors[];   // [token of the CTA][pair], then the places
  const int half = rot / 2, heads = a.heads[0] + a.heads[1] + a.heads[2];
  const int first = blockIdx.x * per, count = min(per, a.tokens - first);
  TokenPlace* places = reinterpret_cast<TokenPlace*>(factors + per * half);
  for (int t = threadIdx.x; t < count; t += blockDim.x) places[t] = place_of(a, c, first + t);
  __syncthreads();
  for (int i = threadIdx.x; i < count * half; i += blockDim.x) {
    const int t = i / half, j = i - t * half;
    factors[i] = rotary::cos_sin((double)places[t].position, __ldg(freqs + j), scale, 1.0f);
  }
  __syncthreads();

  // the unit's columns col and col + apart, its pairs from `pair` on; turn = false: a copied vector
  const int group = threadIdx.x / units, groups = blockDim.x / units, unit = threadIdx.x - group * units;
  if (group >= groups) return;
  const int rotated = kAdjacent ? rot / kVec : half / kVec;
  const bool turn = unit < rotated;
  const int col = kAdjacent ? unit * kVec : turn ? (interleaved ? 2 * unit : unit * kVec) : rot + (unit - rotated) * kVec;
  const int apart = interleaved ? 1 : half, pair = unit * U::kPairs;
  int t = 0, head = group;
  const auto wrap = [&] {
    while (head >= heads) head -= heads, ++t;
  };
  wrap();
  while (t < count) {
    U batch[kBatch];
    int at_t[kBatch], at_head[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      at_t[i] = t, at_head[i] = head;
      if (t < count) {
        const int which = head < a.heads[0] ? 0 : head < a.heads[0] + a.heads[1] ? 1 : 2;
        const int h = head - (which > 0 ? a.heads[0] : 0) - (which > 1 ? a.heads[1] : 0);
        const int64_t in_t = which == 0 ? a.in_t[0] : which == 1 ? a.in_t[1] : a.in_t[2];
        const int64_t in_h = which == 0 ? a.in_h[0] : which == 1 ? a.in_h[1] : a.in_h[2];
        const void* in = which == 0 ? a.in[0] : which == 1 ? a.in[1] : a.in[2];
        batch[i].load(static_cast<const T*>(in) + (first + t) * in_t + h * in_h + col, turn, apart);
      }
      head += groups;
      wrap();
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (at_t[i] >= count) break;
      const TokenPlace p = places[at_t[i]];
      const float2* f = factors + at_t[i] * half + pair;
      int h = at_head[i];
      if (h < a.heads[0]) {
        T* out = static_cast<T*>(a.q_out) + ((int64_t)(first + at_t[i]) * a.heads[0] + h) * dim + col;
        if (p.status != kThere) {
          float x[kVec];
#pragma unroll
          for (int e = 0; e < kVec; ++e) x[e] = p.status == kBad ? __int_as_float(0x7fc00000) : 0.0f;
          const Raw raw = U::V::pack(x);
          *reinterpret_cast<Raw*>(out) = raw;
          if (!kAdjacent && turn) *reinterpret_cast<Raw*>(out + apart) = raw;
        } else if (turn) {
          batch[i].turn(out, apart, f);
        } else {
          batch[i].copy(out);
        }
        continue;
      }
      if (p.status != kThere) continue;
      h -= a.heads[0];
      if (h < a.heads[1]) {
        T* out = static_cast<T*>(c.k) + p.page * c.k_page + p.place * c.k_place + h * c.k_head + col;
        if (turn) batch[i].turn(out, apart, f);
        else batch[i].copy(out);
      } else {
        h -= a.heads[1];
        T* out = static_cast<T*>(c.v) + p.page * c.v_page + p.place * c.v_place + h * c.v_head + col;
        batch[i].copy(out);
        if constexpr (!kAdjacent) {
          if (turn) *reinterpret_cast<Raw*>(out + apart) = batch[i].hi;
        }
      }
    }
  }
}

template <typename T, int kVec, bool kAdjacent>
static cudaError_t launch_append(const Append& a, const Cache& c, const double* freqs, int dim, int rot, int interleaved,
                                 float scale, cudaStream_t stream) {
  const int units = kAdjacent ? dim / kVec : rot / 2 / kVec + (dim - rot) / kVec;
  // few tokens are spread over the SMs; else up to 8 a CTA, within 16 KB of factors
  const int spread = (a.tokens + kSms - 1) / kSms, room = rot > 0 ? (16 << 10) / (rot / 2 * (int)sizeof(float2)) : 8;
  int per = 8;
  per = per < spread ? per : spread;
  per = per < room ? per : room;
  per = per < 1 ? 1 : per;
  append_kernel<T, kVec, kAdjacent><<<(a.tokens + per - 1) / per, kAppendThreads,
                                      per * (rot / 2 * sizeof(float2) + sizeof(TokenPlace)), stream>>>(
      a, c, freqs, dim, rot, interleaved, scale, per, units);
  return cudaGetLastError();
}

// The widest vectors, of 16 bytes at most, that every row start, stride and column range allows.
template <typename T>
static cudaError_t dispatch_append(const Append& a, const Cache& c, const double* freqs, int dim, int rot,
                                   int interleaved, float scale, cudaStream_t stream) {
  uint64_t bits = (uint64_t)dim;  // its low zero bits: the power of two that divides every place
  const auto add = [&](const void* p) { bits |= reinterpret_cast<uintptr_t>(p) / sizeof(T); };
  for (int i = 0; i < 3; ++i)
    if (a.heads[i] > 0) add(a.in[i]), bits |= (uint64_t)a.in_t[i] | (uint64_t)a.in_h[i];
  if (a.heads[0] > 0) add(a.q_out);
  add(c.k), add(c.v);
  bits |= (uint64_t)(c.k_page | c.k_place | c.k_head | c.v_page | c.v_place | c.v_head);
  using std::integral_constant;
  const auto go = [&](auto vec, auto adjacent) {
    return launch_append<T, vec(), adjacent()>(a, c, freqs, dim, rot, interleaved, scale, stream);
  };
  const integral_constant<bool, true> inside{};
  const integral_constant<bool, false> apart{};
  if (interleaved) {
    bits |= (uint64_t)rot;  // a vector is rotated or copied whole
    if (bits % 8 == 0) return go(integral_constant<int, 8>{}, inside);
    if (bits % 2 == 0) return go(integral_constant<int, 2>{}, inside);
    return go(integral_constant<int, 1>{}, apart);
  }
  bits |= (uint64_t)(rot / 2);
  if (bits % 8 == 0) return go(integral_constant<int, 8>{}, apart);
  if (bits % 2 == 0) return go(integral_constant<int, 2>{}, apart);
  return go(integral_constant<int, 1>{}, apart);
}

// ==================================================================== attention
// q [B, n, Hq, D] (n new tokens a sequence, the last n of its lengths[b]) -> o alike: query i of sequence b
// attends keys j <= lengths[b] - n + i.  softmax as in packed_attention.cu.
//
// Bound by memory: K and V of a sequence are read once for the G = Hq / Hk heads that share them (and for
// the n queries), 4 D bytes a key for 4 D G n operations.  The products take mma.sync (m16n8k16): 16 rows
// are all there is, so the tensor cores are idle most of the time whichever instruction feeds them, and
// fragments in registers need no trip through TMEM.
//   * A unit is a sequence, a key head and up to 16 rows (query i, head g), row i G + g.  Its keys come in
//     tiles of 32 KB, a quarter for each of 4 warps (16 keys of 128 columns, 32 of 64: with 16, a step's fixed
//     costs held 64 columns at 0.6 of the memory's rate); a warp loads its own keys into its own ring with
//     cp.async and keeps its own running maximum and sum: no barrier in the loop.
//   * All tiles of all units, in order, are dealt out in equal shares to a fixed number of CTAs (two an
//     SM), whatever the lengths are: a share may end inside a unit and hold several.  A unit that lies in
//     one share is written at once; the pieces of a divided one go to the workspace, two places a CTA, and
//     a second launch joins them in order.  The ring runs on across units.
//   * Where no sequence can have more than kWhole keys (the table's width), a CTA takes one unit and there
//     is no second launch: 16 sequences of 512 keys take 10.9 us so and 14.5 in shares, 16 of 64 keys 4.5 and 9.6,
//     4 of 1,024 keys 18.3 and 10.7, 64 of 1,024 51 and 56 (8 heads of 128).  The host knows the width, not the
//     lengths: 4 sequences of 100 keys take 5.1 us with a table of 112 tokens, 7.5 with one of 4,096.
//   * Keys behind a sequence's end are not read (zero-filled), so what lies there does not matter.
// 131,001 keys of 8 heads of 128, 32 query heads: 88 us (6.1 TB/s), 6 of them the join; 4 sequences of up to 100
// keys in one launch: 4.7 us.
constexpr int kWarps = 4, kThreads = 32 * kWarps, kRows = 16, kCtas = 2 * kSms;
constexpr int kWhole = 512;

struct Queries {
  const void* q;
  int64_t q_b, q_t, q_h;              // strides of sequence, token, head
  int batch, tokens, heads, group;    // heads: of keys
  int row_tiles;                      // of 16 rows, of tokens * group
  int whole;                          // a CTA takes a unit
};

template <int D>
struct Layout {
  static constexpr int kStages = 3;                    // 96 KB a CTA
  static constexpr int kKeys = 2048 / D;               // of a warp's step
  static constexpr int kTile = kWarps * kKeys;
  static constexpr int kWarpBytes = kKeys * D * 2 * 2;  // keys and values
  static constexpr int kRing = kStages * kWarps * kWarpBytes;
  static constexpr int kPitch = D + 4;                 // of a row of the warps' sums, in floats
  static constexpr int kJoin = kWarps * 8 * kPitch * 4, kJoinMl = kWarps * 8 * 8;
  static constexpr int kBytes = kRing + kJoin + kJoinMl;  // two CTAs an SM
};

template <typename T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
  static constexpr float kShift = 0.0f, kLag = 8.0f;
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
};
// fp16's p starts at 2^8 (keys down to 2^-32 of the largest count) and may grow to 2^15 before the maximum
// is raised, as in packed_attention.cu.
template <>
struct Mma<__half> {
  static constexpr float kShift = 8.0f, kLag = 7.0f;
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 p = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void load16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// Keys of sequence b that the table has room for.
__device__ __forceinline__ int length_of(const Cache& c, int b) {
  return min(max(c.lengths[b], 0), c.table_width * c.page_size);
}
template <int kTile>
__device__ __forceinline__ int tiles_of(int length) { return (length + kTile - 1) / kTile; }

// A tile: of sequence b, unit `unit` (key head * row_tiles + row tile) of it.
template <int kTile>
struct Cursor {
  int b, unit, tile, tiles, length;
  __device__ __forceinline__ void enter(const Cache& c, int batch) {  // from b on, the next sequence with keys
    for (; b < batch; ++b) {
      length = length_of(c, b), tiles = tiles_of<kTile>(length);
      if (tiles > 0) return;
    }
  }
  __device__ __forceinline__ void next(const Cache& c, int batch, int units) {
    if (++tile < tiles) return;
    tile = 0;
    if (++unit < units) return;
    unit = 0, ++b;
    enter(c, batch);
  }
};

// `total` tiles of all units, dealt out to `shares` CTAs: CTA i has those from start(i) to start(i + 1).  A share
// has kLeast tiles at least (one, where there are fewer), so none between two others is empty.
constexpr int kLeast = 2;
struct Deal {
  int64_t total;
  int shares;
  __device__ __forceinline__ explicit Deal(int64_t tiles)
      : total(tiles), shares((int)min((int64_t)kCtas, max(tiles / kLeast, (int64_t)1))) {}
  __device__ __forceinline__ int64_t start(int64_t cta) const { return min(cta, (int64_t)shares) * total / shares; }
  __device__ __forceinline__ int owner(int64_t tile) const { return (int)(((tile + 1) * shares - 1) / total); }
};

// The share of this CTA: its first tile, and that tile's sequence with the tiles before it.  All threads; up to
// kThreads sequences take one round, more a second one once the total is known.
struct Share {
  int64_t first, steps, before;
  int b;
};
template <int kTile>
__device__ Share share_of(const Cache& c, int batch, int units, int64_t* scratch) {
  __shared__ int64_t found_before;
  __shared__ int found_b;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Share share = {0, 0, 0, 0};
  int64_t total = 0;
  for (int pass = batch <= kThreads ? 1 : 0; pass < 2; ++pass) {
    int64_t base = 0;
    for (int b0 = 0; b0 < batch; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      const int64_t tiles = b < batch ? (int64_t)tiles_of<kTile>(length_of(c, b)) * units : 0;
      int64_t sum = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      if (lane == 31) scratch[warp] = sum;
      __syncthreads();
      int64_t start = base + sum - tiles;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) start += scratch[w];
        base += scratch[w];
      }
      if (pass == 1) {
        if (batch <= kThreads) total = base;
        const Deal deal(total);
        share.first = deal.start(blockIdx.x), share.steps = deal.start(blockIdx.x + 1) - share.first;
        if (share.steps > 0 && share.first >= start && share.first < start + tiles) found_b = b, found_before = start;
      }
      __syncthreads();
    }
    total = base;
  }
  if (share.steps > 0) share.b = found_b, share.before = found_before;
  return share;
}

// Tiles before sequence b (b = batch: all), summed by the CTA's threads.
template <int kTile>
__device__ int64_t tiles_before(const Cache& c, int b, int units, int64_t* scratch) {
  int64_t sum = 0;
  for (int i = threadIdx.x; i < b; i += kThreads) sum += tiles_of<kTile>(length_of(c, i));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum += scratch[w];
  __syncthreads();
  return sum * units;
}

// Rows of a unit in o, [batch, tokens, heads * group, D].
__device__ __forceinline__ int64_t out_row(const Queries& s, int b, int unit, int row) {
  const int head = unit / s.row_tiles, all = (unit - head * s.row_tiles) * kRows + row, i = all / s.group;
  return ((int64_t)(b * s.tokens + i) * s.heads + head) * s.group + (all - i * s.group);
}
__device__ __forceinline__ int rows_of(const Queries& s, int unit) {
  return min(kRows, s.tokens * s.group - unit % s.row_tiles * kRows);
}
// Whether a row of a unit sees no key of its sequence's `length`.
__device__ __forceinline__ bool sees_none(const Queries& s, int unit, int row, int length) {
  return length - s.tokens + (unit % s.row_tiles * kRows + row) / s.group < 0;
}
// A row's result from its sums: 0 without a key, whatever is in the values that its zeros were multiplied with
// (a sum that is NaN says that a page is wrong), and 0 / 0 where all of its scores are -inf.
template <typename M>
__device__ __forceinline__ uint2 row_result(const float4& acc, float sum, bool none) {
  const float inv = 1.0f / sum;
  uint2 out = make_uint2(M::pack(acc.x * inv, acc.y * inv), M::pack(acc.z * inv, acc.w * inv));
  if (none && sum == 0.0f) out = make_uint2(0u, 0u);
  return out;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
    attention_kernel(const __grid_constant__ Queries s, const __grid_constant__ Cache c, float scale, T* __restrict__ o,
                     float* __restrict__ part_o, float2* __restrict__ part_ml) {
  using L = Layout<D>;
  using M = Mma<T>;
  constexpr int kStages = L::kStages;
  constexpr int kTile = L::kTile, kKeys = L::kKeys;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t scratch[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * L::kWarpBytes;
  constexpr uint32_t kStageBytes = kWarps * L::kWarpBytes;
  float* join = reinterpret_cast<float*>(smem + L::kRing);  // [warp][row of 8]
  float2* join_ml = reinterpret_cast<float2*>(smem + L::kRing + L::kJoin);
  const int units = s.heads * s.row_tiles;

  Cursor<kTile> at = {0, 0, 0, 0, 0};
  int64_t steps;
  if (s.whole) {
    at.b = blockIdx.x / units, at.unit = blockIdx.x - at.b * units;
    at.length = length_of(c, at.b), at.tiles = tiles_of<kTile>(at.length);
    steps = at.tiles;
    if (steps == 0) {  // no keys, or no table for them
      const float x = c.lengths[at.b] > 0 ? __int_as_float(0x7fc00000) : 0.0f;
      const uint32_t w = M::pack(x, x);
      for (int i = threadIdx.x; i < rows_of(s, at.unit) * (D / 8); i += kThreads)
        reinterpret_cast<uint4*>(o + out_row(s, at.b, at.unit, i / (D / 8)) * D)[i % (D / 8)] = make_uint4(w, w, w, w);
      return;
    }
  } else {
    // sequences without keys
    const int64_t chunks = (int64_t)s.tokens * s.heads * s.group * (D / 8);
    for (int b = blockIdx.x; b < s.batch; b += kCtas)
      if (c.lengths[b] <= 0)
        for (int64_t i = threadIdx.x; i < chunks; i += kThreads)
          reinterpret_cast<uint4*>(o + b * chunks * 8)[i] = make_uint4(0, 0, 0, 0);
    const Share share = share_of<kTile>(c, s.batch, units, scratch);
    steps = share.steps;
    if (steps == 0) return;
    at.b = share.b;
    at.length = length_of(c, at.b), at.tiles = tiles_of<kTile>(at.length);
    const int64_t in = share.first - share.before;
    at.unit = (int)(in / at.tiles), at.tile = (int)(in - (int64_t)at.unit * at.tiles);
  }

  // ---- loads: `ahead` is the next tile to load, its table entries on their way.  Lane i looks up key i of the
  // warp's; rows are addressed in 16-byte units (32 bits of them: 64 GiB a cache).
  constexpr uint32_t kAbsent = 0xffffffffu;
  Cursor<kTile> ahead = at;
  int64_t loaded = 0;
  uint32_t bad_stages = 0;  // stages with a page that the cache does not have
  int entry = 0, place = 0;
  bool inside = false;
  const auto look_up = [&] {
    const int key = ahead.tile * kTile + warp * kKeys + (kKeys == 32 ? lane : lane & 15);
    inside = key < ahead.length;
    int e = __umulhi((uint32_t)key, c.page_inverse);  // at most 1 below key / page_size
    place = key - e * c.page_size;
    if (place >= c.page_size) place -= c.page_size, ++e;
    entry = inside ? __ldg(c.table + ahead.b * c.table_row + e) : 0;
  };
  const auto issue = [&](int stage) {
    if (loaded < steps) {
      const bool wrong = inside && (entry < 0 || entry >= c.pages);
      const int head = ahead.unit / s.row_tiles;
      uint32_t k_row = kAbsent, v_row = kAbsent;
      if (inside && !wrong) {
        k_row = (uint32_t)((entry * c.k_page + place * c.k_place + head * c.k_head) >> 3);
        v_row = (uint32_t)((entry * c.v_page + place * c.v_place + head * c.v_head) >> 3);
      }
      bad_stages = (bad_stages & ~(1u << stage)) | ((uint32_t)(__any_sync(0xffffffffu, wrong) != 0) << stage);
      constexpr int kChunks = D / 8, kAtOnce = 32 / kChunks;  // 16-byte chunks of a row; rows of a warp's load
      const int chunk = lane % kChunks;
      const uint32_t dst = ring + stage * kStageBytes;
      const char* const k = static_cast<const char*>(c.k) + chunk * 16;
      const char* const v = static_cast<const char*>(c.v) + chunk * 16;
#pragma unroll
      for (int row0 = 0; row0 < kKeys; row0 += kAtOnce) {
        const int r = row0 + lane / kChunks;
        const uint32_t to = dst + r * (D * 2) + ((chunk ^ (r & 7)) << 4);
        const uint32_t kr = __shfl_sync(0xffffffffu, k_row, r), vr = __shfl_sync(0xffffffffu, v_row, r);
        load16(to, kr != kAbsent ? k + ((uint64_t)kr << 4) : k, kr != kAbsent);
        load16(to + kKeys * D * 2, vr != kAbsent ? v + ((uint64_t)vr << 4) : v, vr != kAbsent);
      }
      ++loaded;
      ahead.next(c, s.batch, units);
      if (loaded < steps) look_up();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  look_up();
  for (int i = 0; i < kStages - 1; ++i) issue(i);

  // ---- one unit's (or piece's) state
  uint32_t qf[D / 16][4];
  float acc[D / 8][4];
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
  int lim0 = 0, lim1 = 0;  // keys that rows lane / 4 and lane / 4 + 8 see
  bool bad = false;
  const int r0 = lane >> 2, c2 = 2 * (lane & 3);
  const auto load_queries = [&](const Cursor<kTile>& u) {
    const int head = u.unit / s.row_tiles, base = (u.unit - head * s.row_tiles) * kRows, all = s.tokens * s.group;
    const T* q = static_cast<const T*>(s.q) + u.b * s.q_b;
    const T* row[2];
    int lim[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // rows behind the last one go along with it
      const int r = min(base + r0 + 8 * i, all - 1), token = r / s.group;
      row[i] = q + token * s.q_t + (head * s.group + (r - token * s.group)) * s.q_h;
      lim[i] = u.length - s.tokens + token + 1;
    }
    lim0 = lim[0], lim1 = lim[1];
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qf[k][i] = *reinterpret_cast<const uint32_t*>(row[i & 1] + 16 * k + 8 * (i >> 1) + c2);
  };
  const auto clear = [&] {
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
    m0 = m1 = -INFINITY, l0 = l1 = 0.0f;
    bad = c.lengths[at.b] > c.table_width * c.page_size;
  };

  int piece_tile = at.tile;     // the piece's first tile
  bool at_start = true;         // ... is the share's first
  load_queries(at);
  clear();
  int stage = 0;
  for (int64_t step = 0; step < steps; ++step, stage = stage + 1 == kStages ? 0 : stage + 1) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    bad |= (bad_stages >> stage) & 1u;
    issue(stage == 0 ? kStages - 1 : stage - 1);  // over the stage of the step before

    const int key0 = at.tile * kTile + warp * kKeys;
    if (key0 < at.length) {
      constexpr int kBlocks = kKeys / 8;
      const uint32_t keys = ring + stage * kStageBytes, values = keys + kKeys * D * 2;
      // S = Q K^T: blocks of 8 keys
      float sc[kBlocks][4] = {};
      {
        const int row = ((lane >> 4) << 3) + (lane & 7), part = (lane >> 3) & 1;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int nb = 0; nb < kBlocks; nb += 2) {
            uint32_t b[4];
            ldmatrix(b, keys + (8 * nb + row) * (D * 2) + (((2 * k + part) ^ (row & 7)) << 4));
            M::run(sc[nb], qf[k], b[0], b[1]);
            M::run(sc[nb + 1], qf[k], b[2], b[3]);
          }
      }
      if (key0 + kKeys > at.length - s.tokens + 1) {
#pragma unroll
        for (int nb = 0; nb < kBlocks; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = key0 + 8 * nb + c2 + e;
            if (key >= lim0) sc[nb][e] = -INFINITY;
            if (key >= lim1) sc[nb][2 + e] = -INFINITY;
          }
      }
      // the running maximum is raised when a score lies 2^kLag above it
      float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb)
        x0 = fmaxf(x0, fmaxf(sc[nb][0], sc[nb][1])), x1 = fmaxf(x1, fmaxf(sc[nb][2], sc[nb][3]));
      x0 = x0 * scale - M::kShift, x1 = x1 * scale - M::kShift;
      if (__any_sync(0xffffffffu, x0 > m0 + M::kLag || x1 > m1 + M::kLag)) {
#pragma unroll
        for (int off = 1; off <= 2; off <<= 1) {
          x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, off));
          x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, off));
        }
        const float n0 = x0 > m0 + M::kLag ? x0 : m0, n1 = x1 > m1 + M::kLag ? x1 : m1;
        const float a0 = n0 == m0 ? 1.0f : ex2(m0 - n0), a1 = n1 == m1 ? 1.0f : ex2(m1 - n1);
        m0 = n0, m1 = n1, l0 *= a0, l1 *= a1;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) acc[i][0] *= a0, acc[i][1] *= a0, acc[i][2] *= a1, acc[i][3] *= a1;
      }
      const float b0 = m0 == -INFINITY ? 0.0f : m0, b1 = m1 == -INFINITY ? 0.0f : m1;
#pragma unroll
      for (int kb = 0; kb < kBlocks; kb += 2) {  // 16 keys of the product with V
        uint32_t p[4], p_rest[4];  // p is taken in two 16-bit parts: the products are there for the taking
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float(&x)[4] = sc[kb + i];
          const float p0 = ex2(fmaf(x[0], scale, -b0)), p1 = ex2(fmaf(x[1], scale, -b0));
          const float p2 = ex2(fmaf(x[2], scale, -b1)), p3 = ex2(fmaf(x[3], scale, -b1));
          l0 += p0 + p1, l1 += p2 + p3;
          p[2 * i] = M::pack(p0, p1), p[2 * i + 1] = M::pack(p2, p3);
          const float2 h0 = M::unpack(p[2 * i]), h1 = M::unpack(p[2 * i + 1]);
          p_rest[2 * i] = M::pack(p0 - h0.x, p1 - h0.y), p_rest[2 * i + 1] = M::pack(p2 - h1.x, p3 - h1.y);
        }
        // O += P V
        const int row = (((lane >> 3) & 1) << 3) + (lane & 7), part = lane >> 4;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          uint32_t b[4];
          ldmatrix_t(b, values + (8 * kb + row) * (D * 2) + (((2 * n + part) ^ (row & 7)) << 4));
          M::run(acc[2 * n], p, b[0], b[1]);
          M::run(acc[2 * n + 1], p, b[2], b[3]);
          M::run(acc[2 * n], p_rest, b[0], b[1]);
          M::run(acc[2 * n + 1], p_rest, b[2], b[3]);
        }
      }
    }

    const bool unit_ends = at.tile + 1 == at.tiles;
    if (!unit_ends && step + 1 < steps) {
      ++at.tile;
      continue;
    }
    // ---- the end of a piece: the four warps' sums, joined in order, 8 rows at a time
    const Cursor<kTile> done = at;
    at.next(c, s.batch, units);
    if (step + 1 < steps) load_queries(at);  // on their way meanwhile
#pragma unroll
    for (int off = 1; off <= 2; off <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, off);
      l1 += __shfl_xor_sync(0xffffffffu, l1, off);
    }
    if (bad) l0 = l1 = __int_as_float(0x7fc00000);
    const int rows = rows_of(s, done.unit);
    const bool whole = piece_tile == 0 && unit_ends;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (8 * half >= rows) break;
      __syncthreads();
      float* to = join + (warp * 8 + r0) * L::kPitch + c2;
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<float2*>(to + 8 * i) = make_float2(acc[i][2 * half], acc[i][2 * half + 1]);
      if ((lane & 3) == 0) join_ml[warp * 8 + r0] = half ? make_float2(m1, l1) : make_float2(m0, l0);
      __syncthreads();
      for (int i = threadIdx.x; i < min(rows - 8 * half, 8) * (D / 4); i += kThreads) {
        const int r = i / (D / 4), col = (i - r * (D / 4)) * 4;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, join_ml[w * 8 + r].x);
        float4 all = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 x = join_ml[w * 8 + r];
          const float4 v = *reinterpret_cast<const float4*>(join + (w * 8 + r) * L::kPitch + col);
          const float f = x.x == -INFINITY ? 0.0f : ex2(x.x - top);
          sum += x.x == -INFINITY ? x.y : x.y * f;  // no key: 0, or NaN for a wrong page
          all.x = fmaf(v.x, f, all.x), all.y = fmaf(v.y, f, all.y), all.z = fmaf(v.z, f, all.z), all.w = fmaf(v.w, f, all.w);
        }
        if (whole) {
          *reinterpret_cast<uint2*>(o + out_row(s, done.b, done.unit, 8 * half + r) * D + col) =
              row_result<M>(all, sum, sees_none(s, done.unit, 8 * half + r, done.length));
        } else {
          const int64_t slot = ((int64_t)blockIdx.x * 2 + (at_start ? 0 : 1)) * kRows + 8 * half + r;
          *reinterpret_cast<float4*>(part_o + slot * D + col) = all;
          if (col == 0) part_ml[slot] = make_float2(top, sum);
        }
      }
    }
    piece_tile = at.tile, at_start = false;
    if (step + 1 < steps) clear();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Joins the pieces of a divided unit: o = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c over the shares that
// hold one, in order.  A CTA takes a row of a unit (one row of 37 pieces each for 8 CTAs took 29 us behind
// 131,001 keys, where the attention takes 83): the pieces' factors first, a thread a piece, then their sums, D / 4
// columns of every kGroups-th piece a thread.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads)
    join_kernel(const __grid_constant__ Queries s, const __grid_constant__ Cache c, T* __restrict__ o,
                const float* __restrict__ part_o, const float2* __restrict__ part_ml) {
  constexpr int kCols = D / 4, kGroups = kThreads / kCols;
  __shared__ int64_t scratch[kWarps];
  __shared__ float factor[kCtas];
  __shared__ float of_warps[2][kWarps];
  __shared__ float4 of_groups[kThreads];
  constexpr int kTile = Layout<D>::kTile;
  const int units = s.heads * s.row_tiles, b = blockIdx.x / units, unit = blockIdx.x - b * units, r = blockIdx.y;
  const int length = length_of(c, b), tiles = tiles_of<kTile>(length);
  const Deal deal(tiles_before<kTile>(c, s.batch, units, scratch));
  const int64_t first = tiles_before<kTile>(c, b, units, scratch) + (int64_t)unit * tiles;
  cudaGridDependencySynchronize();  // in every CTA: what follows in the stream waits for the attention too
  if (tiles == 0 || r >= rows_of(s, unit)) return;
  const int c0 = deal.owner(first), pieces = deal.owner(first + tiles - 1) - c0 + 1;
  if (pieces == 1) return;  // written by that share
  // the first piece is its share's last one, unless it begins there; the others are their shares' first
  const bool inside = deal.start(c0) != first;
  const auto slot = [&](int i) { return ((int64_t)(c0 + i) * 2 + (i == 0 && inside)) * kRows + r; };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float top = -INFINITY;
  for (int i = threadIdx.x; i < pieces; i += kThreads) top = fmaxf(top, part_ml[slot(i)].x);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  if (lane == 0) of_warps[0][warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, of_warps[0][w]);
  float sum = 0.0f;
  for (int i = threadIdx.x; i < pieces; i += kThreads) {
    const float2 x = part_ml[slot(i)];
    const float f = x.x == -INFINITY ? 0.0f : ex2(x.x - top);
    factor[i] = f;
    sum += x.x == -INFINITY ? x.y : x.y * f;  // no key: 0, or NaN for a wrong page
  }
  sum = warp_sum(sum);
  if (lane == 0) of_warps[1][warp] = sum;
  __syncthreads();
  sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum += of_warps[1][w];
  const int col = threadIdx.x % kCols;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = threadIdx.x / kCols; i < pieces; i += kGroups) {
    const float4 v = *reinterpret_cast<const float4*>(part_o + slot(i) * D + col * 4);
    const float f = factor[i];
    acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y), acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
  }
  of_groups[threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.x >= kCols) return;
#pragma unroll
  for (int g = 1; g < kGroups; ++g) {
    const float4 v = of_groups[g * kCols + threadIdx.x];
    acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
  }
  *reinterpret_cast<uint2*>(o + out_row(s, b, unit, r) * D + col * 4) = row_result<Mma<T>>(acc, sum, sees_none(s, unit, r, length));
}

template <typename T, int D>
static cudaError_t launch_attention(Queries s, const Cache& c, float scale, void* o, void* workspace, cudaStream_t stream) {
  const auto kernel = attention_kernel<T, D>;
  constexpr int bytes = Layout<D>::kBytes;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err != cudaSuccess) return err;
  const int all = s.batch * s.heads * s.row_tiles;
  float2* ml = static_cast<float2*>(workspace);
  float* part = reinterpret_cast<float*>(ml + 2 * kCtas * kRows);
  s.whole = (int64_t)c.table_width * c.page_size <= kWhole;
  kernel<<<s.whole ? all : kCtas, kThreads, bytes, stream>>>(s, c, scale, (T*)o, part, ml);
  err = cudaGetLastError();
  if (err != cudaSuccess || s.whole) return err;
  // its launch overlaps the first kernel's end
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute overlap = {};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  config.gridDim = dim3((unsigned)all, (unsigned)min(kRows, s.tokens * s.group)), config.blockDim = dim3(kThreads), config.stream = stream;
  config.attrs = &overlap, config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, join_kernel<T, D>, (const Queries)s, (const Cache)c, (T*)o, (const float*)part, (const float2*)ml);
}

static prism_status_t check_cache(const Cache& c, const int64_t* k_strides, const int64_t* v_strides, int batch,
                                  const char* what) {
  PRISM_CHECK_ARG(c.page_size >= 1 && c.table_width >= 0 && c.pages >= 0 && batch >= 0 &&
                      (int64_t)c.page_size * c.table_width < ((int64_t)1 << 31) - 256,
                  "%s: bad sizes (page size at least 1, fewer than 2^31 keys a sequence)", what);
  PRISM_CHECK_ARG(k_strides && v_strides && (batch == 0 || c.lengths) && (batch == 0 || c.table_width == 0 || c.table) &&
                      (c.pages == 0 || (c.k && c.v)),
                  "%s: null pointer", what);
  return PRISM_OK;
}

// Strides of dimensions of one are never used, and may be anything: 0 then.
static void take_strides(Cache& c, const int64_t* k, const int64_t* v, int heads) {
  c.k_page = c.pages > 1 ? k[0] : 0, c.k_place = c.page_size > 1 ? k[1] : 0, c.k_head = heads > 1 ? k[2] : 0;
  c.v_page = c.pages > 1 ? v[0] : 0, c.v_place = c.page_size > 1 ? v[1] : 0, c.v_head = heads > 1 ? v[2] : 0;
}

}  // namespace paged
}  // namespace prism

using namespace prism;

extern "C" {

prism_status_t prism_append_paged(const void* q, const int64_t* q_strides, int q_heads, const void* k,
                                  const int64_t* k_strides, const void* v, const int64_t* v_strides, int k_heads,
                                  int64_t tokens, int dim, const void* offsets, int offsets_64, int batch, void* k_cache,
                                  const int64_t* k_cache_strides, void* v_cache, const int64_t* v_cache_strides,
                                  int pages, int page_size, const int* page_table, int64_t table_row, int table_width,
                                  const int* lengths, int rot, int interleaved, const double* freqs, float scale,
                                  int dtype, void* q_out, cudaStream_t stream) {
  constexpr const char* what = "prism_append_paged";
  PRISM_CHECK_ARG(tokens >= 0 && tokens < ((int64_t)1 << 30) && dim >= 1 && dim <= paged::kAppendThreads && rot >= 0 && rot % 2 == 0 &&
                      rot <= dim && q_heads >= 0 && k_heads >= 1 &&
                      ((int64_t)q_heads + 2 * (int64_t)k_heads) * dim < ((int64_t)1 << 30),
                  "%s: bad sizes (head dim up to %d, an even part of it rotated)", what, paged::kAppendThreads);
  PRISM_CHECK_ARG(dtype == PRISM_BF16 || dtype == PRISM_FP16, "%s: element type %d (bf16 or fp16)", what, dtype);
  paged::Cache c = {};
  c.k = k_cache, c.v = v_cache, c.table = page_table, c.table_row = table_row, c.table_width = table_width;
  c.page_size = page_size, c.pages = pages, c.lengths = lengths;
  const prism_status_t st = paged::check_cache(c, k_cache_strides, v_cache_strides, batch, what);
  if (st != PRISM_OK) return st;
  PRISM_CHECK_ARG(offsets != nullptr || batch == 0 || tokens % batch == 0, "%s: %lld tokens of %d sequences", what,
                  (long long)tokens, batch);
  if (tokens == 0) return PRISM_OK;
  PRISM_CHECK_ARG(k && v && k_strides && v_strides && (q_heads == 0 || (q && q_strides && q_out)) && (rot == 0 || freqs) &&
                      batch >= 1,
                  "%s: null pointer, or tokens without a sequence", what);
  paged::take_strides(c, k_cache_strides, v_cache_strides, k_heads);
  paged::Append a = {};
  const void* in[3] = {q, k, v};
  const int64_t* strides[3] = {q_strides, k_strides, v_strides};
  const int heads[3] = {q_heads, k_heads, k_heads};
  for (int i = 0; i < 3; ++i) {
    a.heads[i] = heads[i];
    if (heads[i] > 0) a.in[i] = in[i], a.in_t[i] = strides[i][0], a.in_h[i] = strides[i][1];
  }
  a.q_out = q_out, a.offsets = offsets, a.wide = offsets_64, a.count = batch, a.tokens = (int)tokens;
  a.each = offsets != nullptr ? 0 : (int)(tokens / batch);
  const cudaError_t err =
      dtype == PRISM_FP16 ? paged::dispatch_append<__half>(a, c, freqs, dim, rot, interleaved, scale, stream)
                          : paged::dispatch_append<__nv_bfloat16>(a, c, freqs, dim, rot, interleaved, scale, stream);
  PRISM_CHECK_CUDA(err, what);
  return PRISM_OK;
}

size_t prism_paged_attention_workspace_bytes(int D, int page_size, int table_width) {
  if (D < 1 || (int64_t)page_size * table_width <= paged::kWhole) return 0;
  return (size_t)2 * paged::kCtas * paged::kRows * (sizeof(float2) + D * sizeof(float));
}

prism_status_t prism_paged_attention(const void* q, const int64_t* q_strides, int batch, int tokens, int q_heads,
                                     int k_heads, int D, const void* k_cache, const int64_t* k_cache_strides,
                                     const void* v_cache, const int64_t* v_cache_strides, int pages, int page_size,
                                     const int* page_table, int64_t table_row, int table_width, const int* lengths,
                                     float scale, int dtype, void* o, void* workspace, cudaStream_t stream) {
  constexpr const char* what = "prism_paged_attention";
  PRISM_CHECK_ARG(D == 64 || D == 128, "%s: head dim %d not supported (64, 128)", what, D);
  PRISM_CHECK_ARG(k_heads >= 1 && q_heads >= 1 && q_heads % k_heads == 0 && tokens >= 0 && batch >= 0, "%s: bad sizes", what);
  PRISM_CHECK_ARG((int64_t)batch * tokens * q_heads < ((int64_t)1 << 28), "%s: too many rows", what);
  PRISM_CHECK_ARG(dtype == PRISM_BF16 || dtype == PRISM_FP16, "%s: element type %d (bf16 or fp16)", what, dtype);
  PRISM_CHECK_ARG(scale > 0.0f && scale < 1.0e30f, "%s: the scale must be positive and finite", what);
  paged::Cache c = {};
  c.k = const_cast<void*>(k_cache), c.v = const_cast<void*>(v_cache), c.table = page_table, c.table_row = table_row;
  c.table_width = table_width, c.page_size = page_size, c.pages = pages, c.lengths = lengths;
  if (page_size >= 1) c.page_inverse = 0xffffffffu / (uint32_t)page_size;
  const prism_status_t st = paged::check_cache(c, k_cache_strides, v_cache_strides, batch, what);
  if (st != PRISM_OK) return st;
  if ((int64_t)batch * tokens == 0) return PRISM_OK;
  PRISM_CHECK_ARG(q && q_strides && o && (workspace || prism_paged_attention_workspace_bytes(D, page_size, table_width) == 0) && aligned16(o) && aligned16(workspace), "%s: null pointer, or a buffer off 16 bytes", what);
  paged::take_strides(c, k_cache_strides, v_cache_strides, k_heads);
  const int64_t all_strides = c.k_page | c.k_place | c.k_head | c.v_page | c.v_place | c.v_head;
  PRISM_CHECK_ARG(aligned16(k_cache) && aligned16(v_cache) && all_strides >= 0 && (all_strides & 7) == 0,
                  "%s: the caches' rows must start on 16 bytes, with strides that are not negative", what);
  constexpr double kMost = 34359738368.0;  // elements: 2^32 units of 16 bytes
  const auto extent = [&](int64_t page, int64_t place, int64_t head) {
    return (double)(pages - 1) * page + (double)(page_size - 1) * place + (double)(k_heads - 1) * head + D;
  };
  PRISM_CHECK_ARG(extent(c.k_page, c.k_place, c.k_head) <= kMost && extent(c.v_page, c.v_place, c.v_head) <= kMost,
                  "%s: caches of 64 GiB and more", what);
  PRISM_CHECK_ARG(aligned_to(q, 4) && ((q_strides[0] | q_strides[1] | q_strides[2]) & 1) == 0, "%s: q's rows must start on 4 bytes", what);
  paged::Queries s = {q, q_strides[0], q_strides[1], q_strides[2], batch, tokens, k_heads, q_heads / k_heads, 0, 0};
  s.row_tiles = (int)(((int64_t)tokens * s.group + paged::kRows - 1) / paged::kRows);
  const float by = scale * 1.4426950408889634f;
  cudaError_t err;
  if (dtype == PRISM_FP16)
    err = D == 64 ? paged::launch_attention<__half, 64>(s, c, by, o, workspace, stream)
                  : paged::launch_attention<__half, 128>(s, c, by, o, workspace, stream);
  else
    err = D == 64 ? paged::launch_attention<__nv_bfloat16, 64>(s, c, by, o, workspace, stream)
                  : paged::launch_attention<__nv_bfloat16, 128>(s, c, by, o, workspace, stream);
  PRISM_CHECK_CUDA(err, what);
  return PRISM_OK;
}

}  // extern "C"
