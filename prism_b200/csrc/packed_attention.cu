// Dense attention over packed sequences, forward and backward, on the sm_100a tensor cores.
//
// q [T, Hq, D], k and v [Tk, Hk, D]: sequence b is the rows [offsets[b], offsets[b + 1]) of its
// tensors; G = Hq / Hk query heads share a key head.  With n queries and m keys of a sequence, query i
// attends keys j < m, or, causal, j <= i + m - n (the last query is at the last key):
//
//   s_ij = scale q_i . k_j,   p_ij = exp(s_ij - max_j s_ij) / sum_j exp(..),   o_i = sum_j p_ij v_j
//   delta_i = do_i . o_i,   ds_ij = p_ij (do_i . v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij do_i,
//
// dk and dv over the queries of all G heads.  A row without keys has o = 0 and no gradients.
//
// Bound by the tensor cores (4 D operations a score forward, 10 D backward).  What the kernels share:
//   * A tile of 128 rows holds all G heads of n = 128 / G tokens, row (token, head): one TMA box
//     {64 columns, G heads, n tokens}.  Heads that share keys share their loads, a sequence of few
//     tokens fills more of a tile than one head's rows would, and the diagonal of a causal tile is n
//     keys wide instead of 128.  A G that does not divide 128 leaves 128 - n G rows zero.
//   * A step is 128 keys (queries in dK / dV): an M = 128 product costs at least 45 clocks, so
//     N = 128 is needed for the math rate.
//   * Tiles end inside sequences, so a tile's last rows are the next sequence's (or lie behind the
//     tensor: TMA reads zeros there).  Scores of such keys are replaced, not multiplied, and rows that
//     a product sums over (V; K in dQ; Q and dO in dK / dV) are set to zero in shared memory first:
//     a NaN in one sequence stays there, 0 * NaN being NaN.
//   * Scores in log2 units; fp32 statistics and accumulators; P and dS rounded to the inputs' 16 bits
//     for the second products, as the matrix instruction takes them (a second part of P, for what that leaves,
//     would be half as many products again): o is off by 0.0021 of its norm in bf16, 0.00029 in fp16, where one
//     rounding of the result gives 0.0016 and 0.00021.
//   * The tiles of a grid are its CTAs' work items; a grid has the upper bound of tiles that the row counts
//     allow, and its spare items clear the rows that no sequence holds.  Offsets that decrease or leave the
//     tensors give NaN.  The lengths are read on the device only: no host copy, no plan kernel.
//   * A CTA that is running takes over the items of CTAs that have not started (cluster launch control), so
//     that barriers and TMEM are set up once an SM, the next item's loads and first scores run under this
//     one's epilogue, and the hardware's order (long causal tiles first) still balances the SMs.
//
// Warp roles (320 threads): warps 0-7 softmax and epilogue (thread i of a warpgroup owns TMEM lane i),
// warp 8 TMA producer, which also takes the items and finds their sequences, warp 9 MMA issuer (lane 0
// issues; all lanes clear tail rows) and TMEM owner.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <stdint.h>

#include <mutex>
#include <type_traits>

#include "attention_tc.cuh"
#include "prism_common.cuh"
#include "sm100.cuh"

namespace prism {
namespace packed {

using namespace tc;

constexpr int kThreads = 320;
constexpr int kSoftmaxThreads = 256;
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kItemReaders = 9;           // the warps other than the producer
constexpr int kRows = 128;                // of a tile; keys of a step
constexpr size_t kMinSmem = 116 * 1024;   // one CTA an SM: each allocates all of TMEM
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSms = 148;

// First bounded wait that gave up (prism_device_status).
__device__ int g_error = 0;
enum WaitCode : int {
  kErrFwdProducer = 501, kErrFwdMma = 502, kErrFwdSoftmax = 503,
  kErrDkdvProducer = 511, kErrDkdvMma = 512, kErrDkdvSoftmax = 513,
  kErrDqProducer = 521, kErrDqMma = 522, kErrDqSoftmax = 523,
};

__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
  return mbar_wait(bar, parity, abort_flag, &g_error, code);
}
// Warp-uniform result (every lane must agree before a .sync.aligned operation).
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
  const bool ok = __all_sync(0xffffffffu, wait_one(bar, parity, abort_flag, code));
  if (!ok) *abort_flag = 1;
  return ok;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// 32 bytes to global memory: a sector, whole.
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// ------------------------------------------------------------------ element types
// kShift: log2 of the largest p that a fresh maximum gives.  fp16 keeps p >= 2^-24 only, so its maximum is
// put at 2^8 and keys down to 2^-32 of the largest count; kLag more (2^15 in all, below fp16's 65504)
// until the maximum is raised.  kSum: a half step's exponentials below it all are within that; 64 equal
// scores are.
template <typename T>
struct Half;
template <>
struct Half<__nv_bfloat16> {
  static constexpr float kShift = 0.0f, kLag = 8.0f, kSum = 65536.0f;
  static constexpr uint32_t kFormat = 1;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16(lo, hi); }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
};
template <>
struct Half<__half> {
  static constexpr float kShift = 8.0f, kLag = 7.0f, kSum = 32768.0f;
  static constexpr uint32_t kFormat = 0;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
};
// Instruction descriptor as idesc_bf16's, both operands of type T.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int N, bool b_mn) {
  return (1u << 4) | (Half<T>::kFormat << 7) | (Half<T>::kFormat << 10) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}

// ------------------------------------------------------------------ sequences
struct Sequences {
  const void *q, *k;       // offsets, count + 1 of them
  int wide;                // 64-bit
  int count;
  int q_rows, k_rows;      // of the tensors
};
// Heads and the tiles that they give: n = tokens of a tile; pairs = upper bound of the pairs of tiles.
struct Heads {
  int keys, group, tokens, pairs;
};

enum Kind : int { kTile, kSpare, kBad, kStop };  // kStop: no more items

__device__ __forceinline__ int64_t row_at(const void* offsets, int wide, int i) {
  return wide ? static_cast<const long long*>(offsets)[i] : (int64_t)static_cast<const int*>(offsets)[i];
}

// An item without a tile: clears its share of the rows that no sequence holds (kSpare), or fills its share of
// all rows with NaN (kBad).  Rows of `out` are [heads, width] elements; the item has those of key head h:
// `width` elements from h * width on.
template <typename T>
__device__ void fill_rows(int kind, int share, const void* offsets, const Sequences& s, int rows, int per, T* out,
                          int heads, int h, int width) {
  const bool bad = kind == kBad;
  const int head = bad ? 0 : (int)row_at(offsets, s.wide, 0), tail = bad ? 0 : (int)row_at(offsets, s.wide, s.count);
  const int count = bad ? rows : head + rows - tail;
  const int64_t first = (int64_t)share * per;
  const int64_t end = first + per < count ? first + per : count;
  const uint32_t word = bad ? Half<T>::pack(__uint_as_float(0x7fc00000u), __uint_as_float(0x7fc00000u)) : 0u;
  const int chunks = width / 8;
  for (int64_t i = first * chunks + threadIdx.x; i < end * chunks; i += kSoftmaxThreads) {
    const int64_t u = i / chunks;
    const int64_t row = u < head ? u : tail + (u - head);
    *reinterpret_cast<uint4*>(out + (row * heads + h) * width + (i - u * chunks) * 8) = make_uint4(word, word, word, word);
  }
}

// The same for the (maximum, sum) of a part's rows.
__device__ __forceinline__ void fill_parts(int kind, int share, const Sequences& s, int per, float2* ml, const Heads& hd, int h) {
  const bool bad = kind == kBad;
  const int head = bad ? 0 : (int)row_at(s.q, s.wide, 0), tail = bad ? 0 : (int)row_at(s.q, s.wide, s.count);
  const int count = bad ? s.q_rows : head + s.q_rows - tail;
  const int64_t first = (int64_t)share * per, end = first + per < count ? first + per : count;
  for (int64_t i = first * hd.group + threadIdx.x; i < end * hd.group; i += kSoftmaxThreads) {
    const int64_t u = i / hd.group, row = u < head ? u : tail + (u - head);
    ml[(row * hd.keys + h) * hd.group + (i - u * hd.group)] = make_float2(-INFINITY, bad ? __uint_as_float(0x7fc00000u) : 0.0f);
  }
}

// ------------------------------------------------------------------ items
struct Item {
  int kind;
  int q0, nq, k0, nk;   // the sequence's rows
  int tile;             // within the sequence; kSpare, kBad: the share of the rows to fill
  int pairs;            // pairs of query tiles of the sequences before
  int index, h, part;   // the tile's number in the grid, the key head, the part of its steps
};

// What the scan of all offsets finds: whether they are in order, and the tiles and pairs of query tiles.
struct Survey {
  int good, tiles, pairs;
};
template <bool kKeys>
__device__ Survey survey(const Sequences& s, int pair_tokens, int* scratch) {
  int tiles = 0, pairs = 0;
  bool good = true;
  for (int b = threadIdx.x; b < s.count; b += kThreads) {
    const int64_t qa = row_at(s.q, s.wide, b), qb = row_at(s.q, s.wide, b + 1);
    const int64_t ka = row_at(s.k, s.wide, b), kb = row_at(s.k, s.wide, b + 1);
    if (0 <= qa && qa <= qb && qb <= s.q_rows && 0 <= ka && ka <= kb && kb <= s.k_rows) {
      const int p = ((int)(qb - qa) + pair_tokens - 1) / pair_tokens;
      pairs += p, tiles += kKeys ? ((int)(kb - ka) + kRows - 1) / kRows : p;
    } else {
      good = false;
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    pairs += __shfl_xor_sync(0xffffffffu, pairs, o);
  }
  if ((threadIdx.x & 31) == 0) scratch[2 * (threadIdx.x >> 5)] = tiles, scratch[2 * (threadIdx.x >> 5) + 1] = pairs;
  Survey all = {__syncthreads_and(good), 0, 0};
  for (int w = 0; w < kThreads / 32; ++w) all.tiles += scratch[2 * w], all.pairs += scratch[2 * w + 1];
  return all;
}

// A warp's way through the sequences, 32 at a time; items come in order, so that it goes through them once.
template <bool kKeys>
struct Walker {
  int chunk, base, tiles, pairs_base, pairs;  // the 32 sequences, tiles before and in them
  int q0, nq, k0, nk, start, count, pairs_start;  // this lane's sequence
  __device__ __forceinline__ void load(const Sequences& s, int pair_tokens, int lane) {
    const int b = chunk * 32 + lane;
    q0 = nq = k0 = nk = 0;
    if (b < s.count) {
      q0 = (int)row_at(s.q, s.wide, b), nq = (int)row_at(s.q, s.wide, b + 1) - q0;
      k0 = (int)row_at(s.k, s.wide, b), nk = (int)row_at(s.k, s.wide, b + 1) - k0;
    }
    const int p = (nq + pair_tokens - 1) / pair_tokens;
    count = kKeys ? (nk + kRows - 1) / kRows : p;
    int x = count, y = p;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int xo = __shfl_up_sync(0xffffffffu, x, o), yo = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) x += xo, y += yo;
    }
    start = x - count, pairs_start = y - p;  // within the 32
    tiles = __shfl_sync(0xffffffffu, x, 31), pairs = __shfl_sync(0xffffffffu, y, 31);
  }
  __device__ __forceinline__ void begin(const Sequences& s, int pair_tokens, int lane, const Survey& all, int my) {
    const bool back = my > all.tiles / 2;
    chunk = back ? (s.count - 1) / 32 : 0;
    load(s, pair_tokens, lane);
    base = back ? all.tiles - tiles : 0, pairs_base = back ? all.pairs - pairs : 0;
  }
  // tile `my` of good sequences' tiles
  __device__ __forceinline__ void find(const Sequences& s, int pair_tokens, int lane, int my, Item& item) {
    while (my < base) {
      --chunk;
      load(s, pair_tokens, lane);
      base -= tiles, pairs_base -= pairs;
    }
    while (my >= base + tiles) {
      ++chunk, base += tiles, pairs_base += pairs;
      load(s, pair_tokens, lane);
    }
    const int in = my - base;
    const int at = __ffs(__ballot_sync(0xffffffffu, in >= start && in < start + count)) - 1;
    const auto of = [&](int v) { return __shfl_sync(0xffffffffu, v, at); };
    item.q0 = of(q0), item.nq = of(nq), item.k0 = of(k0), item.nk = of(nk);
    item.tile = in - of(start), item.pairs = pairs_base + of(pairs_start);
  }
};

// Asks for an item of a CTA that has not started: 16 bytes to `response`, completing on `bar`.
__device__ __forceinline__ void request_item(uint32_t response, uint32_t bar) {
  mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(response),
               "r"(bar)
               : "memory");
}
// The block index of the CTA that will not start, or -1: none is left.
__device__ __forceinline__ int requested_item(uint32_t response) {
  uint32_t got, index;
  asm volatile(
      "{\n .reg .pred p;\n .reg .b128 r;\n"
      " ld.shared.b128 r, [%2];\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n"
      " selp.u32 %0, 1, 0, p;\n mov.u32 %1, 0;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n}\n"
      : "=r"(got), "=r"(index)
      : "r"(response)
      : "memory");
  return got ? (int)index : -1;
}

// Shared memory of the items, at a 16-byte boundary: two of them in turn, each with a barrier that it is
// there and one that all readers have it.
struct ItemRing {
  static constexpr int RESPONSE = 0, FULL = 16, EMPTY = FULL + 16, ANSWER = EMPTY + 16, ITEMS = ANSWER + 16;
  static constexpr int kBytes = ITEMS + 2 * (int)sizeof(Item);
  __device__ static void init(uint32_t at) {
    for (int i = 0; i < 2; ++i) mbar_init(at + FULL + 8 * i, 1), mbar_init(at + EMPTY + 8 * i, kItemReaders);
    mbar_init(at + ANSWER, 1);
  }
};

// How a grid's items follow from the block index: parts of a tile next to each other, then key heads, then
// tiles, the last ones first where `backwards`.
struct Grid {
  int tiles, parts, backwards;
};

// The producer warp's side.  The next item is asked for when the last load of an item is issued, and not
// before: an item taken early is one that an idle SM does not get (nine causal sequences of up to 4,093
// tokens, 1,200 items: 312 us forward with each item asked for at the start of the one before, 256 so).
template <bool kKeys>
struct ItemSource {
  const Sequences& s;
  const Heads& hd;
  const Grid& grid;
  const Survey& all;
  uint8_t* sm_ring;
  uint32_t ring;
  volatile int* abort_flag;
  int lane, code;
  Walker<kKeys> walker;
  bool begun = false;
  int n = 0;  // items so far

  // The next item, given to the other warps too; false: none, or a wait gave up.
  __device__ __forceinline__ bool next(Item& item) {
    int block = blockIdx.x;
    if (n > 0) {
      if (lane == 0) request_item(ring + ItemRing::RESPONSE, ring + ItemRing::ANSWER);
      __syncwarp();
      if (!wait_warp(ring + ItemRing::ANSWER, (n - 1) & 1, abort_flag, code)) return false;
      block = requested_item(ring + ItemRing::RESPONSE);
      fence_proxy_async_smem();  // read, before the next answer is written over it
      __syncwarp();
    }
    item.kind = kStop;
    if (block >= 0) {
      const int of_head = block / grid.parts, rank = of_head / hd.keys;
      item.part = block - of_head * grid.parts, item.h = of_head - rank * hd.keys;
      const int my = grid.backwards ? grid.tiles - 1 - rank : rank;
      item.index = my;
      item.kind = !all.good ? kBad : my >= all.tiles ? kSpare : kTile;
      item.tile = item.kind == kSpare ? my - all.tiles : my;
      if (item.kind == kTile) {
        if (!begun) walker.begin(s, 2 * hd.tokens, lane, all, my);
        begun = true;
        walker.find(s, 2 * hd.tokens, lane, my, item);
      }
    }
    const int slot = n & 1;
    if (n >= 2 && !wait_warp(ring + ItemRing::EMPTY + 8 * slot, ((n >> 1) - 1) & 1, abort_flag, code)) return false;
    if (lane == 0) {
      *reinterpret_cast<Item*>(sm_ring + ItemRing::ITEMS + slot * sizeof(Item)) = item;
      mbar_arrive(ring + ItemRing::FULL + 8 * slot);
    }
    __syncwarp();
    ++n;
    return item.kind != kStop;
  }
};

__device__ __forceinline__ bool item_ready(int n, uint32_t ring) {
  return mbar_try(ring + ItemRing::FULL + 8 * (n & 1), (n >> 1) & 1);
}
// The next item, for a warp; false: the wait gave up, or there is none.
__device__ __forceinline__ bool next_item(Item& item, int& n, const uint8_t* sm_ring, uint32_t ring,
                                          volatile int* abort_flag, int lane, int code) {
  const int slot = n & 1;
  if (!wait_warp(ring + ItemRing::FULL + 8 * slot, (n >> 1) & 1, abort_flag, code)) return false;
  item = *reinterpret_cast<const Item*>(sm_ring + ItemRing::ITEMS + slot * sizeof(Item));
  __syncwarp();
  if (lane == 0) mbar_arrive(ring + ItemRing::EMPTY + 8 * slot);
  ++n;
  return item.kind != kStop;
}

// Rows [from, 128) of a tile's sub-buffers set to zero, by a group of threads; the caller fences and
// synchronises before the tensor core reads them.
template <int kSub>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int from, int thread, int threads) {
  const int chunks = (kRows - from) * 8;
#pragma unroll
  for (int s = 0; s < kSub; ++s)
    for (int i = thread; i < chunks; i += threads)
      *reinterpret_cast<uint4*>(tile + s * 16384 + from * 128 + i * 16) = make_uint4(0, 0, 0, 0);
}

// r / group for r < 128 and group <= 128: (r * ceil(2^16 / group)) >> 16 is exact, the excess being
// below r / 2^16 < 1 / group.
__device__ __forceinline__ int over_group(int r, uint32_t inverse) { return (int)((uint32_t)r * inverse >> 16); }
__device__ __forceinline__ uint32_t group_inverse(int group) { return (65536u + group - 1) / group; }

// Columns from `lim` on -> -inf.
__device__ __forceinline__ void mask_from(float (&s)[64], int lim) {
#pragma unroll
  for (int c = 0; c < 64; ++c)
    if (c >= lim) s[c] = -INFINITY;
}

// Sums of a row's p: before their rounding, and after it where kRounded.
template <bool kRounded>
struct RowSum {
  float exact, rounded;
  __device__ __forceinline__ void scale(float by) {
    exact *= by;
    if constexpr (kRounded) rounded *= by;
  }
  __device__ __forceinline__ void add(const RowSum& x) {
    exact += x.exact;
    if constexpr (kRounded) rounded += x.rounded;
  }
  __device__ __forceinline__ float of_products() const { return kRounded ? rounded : exact; }
};

// p = exp2(s * scale - m) of 64 scores as 32 pairs of T; returns their fp32 sums.
// m is a maximum of earlier scores, so a row's largest p is no power of two and its rounding is off by half a
// step; where that p is nearly all of its row, o = sum p v / sum p is right only if both sums have the same p.  o
// itself is rounded as coarsely, but delta = dO . o is subtracted from a nearly equal dO . v: for training only
// (8,192 causal tokens of 32 + 8 heads at 128 columns: 475 us, 515 so and with o's remainder written).  lse is that of
// the p before rounding.
template <typename T, bool kRounded>
__device__ __forceinline__ RowSum<kRounded> exp_pairs(const float (&s)[64], float scale, float m, uint32_t (&pk)[32]) {
  const float2 sc = make_float2(scale, scale), nm = make_float2(-m, -m), zero = make_float2(0.f, 0.f);
  float2 even = zero, odd = zero, even_r = zero, odd_r = zero;
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    const float2 x = __ffma2_rn(make_float2(s[2 * c], s[2 * c + 1]), sc, nm);
    const float2 p = make_float2(ex2(x.x), ex2(x.y));
    if (c & 1) odd = __fadd2_rn(odd, p);
    else even = __fadd2_rn(even, p);
    pk[c] = Half<T>::pack(p.x, p.y);
    if constexpr (kRounded) {
      const float2 r = Half<T>::unpack(pk[c]);
      if (c & 1) odd_r = __fadd2_rn(odd_r, r);
      else even_r = __fadd2_rn(even_r, r);
    }
  }
  return {(even.x + even.y) + (odd.x + odd.y), (even_r.x + even_r.y) + (odd_r.x + odd_r.y)};
}

// ===================================================================== forward
// An item: two tiles of 128 rows (groups 0 and 1) of one key head, which share the stream of K and V steps, so
// that the tensor core works on one group's products while the other group's softmax runs.  Where there are
// few tiles and long keys, an item is a part of the steps, and join_kernel adds the parts up.
//
// 8,192 causal tokens of 32 + 8 heads: 475 us at 128 columns (1,155 TFLOP/s, the tensor pipe 53 % busy), 390 at 64
// (705 TFLOP/s, 30 %).  Bound by the softmax warps between the products: 2^x of every score alone takes 240 us at
// 16 a clock and SM, and the multiplications, conversions and TMEM traffic around it have the same issue slots.
template <int D>
struct FwdLayout {
  // 64 columns leave room in TMEM for a third S: that of a group's next step is issued before its P is there
  static constexpr int kScores = D == 64 ? 3 : 2;
  static constexpr int kRing = 2;
  static constexpr int kSub = D / 64;
  static constexpr int kTileBytes = kSub * 16384;
  static constexpr int Q = 0;
  static constexpr int K = Q + 2 * kTileBytes;
  static constexpr int V = K + kRing * kTileBytes;
  static constexpr int ITEMS = V + kRing * kTileBytes;
  static constexpr int BAR = ITEMS + (ItemRing::kBytes + 15) / 16 * 16;
  static constexpr int B_QF = 0, B_QE = 2,    // [g]: Q of the group; its last S done
                       B_KF = 4, B_KE = B_KF + kRing, B_VF = B_KE + kRing, B_VE = B_VF + kRing,
                       B_SF = B_VE + kRing,   // [barrier()]: S of the group
                       B_PF = B_SF + 4,       // [barrier()]: P in TMEM (and O rescaled)
                       B_PV = B_PF + 4,       // [g]: P V done
                       B_OF = B_PV + 2,       // [g]: last P V of an item done
                       B_DRAIN = B_OF + 2, NBAR = B_DRAIN + 1;
  static constexpr int TMEM_SLOT = BAR + NBAR * 8;
  static constexpr int ABORT = TMEM_SLOT + 4;
  static constexpr int SCRATCH = ABORT + 4;
  static constexpr size_t kNeed = 1024 + SCRATCH + 2 * 4 * (kThreads / 32);
  static constexpr size_t kBytes = kNeed > kMinSmem ? kNeed : kMinSmem;
  // TMEM: O of each group (D columns), then the S (128 fp32 columns each; P as pairs over the first 64)
  static constexpr int T_O = 0, T_S = 2 * D;
  static_assert(T_S + 128 * kScores <= 512, "TMEM budget");
  // With three S a group may be a step ahead of what the issuer has waited for: its steps take two barriers in
  // turn, or a second phase would look like none.
  static __device__ __forceinline__ int barrier(int g, int step) { return 2 * g + (kScores > 2 ? step & 1 : 0); }
  static __device__ __forceinline__ int phase(int step) { return (kScores > 2 ? step >> 1 : step) & 1; }
};

// The steps of an item: groups' last tokens, the part's first step and each group's number of them.
struct FwdSteps {
  int tok0, shift, last[2], from, n[2], total;
  __device__ __forceinline__ FwdSteps(const Item& at, int n_tok, int causal, int parts) {
    tok0 = at.tile * 2 * n_tok, shift = at.nk - at.nq;
    int all[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      last[g] = min(tok0 + (g + 1) * n_tok, at.nq) - 1;
      const int keys = tok0 + g * n_tok >= at.nq ? 0 : causal ? min(max(last[g] + shift + 1, 0), at.nk) : at.nk;
      all[g] = (keys + kRows - 1) / kRows;
    }
    const int most = max(all[0], all[1]);
    from = (int)((int64_t)most * at.part / parts);
    const int end = (int)((int64_t)most * (at.part + 1) / parts);
#pragma unroll
    for (int g = 0; g < 2; ++g) n[g] = max(0, min(end, all[g]) - from);
    total = max(n[0], n[1]);
  }
};

// What a forward leaves besides o: nothing; what the backward reads; a part's sums in o's place.
enum Mode : int { kInfer, kTrain, kPart };

// What rounding an fp32 value to bf16 leaves, in 8 bits: the second byte of its bit pattern, signed.  The
// lower half of the pattern is what was rounded off, up where its first bit is set -- but for a value in the very
// middle that went down to the even side, which would come back a place too low (+128 is no signed byte).  Of
// means of two bf16 values a tenth lie there.  So 1 / l is taken kAbove times as large, within the sums' fp32 error:
// such a mean lies 2 to 4 of fp32's last places above the middle and goes up, and the middle is left to one value in
// 2^17 (75,600 queries on 512 keys: 980 us, 1,042 with a test of each value's lower bits).  A bf16 value, 2 to 4 places
// above itself, still comes back as it was.  The bytes of four values:
constexpr float kAbove = 1.0f + 1.0f / 4194304.0f;
__device__ __forceinline__ uint32_t rest_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0051), __byte_perm(c, d, 0x0051), 0x5410);
}
// ... and a value again, from its bf16 and byte i of `left`, to 2^-8 of bf16's last place; one that is a bf16
// comes back as it was.
__device__ __forceinline__ float with_rest(uint32_t high, uint32_t left, int i) {
  return __uint_as_float(high + (uint32_t)((int)(int8_t)(left >> (8 * i)) * 256));
}

// What the parts of a row leave: sums [part][row][head][D] and (maximum, sum) [part][row][head].
struct Parts {
  float* o;
  float2* ml;
};

template <typename T, int D, int kMode>
__global__ void __launch_bounds__(kThreads, 1)
    fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Sequences seqs,
               const __grid_constant__ Heads hd, const __grid_constant__ Grid grid, int causal, float qk_scale,
               T* __restrict__ o, float* __restrict__ lse, int8_t* __restrict__ rest, Parts parts) {
  using L = FwdLayout<D>;
  using H = Half<T>;
  constexpr int R = L::kRing;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = align1024(smem_raw);
  const uint32_t sb = smem_u32(sm);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_tok = hd.tokens, rows = n_tok * hd.group;
  auto bar = [&](int i) { return sb + L::BAR + 8 * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::ABORT);
  const uint32_t ring = sb + L::ITEMS;

  if (threadIdx.x == 0) {
    ItemRing::init(ring);
    for (int i = 0; i < R; ++i) {
      mbar_init(bar(L::B_KF + i), 1);
      mbar_init(bar(L::B_KE + i), 1);
      mbar_init(bar(L::B_VF + i), 1);
      mbar_init(bar(L::B_VE + i), 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(bar(L::B_QF + g), 1);
      mbar_init(bar(L::B_QE + g), 1);
      mbar_init(bar(L::B_SF + 2 * g), 1);
      mbar_init(bar(L::B_SF + 2 * g + 1), 1);
      mbar_init(bar(L::B_PF + 2 * g), 4);
      mbar_init(bar(L::B_PF + 2 * g + 1), 4);
      mbar_init(bar(L::B_PV + g), 1);
      mbar_init(bar(L::B_OF + g), 1);
    }
    mbar_init(bar(L::B_DRAIN), 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (rows < kRows) {  // rows that no load fills
    zero_rows<L::kSub>(sm + L::Q, rows, threadIdx.x, kThreads);
    zero_rows<L::kSub>(sm + L::Q + L::kTileBytes, rows, threadIdx.x, kThreads);
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(sb + L::TMEM_SLOT, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  const Survey all = survey<false>(seqs, 2 * n_tok, reinterpret_cast<int*>(sm + L::SCRATCH));
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + L::TMEM_SLOT);

  Item at;
  int items = 0;
  if (warp == kProducerWarp) {
    // ------------------------------------------------------------ producer
    int nk = 0, nv = 0, nq[2] = {0, 0};
    bool ok = true;
    ItemSource<false> source = {seqs, hd, grid, all, sm + L::ITEMS, ring, abort_flag, lane, kErrFwdProducer};
    while (ok && source.next(at)) {
      if (at.kind != kTile) continue;
      const FwdSteps w(at, n_tok, causal, grid.parts);
      if (lane == 0) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (!ok || w.n[g] == 0) continue;
          ok = nq[g] == 0 || wait_one(bar(L::B_QE + g), (nq[g] - 1) & 1, abort_flag, kErrFwdProducer);
          if (!ok) continue;
          mbar_expect_tx(bar(L::B_QF + g), rows * D * 2);
#pragma unroll
          for (int s = 0; s < L::kSub; ++s)
            tma_load_3d(sb + L::Q + g * L::kTileBytes + s * 16384, &tm_q, s * 64, at.h * hd.group,
                        at.q0 + w.tok0 + g * n_tok, bar(L::B_QF + g));
          ++nq[g];
        }
        for (int n = 0; ok && n < w.total; ++n) {
          const int key = at.k0 + (w.from + n) * kRows;
          ok = nk < R || wait_one(bar(L::B_KE + nk % R), ((nk / R) - 1) & 1, abort_flag, kErrFwdProducer);
          if (!ok) break;
          mbar_expect_tx(bar(L::B_KF + nk % R), L::kTileBytes);
#pragma unroll
          for (int s = 0; s < L::kSub; ++s)
            tma_load_3d(sb + L::K + (nk % R) * L::kTileBytes + s * 16384, &tm_k, s * 64, at.h, key, bar(L::B_KF + nk % R));
          ++nk;
          ok = nv < R || wait_one(bar(L::B_VE + nv % R), ((nv / R) - 1) & 1, abort_flag, kErrFwdProducer);
          if (!ok) break;
          mbar_expect_tx(bar(L::B_VF + nv % R), L::kTileBytes);
#pragma unroll
          for (int s = 0; s < L::kSub; ++s)
            tma_load_3d(sb + L::V + (nv % R) * L::kTileBytes + s * 16384, &tm_v, s * 64, at.h, key, bar(L::B_VF + nv % R));
          ++nv;
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
    }
    if (lane == 0) {  // every load has landed before the CTA may leave
      for (int m = max(nk - R, 0); m < nk; ++m) wait_one(bar(L::B_KF + m % R), (m / R) & 1, abort_flag, kErrFwdProducer);
      for (int m = max(nv - R, 0); m < nv; ++m) wait_one(bar(L::B_VF + m % R), (m / R) & 1, abort_flag, kErrFwdProducer);
#pragma unroll
      for (int g = 0; g < 2; ++g)
        if (nq[g] > 0) wait_one(bar(L::B_QF + g), (nq[g] - 1) & 1, abort_flag, kErrFwdProducer);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------- MMA issuer
    // Steps of both groups and of all items in one stream, by lane 0: every instruction between a P and its
    // products is time that the tensor core idles (32,768 causal tokens took 8.9 ms with votes of the warp in
    // each wait).  One thread's products run in issue order.  An item's first P V overwrites an O that the
    // epilogue of the item before has read: the P that it waits for is written after it.
    constexpr uint32_t kIdS = idesc<T>(kRows, false), kIdO = idesc<T>(D, true);
    const uint64_t dQ = desc_k_sw128(sb + L::Q), dK = desc_k_sw128(sb + L::K), dV = desc_mn_sw128(sb + L::V, 16384);
    constexpr uint32_t kSlot = L::kTileBytes >> 4;
    int v_rows = kRows, steps = 0;                 // keys of the last item's last step; all steps so far
    const auto wait = [&](int i, int parity) { return wait_one(bar(i), parity & 1, abort_flag, kErrFwdMma); };
    // the items: item_steps issues an item's steps, finish what is still open
    const auto run = [&](const auto& item_steps, const auto& finish) {
      // all lanes: the last item's last V is there, its rows behind the sequence zero
      const auto clear_tail = [&]() -> bool {
        if (v_rows == kRows) return true;
        const int slot = (steps - 1) % R;
        const bool ok = wait_warp(bar(L::B_VF + slot), ((steps - 1) / R) & 1, abort_flag, kErrFwdMma);
        if (ok) {
          zero_rows<L::kSub>(sm + L::V + slot * L::kTileBytes, v_rows, lane, 32);
          fence_proxy_async_smem();
        }
        v_rows = kRows;
        __syncwarp();
        return ok;
      };
      const auto flush = [&]() -> bool {
        bool ok = clear_tail();
        if (lane == 0 && ok) ok = finish();
        return __all_sync(0xffffffffu, ok);
      };
      bool ok = true;
      while (ok) {
        // an item that is not there yet is not waited for with products to issue
        if (!__any_sync(0xffffffffu, item_ready(items, ring))) ok = flush();
        if (!ok || !next_item(at, items, sm + L::ITEMS, ring, abort_flag, lane, kErrFwdMma)) break;
        if (at.kind != kTile) continue;
        const FwdSteps w(at, n_tok, causal, grid.parts);
        if (w.total == 0) continue;
        ok = clear_tail();
        if (lane == 0 && ok) ok = item_steps(w.n[0], w.n[1]);
        ok = __all_sync(0xffffffffu, ok);
        steps += w.total;
        v_rows = min(at.nk - (w.from + w.total - 1) * kRows, kRows);
      }
      if (ok) flush();
    };
    if constexpr (L::kScores == 2) {
      // Step n, group by group: P V of the group's step before it, then S of step n over the columns that held
      // that P.
      int ns = 0;                                    // steps so far
      int n_s[2] = {0, 0}, n_q[2] = {0, 0};
      bool waiting[2] = {false, false}, first[2] = {}, last[2] = {};  // P V of the last step still to come
      const auto pv = [&](int g) -> bool {
        const int before = (ns - 1) % R;
        const uint32_t t_o = tmem + L::T_O + g * D, t_s = tmem + L::T_S + 128 * g;
        if (!wait(L::B_PF + 2 * g, n_s[g] - 1)) return false;
        tc_fence_after();
        const uint64_t b = dV + before * kSlot;
        mma_ts_k64_mn(t_o, t_s, b, kIdO, first[g] ? 0u : 1u);
        mma_ts_k64_mn(t_o, t_s + 32, b + (8192 >> 4), kIdO, 1u);
        if (last[g]) mma_commit(bar(L::B_OF + g));
        waiting[g] = false;
        return true;
      };
      const auto step = [&](int n, int n0, int n1) -> bool {
        const int st = ns % R, before = (ns - 1) % R;
        const bool any = waiting[0] || waiting[1];
        if (!wait(L::B_KF + st, ns / R) || (any && !wait(L::B_VF + before, (ns - 1) / R))) return false;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int of_group = g ? n1 : n0;
          if (waiting[g] && !pv(g)) return false;
          if (n >= of_group) continue;
          first[g] = n == 0, last[g] = n + 1 == of_group;
          if (first[g]) {
            if (!wait(L::B_QF + g, n_q[g])) return false;
            tc_fence_after();
          }
          mma_kd<L::kSub, 16384, 16384>(tmem + L::T_S + 128 * g, dQ + g * kSlot, dK + st * kSlot, kIdS, 0u);
          mma_commit(bar(L::B_SF + 2 * g));
          if (last[g]) mma_commit(bar(L::B_QE + g)), ++n_q[g];
          ++n_s[g];
          waiting[g] = true;
        }
        mma_commit(bar(L::B_KE + st));
        if (any) mma_commit(bar(L::B_VE + before));
        ++ns;
        return true;
      };
      // a step that is neither the first two nor the last one of either group: the same, without the cases
      const auto inner = [&]() -> bool {
        const int st = ns % R, before = (ns - 1) % R;
        if (!wait(L::B_KF + st, ns / R) || !wait(L::B_VF + before, (ns - 1) / R)) return false;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const uint32_t t_o = tmem + L::T_O + g * D, t_s = tmem + L::T_S + 128 * g;
          if (!wait(L::B_PF + 2 * g, n_s[g] - 1)) return false;
          tc_fence_after();
          const uint64_t b = dV + before * kSlot;
          mma_ts_k64_mn(t_o, t_s, b, kIdO, 1u);
          mma_ts_k64_mn(t_o, t_s + 32, b + (8192 >> 4), kIdO, 1u);
          mma_kd<L::kSub, 16384, 16384>(t_s, dQ + g * kSlot, dK + st * kSlot, kIdS, 0u);
          mma_commit(bar(L::B_SF + 2 * g));
          ++n_s[g];
        }
        mma_commit(bar(L::B_KE + st));
        mma_commit(bar(L::B_VE + before));
        ++ns;
        return true;
      };
      const auto item_steps = [&](int n0, int n1) -> bool {
        const int total = max(n0, n1), both = min(n0, n1);
        for (int n = 0; n < total; ++n) {
          if (!step(n, n0, n1)) return false;
          if (n == 1)
            for (; n + 2 < both; ++n)
              if (!inner()) return false;
        }
        return true;
      };
      const auto finish = [&]() -> bool {
        if (!waiting[0] && !waiting[1]) return true;
        const int before = (ns - 1) % R;
        if (!wait(L::B_VF + before, (ns - 1) / R)) return false;
#pragma unroll
        for (int g = 0; g < 2; ++g)
          if (waiting[g] && !pv(g)) return false;
        mma_commit(bar(L::B_VE + before));
        return true;
      };
      run(item_steps, finish);
    } else {
      // S goes to the three buffers in turn; one is free again when the P V that read its P is issued, so that
      // S of a group's next step is issued before its P is there (8,192 tokens, 32 + 8 heads: 859 -> 728 us).
      // What is known of an open P V, 8 bits each, the oldest first
      constexpr uint32_t kGroup = 1, kFirst = 2, kLast = 4, kNewV = 8, kEndV = 16;
      uint32_t queue = 0, s_at = 0, p_at = 0;        // ... the buffers of the next S and of the oldest P
      int open = 0, n_k = 0, n_v = 0;                // steps whose S, whose P V are all issued
      int s0 = 0, s1 = 0, p0 = 0, p1 = 0, q0 = 0, q1 = 0;  // S, P V and items of the two groups
      const auto next = [](uint32_t i) { return i + 1 == L::kScores ? 0u : i + 1; };
      // P V of group g, its P the oldest; the step's V is in slot n_v % R
      const auto pv = [&](int g, bool first) -> bool {
        const int j = g ? p1++ : p0++;
        if (!wait(L::B_PF + L::barrier(g, j), L::phase(j))) return false;
        tc_fence_after();
        const uint64_t b = dV + ((uint32_t)n_v % R) * kSlot;
        const uint32_t o_at = tmem + L::T_O + g * D, p = tmem + L::T_S + 128 * p_at;
        mma_ts_k64_mn(o_at, p, b, kIdO, first ? 0u : 1u);
        mma_ts_k64_mn(o_at, p + 32, b + (8192 >> 4), kIdO, 1u);
        mma_commit(bar(L::B_PV + g));
        p_at = next(p_at);
        return true;
      };
      const auto wait_v = [&] { return wait(L::B_VF + n_v % R, n_v / R); };
      const auto end_v = [&] { mma_commit(bar(L::B_VE + n_v % R)), ++n_v; };
      // S of group g's next step, K in slot n_k % R
      const auto scores = [&](int g) {
        const int j = g ? s1++ : s0++;
        mma_kd<L::kSub, 16384, 16384>(tmem + L::T_S + 128 * s_at, dQ + g * kSlot, dK + ((uint32_t)n_k % R) * kSlot, kIdS, 0u);
        mma_commit(bar(L::B_SF + L::barrier(g, j)));
        s_at = next(s_at);
      };
      const auto end_k = [&] { mma_commit(bar(L::B_KE + n_k % R)), ++n_k; };
      // the oldest open P V
      const auto close = [&]() -> bool {
        const uint32_t info = queue & 255u;
        queue >>= 8, --open;
        if ((info & kNewV) && !wait_v()) return false;
        if (!pv((info & kGroup) != 0, (info & kFirst) != 0)) return false;
        if (info & kLast) mma_commit(bar(L::B_OF + (info & kGroup)));
        if (info & kEndV) end_v();
        return true;
      };
      // The next K is loaded behind the last V, and that one when the V of kRing steps before is free: more steps
      // than that may not be open when it is waited for (three, where one group alone takes every S).
      const auto within_ring = [&]() -> bool {
        while (n_k - n_v > R)
          if (!close()) return false;
        return true;
      };
      const auto item_steps = [&](int n0, int n1) -> bool {
        const int total = max(n0, n1), both = min(n0, n1);
        for (int n = 0; n < total; ++n) {
          if (!within_ring() || !wait(L::B_KF + n_k % R, n_k / R)) return false;
          tc_fence_after();
          if (n >= L::kScores && n + 1 < both) {
            // neither group's first or last step, nor are the open ones first steps: the same as below, and the
            // queue stays what it is
            if (!pv(1, false)) return false;
            end_v();
            scores(0);
            if (!wait_v() || !pv(0, false)) return false;
            scores(1);
            end_k();
            continue;
          }
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int mine = g ? n1 : n0, other = g ? n0 : n1;
            if (n >= mine) continue;
            const bool alone = n >= other;
            if (n == 0) {
              if (!wait(L::B_QF + g, g ? q1 : q0)) return false;
              tc_fence_after();
            }
            // a buffer, and no third step of one group: it has two barriers
            while (open == L::kScores || (g ? s1 - p1 : s0 - p0) == 2)
              if (!close()) return false;
            scores(g);
            const bool last = n + 1 == mine;
            if (last) mma_commit(bar(L::B_QE + g)), g ? ++q1 : ++q0;
            queue |= ((uint32_t)g | (n == 0 ? kFirst : 0) | (last ? kLast : 0) | (g == 0 || alone ? kNewV : 0) |
                      (g == 1 || alone ? kEndV : 0)) << (8 * open);
            ++open;
            if (g == 1 || alone) end_k();
          }
        }
        return within_ring();
      };
      const auto finish = [&]() -> bool {
        while (open > 0)
          if (!close()) return false;
        return true;
      };
      run(item_steps, finish);
    }
    // every product is done before TMEM is released
    if (lane == 0) {
      mma_commit(bar(L::B_DRAIN));
      wait_one(bar(L::B_DRAIN), 0, abort_flag, kErrFwdMma);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------ softmax warps
    const int g = warp >> 2;
    const int r = (warp & 3) * 32 + lane;  // row of the tile == TMEM lane
    const int t_of_row = over_group(r, group_inverse(hd.group)), head_of_row = r - t_of_row * hd.group;
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16), t_o = t_lane + L::T_O + g * D;
    const int heads = hd.keys * hd.group;
    int n_s = 0, n_o = 0;
    uint32_t before = 0;  // steps of both groups in the items before
    bool ok = true;
    while (ok && next_item(at, items, sm + L::ITEMS, ring, abort_flag, lane, kErrFwdSoftmax)) {
      if (at.kind != kTile) {
        if constexpr (kMode != kPart) {
          fill_rows(at.kind, at.tile, seqs.q, seqs, seqs.q_rows, 2 * n_tok, o, hd.keys, at.h, hd.group * D);
        } else {  // rows without a key in this part, or NaN
          fill_parts(at.kind, at.tile, seqs, 2 * n_tok, parts.ml + (int64_t)at.part * seqs.q_rows * heads, hd, at.h);
        }
        continue;
      }
      const FwdSteps w(at, n_tok, causal, grid.parts);
      const int n_steps = g ? w.n[1] : w.n[0], of_other = g ? w.n[0] : w.n[1], last = g ? w.last[1] : w.last[0];
      const int tok = w.tok0 + g * n_tok + t_of_row;
      const bool valid = r < rows && tok < at.nq;
      // keys that this row sees; rows without a token go along with the last one
      const int seen = causal ? min(max(min(tok, last) + w.shift + 1, 0), at.nk) : at.nk;
      using Sum = RowSum<kMode == kTrain>;
      float m = -INFINITY;
      Sum l = {1.0f, 1.0f};
      for (int n = 0; n < n_steps; ++n) {
        // keys of the two halves of the step that the row sees; all / none of them for every row of the warp
        const int lim0 = seen - (w.from + n) * kRows, lim1 = lim0 - 64;
        const bool all0 = __all_sync(0xffffffffu, lim0 >= 64), all1 = __all_sync(0xffffffffu, lim1 >= 64);
        const bool none0 = __all_sync(0xffffffffu, lim0 <= 0), none1 = __all_sync(0xffffffffu, lim1 <= 0);
        if (!wait_warp(bar(L::B_SF + L::barrier(g, n_s)), L::phase(n_s), abort_flag, kErrFwdSoftmax)) {
          ok = false;
          break;
        }
        ++n_s;
        tc_fence_after();
        // its S: the group's, or, of three, the steps of both groups take them in turn
        const uint32_t t_s =
            t_lane + L::T_S + 128 * (L::kScores == 2 ? (uint32_t)g : (before + n + min(n + g, of_other)) % 3);
        // before O is touched, the group's P V before is done: with two S, the step's own S was issued after it
        const auto o_settled = [&] {
          if (L::kScores > 2 && n > 0) ok = wait_warp(bar(L::B_PV + g), n_s & 1, abort_flag, kErrFwdSoftmax);
        };
        const auto scores = [&](int u, float(&s)[64]) {
          tmem_load<2>(t_s + u * 64, s);
          if (!(u ? all1 : all0)) mask_from(s, u ? lim1 : lim0);
        };
        Sum sum0 = {0.f, 0.f}, sum1 = {0.f, 0.f};
        // Exponentials against the running maximum in one pass over S; a row's first maximum is that of its
        // first half step.  A first half whose exponentials sum past kSum, and a row that has seen no key yet,
        // take two passes (maximum, then exponentials; S is intact).  If only the second half passes the limit,
        // P of the first half, l and O are scaled to the new maximum.  The two ways raise a maximum at different
        // scores, so only the sequence's own rows have a vote: what lies behind it in the tile must not choose the
        // rounding of its P.
        bool two_pass = false;
        uint32_t pk0[32];
        if (none0) {
          two_pass = __any_sync(0xffffffffu, valid && m == -INFINITY);
#pragma unroll
          for (int i = 0; i < 32; ++i) pk0[i] = 0u;
        } else {
          float s[64];
          scores(0, s);
          if (__any_sync(0xffffffffu, valid && m == -INFINITY)) {
            if (m == -INFINITY) m = tile_max(s) * qk_scale - H::kShift, l = {0.0f, 0.0f};
            if (m == -INFINITY) l = {1.0f, 1.0f};
            two_pass = __any_sync(0xffffffffu, valid && m == -INFINITY);
          }
          sum0 = exp_pairs<T, kMode == kTrain>(s, qk_scale, m, pk0);
          two_pass = two_pass || __any_sync(0xffffffffu, valid && !(sum0.exact <= H::kSum));
        }
        if (two_pass) {
          sum0 = {0.f, 0.f};
          float mx = -INFINITY;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (u ? none1 : none0) continue;
            float s[64];
            scores(u, s);
            mx = fmaxf(mx, tile_max(s));
          }
          mx = mx * qk_scale - H::kShift;
          const bool need = valid && mx > m + H::kLag;  // m = -inf: any key
          if (__any_sync(0xffffffffu, need)) {
            const float m_new = need ? mx : m;
            const float alpha = need ? ex2(m - m_new) : 1.0f;  // m = -inf -> 0
            const bool o_live = __any_sync(0xffffffffu, need && m != -INFINITY);
            l.scale(alpha);
            m = m_new;
            if (n > 0 && o_live) {
              o_settled();
              scale_tmem_rows<D / 32>(t_o, alpha);
            }
          }
          const float mb = (m == -INFINITY) ? 0.0f : m;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t pk[32];
            if (u ? none1 : none0) {
#pragma unroll
              for (int i = 0; i < 32; ++i) pk[i] = 0u;
            } else {
              float s[64];
              scores(u, s);
              const Sum t = exp_pairs<T, kMode == kTrain>(s, qk_scale, mb, pk);
              if (u) sum1 = t; else sum0 = t;
            }
            tmem_st32(t_s + u * 32, pk);  // over scores of the first half, which are read
          }
        } else {
          tmem_st32(t_s, pk0);
          uint32_t pk1[32];
          if (none1) {
#pragma unroll
            for (int i = 0; i < 32; ++i) pk1[i] = 0u;
          } else {
            float s[64];
            scores(1, s);
            sum1 = exp_pairs<T, kMode == kTrain>(s, qk_scale, m, pk1);
          }
          const bool need = valid && !(sum1.exact <= H::kSum);
          if (__any_sync(0xffffffffu, need)) {  // rare
            float s[64];
            scores(1, s);
            const float m_new = need ? fmaxf(m, tile_max(s) * qk_scale - H::kShift) : m;
            const float alpha = ex2(m - m_new);
            o_settled();
            if (n > 0) scale_tmem_rows<D / 32>(t_o, alpha);
            tmem_wait_st();
            uint32_t raw[32];
            float again = 0.f;
            tmem_ld32(t_s, raw);
            tmem_wait_ld_dep(raw);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float2 p = H::unpack(raw[i]);
              raw[i] = H::pack(p.x * alpha, p.y * alpha);
              if (kMode == kTrain) {  // rounded a second time
                p = H::unpack(raw[i]);
                again += p.x + p.y;
              }
            }
            tmem_st32(t_s, raw);
            l.scale(alpha);
            l.add({sum0.exact * alpha, again});
            sum0 = {0.f, 0.f};
            m = m_new;
            sum1 = exp_pairs<T, kMode == kTrain>(s, qk_scale, m, pk1);
          }
          tmem_st32(t_s + 32, pk1);
        }
        sum0.add(sum1), l.add(sum0);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::B_PF + L::barrier(g, n_s - 1)));
        if (!ok) break;
      }
      before += w.n[0] + w.n[1];
      if (!ok) break;
      // epilogue
      // No key here, which gives 0, is told by the mask: a row all of whose scores are -inf or NaN has no maximum
      // either, and its softmax is undefined.
      const bool empty = n_steps == 0 || seen <= w.from * kRows, undefined = !empty && m == -INFINITY;
      const float nan = __uint_as_float(0x7fc00000u);
      const int64_t out_row = (int64_t)(at.q0 + tok) * heads + at.h * hd.group + head_of_row;
      if constexpr (kMode == kTrain)
        lse[(((int64_t)at.h * hd.pairs + at.index) * 2 + g) * kRows + r] =
            !valid || empty ? INFINITY : undefined ? nan : m + __log2f(l.exact);
      if (kMode == kPart && valid)  // undefined: the sum is 1, or NaN with a NaN among the scores
        parts.ml[(int64_t)at.part * seqs.q_rows * heads + out_row] = make_float2(empty ? -INFINITY : m, empty ? 0.0f : l.of_products());
      if (n_steps > 0) {
        if (!wait_warp(bar(L::B_OF + g), n_o & 1, abort_flag, kErrFwdSoftmax)) {
          ok = false;
          break;
        }
        ++n_o;
        tc_fence_after();
        const float inv = undefined ? nan : (kMode == kTrain ? kAbove : 1.0f) / l.of_products();
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t raw[32];
          tmem_ld32(t_o + c * 32, raw);
          tmem_wait_ld_dep(raw);
          if constexpr (kMode == kPart) {
            float* dst = parts.o + ((int64_t)at.part * seqs.q_rows * heads + out_row) * D + c * 32;
            if (valid) {
#pragma unroll
              for (int i = 0; i < 4; ++i) store32(dst + 8 * i, raw + 8 * i);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) raw[i] = __float_as_uint(u2f(raw[i]) * inv);
            if (__any_sync(0xffffffffu, empty)) {
#pragma unroll
              for (int i = 0; i < 32; ++i) raw[i] = empty ? 0u : raw[i];
            }
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) pk[i] = H::pack(u2f(raw[2 * i]), u2f(raw[2 * i + 1]));
            if (valid) {
              T* dst = o + out_row * D + c * 32;
              store32(dst, pk), store32(dst + 16, pk + 8);
            }
            if constexpr (kMode == kTrain) {
              uint32_t left[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) left[i] = rest_bytes(raw[4 * i], raw[4 * i + 1], raw[4 * i + 2], raw[4 * i + 3]);
              if (valid) store32(rest + out_row * D + c * 32, left);
            }
          }
        }
        tc_fence_before();
      } else if (kMode != kPart && valid) {
        uint4* dst = reinterpret_cast<uint4*>(o + out_row * D);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) dst[i] = make_uint4(0, 0, 0, 0);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over a row's parts, in order; D / 4 threads a row.  Bound by
// memory.
constexpr int kJoinThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(Parts parts, int count, int64_t rows, T* __restrict__ o) {
  const int64_t i = (int64_t)blockIdx.x * kJoinThreads + threadIdx.x, row = i / (D / 4);
  const int col = (int)(i - row * (D / 4)) * 4;
  if (row >= rows) return;
  float top = -INFINITY;
#pragma unroll 4
  for (int p = 0; p < count; ++p) top = fmaxf(top, parts.ml[p * rows + row].x);
  float sum = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int p = 0; p < count; ++p) {
    const float2 x = parts.ml[p * rows + row];
    if (x.x == -INFINITY) {
      // no key (0; its sums were not written), scores of -inf only (1: undefined if the others have none either),
      // or NaN for a NaN among them and for wrong offsets
      if (!(x.y == 0.0f) && (top == -INFINITY || x.y != x.y)) sum = __uint_as_float(0x7fc00000u);
      continue;
    }
    const float f = ex2(x.x - top);
    const float4 v = *reinterpret_cast<const float4*>(parts.o + (p * rows + row) * D + col);
    sum = fmaf(x.y, f, sum);
    acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y), acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  *reinterpret_cast<uint2*>(o + row * D + col) =
      make_uint2(Half<T>::pack(acc.x * inv, acc.y * inv), Half<T>::pack(acc.z * inv, acc.w * inv));
}

// Pair `my` of the query tiles (of `per` tokens), for kernels whose CTAs each have one: found by all threads;
// scratch: one int a warp.  Not there: more pairs than that, or offsets that are not in order.
struct Place {
  int there, q0, nq, tile;
};
__device__ void find_place(const Sequences& s, int my, int per, Place* place, int* scratch) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  int base = 0;
  bool good = true;
  if (tid == 0) place->there = 0;
  for (int b0 = 0; b0 < s.count; b0 += blockDim.x) {
    const int b = b0 + tid;
    int q0 = 0, nq = 0;
    bool fine = true;
    if (b < s.count) {
      const int64_t qa = row_at(s.q, s.wide, b), qb = row_at(s.q, s.wide, b + 1);
      const int64_t ka = row_at(s.k, s.wide, b), kb = row_at(s.k, s.wide, b + 1);
      fine = 0 <= qa && qa <= qb && qb <= s.q_rows && 0 <= ka && ka <= kb && kb <= s.k_rows;
      if (fine) q0 = (int)qa, nq = (int)(qb - qa);
    }
    const int tiles = (nq + per - 1) / per;
    int x = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int xo = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += xo;
    }
    if (lane == 31) scratch[warp] = x;
    good = __syncthreads_and(fine) && good;
    int before = base + x - tiles;
    for (int w = 0; w < warps; ++w) {
      if (w < warp) before += scratch[w];
      base += scratch[w];
    }
    if (my >= before && my < before + tiles) *place = {1, q0, nq, my - before};
    __syncthreads();
  }
  if (tid == 0 && !good) place->there = 0;
  __syncthreads();
}

// ===================================================================== delta
// delta = dO . O of every row of every tile, 0 for rows without a token, in the forward's tile order: D / 8
// threads a row.  O with the 8 bits that the forward kept of what its rounding left: delta enters ds next to
// do . v, and o's rounding alone would be as large an error as that of ds.  Bound by memory: 75,600 tokens of 40
// heads of 128 take 291 us (6.6 TB/s).
constexpr int kDeltaThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kDeltaThreads)
    delta_kernel(const __grid_constant__ Sequences seqs, Heads hd, const T* __restrict__ o,
                 const int8_t* __restrict__ rest, const T* __restrict__ go, int64_t go_row, int64_t go_head,
                 float* __restrict__ delta) {
  __shared__ Place shared_place;
  __shared__ int scratch[kDeltaThreads / 32];
  const int pair = blockIdx.x / hd.keys, h = blockIdx.x % hd.keys;
  find_place(seqs, pair, 2 * hd.tokens, &shared_place, scratch);
  const Place at = shared_place;
  if (!at.there) return;
  constexpr int kLanes = D / 8, kStep = kDeltaThreads / kLanes;
  const int lane = threadIdx.x % kLanes;
  const uint32_t inverse = group_inverse(hd.group);
#pragma unroll 4
  for (int i = threadIdx.x / kLanes; i < 2 * kRows; i += kStep) {
    const int g = i / kRows, r = i % kRows, t = over_group(r, inverse);
    const int tok = (at.tile * 2 + g) * hd.tokens + t, head = h * hd.group + r - t * hd.group;
    float sum = 0.0f;
    if (t < hd.tokens && tok < at.nq) {
      const int64_t row = at.q0 + tok, place = (row * hd.keys * hd.group + head) * D + lane * 8;
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(o + place));
      const uint2 e = __ldg(reinterpret_cast<const uint2*>(rest + place));
      const uint4 b = __ldg(reinterpret_cast<const uint4*>(go + row * go_row + head * go_head + lane * 8));
      const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w}, left[2] = {e.x, e.y};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t high = (j & 1) ? x[j / 2] & 0xffff0000u : x[j / 2] << 16;
        const float2 q = Half<T>::unpack(y[j / 2]);
        sum = fmaf(with_rest(high, left[j / 4], j % 4), (j & 1) ? q.y : q.x, sum);
      }
    }
#pragma unroll
    for (int off = kLanes / 2; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) delta[((int64_t)h * hd.pairs + pair) * 2 * kRows + i] = sum;
  }
}

// ================================================================== dK and dV
// An item: 128 keys of one key head and a part of the tiles of 128 query rows that see them (all of them,
// unless there are few key tiles); a step is one such tile, so the sum over the heads that share the keys is
// the products' own (no atomics, a fixed order).  S^T = K Q^T, dP^T = V dO^T; P^T and dS^T are written over
// them in TMEM; dV += P^T dO, dK += dS^T Q.  Rows without a token have lse = +inf: p = 0.
//
// The softmax reads the 16x256b TMEM layout: a thread holds, in each 16-lane half, key lanes a and a + 8
// (a = lane / 4) at columns 8 j + 2 (lane % 4) + {0, 1}, so that it needs 16 of a half tile's 64 lse and
// delta values instead of all of them.
//
// 8,192 causal tokens of 32 + 8 heads: 945 us at 128 columns (8 D operations a score: 1,165 TFLOP/s, the tensor pipe
// 56 % busy), 720 at 64 (765 TFLOP/s, 36 %).  Bound by the chain S, P, dP, dS of a step through the softmax warps
// (two TMEM reads, two writes and a 2^x a score), which the four products of the step before cover only in part.
template <int D>
struct DkdvLayout {
  // 64 columns leave room in TMEM for a second S^T: that of step n + 1 is issued before P^T of step n is there
  static constexpr bool kEarly = D == 64;
  static constexpr int kScores = kEarly ? 2 : 1;
  static constexpr int kRing = kEarly ? 3 : 2;
  static constexpr int kSub = D / 64;
  static constexpr int kTileBytes = kSub * 16384;
  static constexpr int K = 0;
  static constexpr int V = K + kTileBytes;
  static constexpr int Q = V + kTileBytes;
  static constexpr int DO = Q + kRing * kTileBytes;
  static constexpr int M = DO + kRing * kTileBytes;  // lse
  static constexpr int DL = M + kRing * 512;         // delta
  static constexpr int TOKENS = DL + kRing * 512;    // of a tile's rows
  static constexpr int ITEMS = TOKENS + kRows * 4;
  static constexpr int BAR = ITEMS + (ItemRing::kBytes + 15) / 16 * 16;
  static constexpr int B_KV = 0, B_KVE = 1,   // an item's keys; its last S^T and dP^T done
                       B_QF = 2, B_QE = B_QF + kRing,
                       B_SF = B_QE + kRing,   // [buffer]
                       B_DPF = B_SF + kScores,
                       B_PF = B_DPF + 1,      // [buffer]: a warp may be at P^T of the next S^T before all are at this one
                       B_DSF = B_PF + kScores, B_FIN = B_DSF + 1, B_DRAIN = B_FIN + 1, NBAR = B_DRAIN + 1;
  static constexpr int TMEM_SLOT = BAR + NBAR * 8;
  static constexpr int ABORT = TMEM_SLOT + 4;
  static constexpr int SCRATCH = ABORT + 4;
  static constexpr size_t kNeed = 1024 + SCRATCH + 2 * 4 * (kThreads / 32);
  static constexpr size_t kBytes = kNeed > kMinSmem ? kNeed : kMinSmem;
  static constexpr int T_DK = 0, T_DV = D, T_S = 2 * D, T_DP = T_S + 128 * kScores;
  static_assert(T_DP + 128 <= 512, "TMEM budget");
};

// The steps of an item: its first key, and the first of its query tiles and their number.
struct DkdvSteps {
  int key0, shift, first, steps;
  bool tail;  // the last one ends with another sequence's rows
  __device__ __forceinline__ DkdvSteps(const Item& at, int n_tok, int causal, int parts) {
    key0 = at.tile * kRows, shift = at.nk - at.nq;
    const int tiles = (at.nq + n_tok - 1) / n_tok;
    // causal: from the tile that sees the first key
    const int from = causal ? min(max(key0 - shift, 0) / n_tok, tiles) : 0, all = tiles - from;
    first = from + (int)((int64_t)all * at.part / parts);
    const int end = from + (int)((int64_t)all * (at.part + 1) / parts);
    steps = end - first;
    tail = end == tiles && tiles * n_tok > at.nq;
  }
};

// p = exp2(s scale - lse) of 64 columns for this warp's lanes, written as pairs over the first 32 columns.
// kMasked: key lane `key` + 16 hl + 8 kk is 0 in columns whose `beyond` is not above it.
template <typename T, bool kMasked>
__device__ __forceinline__ void dkdv_p(uint32_t t_tile, const float* __restrict__ lse, float qk_scale, int lane,
                                       const int* __restrict__ beyond, int key, float (&p)[64]) {
  const int c2 = 2 * (lane & 3);
  const float2 sc = make_float2(qk_scale, qk_scale);
#pragma unroll
  for (int hl = 0; hl < 2; ++hl) {
    uint32_t raw[32], pk[16];
    tmem_ld_16x256b_x8(t_tile + ((uint32_t)(16 * hl) << 16), raw);
    tmem_wait_ld_dep(raw);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 ls = *reinterpret_cast<const float2*>(lse + 8 * j + c2), nl = make_float2(-ls.x, -ls.y);
      int2 seen = make_int2(0, 0);
      if constexpr (kMasked) seen = *reinterpret_cast<const int2*>(beyond + 8 * j + c2);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const float2 x = __ffma2_rn(make_float2(u2f(raw[4 * j + 2 * kk]), u2f(raw[4 * j + 2 * kk + 1])), sc, nl);
        float e0 = ex2(x.x), e1 = ex2(x.y);
        if constexpr (kMasked) {
          const int row = key + 16 * hl + 8 * kk;
          e0 = row < seen.x ? e0 : 0.0f;
          e1 = row < seen.y ? e1 : 0.0f;
        }
        p[32 * hl + 4 * j + 2 * kk] = e0;
        p[32 * hl + 4 * j + 2 * kk + 1] = e1;
        pk[2 * j + kk] = Half<T>::pack(e0, e1);
      }
    }
    tmem_st_16x128b_x8(t_tile + ((uint32_t)(16 * hl) << 16), pk);
  }
}

// ds = p (dp - delta) as pairs over the first 32 columns of dP^T; 0 where p is 0 by the mask.
template <typename T, bool kMasked>
__device__ __forceinline__ void dkdv_ds(uint32_t t_tile, const float* __restrict__ delta, int lane,
                                        const float (&p)[64]) {
  const int c2 = 2 * (lane & 3);
  const float2 neg1 = make_float2(-1.0f, -1.0f);
#pragma unroll
  for (int hl = 0; hl < 2; ++hl) {
    uint32_t raw[32], pk[16];
    tmem_ld_16x256b_x8(t_tile + ((uint32_t)(16 * hl) << 16), raw);
    tmem_wait_ld_dep(raw);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 d2 = *reinterpret_cast<const float2*>(delta + 8 * j + c2);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int i = 32 * hl + 4 * j + 2 * kk;
        float2 ds = __fmul2_rn(make_float2(p[i], p[i + 1]),
                               __ffma2_rn(d2, neg1, make_float2(u2f(raw[4 * j + 2 * kk]), u2f(raw[4 * j + 2 * kk + 1]))));
        if constexpr (kMasked) ds = make_float2(p[i] == 0.0f ? 0.0f : ds.x, p[i + 1] == 0.0f ? 0.0f : ds.y);
        pk[2 * j + kk] = Half<T>::pack(ds.x, ds.y);
      }
    }
    tmem_st_16x128b_x8(t_tile + ((uint32_t)(16 * hl) << 16), pk);
  }
}

// kParts: sums of a part, fp32, to sums[part][0: dK, 1: dV][row][key head][D]; else dk and dv.
template <typename T, int D, bool kParts>
__global__ void __launch_bounds__(kThreads, 1)
    dkdv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                const __grid_constant__ Sequences seqs, const __grid_constant__ Heads hd,
                const __grid_constant__ Grid grid, int causal, float qk_scale, float scale,
                const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ dk,
                T* __restrict__ dv, float* __restrict__ sums) {
  using L = DkdvLayout<D>;
  constexpr int R = L::kRing;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = align1024(smem_raw);
  const uint32_t sb = smem_u32(sm);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_tok = hd.tokens, rows = n_tok * hd.group;
  auto bar = [&](int i) { return sb + L::BAR + 8 * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::ABORT);
  const uint32_t ring = sb + L::ITEMS;
  int* tokens = reinterpret_cast<int*>(sm + L::TOKENS);

  if (threadIdx.x == 0) {
    ItemRing::init(ring);
    mbar_init(bar(L::B_KV), 1);
    mbar_init(bar(L::B_KVE), 1);
    for (int i = 0; i < R; ++i) {
      mbar_init(bar(L::B_QF + i), 1);
      mbar_init(bar(L::B_QE + i), 1);
    }
    for (int i = 0; i < L::kScores; ++i) {
      mbar_init(bar(L::B_SF + i), 1);
      mbar_init(bar(L::B_PF + i), 8);
    }
    mbar_init(bar(L::B_DPF), 1);
    mbar_init(bar(L::B_DSF), 8);
    mbar_init(bar(L::B_FIN), 1);
    mbar_init(bar(L::B_DRAIN), 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x < kRows) tokens[threadIdx.x] = over_group(threadIdx.x, group_inverse(hd.group));
  if (rows < kRows) {  // rows that no load fills
    for (int i = 0; i < R; ++i) {
      zero_rows<L::kSub>(sm + L::Q + i * L::kTileBytes, rows, threadIdx.x, kThreads);
      zero_rows<L::kSub>(sm + L::DO + i * L::kTileBytes, rows, threadIdx.x, kThreads);
    }
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(sb + L::TMEM_SLOT, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  const Survey all = survey<true>(seqs, 2 * n_tok, reinterpret_cast<int*>(sm + L::SCRATCH));
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + L::TMEM_SLOT);

  Item at;
  int items = 0;
  if (warp == kProducerWarp) {
    // ------------------------------------------------------------ producer
    int ns = 0, n_kv = 0;
    bool ok = true;
    ItemSource<true> source = {seqs, hd, grid, all, sm + L::ITEMS, ring, abort_flag, lane, kErrDkdvProducer};
    while (ok && source.next(at)) {
      if (at.kind != kTile) continue;
      const DkdvSteps w(at, n_tok, causal, grid.parts);
      if (w.steps == 0) continue;
      if (lane == 0) {
        ok = n_kv == 0 || wait_one(bar(L::B_KVE), (n_kv - 1) & 1, abort_flag, kErrDkdvProducer);
        if (ok) {
          mbar_expect_tx(bar(L::B_KV), 2 * L::kTileBytes);
#pragma unroll
          for (int s = 0; s < L::kSub; ++s) {
            tma_load_3d(sb + L::K + s * 16384, &tm_k, s * 64, at.h, at.k0 + w.key0, bar(L::B_KV));
            tma_load_3d(sb + L::V + s * 16384, &tm_v, s * 64, at.h, at.k0 + w.key0, bar(L::B_KV));
          }
          ++n_kv;
        }
        const int64_t stat0 = (((int64_t)at.h * hd.pairs + at.pairs) * 2 + w.first) * kRows;
        for (int n = 0; ok && n < w.steps; ++n) {
          const int st = ns % R, tok = at.q0 + (w.first + n) * n_tok;
          ok = ns < R || wait_one(bar(L::B_QE + st), ((ns / R) - 1) & 1, abort_flag, kErrDkdvProducer);
          if (!ok) break;
          mbar_expect_tx(bar(L::B_QF + st), 2 * rows * D * 2 + 2 * 512);
#pragma unroll
          for (int s = 0; s < L::kSub; ++s) {
            tma_load_3d(sb + L::Q + st * L::kTileBytes + s * 16384, &tm_q, s * 64, at.h * hd.group, tok, bar(L::B_QF + st));
            tma_load_3d(sb + L::DO + st * L::kTileBytes + s * 16384, &tm_do, s * 64, at.h * hd.group, tok, bar(L::B_QF + st));
          }
          bulk_load(sb + L::M + st * 512, lse + stat0 + (int64_t)n * kRows, 512, bar(L::B_QF + st));
          bulk_load(sb + L::DL + st * 512, delta + stat0 + (int64_t)n * kRows, 512, bar(L::B_QF + st));
          ++ns;
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
    }
    if (lane == 0) {  // every load has landed before the CTA may leave
      for (int m = max(ns - R, 0); m < ns; ++m) wait_one(bar(L::B_QF + m % R), (m / R) & 1, abort_flag, kErrDkdvProducer);
      if (n_kv > 0) wait_one(bar(L::B_KV), (n_kv - 1) & 1, abort_flag, kErrDkdvProducer);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------- MMA issuer
    // Steps of all items in one stream: S^T(n) | dK(n-1) | dP^T(n) | dV(n), or, with two S^T, within an item
    // dK(n-1) | S^T(n+1) | dP^T(n) | dV(n).  The softmax computes P^T(n) while dK(n-1) and dP^T(n) run, dS^T(n)
    // while dV(n) and S^T(n+1) do.  S^T(n) overwrites P^T(n-1), read by
    // dV(n-1), dP^T(n) overwrites dS^T(n-1), read by dK(n-1): issued earlier, and one thread's products run in
    // issue order.  An item's first dV and dK overwrite sums that the epilogue of the item before has read: the
    // P^T and dS^T that they wait for are written after it.
    constexpr uint32_t kIdS = idesc<T>(kRows, false), kIdG = idesc<T>(D, true);
    const uint64_t dK = desc_k_sw128(sb + L::K), dV = desc_k_sw128(sb + L::V), dQk = desc_k_sw128(sb + L::Q),
                   dDOk = desc_k_sw128(sb + L::DO), dQmn = desc_mn_sw128(sb + L::Q, 16384),
                   dDOmn = desc_mn_sw128(sb + L::DO, 16384);
    constexpr uint32_t kSlot = L::kTileBytes >> 4;
    int ns = 0, n_kv = 0;
    bool waiting = false, first = false, last = false;  // dK of the last step still to come
    const auto wait = [&](int i, int parity) { return wait_one(bar(i), parity & 1, abort_flag, kErrDkdvMma); };
    const auto dk_step = [&]() -> bool {
      const uint32_t st = (uint32_t)(ns - 1) % R;
      if (!wait(L::B_DSF, ns - 1)) return false;
      tc_fence_after();
      mma_ts_k64_mn(tmem + L::T_DK, tmem + L::T_DP, dQmn + st * kSlot, kIdG, first ? 0u : 1u);
      mma_ts_k64_mn(tmem + L::T_DK, tmem + L::T_DP + 64, dQmn + st * kSlot + 512, kIdG, 1u);
      mma_commit(bar(L::B_QE + st));
      if (last) mma_commit(bar(L::B_FIN));
      waiting = false;
      return true;
    };
    const auto scores = [&](int j) -> bool {  // S^T of step j
      const uint32_t st = (uint32_t)j % R, buffer = (uint32_t)j % L::kScores;
      if (!wait(L::B_QF + st, j / R)) return false;
      tc_fence_after();
      mma_kd<L::kSub, 16384, 16384>(tmem + L::T_S + 128 * buffer, dK, dQk + st * kSlot, kIdS, 0u);
      mma_commit(bar(L::B_SF + buffer));
      return true;
    };
    // step n of `steps`; early: S^T of it is issued; next: S^T of the one behind it may be
    const auto step = [&](int n, int steps, bool early, bool next) -> bool {
      const uint32_t st = (uint32_t)ns % R;
      if (n == 0) {  // keys that are not there yet are not waited for with a product to issue
        if (waiting && !mbar_try(bar(L::B_KV), n_kv & 1) && !dk_step()) return false;
        if (!wait(L::B_KV, n_kv)) return false;
      }
      if (!early && !scores(ns)) return false;
      if (waiting && !dk_step()) return false;
      if (next && !scores(ns + 1)) return false;
      mma_kd<L::kSub, 16384, 16384>(tmem + L::T_DP, dV, dDOk + st * kSlot, kIdS, 0u);
      mma_commit(bar(L::B_DPF));
      first = n == 0, last = n + 1 == steps;
      if (last) mma_commit(bar(L::B_KVE)), ++n_kv;
      const uint32_t buffer = (uint32_t)ns % L::kScores, p = tmem + L::T_S + 128 * buffer;
      if (!wait(L::B_PF + buffer, ns / L::kScores)) return false;
      tc_fence_after();
      mma_ts_k64_mn(tmem + L::T_DV, p, dDOmn + st * kSlot, kIdG, first ? 0u : 1u);
      mma_ts_k64_mn(tmem + L::T_DV, p + 64, dDOmn + st * kSlot + 512, kIdG, 1u);
      ++ns;
      waiting = true;
      return true;
    };
    bool ok = true, any = false;
    while (ok) {
      // an item that is not there yet is not waited for with products to issue
      if (any && !__any_sync(0xffffffffu, item_ready(items, ring))) {
        if (lane == 0 && waiting) ok = dk_step();
        ok = __all_sync(0xffffffffu, ok), any = false;
      }
      if (!ok || !next_item(at, items, sm + L::ITEMS, ring, abort_flag, lane, kErrDkdvMma)) break;
      if (at.kind != kTile) continue;
      const DkdvSteps w(at, n_tok, causal, grid.parts);
      if (w.steps == 0) continue;
      any = true;
      const int plain = w.tail ? w.steps - 1 : w.steps;
      if (lane == 0)
        for (int n = 0; ok && n < plain; ++n)
          ok = step(n, w.steps, L::kEarly && n > 0, L::kEarly && n + 1 < plain);
      ok = __all_sync(0xffffffffu, ok);
      if (lane != 0) ns += plain;
      if (w.tail && ok) {  // the next sequence's rows, which dK and dV sum over
        const int st = ns % R;
        ok = wait_warp(bar(L::B_QF + st), (ns / R) & 1, abort_flag, kErrDkdvMma);
        const int valid = (at.nq - (w.first + plain) * n_tok) * hd.group;
        if (ok) {
          zero_rows<L::kSub>(sm + L::Q + st * L::kTileBytes, valid, lane, 32);
          zero_rows<L::kSub>(sm + L::DO + st * L::kTileBytes, valid, lane, 32);
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0 && ok) ok = step(plain, w.steps, false, false);
        ok = __all_sync(0xffffffffu, ok);
        if (lane != 0) ++ns;
      }
    }
    if (lane == 0) {
      if (ok && waiting) dk_step();
      mma_commit(bar(L::B_DRAIN));
      wait_one(bar(L::B_DRAIN), 0, abort_flag, kErrDkdvMma);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------ softmax warps
    // warpgroup w: columns [64 w, 64 w + 64) of each tile
    const int wg = warp >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;  // key row of the epilogue == TMEM lane
    const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16);
    const int key = quarter * 32 + (lane >> 2), tcol = wg * 64;  // this thread's first key lane
    const float* sM = reinterpret_cast<const float*>(sm + L::M) + tcol;
    const float* sDl = reinterpret_cast<const float*>(sm + L::DL) + tcol;
    const int64_t part_rows = (int64_t)seqs.k_rows * hd.keys;
    int ns = 0, n_fin = 0;
    bool ok = true;
    while (ok && next_item(at, items, sm + L::ITEMS, ring, abort_flag, lane, kErrDkdvSoftmax)) {
      float* part = kParts ? sums + (int64_t)at.part * 2 * part_rows * D : nullptr;
      if (at.kind != kTile) {
        if constexpr (kParts) {  // fp32 zeros or NaN, as pairs of 16-bit ones
          fill_rows(at.kind, at.tile, seqs.k, seqs, seqs.k_rows, kRows, reinterpret_cast<T*>(part), hd.keys, at.h, 2 * D);
          fill_rows(at.kind, at.tile, seqs.k, seqs, seqs.k_rows, kRows, reinterpret_cast<T*>(part + part_rows * D), hd.keys, at.h, 2 * D);
        } else {
          fill_rows(at.kind, at.tile, seqs.k, seqs, seqs.k_rows, kRows, dk, hd.keys, at.h, D);
          fill_rows(at.kind, at.tile, seqs.k, seqs, seqs.k_rows, kRows, dv, hd.keys, at.h, D);
        }
        continue;
      }
      const DkdvSteps w(at, n_tok, causal, grid.parts);
      for (int n = 0; n < w.steps; ++n) {
        const int st = ns % R;
        // the keys that the tile's first row sees, from the item's first one on: all of them, or masked
        const int seen = (w.first + n) * n_tok + w.shift + 1 - w.key0;
        const bool masked = causal && seen < kRows;
        if (!wait_warp(bar(L::B_QF + st), (ns / R) & 1, abort_flag, kErrDkdvSoftmax) ||
            !wait_warp(bar(L::B_SF + ns % L::kScores), (ns / L::kScores) & 1, abort_flag, kErrDkdvSoftmax)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float p[64];
        const uint32_t t_scores = t_lane + L::T_S + 128 * (ns % L::kScores) + tcol;
        // key < seen + tokens[column]
        if (masked) dkdv_p<T, true>(t_scores, sM + st * 128, qk_scale, lane, tokens + tcol, key - seen, p);
        else dkdv_p<T, false>(t_scores, sM + st * 128, qk_scale, lane, nullptr, 0, p);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::B_PF + ns % L::kScores));
        if (!wait_warp(bar(L::B_DPF), ns & 1, abort_flag, kErrDkdvSoftmax)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (masked) dkdv_ds<T, true>(t_lane + L::T_DP + tcol, sDl + st * 128, lane, p);
        else dkdv_ds<T, false>(t_lane + L::T_DP + tcol, sDl + st * 128, lane, p);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::B_DSF));
        ++ns;
      }
      if (!ok) break;
      // epilogue: warpgroup 0 writes dK, 1 dV
      const bool valid = w.key0 + r < at.nk;
      const int64_t row = (int64_t)(at.k0 + w.key0 + r) * hd.keys + at.h;
      T* out = (wg == 0 ? dk : dv) + row * D;
      float* sum = kParts ? part + (wg * part_rows + row) * D : nullptr;
      const float by = wg == 0 ? scale : 1.0f;
      if (w.steps > 0 && !wait_warp(bar(L::B_FIN), n_fin & 1, abort_flag, kErrDkdvSoftmax)) {
        ok = false;
        break;
      }
      if (w.steps > 0) ++n_fin;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t raw[32];
        if (w.steps > 0) {
          tmem_ld32(t_lane + (wg == 0 ? L::T_DK : L::T_DV) + c * 32, raw);
          tmem_wait_ld_dep(raw);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) raw[i] = 0u;
        }
        if (!valid) continue;
        if constexpr (kParts) {
#pragma unroll
          for (int i = 0; i < 4; ++i) store32(sum + c * 32 + 8 * i, raw + 8 * i);
        } else {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[i] = Half<T>::pack(u2f(raw[2 * i]) * by, u2f(raw[2 * i + 1]) * by);
          store32(out + c * 32, pk), store32(out + c * 32 + 16, pk + 8);
        }
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dK and dV from the sums of their parts, in order.  Bound by memory: 42 us for 12 parts of 512 keys of 40 heads of
// 128 (252 MB, L2 holding some of it).
template <typename T>
__global__ void __launch_bounds__(kJoinThreads)
    add_parts_kernel(const float* __restrict__ sums, int parts, int64_t count, float scale, T* __restrict__ dk,
                     T* __restrict__ dv) {
  const int64_t i = ((int64_t)blockIdx.x * kJoinThreads + threadIdx.x) * 4;
  const int which = blockIdx.y;  // 0: dK, 1: dV
  if (i >= count) return;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    const float4 v = *reinterpret_cast<const float4*>(sums + (2 * p + which) * count + i);
    acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
  }
  const float by = which == 0 ? scale : 1.0f;
  *reinterpret_cast<uint2*>((which == 0 ? dk : dv) + i) =
      make_uint2(Half<T>::pack(acc.x * by, acc.y * by), Half<T>::pack(acc.z * by, acc.w * by));
}

// ======================================================================= dQ
// An item: one tile of 128 query rows; a step is 128 keys: S = Q K^T and dP = dO V^T in TMEM, the softmax
// warpgroups (64 keys each) write dS = P (dP - delta) into columns of its own, dQ += dS K reads them from
// there.  S and dP of step n + 1 are issued as soon as those of step n are read.
//
// 8,192 causal tokens of 32 + 8 heads: 690 to 700 us at 128 columns (6 D operations a score: 1,190 TFLOP/s, the tensor
// pipe 55 % busy), 585 at 64 (705 TFLOP/s, 32 %).  Bound as dK and dV are.
template <int D>
struct DqLayout {
  static constexpr int kRingK = 3, kRingV = 2;  // K serves two products
  static constexpr int kSub = D / 64;
  static constexpr int kTileBytes = kSub * 16384;
  static constexpr int Q = 0;
  static constexpr int DO = Q + kTileBytes;
  static constexpr int K = DO + kTileBytes;
  static constexpr int V = K + kRingK * kTileBytes;
  static constexpr int ITEMS = V + kRingV * kTileBytes;
  static constexpr int BAR = ITEMS + (ItemRing::kBytes + 15) / 16 * 16;
  static constexpr int B_QD = 0, B_QE = 1,   // an item's rows; its last S and dP done
                       B_KF = 2, B_KE = B_KF + kRingK, B_VF = B_KE + kRingK, B_VE = B_VF + kRingV,
                       B_SF = B_VE + kRingV, B_DPF = B_SF + 1, B_DPE = B_DPF + 1, B_DSF = B_DPE + 1,
                       B_DSE = B_DSF + 1, B_FIN = B_DSE + 1, B_DRAIN = B_FIN + 1, NBAR = B_DRAIN + 1;
  static constexpr int TMEM_SLOT = BAR + NBAR * 8;
  static constexpr int ABORT = TMEM_SLOT + 4;
  static constexpr int SCRATCH = ABORT + 4;
  static constexpr size_t kNeed = 1024 + SCRATCH + 2 * 4 * (kThreads / 32);
  static constexpr size_t kBytes = kNeed > kMinSmem ? kNeed : kMinSmem;
  // dQ (D columns), S and dP (128 fp32 columns each), dS (64 columns of pairs)
  static constexpr int T_DQ = 0, T_S = 128, T_DP = 256, T_DS = 384;
};

// The steps of an item (its part: which tile of the pair).
struct DqSteps {
  int tok0, shift, last, steps;
  bool tail;  // the last one ends with another sequence's keys
  __device__ __forceinline__ DqSteps(const Item& at, int n_tok, int causal) {
    tok0 = (at.tile * 2 + at.part) * n_tok, shift = at.nk - at.nq;
    last = min(tok0 + n_tok, at.nq) - 1;
    const int keys = tok0 >= at.nq ? 0 : causal ? min(max(last + shift + 1, 0), at.nk) : at.nk;
    steps = (keys + kRows - 1) / kRows;
    tail = steps * kRows > at.nk;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
              const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
              const __grid_constant__ Sequences seqs, const __grid_constant__ Heads hd,
              const __grid_constant__ Grid grid, int causal, float qk_scale, float scale,
              const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ dq) {
  using L = DqLayout<D>;
  constexpr int RK = L::kRingK, RV = L::kRingV;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = align1024(smem_raw);
  const uint32_t sb = smem_u32(sm);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_tok = hd.tokens, rows = n_tok * hd.group;
  auto bar = [&](int i) { return sb + L::BAR + 8 * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::ABORT);
  const uint32_t ring = sb + L::ITEMS;

  if (threadIdx.x == 0) {
    ItemRing::init(ring);
    mbar_init(bar(L::B_QD), 1);
    mbar_init(bar(L::B_QE), 1);
    for (int i = 0; i < RK; ++i) {
      mbar_init(bar(L::B_KF + i), 1);
      mbar_init(bar(L::B_KE + i), 1);
    }
    for (int i = 0; i < RV; ++i) {
      mbar_init(bar(L::B_VF + i), 1);
      mbar_init(bar(L::B_VE + i), 1);
    }
    mbar_init(bar(L::B_SF), 1);
    mbar_init(bar(L::B_DPF), 1);
    mbar_init(bar(L::B_DPE), 8);
    mbar_init(bar(L::B_DSF), 8);
    mbar_init(bar(L::B_DSE), 1);
    mbar_init(bar(L::B_FIN), 1);
    mbar_init(bar(L::B_DRAIN), 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (rows < kRows) {  // rows that no load fills
    zero_rows<L::kSub>(sm + L::Q, rows, threadIdx.x, kThreads);
    zero_rows<L::kSub>(sm + L::DO, rows, threadIdx.x, kThreads);
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(sb + L::TMEM_SLOT, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  const Survey all = survey<false>(seqs, 2 * n_tok, reinterpret_cast<int*>(sm + L::SCRATCH));
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + L::TMEM_SLOT);

  Item at;
  int items = 0;
  if (warp == kProducerWarp) {
    // ------------------------------------------------------------ producer
    int nk = 0, nv = 0, n_q = 0;
    bool ok = true;
    ItemSource<false> source = {seqs, hd, grid, all, sm + L::ITEMS, ring, abort_flag, lane, kErrDqProducer};
    while (ok && source.next(at)) {
      if (at.kind != kTile) continue;
      const DqSteps w(at, n_tok, causal);
      if (w.steps == 0) continue;
      if (lane == 0) {
        ok = n_q == 0 || wait_one(bar(L::B_QE), (n_q - 1) & 1, abort_flag, kErrDqProducer);
        if (ok) {
          mbar_expect_tx(bar(L::B_QD), 2 * rows * D * 2);
#pragma unroll
          for (int s = 0; s < L::kSub; ++s) {
            tma_load_3d(sb + L::Q + s * 16384, &tm_q, s * 64, at.h * hd.group, at.q0 + w.tok0, bar(L::B_QD));
            tma_load_3d(sb + L::DO + s * 16384, &tm_do, s * 64, at.h * hd.group, at.q0 + w.tok0, bar(L::B_QD));
          }
          ++n_q;
        }
        for (int n = 0; ok && n < w.steps; ++n) {
          const int sk = nk % RK, sv = nv % RV, key = at.k0 + n * kRows;
          ok = nk < RK || wait_one(bar(L::B_KE + sk), ((nk / RK) - 1) & 1, abort_flag, kErrDqProducer);
          if (!ok) break;
          mbar_expect_tx(bar(L::B_KF + sk), L::kTileBytes);
#pragma unroll
          for (int s = 0; s < L::kSub; ++s)
            tma_load_3d(sb + L::K + sk * L::kTileBytes + s * 16384, &tm_k, s * 64, at.h, key, bar(L::B_KF + sk));
          ++nk;
          ok = nv < RV || wait_one(bar(L::B_VE + sv), ((nv / RV) - 1) & 1, abort_flag, kErrDqProducer);
          if (!ok) break;
          mbar_expect_tx(bar(L::B_VF + sv), L::kTileBytes);
#pragma unroll
          for (int s = 0; s < L::kSub; ++s)
            tma_load_3d(sb + L::V + sv * L::kTileBytes + s * 16384, &tm_v, s * 64, at.h, key, bar(L::B_VF + sv));
          ++nv;
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
    }
    if (lane == 0) {  // every load has landed before the CTA may leave
      for (int m = max(nk - RK, 0); m < nk; ++m) wait_one(bar(L::B_KF + m % RK), (m / RK) & 1, abort_flag, kErrDqProducer);
      for (int m = max(nv - RV, 0); m < nv; ++m) wait_one(bar(L::B_VF + m % RV), (m / RV) & 1, abort_flag, kErrDqProducer);
      if (n_q > 0) wait_one(bar(L::B_QD), (n_q - 1) & 1, abort_flag, kErrDqProducer);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------- MMA issuer
    // Steps of all items in one stream: S(0) dP(0) | S(1) dP(1) dQ(0) | S(2) dP(2) dQ(1) | ...  An item's first
    // dQ overwrites one that the epilogue of the item before has read: the dS that it waits for is written
    // after it.
    constexpr uint32_t kIdS = idesc<T>(kRows, false), kIdG = idesc<T>(D, true);
    const uint64_t dQ = desc_k_sw128(sb + L::Q), dDO = desc_k_sw128(sb + L::DO), dKk = desc_k_sw128(sb + L::K),
                   dVk = desc_k_sw128(sb + L::V), dKmn = desc_mn_sw128(sb + L::K, 16384);
    constexpr uint32_t kSlot = L::kTileBytes >> 4;
    int ns = 0, n_q = 0;
    bool waiting = false, first = false, last = false;  // dQ of the last step still to come
    const auto wait = [&](int i, int parity) { return wait_one(bar(i), parity & 1, abort_flag, kErrDqMma); };
    const auto dq_step = [&](int j, bool begins, bool ends) -> bool {
      if (!wait(L::B_DSF, j)) return false;
      tc_fence_after();
      const uint64_t b = dKmn + (j % RK) * kSlot;
      mma_ts_k64_mn(tmem + L::T_DQ, tmem + L::T_DS, b, kIdG, begins ? 0u : 1u);
      mma_ts_k64_mn(tmem + L::T_DQ, tmem + L::T_DS + 32, b + (8192 >> 4), kIdG, 1u);
      mma_commit(bar(L::B_DSE));
      mma_commit(bar(L::B_KE + j % RK));
      if (ends) mma_commit(bar(L::B_FIN));
      return true;
    };
    const auto step = [&](int n, int steps) -> bool {
      const int sk = ns % RK, sv = ns % RV;
      if (n == 0) {  // rows that are not there yet are not waited for with a product to issue
        if (waiting && !mbar_try(bar(L::B_QD), n_q & 1)) {
          if (!dq_step(ns - 1, first, last)) return false;
          waiting = false;
        }
        if (!wait(L::B_QD, n_q)) return false;
      }
      if (!wait(L::B_KF + sk, ns / RK) || (ns > 0 && !wait(L::B_DPE, ns - 1))) return false;
      tc_fence_after();
      mma_kd<L::kSub, 16384, 16384>(tmem + L::T_S, dQ, dKk + sk * kSlot, kIdS, 0u);
      mma_commit(bar(L::B_SF));
      if (!wait(L::B_VF + sv, ns / RV)) return false;
      tc_fence_after();
      mma_kd<L::kSub, 16384, 16384>(tmem + L::T_DP, dDO, dVk + sv * kSlot, kIdS, 0u);
      mma_commit(bar(L::B_DPF));
      mma_commit(bar(L::B_VE + sv));
      const bool ends = n + 1 == steps;
      if (ends) mma_commit(bar(L::B_QE)), ++n_q;
      if (waiting && !dq_step(ns - 1, first, last)) return false;
      ++ns;
      waiting = true, first = n == 0, last = ends;
      return true;
    };
    bool ok = true, any = false;
    while (ok) {
      // an item that is not there yet is not waited for with products to issue
      if (any && !__any_sync(0xffffffffu, item_ready(items, ring))) {
        if (lane == 0 && waiting) ok = dq_step(ns - 1, first, last), waiting = false;
        ok = __all_sync(0xffffffffu, ok), any = false;
      }
      if (!ok || !next_item(at, items, sm + L::ITEMS, ring, abort_flag, lane, kErrDqMma)) break;
      if (at.kind != kTile) continue;
      const DqSteps w(at, n_tok, causal);
      if (w.steps == 0) continue;
      any = true;
      const int plain = w.tail ? w.steps - 1 : w.steps;
      if (lane == 0)
        for (int n = 0; ok && n < plain; ++n) ok = step(n, w.steps);
      ok = __all_sync(0xffffffffu, ok);
      if (lane != 0) ns += plain;
      if (w.tail && ok) {  // the next sequence's keys, which dQ sums over
        const int sk = ns % RK;
        ok = wait_warp(bar(L::B_KF + sk), (ns / RK) & 1, abort_flag, kErrDqMma);
        if (ok) {
          zero_rows<L::kSub>(sm + L::K + sk * L::kTileBytes, at.nk - plain * kRows, lane, 32);
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0 && ok) ok = step(plain, w.steps);
        ok = __all_sync(0xffffffffu, ok);
        if (lane != 0) ++ns;
      }
    }
    if (lane == 0) {
      if (ok && waiting) dq_step(ns - 1, first, last);
      mma_commit(bar(L::B_DRAIN));
      wait_one(bar(L::B_DRAIN), 0, abort_flag, kErrDqMma);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------ softmax warps
    // warpgroup w: keys [64 w, 64 w + 64) of each step
    const int wg = warp >> 2;
    const int r = (warp & 3) * 32 + lane;  // row of the tile == TMEM lane
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int t = over_group(r, group_inverse(hd.group)), head = r - t * hd.group;
    int ns = 0, n_fin = 0;
    bool ok = true;
    while (ok && next_item(at, items, sm + L::ITEMS, ring, abort_flag, lane, kErrDqSoftmax)) {
      if (at.kind != kTile) {
        if (at.part == 0) fill_rows(at.kind, at.tile, seqs.q, seqs, seqs.q_rows, 2 * n_tok, dq, hd.keys, at.h, hd.group * D);
        continue;
      }
      const DqSteps w(at, n_tok, causal);
      const int tok = w.tok0 + t;
      const bool valid = r < rows && tok < at.nq;
      const int seen = causal ? min(max(min(tok, w.last) + w.shift + 1, 0), at.nk) : at.nk;
      const int64_t stat = (((int64_t)at.h * hd.pairs + at.index) * 2 + at.part) * kRows + r;
      const float mrow = lse[stat], drow = delta[stat];
      for (int n = 0; n < w.steps; ++n) {
        const int lim = seen - n * kRows - wg * 64;
        const bool all_seen = __all_sync(0xffffffffu, lim >= 64), none = __all_sync(0xffffffffu, lim <= 0);
        if (!wait_warp(bar(L::B_SF), ns & 1, abort_flag, kErrDqSoftmax)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // S and dP are both read before the exponentials and released at once; dS overwrites that of the step
        // before, so its stores wait for that step's dQ; it is written in two parts to bound registers
        float p[64], dp[64];
        if (!none) tmem_load<2>(t_lane + L::T_S + wg * 64, p);
        if (!wait_warp(bar(L::B_DPF), ns & 1, abort_flag, kErrDqSoftmax)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (!none) tmem_load<2>(t_lane + L::T_DP + wg * 64, dp);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::B_DPE));
        if (!none && !all_seen) {  // masked keys: p = 0, whatever their V rows hold
          mask_from(p, lim);
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (c >= lim) dp[c] = 0.0f;
        }
        const float2 sc = make_float2(qk_scale, qk_scale), nm = make_float2(-mrow, -mrow), nd = make_float2(-drow, -drow);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t pk[16];
          if (!none) {
#pragma unroll
            for (int c = 32 * half; c < 32 * half + 32; c += 2) {
              const float2 x = __ffma2_rn(make_float2(p[c], p[c + 1]), sc, nm);
              const float2 ds = __fmul2_rn(make_float2(ex2(x.x), ex2(x.y)), __fadd2_rn(make_float2(dp[c], dp[c + 1]), nd));
              pk[(c - 32 * half) / 2] = Half<T>::pack(ds.x, ds.y);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) pk[i] = 0u;
          }
          if (half == 0) {
            if (ns > 0 && !wait_warp(bar(L::B_DSE), (ns - 1) & 1, abort_flag, kErrDqSoftmax)) {
              ok = false;
              break;
            }
            tc_fence_after();
          }
          tmem_st16(t_lane + L::T_DS + wg * 32 + 16 * half, pk);
        }
        if (!ok) break;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::B_DSF));
        ++ns;
      }
      if (!ok) break;
      // epilogue: warpgroup w writes columns [w D / 2, (w + 1) D / 2); a row without keys has none of its own
      const bool empty = seen == 0;
      T* row = dq + ((int64_t)(at.q0 + tok) * hd.keys * hd.group + at.h * hd.group + head) * D + wg * (D / 2);
      if (w.steps > 0) {
        if (!wait_warp(bar(L::B_FIN), n_fin & 1, abort_flag, kErrDqSoftmax)) {
          ok = false;
          break;
        }
        ++n_fin;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          uint32_t raw[32], pk[16];
          tmem_ld32(t_lane + L::T_DQ + wg * (D / 2) + c * 32, raw);
          tmem_wait_ld_dep(raw);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            pk[i] = empty ? 0u : Half<T>::pack(u2f(raw[2 * i]) * scale, u2f(raw[2 * i + 1]) * scale);
          if (valid) store32(row + c * 32, pk), store32(row + c * 32 + 16, pk + 8);
        }
        tc_fence_before();
      } else if (valid) {
        uint4* dst = reinterpret_cast<uint4*>(row);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) dst[i] = make_uint4(0, 0, 0, 0);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ================================================================ host side
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

// Makes the device's context the thread's: encoding a tensor map needs one, and a thread of autograd's whose
// first call this is has none yet.
static prism_status_t bind_context(const char* what) {
  int device = 0;
  PRISM_CHECK_CUDA(cudaGetDevice(&device), what);
  PRISM_CHECK_CUDA(cudaSetDevice(device), what);
  return PRISM_OK;
}

// [rows, heads, D] with row and head strides in elements; boxes of 64 columns x box_heads x box_rows.
static prism_status_t make_map(CUtensorMap* map, const void* ptr, int64_t rows, int heads, int D, const int64_t* strides,
                               int box_heads, int box_rows, int dtype) {
  EncodeFn enc = encode_fn();
  if (enc == nullptr) {
    set_error("prism_packed_attention: cuTensorMapEncodeTiled is unavailable from the driver");
    return PRISM_ERR_CUDA;
  }
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t bytes[2] = {(cuuint64_t)strides[1] * 2, (cuuint64_t)strides[0] * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(map, dtype == PRISM_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                   const_cast<void*>(ptr), dims, bytes, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("prism_packed_attention: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return PRISM_ERR_CUDA;
  }
  return PRISM_OK;
}

static int64_t pair_bound(int64_t rows, int64_t count, int group) {
  const int64_t per = 2 * (kRows / group);
  return (rows + per - 1) / per + count;
}

struct Shape {
  const void *q_offsets, *k_offsets;
  int wide;
  int64_t count, q_rows, k_rows;
  int q_heads, k_heads, D, causal, dtype;
  float scale;
  Sequences sequences() const {
    return {q_offsets, k_offsets, wide, (int)count, (int)q_rows, (int)k_rows};
  }
  Heads heads() const {
    const int group = q_heads / k_heads;
    return {k_heads, group, kRows / group, (int)pair_bound(q_rows, count, group)};
  }
  int64_t key_tiles() const { return (k_rows + kRows - 1) / kRows + count; }
  // Values of lse, or of delta: of all rows of all tiles.
  int64_t stats() const { return pair_bound(q_rows, count, q_heads / k_heads) * 2 * kRows * k_heads; }
  // Parts that the steps of `items` items are divided into: those for which the SMs' rounds of them take the
  // fewest steps, with 2.5 a round for an item's own costs and, where the parts are added up, 1.3 for reading
  // their sums and 4 for the launch.  Not divided where the items fill a round (16 sequences of 16 queries on
  // 4,096 keys: 66 us, 87 in seven parts), divided where they do not (128 queries on 32,768 keys, 8 items: 402 us,
  // 71 in 16 parts) or leave much of the last one idle, up to 16 rounds (310 MB of sums).
  static int parts(int64_t items, int64_t steps) {
    int best = 1;
    double least = 0.0;
    for (int p = 1; p <= 16 && (p == 1 || (steps >= 4 * p && items * p <= 16 * kSms)); ++p) {
      const double rounds = (double)((items * p + kSms - 1) / kSms);
      const double cost = rounds * ((double)steps / p + (p > 1 ? 3.8 : 2.5)) + (p > 1 ? 4.0 : 0.0);
      if (p == 1 || cost < least) best = p, least = cost;
    }
    return best;
  }
  // Tiles of `per` rows in `rows` rows of count sequences, half a tile too many each, and of an average sequence.
  int64_t tiles(int64_t rows, int64_t per) const {
    const int64_t n = rows / per + count / 2;
    return n > count ? n : count;
  }
  int forward_parts() const {
    if (count == 0) return 1;
    return parts(tiles(q_rows, 2 * (kRows / (q_heads / k_heads))) * k_heads, k_rows / count / kRows);
  }
  int dkdv_parts() const {
    if (count == 0) return 1;
    return parts(tiles(k_rows, kRows) * k_heads, q_rows / count / (kRows / (q_heads / k_heads)));
  }
};

static prism_status_t check(const Shape& s, const char* what) {
  constexpr int64_t kMost = (int64_t)1 << 30;
  PRISM_CHECK_ARG(s.D == 64 || s.D == 128, "%s: head dim %d not supported (64, 128)", what, s.D);
  PRISM_CHECK_ARG(s.k_heads >= 1 && s.q_heads >= 1 && s.q_heads % s.k_heads == 0 && s.q_heads / s.k_heads <= kRows,
                  "%s: %d query heads do not share %d key heads in equal groups of up to %d", what, s.q_heads,
                  s.k_heads, kRows);
  PRISM_CHECK_ARG(s.dtype == PRISM_BF16 || s.dtype == PRISM_FP16, "%s: element type %d (bf16 or fp16)", what, s.dtype);
  PRISM_CHECK_ARG(s.count >= 0 && s.q_rows >= 0 && s.k_rows >= 0 && s.count < kMost && s.q_rows < kMost && s.k_rows < kMost,
                  "%s: bad sizes", what);
  // the grids, the largest of which has two CTAs a pair of tiles and key head
  PRISM_CHECK_ARG(2 * pair_bound(s.q_rows, s.count, s.q_heads / s.k_heads) * s.k_heads < 2 * kMost &&
                      s.key_tiles() * s.k_heads < 2 * kMost,
                  "%s: too many rows, sequences or heads", what);
  PRISM_CHECK_ARG(s.scale > 0.0f && s.scale < 1.0e30f, "%s: the scale must be positive and finite", what);
  return PRISM_OK;
}

// Row and head strides, in elements, that a tensor map takes.
static prism_status_t check_rows(const void* p, const int64_t* strides, const char* what, const char* name) {
  PRISM_CHECK_ARG(p != nullptr && strides != nullptr, "%s: null pointer (%s)", what, name);
  PRISM_CHECK_ARG(aligned16(p) && strides[0] > 0 && strides[1] > 0 && strides[0] % 8 == 0 && strides[1] % 8 == 0 &&
                      strides[0] < ((int64_t)1 << 38) && strides[1] < ((int64_t)1 << 38),
                  "%s: %s must start on 16 bytes, with positive row and head strides of whole 16 bytes", what, name);
  return PRISM_OK;
}

#define PRISM_TRY(x)                       \
  do {                                     \
    prism_status_t st_ = (x);              \
    if (st_ != PRISM_OK) return st_;       \
  } while (0)

struct Input {
  const void* p;
  const int64_t* strides;
};

template <typename T, int D>
static prism_status_t launch_fwd(const Shape& s, const Input& q, const Input& k, const Input& v, void* o, float* lse,
                                 int8_t* rest, void* workspace, cudaStream_t stream) {
  constexpr const char* what = "prism_packed_attention";
  const Heads hd = s.heads();
  PRISM_TRY(bind_context(what));
  CUtensorMap mq, mk, mv;
  PRISM_TRY(make_map(&mq, q.p, s.q_rows, s.q_heads, D, q.strides, hd.group, hd.tokens, s.dtype));
  // without key rows nothing is loaded: any valid map does
  const Input& kk = s.k_rows > 0 ? k : q;
  const Input& vv = s.k_rows > 0 ? v : q;
  const int64_t k_rows = s.k_rows > 0 ? s.k_rows : s.q_rows;
  PRISM_TRY(make_map(&mk, kk.p, k_rows, s.k_heads, D, kk.strides, 1, kRows, s.dtype));
  PRISM_TRY(make_map(&mv, vv.p, k_rows, s.k_heads, D, vv.strides, 1, kRows, s.dtype));
  constexpr size_t bytes = FwdLayout<D>::kBytes;
  static_assert(bytes <= 227 * 1024, "shared memory");
  const Grid grid = {hd.pairs, lse != nullptr ? 1 : s.forward_parts(), s.causal};
  const int64_t rows = s.q_rows * s.q_heads;
  Parts parts = {nullptr, nullptr};
  auto kernel = fwd_kernel<T, D, kInfer>;
  if (grid.parts > 1) {
    parts.o = static_cast<float*>(workspace), parts.ml = reinterpret_cast<float2*>(parts.o + grid.parts * rows * D);
    kernel = fwd_kernel<T, D, kPart>;
  }
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    if (lse != nullptr) kernel = fwd_kernel<T, D, kTrain>;
  PRISM_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), what);
  kernel<<<(unsigned)(hd.pairs * hd.keys * grid.parts), kThreads, bytes, stream>>>(
      mq, mk, mv, s.sequences(), hd, grid, s.causal, s.scale * kLog2e, (T*)o, lse, rest, parts);
  PRISM_CHECK_LAUNCH(what);
  if (grid.parts > 1) {
    join_kernel<T, D><<<(unsigned)((rows * (D / 4) + kJoinThreads - 1) / kJoinThreads), kJoinThreads, 0, stream>>>(
        parts, grid.parts, rows, (T*)o);
    PRISM_CHECK_LAUNCH(what);
  }
  return PRISM_OK;
}

template <typename T, int D>
static prism_status_t launch_bwd(const Shape& s, const Input& q, const Input& k, const Input& v, const void* o,
                                 const int8_t* rest, const Input& go, const float* lse, void* workspace, void* dq,
                                 void* dk, void* dv, cudaStream_t stream) {
  constexpr const char* what = "prism_packed_attention_bwd";
  const Heads hd = s.heads();
  const Sequences seqs = s.sequences();
  float* delta = static_cast<float*>(workspace);
  float* sums = delta + s.stats();
  PRISM_TRY(bind_context(what));
  CUtensorMap mq, mk, mv, mdo;
  PRISM_TRY(make_map(&mq, q.p, s.q_rows, s.q_heads, D, q.strides, hd.group, hd.tokens, s.dtype));
  PRISM_TRY(make_map(&mdo, go.p, s.q_rows, s.q_heads, D, go.strides, hd.group, hd.tokens, s.dtype));
  PRISM_TRY(make_map(&mk, k.p, s.k_rows, s.k_heads, D, k.strides, 1, kRows, s.dtype));
  PRISM_TRY(make_map(&mv, v.p, s.k_rows, s.k_heads, D, v.strides, 1, kRows, s.dtype));
  delta_kernel<T, D><<<(unsigned)(hd.pairs * hd.keys), kDeltaThreads, 0, stream>>>(
      seqs, hd, (const T*)o, rest, (const T*)go.p, go.strides[0], go.strides[1], delta);
  PRISM_CHECK_LAUNCH(what);
  if (dk != nullptr) {
    constexpr size_t bytes = DkdvLayout<D>::kBytes;
    static_assert(bytes <= 227 * 1024, "shared memory");
    const Grid grid = {(int)s.key_tiles(), s.dkdv_parts(), 0};
    const auto kernel = grid.parts > 1 ? dkdv_kernel<T, D, true> : dkdv_kernel<T, D, false>;
    PRISM_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), what);
    kernel<<<(unsigned)(grid.tiles * hd.keys * grid.parts), kThreads, bytes, stream>>>(
        mq, mk, mv, mdo, seqs, hd, grid, s.causal, s.scale * kLog2e, s.scale, lse, delta, (T*)dk, (T*)dv, sums);
    PRISM_CHECK_LAUNCH(what);
    if (grid.parts > 1) {
      const int64_t count = s.k_rows * s.k_heads * D;
      const unsigned blocks = (unsigned)((count / 4 + kJoinThreads - 1) / kJoinThreads);
      add_parts_kernel<T><<<dim3(blocks, 2), kJoinThreads, 0, stream>>>(sums, grid.parts, count, s.scale, (T*)dk, (T*)dv);
      PRISM_CHECK_LAUNCH(what);
    }
  }
  if (dq != nullptr) {
    constexpr size_t bytes = DqLayout<D>::kBytes;
    static_assert(bytes <= 227 * 1024, "shared memory");
    const auto kernel = dq_kernel<T, D>;
    const Grid grid = {hd.pairs, 2, s.causal};
    PRISM_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), what);
    kernel<<<(unsigned)(2 * hd.pairs * hd.keys), kThreads, bytes, stream>>>(
        mq, mk, mv, mdo, seqs, hd, grid, s.causal, s.scale * kLog2e, s.scale, lse, delta, (T*)dq);
    PRISM_CHECK_LAUNCH(what);
  }
  return PRISM_OK;
}

}  // namespace packed
}  // namespace prism

using namespace prism;

int prism_packed_device_status_internal(void) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, packed::g_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(packed::g_error, &zero, sizeof(int));
  }
  return v;
}

extern "C" {

size_t prism_packed_attention_stats_bytes(int64_t q_rows, int64_t count, int q_heads, int k_heads) {
  if (q_rows < 0 || count < 0 || k_heads < 1 || q_heads < k_heads || q_heads / k_heads > packed::kRows) return 0;
  return (size_t)packed::pair_bound(q_rows, count, q_heads / k_heads) * 2 * packed::kRows * k_heads * sizeof(float);
}

size_t prism_packed_attention_workspace_bytes(int64_t q_rows, int64_t k_rows, int64_t count, int q_heads, int k_heads,
                                              int D) {
  if (q_rows < 0 || k_rows < 0 || count < 0 || D < 1 || k_heads < 1 || q_heads < k_heads || q_heads / k_heads > packed::kRows)
    return 0;
  const packed::Shape s = {nullptr, nullptr, 0, count, q_rows, k_rows, q_heads, k_heads, D, 0, PRISM_BF16, 1.0f};
  const int parts = s.forward_parts();
  return parts == 1 ? 0 : (size_t)parts * q_rows * q_heads * (D * sizeof(float) + sizeof(float2));
}

prism_status_t prism_packed_attention(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                      const void* v, const int64_t* v_strides, const void* q_offsets,
                                      const void* k_offsets, int offsets_64, int64_t count, int64_t q_rows,
                                      int64_t k_rows, int q_heads, int k_heads, int D, int causal, float scale,
                                      int dtype, void* o, float* lse, void* rest, void* workspace, cudaStream_t stream) {
  constexpr const char* what = "prism_packed_attention";
  const packed::Shape s = {q_offsets, k_offsets, offsets_64, count, q_rows, k_rows,
                           q_heads,   k_heads,   D,          causal != 0, dtype, scale};
  PRISM_TRY(packed::check(s, what));
  if (q_rows == 0) return PRISM_OK;
  PRISM_CHECK_ARG(q_offsets && k_offsets && o && aligned_to(o, 32) && aligned16(lse), "%s: null pointer, or o off 32 bytes", what);
  PRISM_CHECK_ARG((lse == nullptr) == (rest == nullptr) && (!lse || (dtype == PRISM_BF16 && aligned_to(rest, 32))),
                  "%s: lse and rest belong together, of bf16", what);
  PRISM_CHECK_ARG(lse || s.forward_parts() == 1 || (workspace && aligned_to(workspace, 32)), "%s: no workspace, or one off 32 bytes", what);
  PRISM_TRY(packed::check_rows(q, q_strides, what, "q"));
  if (k_rows > 0) {
    PRISM_TRY(packed::check_rows(k, k_strides, what, "k"));
    PRISM_TRY(packed::check_rows(v, v_strides, what, "v"));
  }
  const packed::Input iq = {q, q_strides}, ik = {k, k_strides}, iv = {v, v_strides};
  if (dtype == PRISM_FP16)
    return D == 64 ? packed::launch_fwd<__half, 64>(s, iq, ik, iv, o, lse, (int8_t*)rest, workspace, stream)
                   : packed::launch_fwd<__half, 128>(s, iq, ik, iv, o, lse, (int8_t*)rest, workspace, stream);
  return D == 64 ? packed::launch_fwd<__nv_bfloat16, 64>(s, iq, ik, iv, o, lse, (int8_t*)rest, workspace, stream)
                 : packed::launch_fwd<__nv_bfloat16, 128>(s, iq, ik, iv, o, lse, (int8_t*)rest, workspace, stream);
}

size_t prism_packed_attention_bwd_workspace_bytes(int64_t q_rows, int64_t k_rows, int64_t count, int q_heads,
                                                  int k_heads, int D) {
  if (q_rows < 0 || k_rows < 0 || count < 0 || D < 1 || k_heads < 1 || q_heads < k_heads || q_heads / k_heads > packed::kRows)
    return 0;
  const packed::Shape s = {nullptr, nullptr, 0, count, q_rows, k_rows, q_heads, k_heads, D, 0, PRISM_BF16, 1.0f};
  const int parts = s.dkdv_parts();
  return (size_t)(s.stats() + (parts == 1 ? 0 : 2 * (int64_t)parts * k_rows * k_heads * D)) * sizeof(float);
}

prism_status_t prism_packed_attention_bwd(const void* q, const int64_t* q_strides, const void* k,
                                          const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                          const void* o, const void* rest, const void* dout,
                                          const int64_t* dout_strides, const float* lse, const void* q_offsets, const void* k_offsets,
                                          int offsets_64, int64_t count, int64_t q_rows, int64_t k_rows, int q_heads,
                                          int k_heads, int D, int causal, float scale, void* workspace, void* dq,
                                          void* dk, void* dv, cudaStream_t stream) {
  constexpr const char* what = "prism_packed_attention_bwd";
  const packed::Shape s = {q_offsets, k_offsets, offsets_64, count, q_rows, k_rows,
                           q_heads,   k_heads,   D,          causal != 0, PRISM_BF16, scale};
  PRISM_TRY(packed::check(s, what));
  PRISM_CHECK_ARG(q_rows > 0 && k_rows > 0, "%s: no rows (all gradients are zero)", what);
  PRISM_CHECK_ARG(q_offsets && k_offsets && o && rest && lse && workspace && (dk == nullptr) == (dv == nullptr),
                  "%s: null pointer", what);
  PRISM_CHECK_ARG(aligned16(o) && aligned16(rest) && aligned16(lse) && aligned_to(workspace, 32) && aligned_to(dq, 32) && aligned_to(dk, 32) &&
                      aligned_to(dv, 32),
                  "%s: buffers must start on 32 bytes", what);
  PRISM_TRY(packed::check_rows(q, q_strides, what, "q"));
  PRISM_TRY(packed::check_rows(k, k_strides, what, "k"));
  PRISM_TRY(packed::check_rows(v, v_strides, what, "v"));
  PRISM_TRY(packed::check_rows(dout, dout_strides, what, "dout"));
  const packed::Input iq = {q, q_strides}, ik = {k, k_strides}, iv = {v, v_strides}, ig = {dout, dout_strides};
  return D == 64 ? packed::launch_bwd<__nv_bfloat16, 64>(s, iq, ik, iv, o, (const int8_t*)rest, ig, lse, workspace, dq, dk, dv, stream)
                 : packed::launch_bwd<__nv_bfloat16, 128>(s, iq, ik, iv, o, (const int8_t*)rest, ig, lse, workspace, dq, dk, dv, stream);
}

}  // extern "C"
