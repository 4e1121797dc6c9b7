// Shared by the kernels of cross_attention.hip and cross_attention_bwd.hip:
// the matrix instructions on channels-first tiles, the position bias, and
// the host's checks.
#pragma once

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <climits>

#include "sa_common.h"
#include "sa_tensor.h"

namespace attend {

using bf16x8 = __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16;
using s16x4 = __attribute__((__vector_size__(4 * sizeof(short)))) short;
using f32x4 = __attribute__((__vector_size__(4 * sizeof(float)))) float;
using f32x16 = __attribute__((__vector_size__(16 * sizeof(float)))) float;
using lds_s16x4 = s16x4 __attribute__((address_space(3)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxThresholds = 16;
constexpr int kMaxBuckets = 64;
constexpr int kMaxDistance = 1024;
// a bias at or under this takes its pair out of the softmax
constexpr float kOut = -1e30f;

struct Bias {
  const void* table;  // (H, buckets), null without
  int buckets, exact, max_distance, key_step, query_start;
  int threshold[kMaxThresholds];  // those there are not: INT_MAX
};

struct Args {
  const void *q, *k, *v, *o, *dout;
  void *out, *dk, *dv;
  float* lse;      // (N, H, Lq), log2; +inf where a query has no key
  float* delta;    // (N, H, Lq)
  float* deltas;   // (splits, 2, N, H, Lq), shares of sum p dp and of sum p
  float* part;     // split results, fp32
  float* stat;     // split maxima and sums
  float* dbias;    // (N * splits, H, tiles of 128 rows, buckets)
  const int* lengths;
  long qn, qh, qe, kn, kh, ke, vn, vh, ve, dn, dh, de;
  int N, H, Hkv, G, E, Lq, Lk;
  int pad;         // rows a head takes: Lq, or Lq rounded up to whole tiles
  int tiles;       // row (or key) tiles of a workgroup's size
  int splits, per_split;
  float scale;     // times log2(e) in the scores, plain in the gradients
  Bias bias;
};

// --- matrix instructions and the staged tile ------------------------------

template <typename T>
struct Mma;

// Lane l has column l%32 and half h = l/32. Of the 32x32 result it holds 16
// rows; seq(i, h) is the position that the i-th of them stands for.
template <>
struct Mma<__bf16> {
  static constexpr int kVec = 8;        // elements of 16 bytes
  static constexpr int kDepth = 16;     // channels of one first product
  using Op = bf16x8;
  __device__ static int seq(int i, int h) { return 16 * (i / 8) + 8 * h + i % 8; }
  __device__ static float get(const Op& op, int j) { return (float)op[j]; }

  // channels 16*kk.. of positions col..col+31, positions along the rows. The
  // transposing load gives lane i of 16 its column of a 4 x 16 block that the
  // 16 lanes address in pieces of 4; pieces 1 and 2 are swapped, so that the
  // rows of the product are in the order seq() says; a right operand's
  // columns (SWAP false) stay in the lanes' order.
  template <int STRIDE, bool SWAP = true>
  __device__ static Op first(const __bf16* tile, int kk, int col) {
    const int l = threadIdx.x & 63, i = l & 15, t = (l >> 4) & 1, h = l >> 5;
    const int c = i & 3;
    const int piece = SWAP ? ((c & 1) << 1) | (c >> 1) : c;
    const __bf16* at = tile + (16 * kk + 8 * h + (i >> 2)) * STRIDE + col +
                       16 * t + 4 * piece;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(at + 4 * STRIDE));
    union { s16x4 s[2]; Op op; } u;
    u.s[0] = lo;
    u.s[1] = hi;
    return u.op;
  }
  __device__ static f32x16 mul(Op a, Op b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // the second product's left operand: channels row..+31 by 32 positions
  struct Left { Op a[2]; };
  template <int STRIDE, int ROWS>
  __device__ static Left second(const __bf16* tile, int row, int col) {
    const int l = threadIdx.x & 63, h = l >> 5;
    const __bf16* at = tile + (row + (l & (ROWS < 32 ? ROWS - 1 : 31))) * STRIDE
                       + col + 8 * h;
    return {{*(const Op*)at, *(const Op*)(at + 16)}};
  }
  __device__ static f32x16 mul(const Left& a, const Op (&p)[2], f32x16 c) {
    return mul(a.a[1], p[1], mul(a.a[0], p[0], c));
  }
  using Right = Op[2];
  __device__ static void right(Op (&p)[2], const float (&s)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i / 8][i % 8] = (__bf16)s[i];
  }
};

template <>
struct Mma<float> {
  static constexpr int kVec = 4;
  static constexpr int kDepth = 2;
  using Op = float;
  __device__ static int seq(int i, int h) { return 8 * (i / 4) + 4 * h + i % 4; }
  __device__ static float get(const Op& op, int) { return op; }
  template <int STRIDE, bool SWAP = true>
  __device__ static Op first(const float* tile, int kk, int col) {
    const int l = threadIdx.x & 63;
    return tile[(2 * kk + (l >> 5)) * STRIDE + col + (l & 31)];
  }
  __device__ static f32x16 mul(Op a, Op b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
  }
  struct Left { f32x4 a[4]; };
  template <int STRIDE, int ROWS>
  __device__ static Left second(const float* tile, int row, int col) {
    const int l = threadIdx.x & 63, h = l >> 5;
    const float* at = tile + (row + (l & (ROWS < 32 ? ROWS - 1 : 31))) * STRIDE
                      + col + 4 * h;
    Left r;
#pragma unroll
    for (int g = 0; g < 4; ++g) r.a[g] = *(const f32x4*)(at + 8 * g);
    return r;
  }
  __device__ static f32x16 mul(const Left& a, const float (&p)[16],
                               f32x16 c) {
#pragma unroll
    for (int i = 0; i < 16; ++i) c = mul(a.a[i / 4][i % 4], p[i], c);
    return c;
  }
  using Right = float[16];
  __device__ static void right(float (&p)[16], const float (&s)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = s[i];
  }
};

// A tile of ED channels by POS positions in LDS. Rows are padded by 16
// bytes, which spreads the second product's 16-byte reads of 8 consecutive
// rows over all banks. NT threads stage it, through registers, so that a
// tile is on its way while the one before it is worked on.
template <typename T, int ED, int POS, int NT>
struct Tile {
  static constexpr int kVec = Mma<T>::kVec;
  static constexpr int kStride = POS + kVec;
  static constexpr int kPerRow = POS / kVec;
  static constexpr int kChunks = ED * kPerRow;
  static constexpr int kOwn = (kChunks + NT - 1) / NT;
  static constexpr int kBytes = ED * kStride * sizeof(T);
  struct alignas(16) Chunk { unsigned long long v[2]; };
  Chunk c[kOwn];
  unsigned at[kOwn];  // bytes from a tile's first position in channel 0

  __device__ static int row_of(int tid, int o) {
    return (tid + o * NT) / kPerRow;
  }
  __device__ static int col_of(int tid, int o) {
    return (tid + o * NT) % kPerRow * kVec;
  }

  // A channel's rows are `stride` apart; all of a head's E channels lie
  // within 4 GiB. Rows past them repeat the last one and are not stored.
  __device__ __forceinline__ void place(long stride, int E, int tid) {
#pragma unroll
    for (int o = 0; o < kOwn; ++o)
      at[o] = (unsigned)(min(row_of(tid, o), E - 1) * (unsigned)stride +
                         col_of(tid, o)) * sizeof(T);
  }

  // positions first.. of a sequence of `count` that starts at `base`;
  // positions past the end are zero, so that nothing that stands there is
  // ever seen. Rows start anywhere, so the 16-byte loads are not aligned.
  __device__ __forceinline__ void load(const T* base, int first, int count,
                                       int tid) {
    const char* tile = (const char*)(base + first);
    if (first + POS <= count) {
#pragma unroll
      for (int o = 0; o < kOwn; ++o)
        __builtin_memcpy(&c[o], tile + at[o], sizeof(Chunk));
    } else if (count >= kVec) {
      // what would pass the end is read from the last whole 16 bytes
      // before it, and shifted
#pragma unroll
      for (int o = 0; o < kOwn; ++o) {
        const int over =
            max(0, first + col_of(tid, o) + kVec - count);  // elements
        __builtin_memcpy(&c[o], tile + at[o] - (long)over * (int)sizeof(T),
                         sizeof(Chunk));
      }
#pragma unroll
      for (int o = 0; o < kOwn; ++o) {
        const int over = max(0, first + col_of(tid, o) + kVec - count);
        const int bits = min(over, kVec) * 8 * (int)sizeof(T);
        unsigned long long lo = c[o].v[0], hi = c[o].v[1];
        if (bits >= 64) lo = hi, hi = 0;
        const int left = bits & 63;
        c[o].v[0] = bits >= 128 ? 0 : (lo >> left) | (hi << 1 << (63 - left));
        c[o].v[1] = hi >> left;
      }
    } else {  // a sequence shorter than 16 bytes
#pragma unroll
      for (int o = 0; o < kOwn; ++o) c[o] = Chunk{};
#pragma unroll 1
      for (int j = 0; j < count && first == 0; ++j) {
        const int bit = j * 8 * sizeof(T);
#pragma unroll
        for (int o = 0; o < kOwn; ++o) {
          if (col_of(tid, o) != 0) continue;
          unsigned v = 0;
          __builtin_memcpy(&v, tile + at[o] + j * sizeof(T), sizeof(T));
          const unsigned long long w = (unsigned long long)v << (bit & 63);
          c[o].v[0] |= bit < 64 ? w : 0;
          c[o].v[1] |= bit < 64 ? 0 : w;
        }
      }
    }
  }
  __device__ __forceinline__ void store(T* lds, int E, int tid) const {
#pragma unroll
    for (int o = 0; o < kOwn; ++o)
      if (row_of(tid, o) < E)
        *(Chunk*)(lds + row_of(tid, o) * kStride + col_of(tid, o)) = c[o];
  }
  // the rows that store() leaves out, once
  __device__ static void blank(T* lds, int E, int tid) {
#pragma unroll
    for (int o = 0; o < kOwn; ++o)
      if (row_of(tid, o) >= E && row_of(tid, o) < ED)
        *(Chunk*)(lds + row_of(tid, o) * kStride + col_of(tid, o)) = Chunk{};
  }
};

// LDS written and read by one wave alone: its accesses are carried out in
// order, so only the compiler has to keep them so
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The wave's own 32 columns as right operands: positions first.. of a
// sequence of `count`, by way of `lds`, which is this wave's.
template <typename T, int ED>
using Columns = Tile<T, ED, 32, 64>;

template <typename T, int ED>
__device__ __forceinline__ void own_columns(
    typename Mma<T>::Op (&op)[ED / Mma<T>::kDepth], T* lds, const T* base,
    long stride, int E, int first, int count) {
  const int lane = threadIdx.x & 63;
  Columns<T, ED> t;
  t.place(stride, E, lane);
  t.load(base, first, count, lane);
  wave_fence();
  t.store(lds, E, lane);
  if (E < ED) t.blank(lds, E, lane);
  wave_fence();
#pragma unroll
  for (int kk = 0; kk < ED / Mma<T>::kDepth; ++kk)
    op[kk] = Mma<T>::template first<Columns<T, ED>::kStride, false>(lds, kk,
                                                                    0);
}

// A wave's 32 columns of channels, as the second product leaves them, out to
// memory: `to` is channel 0 of the first column, `count` columns are there.
// By way of `lds`, which is this wave's, so that 16 bytes go out at a time
// and not an element (bf16: 64 lanes then write 1 KB and not 128 bytes).
template <typename T, int ED, int DB>
__device__ __forceinline__ void put_columns(T* lds, const f32x16 (&acc)[DB],
                                            float by, T* to, long stride,
                                            int E, int count) {
  using C = Columns<T, ED>;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  wave_fence();
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int e = 32 * d + 8 * (j / 4) + 4 * h + j % 4;
      if (ED % 32 == 0 || e < ED)
        lds[e * C::kStride + (lane & 31)] = (T)(acc[d][j] * by);
    }
  wave_fence();
#pragma unroll
  for (int o = 0; o < C::kOwn; ++o) {
    const int e = C::row_of(lane, o), col = C::col_of(lane, o);
    if (e >= E) continue;
    const T* from = lds + e * C::kStride + col;
    T* at = to + e * stride + col;
    if (col + C::kVec <= count) {
      const typename C::Chunk c = *(const typename C::Chunk*)from;
      __builtin_memcpy(at, &c, sizeof(c));
    } else {
#pragma unroll 1
      for (int j = 0; col + j < count; ++j) at[j] = from[j];
    }
  }
}

// over the two lanes that a column has, one in each half of the wave
__device__ __forceinline__ float both_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(
      __float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(
      __float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// --- position bias ---------------------------------------------------------

__device__ __forceinline__ int bucket_of(const Bias& b, int d) {
  const int n = d < 0 ? -d : d;
  int at = n;
  if (n >= b.exact) {
    at = b.exact;
#pragma unroll
    for (int m = 0; m < kMaxThresholds; ++m) at += n >= b.threshold[m];
  }
  return d > 0 ? at + b.buckets / 2 : at;
}

template <typename T>
__device__ __forceinline__ float bias_of(const Bias& b, int head, int d) {
  const float v = (float)((const T*)b.table)[head * b.buckets +
                                             bucket_of(b, d)];
  return v <= kOut ? -INFINITY : v * kLog2e;
}

// One of a head's entries for each lane, loaded early and looked at late: a
// wave whose head has one at or under kOut takes pairs out. Those are out
// whatever their scores are, and a NaN or an infinity plus -inf need not be
// -inf; so such a wave looks the bias up once more for each score. For the
// others that is a branch: pooled keys go from 28.5 to 29.7 us, training with
// a bias stays at 273, and with a comparison and a selection for every score
// they take 31.2 and 284.
template <typename T>
__device__ __forceinline__ float entry_of_lane(const Bias& b, int head) {
  const int lane = threadIdx.x & 63;
  return (float)((const T*)b.table)[head * b.buckets +
                                    min(lane, b.buckets - 1)];
}
__device__ __forceinline__ bool takes_out(float entry) {
  return __any(entry <= kOut);
}

// a value that the compiler takes for a new one, so that it computes what
// follows from it once more and keeps no registers for it in between
__device__ __forceinline__ int anew(int v) {
  asm("" : "+v"(v));
  return v;
}

// Where a distance's entry stands in a line of them. PADDED leaves out one
// place in 16, so that lanes whose distances are 16 apart (keys pooled by 16)
// do not all read the same banks.
template <bool PADDED>
__device__ __forceinline__ int line_at(int d) {
  return PADDED ? d + (d >> 4) : d;
}
__host__ __device__ inline int line_floats(int max_distance, bool padded) {
  return 2 * max_distance + 1 + (padded ? max_distance / 8 + 2 : 0);
}
// of distance 0 in such a line
__host__ __device__ inline int line_middle(int max_distance, bool padded) {
  return max_distance + (padded ? max_distance / 16 + 1 : 0);
}

// A line in LDS by the address that an entry has: 4 times the distance from
// distance 0's, held to the line's ends, so that a score's bias costs an
// addition, a comparison of three and the load. Distances stay under 2^28.
struct Line {
  int zero, low, high;
  __device__ __forceinline__ Line(const float* middle, int most) {
    zero = (int)(size_t)(const __attribute__((address_space(3))) float*)
        middle;
    low = zero - 4 * most;
    high = zero + 4 * most;
  }
  __device__ __forceinline__ int at(int distance) const {
    return zero + 4 * distance;
  }
  __device__ __forceinline__ float get(int at) const {
    int held;
    asm("v_med3_i32 %0, %1, %2, %3"
        : "=v"(held)
        : "v"(at), "v"(low), "v"(high));
    return *(const __attribute__((address_space(3))) float*)(size_t)held;
  }
};

// 32 columns of queries (or keys) against `span` positions of the other
// sequence: whether every distance is past the last bucket's start. `least`
// and `most` bound the distances; +1 and -1 say on which side.
__device__ __forceinline__ int beyond(const Bias& b, int least, int most) {
  return least >= b.max_distance ? 1 : most <= -b.max_distance ? -1 : 0;
}

// a head's bias by distance, -max_distance .. max_distance, at `line` for
// distance 0; `lane` of `lanes` fill it
template <typename T, bool PADDED>
__device__ __forceinline__ void spread_bias(const Bias& b, int head,
                                            float* line, int lane,
                                            int lanes) {
  for (int n = lane; n <= b.max_distance; n += lanes) {
    line[line_at<PADDED>(-n)] = bias_of<T>(b, head, -n);
    if (n > 0) line[line_at<PADDED>(n)] = bias_of<T>(b, head, n);
  }
}

__device__ __forceinline__ int key_count(const Args& p, int n) {
  if (p.lengths == nullptr) return p.Lk;
  return max(0, min(p.lengths[n], p.Lk));
}

// Which work a workgroup has: its place among the `inner` workgroups of a
// (record, key head) pair. Consecutive workgroups go to the 8 dies in turn;
// a pair's share keys and values (or queries), so they are given to one die,
// whose L2 then holds those, and neighbouring pairs to different dies, since
// the heads of a long record are all long.
struct Place {
  int nh, at;
  __device__ __forceinline__ Place(const Args& p, int inner) {
    const unsigned block = blockIdx.x;
    const unsigned even = (unsigned)(p.N * p.Hkv / 8) * 8 * inner;
    const unsigned j = block < even ? block / 8 : block - even;
    const unsigned k = j / inner;
    at = j - k * inner;
    nh = block < even ? k * 8 + block % 8 : even / inner + k;
  }
};

// --- host --------------------------------------------------------------------

template <typename K>
inline void launch(K kernel, long blocks, int threads, size_t lds,
                   const Args& p, hipStream_t stream) {
  // a launch has fewer than 2^32 threads
  TORCH_CHECK_VALUE(blocks * threads < (1L << 32),
                    "cross_attention: too much work for one launch, ", blocks,
                    " workgroups of ", threads, "; split the records");
  if (lds > 64 * 1024)
    SA_CHECK_HIP(hipFuncSetAttribute(
        (const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
        (int)lds));
  kernel<<<dim3(blocks), dim3(threads), lds, stream>>>(p);
  SA_CHECK_HIP(hipGetLastError());
}

// Positions of a staged tile: as many as 8 KB of it hold, from 32 to 128. A
// tile has to be worked on for as long as the next one is on its way, so
// heads of few channels need more positions.
template <typename T, int ED>
constexpr int tile_positions() {
  constexpr int bytes = ED * sizeof(T);
  return bytes > 256 ? 32 : bytes > 64 ? 64 : 128;
}

template <typename F>
inline void with_depth(int E, F f) {
  if (E <= 16) f(std::integral_constant<int, 16>{});
  else if (E <= 32) f(std::integral_constant<int, 32>{});
  else if (E <= 64) f(std::integral_constant<int, 64>{});
  else if (E <= 96) f(std::integral_constant<int, 96>{});
  else f(std::integral_constant<int, 128>{});
}

template <typename F>
inline void with_type(at::ScalarType type, F f) {
  if (type == at::kBFloat16) f((__bf16)0);
  else f((float)0);
}

inline int round_up(long v, int to) { return (int)((v + to - 1) / to * to); }

// Where the workgroups are fewer than two for a compute unit, the long axis
// is cut: into pieces of 256 positions at least, which outweigh the joining.
inline int cut(long blocks, long length, int step, int* per_split) {
  const long want = 512;
  long splits = 1;
  if (blocks < want)
    splits = std::min<long>((want + blocks - 1) / blocks,
                            (length + 255) / 256);
  *per_split = round_up((length + splits - 1) / splits, step);
  return sa::ceil_div(length, *per_split);
}

// A call's tensors, as checked by checked(): unit stride along positions.
struct Call {
  at::Tensor q, k, v, table, lengths;  // the last two may be undefined
  double scale;
  long key_step, query_start, max_distance;
  std::vector<long> thresholds;
};

inline Args args_of(const Call& c) {
  Args p = {};
  p.q = sa::memory_of(c.q);
  p.k = sa::memory_of(c.k);
  p.v = sa::memory_of(c.v);
  p.qn = c.q.stride(0), p.qh = c.q.stride(1), p.qe = c.q.stride(2);
  p.kn = c.k.stride(0), p.kh = c.k.stride(1), p.ke = c.k.stride(2);
  p.vn = c.v.stride(0), p.vh = c.v.stride(1), p.ve = c.v.stride(2);
  p.N = c.q.size(0), p.H = c.q.size(1), p.Hkv = c.k.size(1);
  p.G = p.H / p.Hkv;
  p.E = c.q.size(2), p.Lq = c.q.size(3), p.Lk = c.k.size(3);
  p.scale = (float)c.scale;
  if (c.lengths.defined()) p.lengths = sa::memory_of<int>(c.lengths);
  if (c.table.defined()) {
    Bias& b = p.bias;
    b.table = sa::memory_of(c.table);
    b.buckets = c.table.size(1);
    b.exact = b.buckets / 4;
    b.max_distance = c.max_distance;
    b.key_step = c.key_step;
    b.query_start = c.query_start;
    for (int m = 0; m < kMaxThresholds; ++m)
      b.threshold[m] = m < (int)c.thresholds.size() ? c.thresholds[m]
                                                    : INT_MAX;
  }
  return p;
}

// {out, lse}; lse is empty unless `stats`
std::vector<at::Tensor> forward(const Call& c, bool stats);
// {dq, dk, dv, dtable}; dk and dv empty unless `kv`, dtable unless `table`
std::vector<at::Tensor> backward(const Call& c, const at::Tensor& out,
                                 const at::Tensor& lse,
                                 const at::Tensor& dout, bool kv, bool table);

}  // namespace attend
