// Attention of (N, H, E, Lq) queries to (N, Hkv, E, Lk) keys and values,
// channels-first, H a multiple of Hkv, the first kv_lengths[n] keys of a
// record counting:
//
//   s_ij = scale * q_i . k_j + table[h, bucket(j*key_step - query_start - i)]
//   p_ij = softmax_j(s_ij),  o_i = sum_j p_ij v_j
//
// and its gradient, with delta_i = sum_j p_ij dp_ij, dp_ij = do_i . v_j,
// ds_ij = p_ij (dp_ij - delta_i):
//
//   dv_j = sum_i p_ij do_i,   dk_j = scale * sum_i ds_ij q_i,
//   dq_i = scale * sum_j ds_ij k_j,   dtable[h,b] = sum of ds over b's pairs.
//
// Neither s nor p reaches memory: the forward pass keeps a running maximum
// and sum per query and leaves their joint logarithm, from which the
// backward kernels make p again. Scores are kept in units of log2.
//
// Matrix instructions. A wave owns 32 columns (queries, or keys in the dk/dv
// kernel) and walks tiles of 32 rows of the other sequence. Scores come out
// of v_mfma_f32_32x32 with the wave's columns along the lanes, so softmax
// statistics are in-lane but for one exchange between the wave's halves, and
// a lane's 16 scores are at once the right operand of the second product:
// the rows of the first product are taken in an order (Mma::seq) that makes
// them so, and p and ds never leave registers. The staged tiles keep the
// channels-first layout, (channel, position) with positions contiguous; the
// first product reads them through the transposing LDS load, the second with
// plain 16-byte loads.
//
// bf16: p and ds are rounded to bf16 for the second products, which is the
// type their other operand has; statistics, sums and products are fp32.
// fp32: everything is fp32 on the fp32 matrix instructions.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "sa_common.h"

namespace {

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
  int buckets, exact, steps, max_distance, key_step, query_start;
  int threshold[kMaxThresholds];
};

struct Args {
  const void *q, *k, *v, *o, *dout;
  void *out, *dk, *dv;
  float* lse;      // (N, H, Lq), log2; +inf where a query has no key
  float* delta;    // (N, H, Lq)
  float* part;     // split results, fp32
  float* stat;     // split maxima and sums
  float* dbias;    // (N, Hkv*G, row tiles, buckets)
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
  // channel of element j of the kk-th operand
  __device__ static int channel(int kk, int j, int h) { return 16 * kk + 8 * h + j; }
  __device__ static void put(Op& op, int j, float v) { op[j] = (__bf16)v; }
  __device__ static float get(const Op& op, int j) { return (float)op[j]; }

  // channels 16*kk.. of positions col..col+31, positions along the rows. The
  // transposing load gives lane i of 16 its column of a 4 x 16 block that the
  // 16 lanes address in pieces of 4; pieces 1 and 2 are swapped, so that the
  // rows of the product are in the order seq() says.
  template <int STRIDE>
  __device__ static Op first(const __bf16* tile, int kk, int col) {
    const int l = threadIdx.x & 63, i = l & 15, t = (l >> 4) & 1, h = l >> 5;
    const int c = i & 3;
    const int piece = ((c & 1) << 1) | (c >> 1);
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
  // acc += tile[channel, col + position] * p[position], channels `row`..+31
  template <int STRIDE, int ROWS>
  __device__ static void second(f32x16& acc, const __bf16* tile, int row,
                                int col, const Op (&p)[2]) {
    const int l = threadIdx.x & 63, h = l >> 5;
    const __bf16* at = tile + (row + (l & (ROWS < 32 ? ROWS - 1 : 31))) * STRIDE
                       + col + 8 * h;
    acc = mul(*(const Op*)at, p[0], acc);
    acc = mul(*(const Op*)(at + 16), p[1], acc);
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
  __device__ static int channel(int kk, int j, int h) { return 2 * kk + h; }
  __device__ static void put(Op& op, int, float v) { op = v; }
  __device__ static float get(const Op& op, int) { return op; }
  template <int STRIDE>
  __device__ static Op first(const float* tile, int kk, int col) {
    const int l = threadIdx.x & 63;
    return tile[(2 * kk + (l >> 5)) * STRIDE + col + (l & 31)];
  }
  __device__ static f32x16 mul(Op a, Op b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
  }
  template <int STRIDE, int ROWS>
  __device__ static void second(f32x16& acc, const float* tile, int row,
                                int col, const float (&p)[16]) {
    const int l = threadIdx.x & 63, h = l >> 5;
    const float* at = tile + (row + (l & (ROWS < 32 ? ROWS - 1 : 31))) * STRIDE
                      + col + 4 * h;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 a = *(const f32x4*)(at + 8 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc = mul(a[i], p[4 * g + i], acc);
    }
  }
  using Right = float[16];
  __device__ static void right(float (&p)[16], const float (&s)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = s[i];
  }
};

// A tile of ED channels by POS positions in LDS. Rows are padded by 16
// bytes, which spreads the second product's 16-byte reads of 8 consecutive
// rows over all banks. NT threads stage it.
template <typename T, int ED, int POS, int NT>
struct Tile {
  static constexpr int kVec = Mma<T>::kVec;
  static constexpr int kStride = POS + kVec;
  static constexpr int kPerRow = POS / kVec;
  static constexpr int kChunks = ED * kPerRow;
  static constexpr int kOwn = (kChunks + NT - 1) / NT;
  static constexpr int kBytes = ED * kStride * sizeof(T);
  struct alignas(16) Chunk { T v[kVec]; };
  Chunk c[kOwn];

  // positions first.. of a sequence with `count` of them, rows of `E`
  // channels; what is outside is zero, so that nothing of it is ever seen
  __device__ __forceinline__ void load(const T* base, long stride, int E,
                                       long first, long count) {
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
      const int at = threadIdx.x + o * NT;
      const int row = at / kPerRow;
      const long pos = first + (at % kPerRow) * kVec;
      Chunk t = {};
      if (row < E && (kChunks % NT == 0 || at < kChunks)) {
        const T* p = base + row * stride + pos;
        if (pos + kVec <= count) {
          __builtin_memcpy(&t, p, sizeof(t));  // rows start anywhere
        } else {
#pragma unroll
          for (int j = 0; j < kVec; ++j)
            if (pos + j < count) t.v[j] = p[j];
        }
      }
      c[o] = t;
    }
  }
  __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
      const int at = threadIdx.x + o * NT;
      if (kChunks % NT == 0 || at < kChunks)
        *(Chunk*)(lds + (at / kPerRow) * kStride + (at % kPerRow) * kVec) =
            c[o];
    }
  }
};

// The wave's own columns as right operands, straight from memory: channel d
// of the lane's position is p[d * stride].
template <typename T, int ED>
__device__ __forceinline__ void own_columns(
    typename Mma<T>::Op (&op)[ED / Mma<T>::kDepth], const T* p, long stride,
    int E, bool live) {
  using M = Mma<T>;
  const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int kk = 0; kk < ED / M::kDepth; ++kk)
#pragma unroll
    for (int j = 0; j < M::kDepth / 2; ++j) {
      const int d = M::channel(kk, j, h);
      M::put(op[kk], j, live && d < E ? (float)p[d * stride] : 0.0f);
    }
}

__device__ __forceinline__ float other_half(float v) {
  return __shfl_xor(v, 32);
}

// --- position bias ---------------------------------------------------------

__device__ __forceinline__ int bucket_of(const Bias& b, int d) {
  const int n = d < 0 ? -d : d;
  int at = n;
  if (n >= b.exact) {
    at = b.exact;
    for (int m = 0; m < b.steps; ++m) at += n >= b.threshold[m];
  }
  return d > 0 ? at + b.buckets / 2 : at;
}

template <typename T>
__device__ __forceinline__ float bias_of(const Bias& b, int head, int d) {
  const float v = (float)((const T*)b.table)[head * b.buckets +
                                             bucket_of(b, d)];
  return v <= kOut ? -INFINITY : v * kLog2e;
}

__device__ __forceinline__ int clamped(int d, int most) {
  return max(-most, min(d, most)) + most;
}

// a head's bias by distance, -max_distance .. max_distance; `lane` of
// `lanes` fill it
template <typename T>
__device__ __forceinline__ void spread_bias(const Bias& b, int head,
                                            float* line, int lane,
                                            int lanes) {
  for (int i = lane; i <= 2 * b.max_distance; i += lanes)
    line[i] = bias_of<T>(b, head, i - b.max_distance);
}

// --- forward ---------------------------------------------------------------

enum BiasKind { NONE, LINE, DIRECT };  // LINE: a wave's rows share a head

__device__ __forceinline__ int key_count(const Args& p, int n) {
  if (p.lengths == nullptr) return p.Lk;
  return max(0, min(p.lengths[n], p.Lk));
}

// Consecutive workgroups go to the 8 dies in turn. Those that share keys and
// values are consecutive here, so each die is given one run of them.
__device__ __forceinline__ long spread_block() {
  const long all = gridDim.x, at = blockIdx.x;
  const long run = all / 8, rest = all % 8, die = at % 8;
  return die * run + min(die, rest) + at / 8;
}

template <typename T, int ED, int NW, int POS, BiasKind BIAS>
__global__ __launch_bounds__(NW * 64) void attend_kernel(Args p) {
  using M = Mma<T>;
  using Staged = Tile<T, ED, POS, NW * 64>;
  constexpr int DB = (ED + 31) / 32;
  constexpr int SUBS = POS / 32;
  extern __shared__ char shared[];
  T* tiles[2][2];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int c = 0; c < 2; ++c)
      tiles[b][c] = (T*)(shared + (2 * b + c) * Staged::kBytes);

  long block = spread_block();
  const int tile = block % p.tiles;
  block /= p.tiles;
  const int split = block % p.splits;
  const int nh = block / p.splits;
  const int n = nh / p.Hkv, hk = nh % p.Hkv;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int row = (tile * NW + wave) * 32 + (lane & 31);
  const int g = min(row / p.pad, p.G - 1);
  const int i = row - g * p.pad;
  const bool live = i < p.Lq;
  const int head = hk * p.G + g;
  const int position = p.bias.query_start + i;

  const int total = key_count(p, n);
  const int begin = split * p.per_split;
  const int end = min(total, begin + p.per_split);

  float* line = nullptr;
  if (BIAS == LINE) {
    line = (float*)(shared + 4 * Staged::kBytes) +
           wave * (2 * p.bias.max_distance + 1);
    spread_bias<T>(p.bias, __builtin_amdgcn_readfirstlane(head), line, lane,
                   64);
  }

  typename M::Op q[ED / M::kDepth];
  own_columns<T, ED>(q, (const T*)p.q + n * p.qn + head * p.qh +
                            (live ? i : 0),
                     p.qe, p.E, live);

  f32x16 acc[DB] = {};
  float most = -INFINITY, sum = 0.0f;
  const float scale = p.scale * kLog2e;
  const T* kb = (const T*)p.k + n * p.kn + hk * p.kh;
  const T* vb = (const T*)p.v + n * p.vn + hk * p.vh;

  Staged ks, vs;
  if (begin < end) {
    ks.load(kb, p.ke, p.E, begin, end);
    vs.load(vb, p.ve, p.E, begin, end);
  }
  int buf = 0;
  for (int at = begin; at < end; at += POS, buf ^= 1) {
    ks.store(tiles[buf][0]);
    vs.store(tiles[buf][1]);
    __syncthreads();
    if (at + POS < end) {
      ks.load(kb, p.ke, p.E, at + POS, end);
      vs.load(vb, p.ve, p.E, at + POS, end);
    }
    const T* kt = tiles[buf][0];
    const T* vt = tiles[buf][1];
    float s[SUBS][16];
    float top = -INFINITY;
#pragma unroll
    for (int b = 0; b < SUBS; ++b) {
      f32x16 c = {};
#pragma unroll
      for (int kk = 0; kk < ED / M::kDepth; ++kk)
        c = M::mul(M::template first<Staged::kStride>(kt, kk, 32 * b), q[kk],
                   c);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int key = at + 32 * b + M::seq(j, h);
        float v = c[j] * scale;
        if (BIAS == LINE)
          v += line[clamped(key * p.bias.key_step - position,
                            p.bias.max_distance)];
        if (BIAS == DIRECT)
          v += bias_of<T>(p.bias, head, key * p.bias.key_step - position);
        if (key >= end) v = -INFINITY;
        s[b][j] = v;
        top = fmaxf(top, v);
      }
    }
    top = fmaxf(top, other_half(top));
    if (__any(top > most)) {
      const float next = fmaxf(most, top);
      const float c = next == -INFINITY
                          ? 1.0f
                          : __builtin_amdgcn_exp2f(most - next);
      most = next;
      sum *= c;
#pragma unroll
      for (int d = 0; d < DB; ++d) acc[d] *= c;
    }
    const float base = most == -INFINITY ? 0.0f : most;
#pragma unroll
    for (int b = 0; b < SUBS; ++b) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        s[b][j] = __builtin_amdgcn_exp2f(s[b][j] - base);
        sum += s[b][j];
      }
      typename M::Right pr;
      M::right(pr, s[b]);
#pragma unroll
      for (int d = 0; d < DB; ++d)
        M::template second<Staged::kStride, ED>(acc[d], vt, 32 * d, 32 * b,
                                                pr);
    }
  }
  sum += other_half(sum);

  if (p.splits > 1) {
    const int rows = p.G * p.pad;
    if (row < rows && live) {
      const long at = (long)split * p.N * p.Hkv + nh;
      float* out = p.part + at * p.E * rows + row;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int e = 32 * d + 8 * (j / 4) + 4 * h + j % 4;
          if (e < p.E) out[(long)e * rows] = acc[d][j];
        }
      if (h == 0) {
        p.stat[(at * 2 + 0) * rows + row] = most;
        p.stat[(at * 2 + 1) * rows + row] = sum;
      }
    }
    return;
  }
  if (!live || row >= p.G * p.pad) return;
  const float inv = sum > 0.0f ? 1.0f / sum : sum;  // 0 keeps 0, NaN stays
  T* out = (T*)p.out + ((long)n * p.H + head) * p.E * p.Lq + i;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int e = 32 * d + 8 * (j / 4) + 4 * h + j % 4;
      if (e < p.E) out[(long)e * p.Lq] = (T)(acc[d][j] * inv);
    }
  if (p.lse && h == 0)
    p.lse[((long)n * p.H + head) * p.Lq + i] =
        sum == 0.0f ? INFINITY : most + log2f(sum);
}

// Joins the splits of the keys: one thread for a channel of a query.
template <typename T>
__global__ __launch_bounds__(256) void attend_join_kernel(Args p) {
  const int rows = p.G * p.pad;
  const long at = (long)blockIdx.x * 256 + threadIdx.x;
  const long all = (long)p.N * p.Hkv * p.E * rows;
  if (at >= all) return;
  const int row = at % rows;
  const int e = at / rows % p.E;
  const int nh = at / rows / p.E;
  const int g = row / p.pad, i = row % p.pad;
  if (i >= p.Lq) return;
  const long step = (long)p.N * p.Hkv;
  const float* stat = p.stat + (long)nh * 2 * rows + row;
  float most = -INFINITY;
  for (int s = 0; s < p.splits; ++s)
    most = fmaxf(most, stat[s * step * 2 * rows]);
  const float base = most == -INFINITY ? 0.0f : most;
  float sum = 0.0f, o = 0.0f;
  for (int s = 0; s < p.splits; ++s) {
    const float w =
        __builtin_amdgcn_exp2f(stat[s * step * 2 * rows] - base);
    sum = fmaf(w, stat[(s * step * 2 + 1) * rows], sum);
    o = fmaf(w, p.part[((s * step + nh) * p.E + e) * rows + row], o);
  }
  const int n = nh / p.Hkv, head = nh % p.Hkv * p.G + g;
  const float inv = sum > 0.0f ? 1.0f / sum : sum;
  ((T*)p.out)[(((long)n * p.H + head) * p.E + e) * p.Lq + i] = (T)(o * inv);
  if (p.lse && e == 0)
    p.lse[((long)n * p.H + head) * p.Lq + i] =
        sum == 0.0f ? INFINITY : most + log2f(sum);
}

// --- backward: dq, delta, dtable -------------------------------------------

// A wave's sums of ds by distance (one line for each half) and beyond the
// last one, added up by bucket. `out` is the wave's first row's place.
__device__ __forceinline__ void fold_table(const Args& p, const float* lines,
                                           float before, float behind,
                                           float* out, bool live) {
  const Bias& b = p.bias;
  const int lane = threadIdx.x & 63, half = b.buckets / 2;
  const int wide = 2 * b.max_distance + 1;
#pragma unroll 1
  for (int at = 0; at < b.buckets; ++at) {
    const bool after = at >= half;
    const int m = after ? at - half : at;
    int lo = m, hi = m + 1;
    if (m >= b.exact) {
      lo = m == b.exact ? b.exact : b.threshold[m - b.exact - 1];
      hi = m == half - 1 ? b.max_distance : b.threshold[m - b.exact];
    }
    if (after && lo == 0) lo = 1;
    float v = m < half - 1 ? 0.0f : after ? behind : before;
    for (int n = lo + lane; n < hi; n += 64) {
      const int d = b.max_distance + (after ? n : -n);
      v += lines[d] + lines[wide + d];
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    if (live && lane == 0) out[at] = v;
  }
}

// As the forward kernel, a wave has 32 queries along its lanes. TABLE: the
// gradient of the bias, too. Its entries sum ds over many pairs, and ds of a
// query sums to zero over its keys; a delta made from the rounded output
// would leave a remainder there that outgrows the entries, so bf16 walks the
// keys once more beforehand for the delta that belongs to these p and dp.
template <typename T, int ED, int NW, int POS, bool LINED, bool TABLE>
__global__ __launch_bounds__(NW * 64) void attend_dq_kernel(Args p) {
  using M = Mma<T>;
  using Staged = Tile<T, ED, POS, NW * 64>;
  constexpr int DB = (ED + 31) / 32;
  constexpr int SUBS = POS / 32;
  constexpr bool TWICE = TABLE && sizeof(T) == 2;
  extern __shared__ char shared[];
  T* kt = (T*)shared;
  T* vt = (T*)(shared + Staged::kBytes);

  long block = spread_block();
  const int tile = block % p.tiles;
  block /= p.tiles;
  const int split = block % p.splits;
  const int nh = block / p.splits;
  const int n = nh / p.Hkv, hk = nh % p.Hkv;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int row = (tile * NW + wave) * 32 + (lane & 31);
  const int g = min(row / p.pad, p.G - 1);
  const int i = row - g * p.pad;
  const bool live = i < p.Lq;
  const int head = hk * p.G + g;
  const int position = p.bias.query_start + i;
  const int wide = 2 * p.bias.max_distance + 1;

  const int total = key_count(p, n);
  const int begin = split * p.per_split;
  const int end = min(total, begin + p.per_split);

  float* line = nullptr;
  float* sums = nullptr;  // this half wave's ds by distance
  float before = 0.0f, behind = 0.0f;  // and those beyond the last bucket
  if (LINED) {
    line = (float*)(shared + 2 * Staged::kBytes) + wave * (TABLE ? 3 : 1) * wide;
    spread_bias<T>(p.bias, __builtin_amdgcn_readfirstlane(head), line, lane,
                   64);
    if (TABLE) {
      for (int d = lane; d < 2 * wide; d += 64) line[wide + d] = 0.0f;
      sums = line + (1 + h) * wide;
    }
  }

  typename M::Op q[ED / M::kDepth], go[ED / M::kDepth];
  const long col = live ? i : 0;
  own_columns<T, ED>(q, (const T*)p.q + n * p.qn + head * p.qh + col, p.qe,
                     p.E, live);
  own_columns<T, ED>(go, (const T*)p.dout + n * p.dn + head * p.dh + col,
                     p.de, p.E, live);
  const long stat = ((long)n * p.H + head) * p.Lq + col;
  const float lse = live ? p.lse[stat] : INFINITY;
  float delta = 0.0f;
  if (!TWICE) {
    const T* o = (const T*)p.o + ((long)n * p.H + head) * p.E * p.Lq + col;
#pragma unroll
    for (int kk = 0; kk < ED / M::kDepth; ++kk)
#pragma unroll
      for (int j = 0; j < M::kDepth / 2; ++j) {
        const int d = M::channel(kk, j, h);
        if (d < p.E)
          delta = fmaf(M::get(go[kk], j), (float)o[(long)d * p.Lq], delta);
      }
    delta += other_half(delta);
  }

  f32x16 acc[DB] = {};
  const float scale = p.scale * kLog2e;
  const T* kb = (const T*)p.k + n * p.kn + hk * p.kh;
  const T* vb = (const T*)p.v + n * p.vn + hk * p.vh;

#pragma unroll 1
  for (int walk = TWICE ? 0 : 1; walk < 2; ++walk) {
    Staged ks, vs;
    if (begin < end) {
      ks.load(kb, p.ke, p.E, begin, end);
      vs.load(vb, p.ve, p.E, begin, end);
    }
    for (int at = begin; at < end; at += POS) {
      __syncthreads();
      ks.store(kt);
      vs.store(vt);
      __syncthreads();
      if (at + POS < end) {
        ks.load(kb, p.ke, p.E, at + POS, end);
        vs.load(vb, p.ve, p.E, at + POS, end);
      }
#pragma unroll
      for (int b = 0; b < SUBS; ++b) {
        f32x16 c = {}, dp = {};
#pragma unroll
        for (int kk = 0; kk < ED / M::kDepth; ++kk) {
          c = M::mul(M::template first<Staged::kStride>(kt, kk, 32 * b),
                     q[kk], c);
          dp = M::mul(M::template first<Staged::kStride>(vt, kk, 32 * b),
                      go[kk], dp);
        }
        float ds[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int key = at + 32 * b + M::seq(j, h);
          float v = c[j] * scale;
          if (LINED)
            v += line[clamped(key * p.bias.key_step - position,
                              p.bias.max_distance)];
          const float e =
              key < end ? __builtin_amdgcn_exp2f(v - lse) : 0.0f;
          if (TWICE && walk == 0) delta = fmaf(e, dp[j], delta);
          ds[j] = e * (dp[j] - delta);
        }
        if (TWICE && walk == 0) continue;
        if (TABLE) {
          // the lanes of a half have different distances, and a wave's
          // additions reach LDS in order: the sums come out the same each
          // time
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int key = at + 32 * b + M::seq(j, h);
            const int d = key * p.bias.key_step - position;
            const int where = clamped(d, p.bias.max_distance);
            if (where == 0) before += ds[j];
            else if (where == wide - 1) behind += ds[j];
            else
              __hip_atomic_fetch_add(sums + where, ds[j], __ATOMIC_RELAXED,
                                     __HIP_MEMORY_SCOPE_WORKGROUP);
          }
        }
        typename M::Right pr;
        M::right(pr, ds);
#pragma unroll
        for (int d = 0; d < DB; ++d)
          M::template second<Staged::kStride, ED>(acc[d], kt, 32 * d, 32 * b,
                                                  pr);
      }
    }
    if (TWICE && walk == 0) delta += other_half(delta);
  }
  const int rows = p.G * p.pad;
  if (TABLE) {
    __syncthreads();
    fold_table(p, line + wide, before, behind,
               p.dbias + (((long)n * p.H + head) * (p.pad / 32) + i / 32) *
                             p.bias.buckets,
               row - (lane & 31) < rows);
  }
  if (row >= rows || !live) return;
  if (p.delta && split == 0 && h == 0) p.delta[stat] = delta;
  if (p.splits > 1) {
    float* out = p.part +
        (((long)split * p.N + n) * p.H + head) * p.E * p.Lq + i;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int e = 32 * d + 8 * (j / 4) + 4 * h + j % 4;
        if (e < p.E) out[(long)e * p.Lq] = acc[d][j] * p.scale;
      }
    return;
  }
  T* out = (T*)p.out + ((long)n * p.H + head) * p.E * p.Lq + i;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int e = 32 * d + 8 * (j / 4) + 4 * h + j % 4;
      if (e < p.E) out[(long)e * p.Lq] = (T)(acc[d][j] * p.scale);
    }
}

// --- backward: dk, dv --------------------------------------------------------

// A wave has 32 keys along its lanes and walks the queries of the heads that
// read them, a workgroup staging 64 at a time: so the sum over shared heads
// is made in registers.
template <typename T, int ED, int NW, int POS, bool LINED>
__global__ __launch_bounds__(NW * 64) void attend_dkv_kernel(Args p) {
  using M = Mma<T>;
  using Staged = Tile<T, ED, POS, NW * 64>;
  constexpr int DB = (ED + 31) / 32;
  constexpr int SUBS = POS / 32;
  static_assert(POS <= NW * 64, "one thread stages one query's statistics");
  extern __shared__ char shared[];
  T* qt = (T*)shared;
  T* dt = (T*)(shared + Staged::kBytes);
  float* lses = (float*)(shared + 2 * Staged::kBytes);
  float* deltas = lses + POS;
  float* line = deltas + POS;

  long block = spread_block();
  const int tile = block % p.tiles;
  block /= p.tiles;
  const int split = block % p.splits;
  const int nh = block / p.splits;
  const int n = nh / p.Hkv, hk = nh % p.Hkv;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int key = (tile * NW + wave) * 32 + (lane & 31);
  const int total = key_count(p, n);
  const bool live = key < total;

  const int all = p.G * p.pad;
  const int begin = split * p.per_split;
  const int end = tile * NW * 32 < total ? min(all, begin + p.per_split) : 0;

  typename M::Op k[ED / M::kDepth], v[ED / M::kDepth];
  const long col = live ? key : 0;
  own_columns<T, ED>(k, (const T*)p.k + n * p.kn + hk * p.kh + col, p.ke,
                     p.E, live);
  own_columns<T, ED>(v, (const T*)p.v + n * p.vn + hk * p.vh + col, p.ve,
                     p.E, live);

  f32x16 dk[DB] = {}, dv[DB] = {};
  const float scale = p.scale * kLog2e;
  Staged qs, os;
  float lse = INFINITY, delta = 0.0f;
  auto fetch = [&](int row) {
    const int g = row / p.pad, i = row - g * p.pad, head = hk * p.G + g;
    qs.load((const T*)p.q + n * p.qn + head * p.qh, p.qe, p.E, i, p.Lq);
    os.load((const T*)p.dout + n * p.dn + head * p.dh, p.de, p.E, i, p.Lq);
    lse = INFINITY;
    delta = 0.0f;
    if (threadIdx.x < POS && i + (int)threadIdx.x < p.Lq) {
      const long at = ((long)n * p.H + head) * p.Lq + i + threadIdx.x;
      lse = p.lse[at];
      delta = p.delta[at];
    }
  };
  if (begin < end) fetch(begin);
  int lined = -1;
  for (int row = begin; row < end; row += POS) {
    const int g = row / p.pad, i = row - g * p.pad;
    __syncthreads();
    qs.store(qt);
    os.store(dt);
    if (threadIdx.x < POS) {
      lses[threadIdx.x] = lse;
      deltas[threadIdx.x] = delta;
    }
    if (LINED && g != lined) {
      spread_bias<T>(p.bias, hk * p.G + g, line, threadIdx.x, NW * 64);
      lined = g;
    }
    __syncthreads();
    if (row + POS < end) fetch(row + POS);
#pragma unroll
    for (int b = 0; b < SUBS; ++b) {
      f32x16 c = {}, dp = {};
#pragma unroll
      for (int kk = 0; kk < ED / M::kDepth; ++kk) {
        c = M::mul(M::template first<Staged::kStride>(qt, kk, 32 * b), k[kk],
                   c);
        dp = M::mul(M::template first<Staged::kStride>(dt, kk, 32 * b), v[kk],
                    dp);
      }
      float e[16], ds[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int at = 32 * b + M::seq(j, h);
        float w = c[j] * scale;
        if (LINED)
          w += line[clamped(key * p.bias.key_step - p.bias.query_start - i -
                                at,
                            p.bias.max_distance)];
        e[j] = __builtin_amdgcn_exp2f(w - lses[at]);
        ds[j] = e[j] * (dp[j] - deltas[at]);
      }
      typename M::Right pr, dr;
      M::right(pr, e);
      M::right(dr, ds);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        M::template second<Staged::kStride, ED>(dv[d], dt, 32 * d, 32 * b,
                                                pr);
        M::template second<Staged::kStride, ED>(dk[d], qt, 32 * d, 32 * b,
                                                dr);
      }
    }
  }
  if (key >= p.Lk) return;
  // a key that does not count has gone through with k = v = 0: its column
  // holds numbers of no meaning
  const long first = (long)nh * p.E * p.Lk + key;
  const long whole = (long)p.N * p.Hkv * p.E * p.Lk;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int e = 32 * d + 8 * (j / 4) + 4 * h + j % 4;
      if (e >= p.E) continue;
      const long at = first + (long)e * p.Lk;
      const float a = live ? dk[d][j] * p.scale : 0.0f;
      const float b = live ? dv[d][j] : 0.0f;
      if (p.splits > 1) {
        p.part[split * whole + at] = a;
        p.part[(p.splits + split) * whole + at] = b;
      } else {
        ((T*)p.dk)[at] = (T)a;
        ((T*)p.dv)[at] = (T)b;
      }
    }
}

// out[i] = sum of `splits` runs of `count`
template <typename T>
__global__ __launch_bounds__(256) void sum_splits_kernel(const float* part,
                                                         T* out, long count,
                                                         int splits) {
  const long at = (long)blockIdx.x * 256 + threadIdx.x;
  if (at >= count) return;
  float v = 0.0f;
  for (int s = 0; s < splits; ++s) v += part[s * count + at];
  out[at] = (T)v;
}

// (N, H, tiles, buckets) -> (H, gridDim.y, buckets)
template <typename T>
__global__ __launch_bounds__(256) void sum_table_kernel(const float* in,
                                                        T* out, int N, int H,
                                                        int tiles,
                                                        int buckets) {
  __shared__ float sums[4][kMaxBuckets];
  const int b = threadIdx.x & 63, lane = threadIdx.x >> 6;
  const long rows = (long)N * tiles;
  const long each = (rows + gridDim.y - 1) / gridDim.y;
  const long begin = blockIdx.y * each, end = min(rows, begin + each);
  float v = 0.0f;
  if (b < buckets)
    for (long r = begin + lane; r < end; r += 4)
      v += in[((r / tiles * H + blockIdx.x) * tiles + r % tiles) * buckets +
              b];
  sums[lane][b] = v;
  __syncthreads();
  if (lane == 0 && b < buckets)
    out[((long)blockIdx.x * gridDim.y + blockIdx.y) * buckets + b] =
        (T)((sums[0][b] + sums[1][b]) + (sums[2][b] + sums[3][b]));
}

// --- host --------------------------------------------------------------------

template <typename K>
void launch(K kernel, long blocks, int threads, size_t lds, const Args& p,
            hipStream_t stream) {
  TORCH_CHECK(blocks < (1L << 31), "cross_attention: too many workgroups");
  if (lds > 64 * 1024)
    SA_CHECK_HIP(hipFuncSetAttribute(
        (const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
        (int)lds));
  kernel<<<dim3(blocks), dim3(threads), lds, stream>>>(p);
  SA_CHECK_HIP(hipGetLastError());
}

// positions of a staged tile
template <typename T, int ED>
constexpr int tile_positions() {
  return ED * sizeof(T) >= 512 ? 32 : 64;
}

template <typename F>
void with_depth(int E, F f) {
  if (E <= 16) f(std::integral_constant<int, 16>{});
  else if (E <= 32) f(std::integral_constant<int, 32>{});
  else if (E <= 64) f(std::integral_constant<int, 64>{});
  else f(std::integral_constant<int, 128>{});
}

template <typename F>
void with_type(at::ScalarType type, F f) {
  if (type == at::kBFloat16) f((__bf16)0);
  else f((float)0);
}

int round_up(long v, int to) { return (int)((v + to - 1) / to * to); }

// Where the workgroups are fewer than two for a compute unit, the long axis
// is cut: into pieces of 256 positions at least, which outweigh the joining.
int cut(long blocks, long length, int step, int* per_split) {
  const long want = 512;
  long splits = 1;
  if (blocks < want)
    splits = std::min<long>((want + blocks - 1) / blocks,
                            (length + 255) / 256);
  *per_split = round_up((length + splits - 1) / splits, step);
  return sa::ceil_div(length, *per_split);
}

struct Inputs {
  const at::Tensor &q, &k, &v;
  const c10::optional<at::Tensor>&lengths, &table;
};

Args args_of(const Inputs& in, double scale, long key_step, long query_start,
             long max_distance, const std::vector<long>& thresholds) {
  const auto &q = in.q, &k = in.k, &v = in.v;
  TORCH_CHECK(q.is_cuda() && k.device() == q.device() &&
                  v.device() == q.device(),
              "cross_attention: q, k and v on one GPU required");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.sizes() == k.sizes() &&
                  k.size(0) == q.size(0) && k.size(2) == q.size(2),
              "cross_attention: q (N, H, E, Lq), k and v (N, Hkv, E, Lk) "
              "required");
  TORCH_CHECK((q.scalar_type() == at::kBFloat16 ||
               q.scalar_type() == at::kFloat) &&
                  k.scalar_type() == q.scalar_type() &&
                  v.scalar_type() == q.scalar_type(),
              "cross_attention: q, k and v all bf16 or all fp32 required");
  TORCH_CHECK(q.stride(3) == 1 && k.stride(3) == 1 && v.stride(3) == 1,
              "cross_attention: unit stride along the positions required");
  TORCH_CHECK(k.size(1) >= 1 && q.size(1) % k.size(1) == 0,
              "cross_attention: H a multiple of Hkv required");
  TORCH_CHECK(q.size(2) >= 1 && q.size(2) <= 128,
              "cross_attention: E from 1 to 128 required");
  TORCH_CHECK(q.size(3) < (1L << 28) && k.size(3) < (1L << 28) &&
                  q.size(1) / k.size(1) * (q.size(3) + 128) < (1L << 30),
              "cross_attention: sequences too long");
  Args p = {};
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.qn = q.stride(0), p.qh = q.stride(1), p.qe = q.stride(2);
  p.kn = k.stride(0), p.kh = k.stride(1), p.ke = k.stride(2);
  p.vn = v.stride(0), p.vh = v.stride(1), p.ve = v.stride(2);
  p.N = q.size(0), p.H = q.size(1), p.Hkv = k.size(1), p.G = p.H / p.Hkv;
  p.E = q.size(2), p.Lq = q.size(3), p.Lk = k.size(3);
  p.scale = (float)scale;
  if (in.lengths.has_value()) {
    const auto& l = *in.lengths;
    TORCH_CHECK(l.device() == q.device() && l.scalar_type() == at::kInt &&
                    l.is_contiguous() && l.dim() == 1 && l.size(0) == p.N,
                "cross_attention: contiguous int32 kv_lengths (N) required");
    p.lengths = l.data_ptr<int>();
  }
  if (in.table.has_value()) {
    const auto& t = *in.table;
    TORCH_CHECK(t.device() == q.device() && t.is_contiguous() &&
                    t.dim() == 2 && t.size(0) == p.H &&
                    t.scalar_type() == q.scalar_type(),
                "cross_attention: contiguous bias table (H, buckets) of q's "
                "type required");
    Bias& b = p.bias;
    b.table = t.data_ptr();
    b.buckets = t.size(1);
    b.exact = b.buckets / 4;
    b.steps = thresholds.size();
    TORCH_CHECK(t.size(1) % 2 == 0 && b.buckets >= 4 &&
                    b.buckets <= kMaxBuckets &&
                    b.steps == b.buckets / 2 - b.exact - 1 &&
                    b.steps <= kMaxThresholds,
                "cross_attention: an even number of buckets from 4 to 64 "
                "required");
    TORCH_CHECK(max_distance > b.exact && max_distance <= kMaxDistance,
                "cross_attention: max_distance over buckets/4 and at most ",
                kMaxDistance, " required");
    const long limit = 1L << 30;
    TORCH_CHECK(key_step >= 1 && key_step < limit &&
                    (double)key_step * (p.Lk + 128) < (double)limit &&
                    std::abs(query_start) + p.Lq < limit,
                "cross_attention: positions out of range");
    b.max_distance = max_distance;
    b.key_step = key_step;
    b.query_start = query_start;
    long least = b.exact;
    for (int m = 0; m < b.steps; ++m) {
      TORCH_CHECK(thresholds[m] >= least && thresholds[m] <= max_distance,
                  "cross_attention: bucket thresholds out of order");
      least = b.threshold[m] = thresholds[m];
    }
  }
  return p;
}

}  // namespace

// {out, lse}; lse is empty unless `stats`
std::vector<at::Tensor> cross_attention_fwd(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
    const c10::optional<at::Tensor>& lengths,
    const c10::optional<at::Tensor>& table, double scale, long key_step,
    long query_start, long max_distance, std::vector<long> thresholds,
    bool stats) {
  Args p = args_of({q, k, v, lengths, table}, scale, key_step, query_start,
                   max_distance, thresholds);
  const c10::DeviceGuard guard(q.device());
  const auto f32 = q.options().dtype(at::kFloat);
  auto out = at::empty(q.sizes(), q.options());
  auto lse = at::empty({stats ? p.N : 0, p.H, p.Lq}, f32);
  if (out.numel() == 0) return {out, lse};
  const auto stream = at::hip::getCurrentHIPStream().stream();
  p.out = out.data_ptr();
  p.lse = stats ? lse.data_ptr<float>() : nullptr;
  // few rows for a key head share one wave's 32 columns, whatever their head
  const bool few = (long)p.G * p.Lq <= 32;
  const int waves = few ? 1 : 4;
  p.pad = few ? p.Lq : round_up(p.Lq, 32);
  const long rows = (long)p.G * p.pad;
  p.tiles = sa::ceil_div(rows, 32 * waves);
  const long pairs = (long)p.N * p.Hkv;
  p.splits = cut(pairs * p.tiles, std::max(p.Lk, 1), 64, &p.per_split);
  at::Tensor part, stat;
  if (p.splits > 1) {
    part = at::empty({p.splits * pairs * p.E * rows}, f32);
    stat = at::empty({p.splits * pairs * 2 * rows}, f32);
    p.part = part.data_ptr<float>();
    p.stat = stat.data_ptr<float>();
  }
  const long blocks = pairs * p.splits * p.tiles;
  with_type(q.scalar_type(), [&](auto zero) {
    using T = decltype(zero);
    with_depth(p.E, [&](auto depth) {
      constexpr int ED = decltype(depth)::value;
      if (few) {
        const size_t lds = 4 * Tile<T, ED, 32, 64>::kBytes;
        if (p.bias.table)
          launch(attend_kernel<T, ED, 1, 32, DIRECT>, blocks, 64, lds, p,
                 stream);
        else
          launch(attend_kernel<T, ED, 1, 32, NONE>, blocks, 64, lds, p,
                 stream);
      } else {
        constexpr int POS = tile_positions<T, ED>();
        const size_t lds = 4 * Tile<T, ED, POS, 256>::kBytes;
        const size_t lines = 4 * (2 * p.bias.max_distance + 1) * 4;
        if (p.bias.table)
          launch(attend_kernel<T, ED, 4, POS, LINE>, blocks, 256, lds + lines,
                 p, stream);
        else
          launch(attend_kernel<T, ED, 4, POS, NONE>, blocks, 256, lds, p,
                 stream);
      }
    });
    if (p.splits > 1)
      launch(attend_join_kernel<T>,
             (pairs * p.E * rows + 255) / 256, 256, 0, p, stream);
  });
  return {out, lse};
}

// {dq, dk, dv, dtable}; dk and dv empty unless `kv`, dtable unless `dtable`
std::vector<at::Tensor> cross_attention_bwd(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
    const c10::optional<at::Tensor>& lengths,
    const c10::optional<at::Tensor>& table, const at::Tensor& out,
    const at::Tensor& lse, const at::Tensor& dout, double scale,
    long key_step, long query_start, long max_distance,
    std::vector<long> thresholds, bool kv, bool dtable) {
  Args p = args_of({q, k, v, lengths, table}, scale, key_step, query_start,
                   max_distance, thresholds);
  TORCH_CHECK(dout.sizes() == q.sizes() && dout.stride(3) == 1 &&
                  dout.scalar_type() == q.scalar_type() &&
                  dout.device() == q.device(),
              "cross_attention: dout like q required");
  TORCH_CHECK(out.sizes() == q.sizes() && out.is_contiguous() &&
                  out.scalar_type() == q.scalar_type() &&
                  out.device() == q.device() && lse.is_contiguous() &&
                  lse.numel() == (long)p.N * p.H * p.Lq &&
                  lse.scalar_type() == at::kFloat &&
                  lse.device() == q.device(),
              "cross_attention: the forward pass's results required");
  TORCH_CHECK(!dtable || p.bias.table, "cross_attention: no table given");
  const c10::DeviceGuard guard(q.device());
  const auto f32 = q.options().dtype(at::kFloat);
  auto dq = at::empty(q.sizes(), q.options());
  auto dk = at::empty(kv ? k.sizes() : at::IntArrayRef({0}), q.options());
  auto dv = at::empty(kv ? v.sizes() : at::IntArrayRef({0}), q.options());
  auto dt = at::empty(
      dtable ? table->sizes() : at::IntArrayRef({0}), q.options());
  if (q.numel() == 0 || k.numel() == 0)
    return {dq.zero_(), dk.zero_(), dv.zero_(), dt.zero_()};
  const auto stream = at::hip::getCurrentHIPStream().stream();
  auto delta = at::empty({p.N, p.H, p.Lq}, f32);
  p.o = out.data_ptr();
  p.lse = lse.data_ptr<float>();
  p.delta = delta.data_ptr<float>();
  p.dout = dout.data_ptr();
  p.dn = dout.stride(0), p.dh = dout.stride(1), p.de = dout.stride(2);
  const long pairs = (long)p.N * p.Hkv;

  p.out = dq.data_ptr();
  p.pad = round_up(p.Lq, 32);
  p.tiles = sa::ceil_div((long)p.G * p.pad, 128);
  p.splits = cut(dtable ? 1L << 40 : pairs * p.tiles, p.Lk, 64, &p.per_split);
  at::Tensor part, sums;
  if (p.splits > 1) {
    part = at::empty({p.splits, q.numel()}, f32);
    p.part = part.data_ptr<float>();
  }
  if (dtable) {
    sums = at::empty({p.N, p.H, p.pad / 32, p.bias.buckets}, f32);
    p.dbias = sums.data_ptr<float>();
  }
  const size_t line = (2 * p.bias.max_distance + 1) * 4;
  with_type(q.scalar_type(), [&](auto zero) {
    using T = decltype(zero);
    with_depth(p.E, [&](auto depth) {
      constexpr int ED = decltype(depth)::value;
      constexpr int POS = tile_positions<T, ED>();
      const size_t lds = 2 * Tile<T, ED, POS, 256>::kBytes;
      const long blocks = pairs * p.splits * p.tiles;
      if (dtable)
        launch(attend_dq_kernel<T, ED, 4, POS, true, true>, blocks, 256,
               lds + 12 * line, p, stream);
      else if (p.bias.table)
        launch(attend_dq_kernel<T, ED, 4, POS, true, false>, blocks, 256,
               lds + 4 * line, p, stream);
      else
        launch(attend_dq_kernel<T, ED, 4, POS, false, false>, blocks, 256,
               lds, p, stream);
    });
    if (p.splits > 1) {
      sum_splits_kernel<T><<<sa::ceil_div(q.numel(), 256), 256, 0, stream>>>(
          p.part, (T*)dq.data_ptr(), q.numel(), p.splits);
      SA_CHECK_HIP(hipGetLastError());
    }
    if (dtable) {
      const long rows = (long)p.N * (p.pad / 32);
      const int pieces = (int)std::min<long>((rows + 63) / 64, 256);
      const dim3 grid(p.H, pieces);
      if (pieces == 1) {
        sum_table_kernel<T><<<grid, 256, 0, stream>>>(
            p.dbias, (T*)dt.data_ptr(), p.N, p.H, p.pad / 32,
            p.bias.buckets);
      } else {
        auto some = at::empty({p.H, pieces, p.bias.buckets}, f32);
        sum_table_kernel<float><<<grid, 256, 0, stream>>>(
            p.dbias, some.data_ptr<float>(), p.N, p.H, p.pad / 32,
            p.bias.buckets);
        sum_table_kernel<T><<<dim3(p.H, 1), 256, 0, stream>>>(
            some.data_ptr<float>(), (T*)dt.data_ptr(), 1, p.H, pieces,
            p.bias.buckets);
      }
      SA_CHECK_HIP(hipGetLastError());
    }
  });
  if (!kv) return {dq, dk, dv, dt};

  p.dk = dk.data_ptr();
  p.dv = dv.data_ptr();
  p.tiles = sa::ceil_div(p.Lk, 128);
  with_type(q.scalar_type(), [&](auto zero) {
    using T = decltype(zero);
    with_depth(p.E, [&](auto depth) {
      constexpr int ED = decltype(depth)::value;
      constexpr int POS = tile_positions<T, ED>();
      p.pad = round_up(p.Lq, POS);
      p.splits = cut(pairs * p.tiles, (long)p.G * p.pad, POS, &p.per_split);
      if (p.splits > 1) {
        part = at::empty({2, p.splits, k.numel()}, f32);
        p.part = part.data_ptr<float>();
      }
      const size_t lds = 2 * Tile<T, ED, POS, 256>::kBytes + 2 * POS * 4;
      const long blocks = pairs * p.splits * p.tiles;
      if (p.bias.table)
        launch(attend_dkv_kernel<T, ED, 4, POS, true>, blocks, 256,
               lds + line, p, stream);
      else
        launch(attend_dkv_kernel<T, ED, 4, POS, false>, blocks, 256, lds, p,
               stream);
    });
    if (p.splits > 1) {
      const int grid = sa::ceil_div(k.numel(), 256);
      sum_splits_kernel<T><<<grid, 256, 0, stream>>>(
          p.part, (T*)dk.data_ptr(), k.numel(), p.splits);
      sum_splits_kernel<T><<<grid, 256, 0, stream>>>(
          p.part + p.splits * k.numel(), (T*)dv.data_ptr(), k.numel(),
          p.splits);
      SA_CHECK_HIP(hipGetLastError());
    }
  });
  return {dq, dk, dv, dt};
}
