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

#include "cross_attention.h"

namespace attend {

// A running maximum is only raised once a score passes it by this much (in
// log2): until then p stays under 2^8, which costs no precision, and the
// sums need no rescaling.
constexpr float kSlack = 8.0f;

// The softmax of one more tile for a column's sums: scores in, weights out.
// `add` is a bias common to the tile, SCALED says that the scores already
// are in log2 with theirs.
template <int SUBS, int DB, bool SCALED>
__device__ __forceinline__ void weigh(float (&s)[SUBS][16], float scale,
                                      float add, float& most, float& sum,
                                      f32x16 (&acc)[DB]) {
  float top = s[0][0];
#pragma unroll
  for (int b = 0; b < SUBS; ++b)
#pragma unroll
    for (int j = 0; j < 16; ++j) top = fmaxf(top, s[b][j]);
  top = both_max(top);
  if (!SCALED) top = fmaf(top, scale, add);
  if (__any(top > most + kSlack)) {
    const float next = fmaxf(most, top);
    const float c =
        next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(most - next);
    most = next;
    sum *= c;
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] *= c;
  }
  const float base = most == -INFINITY ? 0.0f : most;
  const float off = SCALED ? -base : add - base;
#pragma unroll
  for (int b = 0; b < SUBS; ++b)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      s[b][j] = __builtin_amdgcn_exp2f(SCALED ? s[b][j] + off
                                              : fmaf(s[b][j], scale, off));
      sum += s[b][j];
    }
}

// Rows are the queries of the heads that share keys, head after head, each
// padded to whole waves: a workgroup of 4 waves stages POS keys at a time for
// 4 x QB x 32 rows. Two blocks of 32 columns for a wave (QB = 2) read a
// tile's operands from LDS once for both; LDS reads bound one block at about
// half of the matrix rate.
//
// Deep heads are bound by the matrix units and what a wave waits between
// them: (4, 16 on 4 heads of 128, 4096 x 4096) bf16 takes 593 us, 927 TFLOP/s.
// Small ones are bound by the vector units, and there by the exponential,
// which goes at a quarter of their rate: 24 heads of 16, 8192 x 8192, take
// 272 us, of which the 1.6e9 exponentials alone fill 164.
template <typename T, int ED, int QB, int POS, bool BIASED>
__global__ __launch_bounds__(
    256, ED * QB * (BIASED ? 2 : 1) * sizeof(T) <= 256 ? 2 : 1) void
attend_kernel(Args p) {
  using M = Mma<T>;
  using Staged = Tile<T, ED, POS, 256>;
  constexpr int DB = (ED + 31) / 32;
  constexpr int STEP = POS < 64 ? POS : 64;  // keys worked on at once
  constexpr int SUBS = STEP / 32;
  extern __shared__ char shared[];

  const Place place(p, p.tiles * p.splits);
  const int split = place.at / p.tiles, tile = place.at % p.tiles;
  const int nh = place.nh;
  const int n = nh / p.Hkv, hk = nh % p.Hkv;

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int total = key_count(p, n);
  const int begin = split * p.per_split;
  const int end = min(total, begin + p.per_split);

  const float scale = p.scale * kLog2e;
  const T* kb = (const T*)p.k + n * p.kn + hk * p.kh;
  const T* vb = (const T*)p.v + n * p.vn + hk * p.vh;
  Staged ks, vs;
  ks.place(p.ke, p.E, tid);
  vs.place(p.ve, p.E, tid);
  if (begin < end) {
    ks.load(kb, begin, end, tid);
    vs.load(vb, begin, end, tid);
  }

  float* line = (float*)(shared + 4 * Staged::kBytes) +
                line_middle(p.bias.max_distance, false);
  const int first = (tile * 4 + wave) * 32 * QB;  // this wave's first row
  const int g = min(first / p.pad, p.G - 1);
  const int head = hk * p.G + g;
  const int i0 = first - g * p.pad + (lane & 31);
  float before = 0.0f, behind = 0.0f, entry = 0.0f;
  if (BIASED) {  // the workgroup's rows are one head's
    entry = entry_of_lane<T>(p.bias, head);
    spread_bias<T, false>(p.bias, head, line, tid, 256);
    before = bias_of<T>(p.bias, head, -p.bias.max_distance);
    behind = bias_of<T>(p.bias, head, p.bias.max_distance);
  }
  typename M::Op q[QB][ED / M::kDepth];
#pragma unroll
  for (int c = 0; c < QB; ++c)
    own_columns<T, ED>(
        q[c], (T*)shared + wave * (Columns<T, ED>::kBytes / sizeof(T)),
        (const T*)p.q + n * p.qn + head * p.qh, p.qe, p.E,
        first - g * p.pad + 32 * c, p.Lq);
  __syncthreads();
  if (p.E < ED)
    for (int b = 0; b < 4; ++b)
      Staged::blank((T*)(shared + b * Staged::kBytes), p.E, tid);

  const Line bias_line(line, p.bias.max_distance);
  const bool holes = BIASED && takes_out(entry);
  f32x16 acc[QB][DB] = {};
  float most[QB], sum[QB];
#pragma unroll
  for (int c = 0; c < QB; ++c) most[c] = -INFINITY, sum[c] = 0.0f;
  int buf = 0;
  for (int at = begin; at < end; at += POS, buf ^= 1) {
    T* kt = (T*)(shared + 2 * buf * Staged::kBytes);
    T* vt = (T*)(shared + (2 * buf + 1) * Staged::kBytes);
    ks.store(kt, p.E, tid);
    vs.store(vt, p.E, tid);
    __syncthreads();
    if (at + POS < end) {
      ks.load(kb, at + POS, end, tid);
      vs.load(vb, at + POS, end, tid);
    }
    if (first - g * p.pad >= p.Lq) continue;  // no query of this wave's
#pragma unroll 1
    for (int col = 0; col < POS && at + col < end; col += STEP) {
      const int key0 = at + col;
      int side = 2;
      float add = 0.0f;
      if (BIASED) {
        const int from = first - g * p.pad + p.bias.query_start;
        side = beyond(p.bias, key0 * p.bias.key_step - (from + 32 * QB - 1),
                      (key0 + STEP - 1) * p.bias.key_step - from);
        add = side > 0 ? behind : before;
        if (side != 0 && add == -INFINITY) continue;  // all pairs are out
      }
      float s[QB][SUBS][16];
#pragma unroll
      for (int b = 0; b < SUBS; ++b) {
        f32x16 c[QB] = {};
#pragma unroll
        for (int kk = 0; kk < ED / M::kDepth; ++kk) {
          const auto a =
              M::template first<Staged::kStride>(kt, kk, col + 32 * b);
#pragma unroll
          for (int o = 0; o < QB; ++o) c[o] = M::mul(a, q[o][kk], c[o]);
        }
#pragma unroll
        for (int o = 0; o < QB; ++o)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[o][b][j] = c[o][j];
      }
      if (key0 + STEP > end) {
#pragma unroll
        for (int b = 0; b < SUBS; ++b)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (key0 + 32 * b + M::seq(j, h) >= end)
#pragma unroll
              for (int o = 0; o < QB; ++o) s[o][b][j] = -INFINITY;
      }
      if (BIASED && side == 0) {
#pragma unroll
        for (int o = 0; o < QB; ++o) {
          // the lane's own part of a distance; the rest is the wave's
          const int a0 = bias_line.at((key0 + M::seq(0, h)) * p.bias.key_step -
                                      (i0 + 32 * o + p.bias.query_start));
#pragma unroll
          for (int b = 0; b < SUBS; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j)
              s[o][b][j] = fmaf(
                  s[o][b][j], scale,
                  bias_line.get(a0 + 4 * (32 * b + M::seq(j, 0)) *
                                         p.bias.key_step));
          if (holes) {
            const int a1 = anew(a0);
#pragma unroll
            for (int b = 0; b < SUBS; ++b)
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (bias_line.get(a1 + 4 * (32 * b + M::seq(j, 0)) *
                                           p.bias.key_step) == -INFINITY)
                  s[o][b][j] = -INFINITY;
          }
          weigh<SUBS, DB, true>(s[o], 1.0f, 0.0f, most[o], sum[o], acc[o]);
        }
      } else {
#pragma unroll
        for (int o = 0; o < QB; ++o)
          weigh<SUBS, DB, false>(s[o], scale, add, most[o], sum[o], acc[o]);
      }
#pragma unroll
      for (int b = 0; b < SUBS; ++b) {
        typename M::Right pr[QB];
#pragma unroll
        for (int o = 0; o < QB; ++o) M::right(pr[o], s[o][b]);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const auto a =
              M::template second<Staged::kStride, ED>(vt, 32 * d, col + 32 * b);
#pragma unroll
          for (int o = 0; o < QB; ++o)
            acc[o][d] = M::mul(a, pr[o], acc[o][d]);
        }
      }
    }
  }

  __syncthreads();  // the results pass through where the tiles were
  if (first - g * p.pad >= p.Lq || first >= p.G * p.pad) return;
#pragma unroll
  for (int o = 0; o < QB; ++o) {
    const float all = both_sum(sum[o]);
    const int i = i0 + 32 * o;
    const long to = (long)n * p.H + head;
    if (p.splits > 1) {
      const int rows = p.G * p.pad, row = first + 32 * o + (lane & 31);
      if (i >= p.Lq) continue;
      const long at = (long)split * p.N * p.Hkv + nh;
      float* out = p.part + at * p.E * rows + row;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int e = 32 * d + 8 * (j / 4) + 4 * h + j % 4;
          if (e < p.E) out[(long)e * rows] = acc[o][d][j];
        }
      if (h == 0) {
        p.stat[(at * 2 + 0) * rows + row] = most[o];
        p.stat[(at * 2 + 1) * rows + row] = all;
      }
      continue;
    }
    const float inv = all > 0.0f ? 1.0f / all : all;  // 0 stays, NaN stays
    const int from = first - g * p.pad + 32 * o;
    put_columns<T, ED>(
        (T*)shared + wave * (Columns<T, ED>::kBytes / sizeof(T)), acc[o], inv,
        (T*)p.out + to * p.E * p.Lq + from, p.Lq, p.E, p.Lq - from);
    if (p.lse && h == 0 && i < p.Lq)
      p.lse[to * p.Lq + i] = all == 0.0f ? INFINITY : most[o] + log2f(all);
  }
}

// At most 32 rows for a key head, as when one query comes at a time: all of
// them, whatever their heads, are one wave's columns, and the 4 waves of a
// workgroup take the keys in turn, 32 at a time, each staging its own. What
// bounds it is reading keys and values, so many waves with a tile in flight
// each are what counts; they meet once, at the end, in LDS. One query of 16
// records, 8 heads on 2 of 64, 4096 keys in bf16: 9.5 us, 3.5 TB/s, and 3.9
// for the joining.
template <typename T, int ED, bool BIASED>
__global__ __launch_bounds__(
    256, ED * (BIASED ? 2 : 1) * sizeof(T) <= 256 ? 2 : 1) void
attend_few_kernel(Args p) {
  using M = Mma<T>;
  using Staged = Tile<T, ED, 32, 64>;
  constexpr int DB = (ED + 31) / 32;
  constexpr int BYTES = 2 * Staged::kBytes;  // of a wave
  static_assert(ED * 32 * sizeof(float) <= BYTES, "a wave's sums fit");
  extern __shared__ char shared[];

  const Place place(p, p.splits);
  const int split = place.at, nh = place.nh;
  const int n = nh / p.Hkv, hk = nh % p.Hkv;

  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = p.G * p.Lq;
  const int row = min(lane & 31, rows - 1);
  const int g = row / p.Lq, i = row - g * p.Lq;
  const int head = hk * p.G + g;
  const int position = p.bias.query_start + i;

  const int total = key_count(p, n);
  const int begin = split * p.per_split;
  const int end = min(total, begin + p.per_split);

  T* kt = (T*)(shared + wave * BYTES);
  T* vt = (T*)(shared + wave * BYTES + Staged::kBytes);
  const float scale = p.scale * kLog2e;
  const T* kb = (const T*)p.k + n * p.kn + hk * p.kh;
  const T* vb = (const T*)p.v + n * p.vn + hk * p.vh;

  Staged ks, vs;
  int at = begin + 32 * wave;
  ks.place(p.ke, p.E, lane);
  vs.place(p.ve, p.E, lane);
  if (at < end) {
    ks.load(kb, at, end, lane);
    vs.load(vb, at, end, lane);
  }
  float* stats = (float*)(shared + 4 * BYTES);  // (4, 2, 32)
  float* table = stats + 256;                   // (G, buckets), log2
  unsigned char* ids =                          // buckets by distance
      (unsigned char*)(table + p.G * p.bias.buckets);
  float before = 0.0f, behind = 0.0f;
  if (BIASED) {
    const T* t = (const T*)p.bias.table + hk * p.G * p.bias.buckets;
    for (int b = threadIdx.x; b < p.G * p.bias.buckets; b += 256) {
      const float v = (float)t[b];
      table[b] = v <= kOut ? -INFINITY : v * kLog2e;
    }
    for (int d = threadIdx.x; d <= 2 * p.bias.max_distance; d += 256)
      ids[d] = bucket_of(p.bias, d - p.bias.max_distance);
    table += g * p.bias.buckets;
    ids += p.bias.max_distance;
    before = bias_of<T>(p.bias, head, -p.bias.max_distance);
    behind = bias_of<T>(p.bias, head, p.bias.max_distance);
  }

  typename M::Op q[ED / M::kDepth];
  {
    T* qt = (T*)shared;  // (ED, 32), the rows as columns
    const int r = threadIdx.x & 31, from = min(r, rows - 1);
    const T* p0 = (const T*)p.q + n * p.qn +
                  (hk * p.G + from / p.Lq) * p.qh + from % p.Lq;
#pragma unroll
    for (int o = 0; o < ED / 8; ++o) {
      const int e = o * 8 + (threadIdx.x >> 5);
      const T v = p0[min(e, p.E - 1) * p.qe];
      qt[e * Staged::kStride + r] = e < p.E && r < rows ? v : (T)0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < ED / M::kDepth; ++kk)
      q[kk] = M::template first<Staged::kStride, false>(qt, kk, 0);
    __syncthreads();
  }
  f32x16 acc[DB] = {};
  float most = -INFINITY, sum = 0.0f;
  if (p.E < ED && at < end) {
    Staged::blank(kt, p.E, lane);
    Staged::blank(vt, p.E, lane);
  }
  for (; at < end; at += 128) {
    wave_fence();
    ks.store(kt, p.E, lane);
    vs.store(vt, p.E, lane);
    wave_fence();
    if (at + 128 < end) {
      ks.load(kb, at + 128, end, lane);
      vs.load(vb, at + 128, end, lane);
    }
    f32x16 c = {};
#pragma unroll
    for (int kk = 0; kk < ED / M::kDepth; ++kk)
      c = M::mul(M::template first<Staged::kStride>(kt, kk, 0), q[kk], c);
    float s[1][16];
#pragma unroll
    for (int j = 0; j < 16; ++j)
      s[0][j] = at + M::seq(j, h) < end ? c[j] : -INFINITY;
    int side = 2;
    if (BIASED) {
      const int from = p.bias.query_start;
      side = beyond(p.bias, at * p.bias.key_step - (from + p.Lq - 1),
                    (at + 31) * p.bias.key_step - from);
    }
    if (BIASED && side == 0) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int d = (at + M::seq(j, h)) * p.bias.key_step - position;
        const float b = table[ids[max(-p.bias.max_distance,
                                      min(d, p.bias.max_distance))]];
        s[0][j] = b == -INFINITY ? b : fmaf(s[0][j], scale, b);
      }
      weigh<1, DB, true>(s, 1.0f, 0.0f, most, sum, acc);
    } else {
      const float add = !BIASED ? 0.0f : side > 0 ? behind : before;
      if (BIASED && add == -INFINITY) {  // of this lane's head
#pragma unroll
        for (int j = 0; j < 16; ++j) s[0][j] = 0.0f;
      }
      weigh<1, DB, false>(s, scale, add, most, sum, acc);
    }
    typename M::Right pr;
    M::right(pr, s[0]);
#pragma unroll
    for (int d = 0; d < DB; ++d)
      acc[d] = M::mul(M::template second<Staged::kStride, ED>(vt, 32 * d, 0),
                      pr, acc[d]);
  }

  // the four waves' sums, where their tiles were
  sum = both_sum(sum);
  wave_fence();
  float* own = (float*)(shared + wave * BYTES);  // (ED, 32)
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int e = 32 * d + 8 * (j / 4) + 4 * h + j % 4;
      if (ED % 32 == 0 || e < ED) own[e * 32 + (lane & 31)] = acc[d][j];
    }
  if (h == 0) {
    stats[wave * 64 + lane] = most;
    stats[wave * 64 + 32 + lane] = sum;
  }
  __syncthreads();
  const int column = threadIdx.x & 31;
  if (column >= rows) return;
  float w[4], all = 0.0f, top = -INFINITY;
#pragma unroll
  for (int o = 0; o < 4; ++o) top = fmaxf(top, stats[o * 64 + column]);
  const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int o = 0; o < 4; ++o) {
    w[o] = __builtin_amdgcn_exp2f(stats[o * 64 + column] - base);
    all = fmaf(w[o], stats[o * 64 + 32 + column], all);
  }
  const int og = column / p.Lq, oi = column - og * p.Lq;
  const long where = (long)n * p.H + hk * p.G + og;
  const long at_split = (long)split * p.N * p.Hkv + nh;
  const float inv = all > 0.0f ? 1.0f / all : all;
  for (int e = threadIdx.x >> 5; e < p.E; e += 8) {
    float v = 0.0f;
#pragma unroll
    for (int o = 0; o < 4; ++o)
      v = fmaf(w[o], ((const float*)(shared + o * BYTES))[e * 32 + column], v);
    if (p.splits > 1)
      p.part[(at_split * p.E + e) * rows + column] = v;
    else
      ((T*)p.out)[(where * p.E + e) * p.Lq + oi] = (T)(v * inv);
  }
  if (threadIdx.x >= 32) return;
  if (p.splits > 1) {
    p.stat[(at_split * 2 + 0) * rows + column] = top;
    p.stat[(at_split * 2 + 1) * rows + column] = all;
  } else if (p.lse) {
    p.lse[where * p.Lq + oi] = all == 0.0f ? INFINITY : top + log2f(all);
  }
}

// Joins the splits of the keys: one thread for a channel of a query.
template <typename T>
__global__ __launch_bounds__(64) void attend_join_kernel(Args p) {
  const int rows = p.G * p.pad;
  const long at = (long)blockIdx.x * 64 + threadIdx.x;
  const long all = (long)p.N * p.Hkv * p.E * rows;
  if (at >= all) return;
  const int row = at % rows;
  const int e = at / rows % p.E;
  const int nh = at / rows / p.E;
  const int g = row / p.pad, i = row % p.pad;
  if (i >= p.Lq) return;
  const long step = (long)p.N * p.Hkv;
  const float* stat = p.stat + (long)nh * 2 * rows + row;
  const float* part = p.part + ((long)nh * p.E + e) * rows + row;
  float most = -INFINITY, sum = 0.0f, o = 0.0f;
  // 8 splits at a time, so that their loads are on the way together
  for (int s0 = 0; s0 < p.splits; s0 += 8) {
    float m[8], l[8], v[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const long s = min(s0 + c, p.splits - 1);
      m[c] = s0 + c < p.splits ? stat[s * step * 2 * rows] : -INFINITY;
      l[c] = stat[(s * step * 2 + 1) * rows];
      v[c] = part[s * step * p.E * rows];
    }
    float next = most;
#pragma unroll
    for (int c = 0; c < 8; ++c) next = fmaxf(next, m[c]);
    const float base = next == -INFINITY ? 0.0f : next;
    const float keep = __builtin_amdgcn_exp2f(most - base);
    sum *= keep;
    o *= keep;
    most = next;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const float w = __builtin_amdgcn_exp2f(m[c] - base);
      sum = fmaf(w, l[c], sum);
      o = fmaf(w, v[c], o);
    }
  }
  const int n = nh / p.Hkv, head = nh % p.Hkv * p.G + g;
  const float inv = sum > 0.0f ? 1.0f / sum : sum;
  ((T*)p.out)[(((long)n * p.H + head) * p.E + e) * p.Lq + i] = (T)(o * inv);
  if (p.lse && e == 0)
    p.lse[((long)n * p.H + head) * p.Lq + i] =
        sum == 0.0f ? INFINITY : most + log2f(sum);
}

template <typename T, int ED, int QB>
void launch_attend(const Args& p, long blocks, hipStream_t stream) {
  constexpr int POS = tile_positions<T, ED>();
  const size_t lds = 4 * Tile<T, ED, POS, 256>::kBytes;
  if constexpr (QB == 1) {
    if (p.bias.table)
      return launch(attend_kernel<T, ED, 1, POS, true>, blocks, 256,
                    lds + 4 * line_floats(p.bias.max_distance, false), p,
                    stream);
  }
  launch(attend_kernel<T, ED, QB, POS, false>, blocks, 256, lds, p, stream);
}

std::vector<at::Tensor> forward(const Call& c, bool stats) {
  Args p = args_of(c);
  const c10::DeviceGuard guard(c.q.device());
  const auto f32 = c.q.options().dtype(at::kFloat);
  auto out = at::empty(c.q.sizes(), c.q.options());
  at::Tensor lse;
  if (stats) lse = at::empty({p.N, p.H, p.Lq}, f32);
  if (out.numel() == 0) return {out, lse};
  const auto stream = at::hip::getCurrentHIPStream().stream();
  p.out = sa::memory_of(out);
  p.lse = stats ? sa::memory_of<float>(lse) : nullptr;
  const long pairs = (long)p.N * p.Hkv;
  const bool few = (long)p.G * p.Lq <= 32;
  // two blocks of columns a wave where that still leaves every compute unit
  // two workgroups and a SIMD two waves (heads up to 64); fp32 matrix
  // products are too slow to wait for LDS
  const bool twice = c.q.scalar_type() == at::kBFloat16 && p.E <= 64 &&
                     !p.bias.table &&
                     pairs * (p.G * (long)p.Lq / 256) >= 512;
  const int columns = twice ? 64 : 32;
  // with a bias, a workgroup's rows are one head's
  p.pad = few ? p.Lq : round_up(p.Lq, p.bias.table ? 4 * columns : columns);
  const long rows = (long)p.G * p.pad;
  p.tiles = few ? 1 : sa::ceil_div(rows, 4 * columns);
  p.splits = cut(pairs * p.tiles, std::max(p.Lk, 1), 128, &p.per_split);
  at::Tensor part;
  if (p.splits > 1) {
    const long sums = p.splits * pairs * p.E * rows;
    part = at::empty({sums + p.splits * pairs * 2 * rows}, f32);
    p.part = sa::memory_of<float>(part);
    p.stat = p.part + sums;
  }
  const long blocks = pairs * p.splits * p.tiles;
  with_type(c.q.scalar_type(), [&](auto zero) {
    using T = decltype(zero);
    with_depth(p.E, [&](auto depth) {
      constexpr int ED = decltype(depth)::value;
      if (few) {
        const size_t lds = 8 * Tile<T, ED, 32, 64>::kBytes + 1024;
        if (p.bias.table)
          launch(attend_few_kernel<T, ED, true>, blocks, 256,
                 lds + 4 * p.G * p.bias.buckets +
                     2 * p.bias.max_distance + 1,
                 p, stream);
        else
          launch(attend_few_kernel<T, ED, false>, blocks, 256, lds, p,
                 stream);
      } else if constexpr (sizeof(T) == 2 && ED <= 64) {
        if (twice) launch_attend<T, ED, 2>(p, blocks, stream);
        else launch_attend<T, ED, 1>(p, blocks, stream);
      } else {
        launch_attend<T, ED, 1>(p, blocks, stream);
      }
    });
    if (p.splits > 1)
      launch(attend_join_kernel<T>, (pairs * p.E * rows + 63) / 64, 64, 0, p,
             stream);
  });
  return {out, lse};
}

namespace {

// Tile::place reaches a head's channels by 32 bits of bytes, up to the end of
// a staged tile of 128 positions in the last one, whether or not so many are
// there.
bool within_reach(const at::Tensor& t, long stride) {
  return (stride * (t.size(2) - 1) + 128) * (long)t.element_size() <=
         (1L << 32);
}

at::Tensor along_positions(const at::Tensor& t) {
  return t.stride(3) == 1 && within_reach(t, t.stride(2)) ? t
                                                          : t.contiguous();
}

std::string shape_of(const at::Tensor& t) {
  return c10::str(t.sizes(), " ", t.scalar_type(), " on ", t.device());
}

// What the kernels take for granted. Lengths outside 0..Lk are held to it by
// the kernels.
Call checked(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
             const c10::optional<at::Tensor>& lengths,
             const c10::optional<at::Tensor>& table,
             c10::optional<double> scale, long key_step, long query_start,
             long max_distance, std::vector<long> thresholds) {
  TORCH_CHECK_VALUE(
      q.dim() == 4 && k.dim() == 4 && v.sizes() == k.sizes() &&
          k.size(0) == q.size(0) && k.size(2) == q.size(2),
      "cross_attention: q (N, H, E, Lq) and k, v (N, Hkv, E, Lk) are needed, "
      "got ", shape_of(q), ", ", shape_of(k), ", ", shape_of(v));
  const auto type = q.scalar_type();
  TORCH_CHECK_VALUE(
      (type == at::kBFloat16 || type == at::kFloat) &&
          k.scalar_type() == type && v.scalar_type() == type,
      "cross_attention: q, k and v have to be all float32 or all bfloat16, "
      "got ", type, ", ", k.scalar_type(), ", ", v.scalar_type());
  TORCH_CHECK_VALUE(q.is_cuda() && k.device() == q.device() &&
                        v.device() == q.device(),
                    "cross_attention: q, k and v have to be on one device");
  TORCH_CHECK(!sa::has_tangent(q) && !sa::has_tangent(k) &&
                  !sa::has_tangent(v) &&
                  !(table.has_value() && sa::has_tangent(*table)),
              "cross_attention: forward-mode derivatives are not available");
  const long H = q.size(1), Hkv = k.size(1), E = q.size(2), Lq = q.size(3),
             Lk = k.size(3);
  TORCH_CHECK_VALUE(Hkv > 0 && H % Hkv == 0, "cross_attention: ", H,
                    " query heads cannot share ", Hkv, " key heads");
  TORCH_CHECK_VALUE(E >= 1 && E <= 128, "cross_attention: heads of 1 to 128 "
                    "channels are needed, got ", E);
  TORCH_CHECK_VALUE(Lq < (1L << 28) && Lk < (1L << 28) &&
                        H / Hkv * (Lq + 256) < (1L << 30),
                    "cross_attention: sequences too long, ", shape_of(q), ", ",
                    shape_of(k));
  Call c = {along_positions(q), along_positions(k), along_positions(v), {},
            {}, scale.value_or(1.0 / std::sqrt((double)E)), key_step,
            query_start, max_distance, std::move(thresholds)};
  TORCH_CHECK_VALUE(c.scale > 0 && std::isfinite((float)c.scale * kLog2e),
                    "cross_attention: scale has to be positive, got ",
                    c.scale);
  for (const auto* t : {&c.q, &c.k, &c.v})
    TORCH_CHECK_VALUE(within_reach(*t, t->stride(2)) &&
                          within_reach(q, Lq),  // the output, read again
                      "cross_attention: a head has to fit into 4 GiB, got ",
                      shape_of(*t));
  if (lengths.has_value()) {
    const auto& l = *lengths;
    TORCH_CHECK_VALUE(
        l.dim() == 1 && l.size(0) == q.size(0) &&
            (l.scalar_type() == at::kInt || l.scalar_type() == at::kLong) &&
            l.device() == q.device(),
        "cross_attention: kv_lengths has to be [", q.size(0),
        "] int32 or int64 on ", q.device(), ", got ", shape_of(l));
    c.lengths = l.scalar_type() == at::kInt
                    ? l.contiguous()
                    : l.clamp(0, Lk).to(at::kInt).contiguous();
  }
  if (table.has_value()) {
    const auto& t = *table;
    TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == H &&
                          t.scalar_type() == type && t.device() == q.device(),
                      "cross_attention: bias_table has to be [", H,
                      ", buckets] ", type, " on ", q.device(), ", got ",
                      shape_of(t));
    const long buckets = t.size(1), exact = buckets / 4;
    TORCH_CHECK_VALUE(buckets % 2 == 0 && buckets >= 4 &&
                          buckets <= kMaxBuckets &&
                          (long)c.thresholds.size() ==
                              buckets / 2 - exact - 1,
                      "cross_attention: an even number of buckets from 4 to ",
                      kMaxBuckets, " is needed, got ", buckets);
    TORCH_CHECK_VALUE(max_distance > exact && max_distance <= kMaxDistance,
                      "cross_attention: max_distance has to be over ", exact,
                      " and at most ", kMaxDistance, ", got ", max_distance);
    long least = exact;
    for (const long m : c.thresholds) {
      TORCH_CHECK_VALUE(m >= least && m <= max_distance,
                        "cross_attention: bucket thresholds out of order");
      least = m;
    }
    TORCH_CHECK_VALUE(key_step >= 1, "cross_attention: key_step has to be 1 "
                      "or more, got ", key_step);
    const long limit = 1L << 27;
    TORCH_CHECK_VALUE(key_step < limit && key_step * (Lk + 128) < limit &&
                          query_start > -limit && query_start < limit &&
                          std::abs(query_start) + Lq + 256 < limit,
                      "cross_attention: positions have to stay under 2**27");
    c.table = t.contiguous();
  }
  return c;
}

// The node keeps the output and one logarithm a query; the backward pass
// makes the scores again.
class CrossAttention : public torch::autograd::Function<CrossAttention> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx,
                            const at::Tensor& q, const at::Tensor& k,
                            const at::Tensor& v,
                            const c10::optional<at::Tensor>& table,
                            const Call& call) {
    auto r = attend::forward(call, true);
    ctx->save_for_backward(
        {q, k, v, call.table, call.lengths, r[0], r[1]});
    ctx->saved_data["scale"] = call.scale;
    ctx->saved_data["where"] = std::vector<int64_t>{
        call.key_step, call.query_start, call.max_distance};
    ctx->saved_data["thresholds"] = std::vector<int64_t>(
        call.thresholds.begin(), call.thresholds.end());
    return r[0];
  }
  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "cross_attention: second derivatives are not available");
    TORCH_CHECK(!sa::has_tangent(grads[0]),
                "cross_attention: forward-mode derivatives are not available");
    const auto s = ctx->get_saved_variables();
    const auto where = ctx->saved_data["where"].toIntVector();
    const auto steps = ctx->saved_data["thresholds"].toIntVector();
    const Call call = {s[0], s[1], s[2], s[3], s[4],
                       ctx->saved_data["scale"].toDouble(), where[0],
                       where[1], where[2],
                       std::vector<long>(steps.begin(), steps.end())};
    const at::Tensor dout = along_positions(grads[0]);
    const bool kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const bool table = call.table.defined() && ctx->needs_input_grad(3);
    auto r = attend::backward(call, s[5], s[6], dout, kv, table);
    return {r[0], r[1], r[2], r[3], at::Tensor()};
  }
};

}  // namespace
}  // namespace attend

// nothing where a call is recorded or a tensor only stands for one
c10::optional<at::Tensor> cross_attention(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
    const c10::optional<at::Tensor>& lengths,
    const c10::optional<at::Tensor>& table, c10::optional<double> scale,
    long key_step, long query_start, long max_distance,
    std::vector<long> thresholds) {
  if (sa::recorded() || sa::stands_in(q) || sa::stands_in(k) ||
      sa::stands_in(v) || sa::stands_in(lengths) || sa::stands_in(table))
    return c10::nullopt;
  const auto call =
      attend::checked(q, k, v, lengths, table, scale, key_step, query_start,
                      max_distance, std::move(thresholds));
  if (at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || v.requires_grad() ||
       (table.has_value() && table->requires_grad())))
    return attend::CrossAttention::apply(
        call.q, call.k, call.v,
        call.table.defined() ? c10::optional<at::Tensor>(call.table)
                             : c10::nullopt,
        call);
  return attend::forward(call, false)[0];
}
