// Backward kernels of the attention in cross_attention.hip, which has the
// formulas.

#include "cross_attention.h"

namespace attend {

// LDS of a workgroup: two pairs of staged tiles and what stands behind them,
// where the four waves' own columns pass through beforehand
template <typename T, int ED>
size_t backward_lds(size_t behind) {
  const size_t staged =
      4 * Tile<T, ED, tile_positions<T, ED>(), 256>::kBytes + behind;
  return std::max<size_t>(staged, 4 * Columns<T, ED>::kBytes);
}

// the same for the kernel whose waves work in pairs, and what they hand over
template <typename T, int ED>
size_t deep_lds(size_t lines) {
  constexpr int POS = tile_positions<T, ED>();
  const size_t staged = 4 * Tile<T, ED, POS, 512>::kBytes + 16 * POS +
                        (lines + 3) / 4 * 16 + 4 * (POS / 32) * 4096;
  return std::max<size_t>(staged, 8 * Columns<T, ED>::kBytes);
}

// A workgroup's sums of ds by distance (a line for each of its 4 waves) and
// beyond the last one (a wave's in each lane), added up by bucket, each
// in the same order every time. `ends`: 8 floats of LDS.
__device__ __forceinline__ void fold_table(const Bias& b, const float* lines,
                                           float before, float behind,
                                           float* ends, float* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int half = b.buckets / 2, wide = 2 * b.max_distance + 1;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    before += __shfl_xor(before, off);
    behind += __shfl_xor(behind, off);
  }
  if (lane == 0) {
    ends[wave] = before;
    ends[4 + wave] = behind;
  }
  __syncthreads();
#pragma unroll 1
  for (int at = wave; at < b.buckets; at += 4) {
    const bool after = at >= half;
    const int m = after ? at - half : at;
    int lo = m, hi = m + 1;
    if (m >= b.exact) {
      lo = m == b.exact ? b.exact : b.threshold[m - b.exact - 1];
      hi = m == half - 1 ? b.max_distance : b.threshold[m - b.exact];
    }
    if (after && lo == 0) lo = 1;
    float v = m == half - 1 && lane < 4 ? ends[4 * after + lane] : 0.0f;
    for (int n = lo + lane; n < hi; n += 64) {
      const int d = b.max_distance + (after ? n : -n);
#pragma unroll
      for (int k = 0; k < 4; ++k) v += lines[k * wide + d];
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    if (lane == 0) out[at] = v;
  }
}

// Adds a wave's ds, 32 keys by 32 queries, to its sums by distance. Adding
// them where they are, an atomic an element, took 224 cycles for 64 lanes; so
// they go through LDS, and a lane sums a whole diagonal of equal distances:
// each distance is then added to once, in the same order every time.
template <typename T>
__device__ __forceinline__ void add_diagonals(const Bias& b,
                                              const float (&ds)[16],
                                              float* tile, float* sums,
                                              int d0, float& before,
                                              float& behind) {
  using M = Mma<T>;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int step = b.key_step, far = b.max_distance;
  auto add = [&](int d, float v) {
    before += d <= -far ? v : 0.0f;
    behind += d >= far ? v : 0.0f;
    if (d > -far && d < far) sums[d] += v;
  };
  if (step >= 32) {  // no two of the tile's distances are equal
#pragma unroll
    for (int j = 0; j < 16; ++j)
      add(d0 + M::seq(j, h) * step - (lane & 31), ds[j]);
    return;
  }
  constexpr int STRIDE = 33;  // a diagonal's reads then fall on other banks
  wave_fence();
#pragma unroll
  for (int j = 0; j < 16; ++j)
    tile[M::seq(j, h) * STRIDE + (lane & 31)] = ds[j];
  wave_fence();
  const float inv = 1.0f / step;
  // r = key * step - query, both within the tile
  for (int r = lane - 31; r <= 31 * step; r += 64) {
    // whole quotients: half a unit is more than what the products are off
    const int from = r > 0 ? (int)((r + step - 0.5f) * inv) : 0;
    const int to = min(31, (int)((r + 31.5f) * inv));
    float v = 0.0f;
    for (int k = from; k <= to; ++k) v += tile[k * STRIDE + k * step - r];
    add(d0 + r, v);
  }
}

// As the forward kernel, a wave has 32 queries along its lanes. What it is to
// find:
// DQ     dq, with delta from the output, or a given one
// DELTA  delta alone, from these p and dp
// TABLE  dq and the gradient of the bias, with a given delta.
// delta is the mean of dp under p. An entry of the bias sums ds over many
// pairs, and ds of a query sums to zero over its keys; a delta made from the
// output, which is rounded and whose p was, would leave a remainder there that
// outgrows the entries. So where the bias has a gradient, the keys are walked
// once more beforehand, and the mean is over what the same weights sum to: a
// logarithm of 13 has steps of 1e-6, and p with it.
// Where a query has 32 keys at most, its p and dp are in registers at once and
// delta is theirs too: with few keys the output is no smaller than a value,
// and so is its rounding.
// In heads of few channels that rounding shows whatever the keys' number: k's
// mean under p is q / E. So for up to 32 channels in bf16 the sums over keys
// of ds and of p k are kept as well: the first would be zero, and times the
// second it is what dq is off by; added to delta, it sets that right. Errors
// of dq against 64 bits, in those that rounding the exact dq leaves: 17 to 32
// channels 1.45 to 1.48 and 1.47 to 1.55 without, for 228 and 205 us of a
// backward pass of 32 x 8 heads, 1024 by 1024 (and a DELTA launch where keys
// are cut).
// Up to 16 channels the roundings of ds meet k's mean as well, and what they
// add up to is taken off with it, whoever found delta: 1.40, the sqrt(2) of
// two independent roundings, where it was 1.48 at 16 channels, 1.6 at 8 and
// 1.65 at 4. TABLE takes 173 and not 144 us (16 x 8 heads of 16, 2048 by 1000).
//
// Bound as the forward kernel is: 4096 x 4096, 64 heads of 128 on 16, 820 us,
// 1006 TFLOP/s; (8, 8, 2048 x 1000 at most) heads of 64 with a bias 43 us for
// DELTA and 96 for TABLE.
enum Find { DQ, DELTA, TABLE };

template <typename T, int ED, int POS, bool LINED, Find FIND>
__global__ __launch_bounds__(
    256, ED * (LINED ? 2 : 1) * (sizeof(T) == 2 ? 2 : 8) <= 256 ? 2 : 1)
void attend_dq_kernel(Args p) {
  using M = Mma<T>;
  using Staged = Tile<T, ED, POS, 256>;
  constexpr int DB = (ED + 31) / 32;
  extern __shared__ char shared[];

  const Place place(p, p.tiles * p.splits);
  const int split = place.at / p.tiles, tile = place.at % p.tiles;
  const int nh = place.nh;
  const int n = nh / p.Hkv, hk = nh % p.Hkv;

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int first = (tile * 4 + wave) * 32;
  const int g = min(first / p.pad, p.G - 1);
  const int head = hk * p.G + g;
  const int i0 = first - g * p.pad;  // the wave's first query
  const int i = i0 + (lane & 31);
  const bool live = i < p.Lq;
  const int from = p.bias.query_start + i0;
  const int far = p.bias.max_distance;

  const int total = key_count(p, n);
  const int begin = split * p.per_split;
  const int end = min(total, begin + p.per_split);

  typename M::Op q[ED / M::kDepth], go[ED / M::kDepth];
  T* own = (T*)shared + wave * (Columns<T, ED>::kBytes / sizeof(T));
  own_columns<T, ED>(q, own, (const T*)p.q + n * p.qn + head * p.qh, p.qe,
                     p.E, i0, p.Lq);
  own_columns<T, ED>(go, own, (const T*)p.dout + n * p.dn + head * p.dh,
                     p.de, p.E, i0, p.Lq);
  const long rows = (long)p.N * p.H * p.Lq;
  const long stat = ((long)n * p.H + head) * p.Lq + i;
  // Where the bias has a gradient, the weights are 2^up times p, so that their
  // logarithms are near zero and not near log2 of the keys' number: a rounding
  // there is an error of each p that the last buckets sum up.
  const int up = FIND == DQ ? 0 : 31 - __clz(total | 1);
  const float down = __builtin_ldexpf(1.0f, -up);
  const float lse = live ? p.lse[stat] - up : INFINITY;
  float delta = 0.0f;
  float weight = 0.0f;  // what the weights sum to
  constexpr bool MEND = FIND == DQ && sizeof(T) == 2 && ED <= 32;
  const bool given = FIND == TABLE || (MEND && p.deltas != nullptr);
  const bool mend = MEND && !given;
  constexpr bool EVEN = FIND != DELTA && sizeof(T) == 2 && ED == 16;
  const bool few = FIND == DQ && !MEND && total <= 32;
  if (given && live) {
    for (int s = 0; s < p.splits; ++s) {
      const float* of = p.deltas + 2 * s * rows + stat;
      delta += of[0];
      weight += of[rows];
    }
    if (weight != 0.0f) delta /= weight;
    weight = 0.0f;
  }
  if (FIND == DQ && !given && !few) {
    typename M::Op o[ED / M::kDepth];
    own_columns<T, ED>(o, own,
                       (const T*)p.o + ((long)n * p.H + head) * p.E * p.Lq,
                       p.Lq, p.E, i0, p.Lq);
#pragma unroll
    for (int kk = 0; kk < ED / M::kDepth; ++kk)
#pragma unroll
      for (int j = 0; j < M::kDepth / 2; ++j)
        delta = fmaf(M::get(go[kk], j), M::get(o[kk], j), delta);
    delta = both_sum(delta);
  }
  __syncthreads();  // the tiles come where the columns were

  float* line = (float*)(shared + 4 * Staged::kBytes) +
                line_middle(far, false);
  float* lines = line + far + 1;  // the waves' ds by distance
  float* ends = lines + 4 * (2 * far + 1);
  float* diagonals = ends + 8 + wave * 32 * 33;
  float before = 0.0f, behind = 0.0f;      // bias past the last bucket
  float ds_before = 0.0f, ds_behind = 0.0f;
  float entry = 0.0f;
  if (LINED) {  // the workgroup's rows are one head's
    entry = entry_of_lane<T>(p.bias, head);
    spread_bias<T, false>(p.bias, head, line, tid, 256);
    before = bias_of<T>(p.bias, head, -far);
    behind = bias_of<T>(p.bias, head, far);
    if (FIND == TABLE)
      for (int d = tid; d < 4 * (2 * far + 1); d += 256) lines[d] = 0.0f;
  }
  float* sums = lines + wave * (2 * far + 1) + far;

  const Line bias_line(line, far);
  const bool holes = LINED && takes_out(entry);
  f32x16 acc[DB] = {};
  f32x16 mean = {};    // sum of p k
  float excess = 0.0f;  // sum of ds
  const float scale = p.scale * kLog2e;
  const T* kb = (const T*)p.k + n * p.kn + hk * p.kh;
  const T* vb = (const T*)p.v + n * p.vn + hk * p.vh;
  Staged ks, vs;
  ks.place(p.ke, p.E, tid);
  vs.place(p.ve, p.E, tid);
  if (p.E < ED)
    for (int b = 0; b < 4; ++b)
      Staged::blank((T*)(shared + b * Staged::kBytes), p.E, tid);

  if (begin < end) {
    ks.load(kb, begin, end, tid);
    vs.load(vb, begin, end, tid);
  }
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
    if (i0 >= p.Lq) continue;  // no query of this wave's
    // Up to 16 channels are half of a product's rows. Ones in the others make
    // the weights' sum of what they weigh, over both halves' keys, in all of
    // rows 16.. (element 8 and its like).
    auto keys_and_ones = [&](int col) {
      auto left = M::template second<Staged::kStride, ED>(kt, 0, col);
      if constexpr (EVEN) {
        if (lane & 16)
#pragma unroll
          for (int j = 0; j < 8; ++j) left.a[0][j] = left.a[1][j] = (__bf16)1.0f;
      }
      return left;
    };
#pragma unroll 1
    for (int col = 0; col < POS && at + col < end; col += 32) {
      const int key0 = at + col;
      int side = 2;
      float add = 0.0f;
      if (LINED) {
        side = beyond(p.bias, key0 * p.bias.key_step - (from + 31),
                      (key0 + 31) * p.bias.key_step - from);
        add = side > 0 ? behind : before;
        if (side != 0 && add == -INFINITY) continue;  // all pairs are out
      }
      f32x16 c = {}, dp = {};
#pragma unroll
      for (int kk = 0; kk < ED / M::kDepth; ++kk) {
        c = M::mul(M::template first<Staged::kStride>(kt, kk, col), q[kk],
                   c);
        dp = M::mul(M::template first<Staged::kStride>(vt, kk, col),
                    go[kk], dp);
      }
      // the lane's own part of a distance; the rest is the wave's
      const int d0 = (key0 + M::seq(0, h)) * p.bias.key_step - from -
                     (lane & 31);
      float ds[16];
      if (LINED && side == 0) {
        const int a0 = bias_line.at(d0);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          ds[j] = fmaf(c[j], scale,
                       bias_line.get(a0 + 4 * M::seq(j, 0) *
                                              p.bias.key_step)) -
                  lse;
        if (holes) {
          const int a1 = anew(a0);
          // a query that is not there is zeros, and NaN by such a key
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (!live || bias_line.get(a1 + 4 * M::seq(j, 0) *
                                                p.bias.key_step) == -INFINITY)
              ds[j] = -INFINITY;
        }
      } else {
        const float off = add - lse;
#pragma unroll
        for (int j = 0; j < 16; ++j) ds[j] = fmaf(c[j], scale, off);
      }
      if (key0 + 32 > end) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (key0 + M::seq(j, h) >= end) ds[j] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) ds[j] = __builtin_amdgcn_exp2f(ds[j]);
      if (mend || EVEN) {
        typename M::Right pr;
        M::right(pr, ds);
        mean = M::mul(keys_and_ones(col), pr, mean);
        if (!EVEN) {
#pragma unroll
          for (int j = 0; j < 16; ++j) weight += ds[j];
        }
      }
      if (FIND == DELTA) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          delta = fmaf(ds[j], dp[j], delta);
          weight += ds[j];
        }
        continue;
      }
      if (few) {
        float all = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          delta = fmaf(ds[j], dp[j], delta);
          all += ds[j];
        }
        all = both_sum(all);
        delta = both_sum(delta);
        if (all != 0.0f) delta /= all;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j)
        ds[j] *= FIND == DQ ? dp[j] - delta : fmaf(dp[j], down, -delta * down);
      if (FIND == TABLE && side == 0) {
        add_diagonals<T>(p.bias, ds, diagonals, sums,
                         key0 * p.bias.key_step - from, ds_before,
                         ds_behind);
      } else if (FIND == TABLE) {
        float all = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) all += ds[j];
        if (side > 0) ds_behind += all;
        else ds_before += all;
      }
      if (mend || EVEN) {
#pragma unroll
        for (int j = 0; j < 16; ++j) excess += ds[j];
      }
      typename M::Right pr;
      M::right(pr, ds);
#pragma unroll
      for (int d = 0; d < DB; ++d)
        acc[d] = M::mul(
            EVEN ? keys_and_ones(col)
                 : M::template second<Staged::kStride, ED>(kt, 32 * d, col),
            pr, acc[d]);
    }
  }
  if (mend || EVEN) {
    excess = both_sum(excess);
    weight = EVEN ? mean[8] : both_sum(weight);
    const float by = weight != 0.0f ? 1.0f / weight : 0.0f;
    float off = excess;
    if (EVEN) off = mend ? acc[0][8] : acc[0][8] - excess;
    if (mend) delta += excess * by;
    acc[0] -= mean * (off * by);
  }
  if (FIND == DELTA) {
    delta = both_sum(delta);
    weight = both_sum(weight);
    if (first < p.G * p.pad && live && h == 0) {
      float* to = p.deltas + 2 * split * rows + stat;
      to[0] = delta;
      to[rows] = weight;
    }
    return;
  }
  if (FIND == TABLE)  // a workgroup's rows are one head's, and there are some
    fold_table(p.bias, lines, ds_before, ds_behind, ends,
               p.dbias + (((long)(n * p.splits + split) * p.H + head) *
                              (p.pad / 128) + i0 / 128) * p.bias.buckets);
  __syncthreads();  // the results pass through where the tiles were
  if (first >= p.G * p.pad || i0 >= p.Lq) return;
  if (live && split == 0 && h == 0) p.delta[stat] = delta;
  const long to = ((long)n * p.H + head) * p.E * p.Lq + i0;
  if (p.splits > 1) {
    if (!live) return;
    float* out = p.part + (long)split * p.N * p.H * p.E * p.Lq + to +
                 (lane & 31);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int e = 32 * d + 8 * (j / 4) + 4 * h + j % 4;
        if (e < p.E) out[(long)e * p.Lq] = acc[d][j] * p.scale;
      }
    return;
  }
  put_columns<T, ED>(own, acc, p.scale, (T*)p.out + to, p.Lq, p.E,
                     p.Lq - i0);
}

// --- backward: dk, dv --------------------------------------------------------

// log2 p of SUBS blocks of 32 queries (rows, from position `from` on, `rows`
// of them there) for a wave's 32 keys: scores, bias and the queries'
// logarithms
template <typename T, int SUBS, bool LINED>
__device__ __forceinline__ void log_weights(const Args& p,
                                            f32x16 (&c)[SUBS],
                                            const float* lses,
                                            const float* line, float before,
                                            float behind, bool holes,
                                            int key0, int from, int rows) {
  using M = Mma<T>;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const float scale = p.scale * kLog2e;
  const int far = p.bias.max_distance, step = p.bias.key_step;
  int side = 2;
  float add = 0.0f;
  if (LINED) {
    side = beyond(p.bias, key0 * step - (from + 32 * SUBS - 1),
                  (key0 + 31) * step - from);
    add = side > 0 ? behind : before;
    if (side != 0 && add == -INFINITY) {  // all pairs are out
#pragma unroll
      for (int b = 0; b < SUBS; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) c[b][j] = -INFINITY;
      return;
    }
  }
#pragma unroll
  for (int b = 0; b < SUBS; ++b) {
    if (LINED && side == 0) {
      const int d0 =
          (key0 + (lane & 31)) * step - from - 32 * b - M::seq(0, h);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 l = *(const f32x4*)(lses + 32 * b + M::seq(4 * g, h));
#pragma unroll
        for (int j = 4 * g; j < 4 * g + 4; ++j) {
          const int d = d0 - M::seq(j, 0);
          c[b][j] = fmaf(c[b][j], scale,
                         line[line_at<true>(max(-far, min(d, far)))]) -
                    l[j & 3];
        }
      }
    } else {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 l = *(const f32x4*)(lses + 32 * b + M::seq(4 * g, h));
#pragma unroll
        for (int j = 4 * g; j < 4 * g + 4; ++j)
          c[b][j] =
              fmaf(c[b][j], scale, LINED ? add - l[j & 3] : -l[j & 3]);
      }
    }
  }
  if (LINED && side == 0 && holes) {
#pragma unroll
    for (int b = 0; b < SUBS; ++b) {
      const int d0 = anew((key0 + (lane & 31)) * step - from - 32 * b -
                          M::seq(0, h));
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int d = d0 - M::seq(j, 0);
        // a query that is not there is zeros, and NaN by such a key
        if (32 * b + M::seq(j, h) >= rows ||
            line[line_at<true>(max(-far, min(d, far)))] == -INFINITY)
          c[b][j] = -INFINITY;
      }
    }
  }
}

// What both kernels below do alike: a workgroup's 128 keys, 32 a wave, walk
// the queries of the heads that read them, so that the sum over shared heads
// is made in registers.
template <typename T, int ED, int POS, int NT, bool LINED>
struct Walk {
  using Staged = Tile<T, ED, POS, NT>;
  const Args& p;
  int nh, n, hk, split, tile, tid, wave, total, begin, end;
  char* shared;
  float *stats, *line;  // (2, 2, POS) lse and delta; bias by distance
  Staged qs, os;
  float lse, delta, before, behind;
  bool holes;  // the head's table takes pairs out
  int lined, buf;
  T *qt, *dt;
  float *lses, *deltas;

  __device__ __forceinline__ Walk(const Args& args, char* lds)
      : p(args), shared(lds) {
    const Place place(p, p.tiles * p.splits);
    split = place.at / p.tiles;
    tile = place.at % p.tiles;
    nh = place.nh;
    n = nh / p.Hkv;
    hk = nh % p.Hkv;
    tid = threadIdx.x;
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    total = key_count(p, n);
    begin = split * p.per_split;
    end = tile * 128 < total ? min(p.G * p.pad, begin + p.per_split) : 0;
    stats = (float*)(shared + 4 * Staged::kBytes);
    line = stats + 4 * POS + line_middle(p.bias.max_distance, true);
    lined = -1;
    buf = 0;
    before = behind = 0.0f;
    holes = false;
    qs.place(p.qe, p.E, tid);
    os.place(p.de, p.E, tid);
  }
  __device__ __forceinline__ void fetch(int row) {
    const int g = row / p.pad, i = row - g * p.pad, head = hk * p.G + g;
    qs.load((const T*)p.q + n * p.qn + head * p.qh, i, p.Lq, tid);
    os.load((const T*)p.dout + n * p.dn + head * p.dh, i, p.Lq, tid);
    lse = INFINITY;
    delta = 0.0f;
    if (tid < POS && i + tid < p.Lq) {
      const long at = ((long)n * p.H + head) * p.Lq + i + tid;
      lse = p.lse[at];
      delta = p.delta[at];
    }
  }
  __device__ __forceinline__ void start() {
    if (p.E < ED)
      for (int b = 0; b < 4; ++b)
        Staged::blank((T*)(shared + b * Staged::kBytes), p.E, tid);
    fetch(begin);
  }
  // puts down the queries row.. and starts on the next ones
  __device__ __forceinline__ void next(int row) {
    qt = (T*)(shared + 2 * buf * Staged::kBytes);
    dt = (T*)(shared + (2 * buf + 1) * Staged::kBytes);
    lses = stats + 2 * buf * POS;
    deltas = lses + POS;
    buf ^= 1;
    qs.store(qt, p.E, tid);
    os.store(dt, p.E, tid);
    if (tid < POS) {
      lses[tid] = lse;
      deltas[tid] = delta;
    }
    if (LINED) {
      const int g = row / p.pad;
      if (g != lined) {  // the next head's
        __syncthreads();
        const float entry = entry_of_lane<T>(p.bias, hk * p.G + g);
        spread_bias<T, true>(p.bias, hk * p.G + g, line, tid, NT);
        before = bias_of<T>(p.bias, hk * p.G + g, -p.bias.max_distance);
        behind = bias_of<T>(p.bias, hk * p.G + g, p.bias.max_distance);
        holes = takes_out(entry);
        lined = g;
      }
    }
    __syncthreads();
    if (row + POS < end) fetch(row + POS);
  }
  // A wave's columns of dk or dv, by way of its own part of the LDS: all
  // waves have to be past the tiles.
  template <int DB>
  __device__ __forceinline__ void store(f32x16 (&acc)[DB], T* out, int half,
                                        int key0, float by) const {
    if (key0 >= p.Lk) return;
    const int lane = tid & 63, h = lane >> 5, key = key0 + (lane & 31);
    // a key that does not count has gone through with k = v = 0: its column
    // holds numbers of no meaning
    if (key >= total) {
#pragma unroll
      for (int d = 0; d < DB; ++d) acc[d] = f32x16{};
    }
    const long to = (long)nh * p.E * p.Lk;
    if (p.splits == 1) {
      put_columns<T, ED>(
          (T*)shared + wave * (Columns<T, ED>::kBytes / sizeof(T)), acc, by,
          out + to + key0, p.Lk, p.E, p.Lk - key0);
      return;
    }
    if (key >= p.Lk) return;
    float* part = p.part + ((long)half * p.splits + split) * p.N * p.Hkv *
                               p.E * p.Lk + to + key;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int e = 32 * d + 8 * (j / 4) + 4 * h + j % 4;
        if (e < p.E) part[(long)e * p.Lk] = acc[d][j] * by;
      }
  }
};

// Heads of up to 64 bf16 or 32 fp32 channels: a wave makes both gradients of
// its keys, whose sums are at most 64 registers each. 256 heads of 32, 1024
// queries to lengths up to 1024: 89 us, of which the exponentials fill 13 and
// the products, at a large one's rate, 28. The lengths are another part: each
// die has 137 workgroups with keys for 64 places, three rounds for 2.1.
template <typename T, int ED, int POS, bool LINED>
__global__ __launch_bounds__(256, 2) void attend_dkv_kernel(Args p) {
  using M = Mma<T>;
  using W = Walk<T, ED, POS, 256, LINED>;
  constexpr int STRIDE = W::Staged::kStride;
  constexpr int DB = (ED + 31) / 32;
  constexpr int STEP = POS < 64 ? POS : 64;
  constexpr int SUBS = STEP / 32;
  extern __shared__ char shared[];
  W w(p, shared);
  const int h = (threadIdx.x & 63) >> 5;
  const int key0 = (w.tile * 4 + w.wave) * 32;

  typename M::Op k[ED / M::kDepth], v[ED / M::kDepth];
  f32x16 dk[DB] = {}, dv[DB] = {};
  if (w.begin < w.end) {
    T* own = (T*)shared + w.wave * (Columns<T, ED>::kBytes / sizeof(T));
    own_columns<T, ED>(k, own, (const T*)p.k + w.n * p.kn + w.hk * p.kh,
                       p.ke, p.E, key0, w.total);
    own_columns<T, ED>(v, own, (const T*)p.v + w.n * p.vn + w.hk * p.vh,
                       p.ve, p.E, key0, w.total);
    __syncthreads();
    w.start();
  }
  for (int row = w.begin; row < w.end; row += POS) {
    w.next(row);
    if (key0 >= w.total) continue;  // no key of this wave's
    const int i0 = row % p.pad;
#pragma unroll 1
    for (int col = 0; col < POS && i0 + col < p.Lq; col += STEP) {
      f32x16 c[SUBS] = {}, dp[SUBS] = {};
#pragma unroll
      for (int b = 0; b < SUBS; ++b)
#pragma unroll
        for (int kk = 0; kk < ED / M::kDepth; ++kk) {
          c[b] = M::mul(M::template first<STRIDE>(w.qt, kk, col + 32 * b),
                        k[kk], c[b]);
          dp[b] = M::mul(M::template first<STRIDE>(w.dt, kk, col + 32 * b),
                         v[kk], dp[b]);
        }
      log_weights<T, SUBS, LINED>(p, c, w.lses + col, w.line, w.before,
                                  w.behind, w.holes, key0,
                                  p.bias.query_start + i0 + col,
                                  p.Lq - i0 - col);
#pragma unroll
      for (int b = 0; b < SUBS; ++b) {
        float e[16], ds[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 dl =
              *(const f32x4*)(w.deltas + col + 32 * b + M::seq(4 * g, h));
#pragma unroll
          for (int j = 4 * g; j < 4 * g + 4; ++j) {
            e[j] = __builtin_amdgcn_exp2f(c[b][j]);
            ds[j] = e[j] * (dp[b][j] - dl[j & 3]);
          }
        }
        typename M::Right pr, dr;
        M::right(pr, e);
        M::right(dr, ds);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          dv[d] = M::mul(
              M::template second<STRIDE, ED>(w.dt, 32 * d, col + 32 * b), pr,
              dv[d]);
          dk[d] = M::mul(
              M::template second<STRIDE, ED>(w.qt, 32 * d, col + 32 * b), dr,
              dk[d]);
        }
      }
    }
  }
  __syncthreads();
  w.template store<DB>(dk, (T*)p.dk, 0, key0, p.scale);
  w.template store<DB>(dv, (T*)p.dv, 1, key0, 1.0f);
}

// For deep heads a wave's k, v, dk and dv alone are 192 registers, and a SIMD
// would hold one wave, with nothing to run beside its waits. So two waves
// share 32 keys: one has k and makes p and dv, the other has v and makes dp,
// ds and dk. p goes from the one to the other through LDS in fp32, each lane
// to its like, and the one's exponentials run beside the other's products.
// 4096 x 4096, 64 heads of 128 on 16: 1440 us, 763 TFLOP/s, and 2129 with one
// wave for all; the matrix units are busy for 29% of it, half of a wave's
// time are waits, for the staged tile and the hand-over. Three tiles in
// flight of half the positions took 1731.
template <typename T, int ED, int POS, bool LINED>
__global__ __launch_bounds__(512, 2) void attend_dkv_pair_kernel(Args p) {
  using M = Mma<T>;
  using W = Walk<T, ED, POS, 512, LINED>;
  constexpr int STRIDE = W::Staged::kStride;
  constexpr int DB = (ED + 31) / 32;
  constexpr int SUBS = POS / 32;
  static_assert(POS <= 64, "one step a tile");
  extern __shared__ char shared[];
  W w(p, shared);
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const bool second = w.wave >= 4;  // the wave with v
  const int pair = w.wave & 3;
  const int key0 = (w.tile * 4 + pair) * 32;
  // (4 pairs, SUBS, 4, 64 lanes) of 4 floats
  f32x4* hand = (f32x4*)(shared + 4 * W::Staged::kBytes + 16 * POS +
                         (LINED ? (line_floats(p.bias.max_distance, true) + 3)
                                          / 4 * 16
                                : 0)) +
                pair * SUBS * 256 + lane;

  typename M::Op own[ED / M::kDepth];
  f32x16 acc[DB] = {};
  if (w.begin < w.end) {
    const T* base = second ? (const T*)p.v + w.n * p.vn + w.hk * p.vh
                           : (const T*)p.k + w.n * p.kn + w.hk * p.kh;
    own_columns<T, ED>(
        own, (T*)shared + w.wave * (Columns<T, ED>::kBytes / sizeof(T)),
        base, second ? p.ve : p.ke, p.E, key0, w.total);
    __syncthreads();
    w.start();
  }
  for (int row = w.begin; row < w.end; row += POS) {
    w.next(row);
    const int i0 = row % p.pad;
    const bool busy = key0 < w.total;
    f32x16 c[SUBS] = {};
    if (busy) {
      const T* tile = second ? w.dt : w.qt;
#pragma unroll
      for (int b = 0; b < SUBS; ++b)
#pragma unroll
        for (int kk = 0; kk < ED / M::kDepth; ++kk)
          c[b] = M::mul(M::template first<STRIDE>(tile, kk, 32 * b), own[kk],
                        c[b]);
      if (!second) {
        log_weights<T, SUBS, LINED>(p, c, w.lses, w.line, w.before, w.behind,
                                    w.holes, key0, p.bias.query_start + i0,
                                    p.Lq - i0);
#pragma unroll
        for (int b = 0; b < SUBS; ++b)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            f32x4 e;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              c[b][4 * g + j] = e[j] =
                  __builtin_amdgcn_exp2f(c[b][4 * g + j]);
            hand[(b * 4 + g) * 64] = e;
          }
      }
    }
    __syncthreads();
    if (!busy) continue;
    const T* tile = second ? w.qt : w.dt;
#pragma unroll
    for (int b = 0; b < SUBS; ++b) {
      float s[16];
      if (second) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 e = hand[(b * 4 + g) * 64];
          const f32x4 dl =
              *(const f32x4*)(w.deltas + 32 * b + M::seq(4 * g, h));
#pragma unroll
          for (int j = 0; j < 4; ++j)
            s[4 * g + j] = e[j] * (c[b][4 * g + j] - dl[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = c[b][j];
      }
      typename M::Right r;
      M::right(r, s);
#pragma unroll
      for (int d = 0; d < DB; ++d)
        acc[d] = M::mul(M::template second<STRIDE, ED>(tile, 32 * d, 32 * b),
                        r, acc[d]);
    }
  }
  __syncthreads();
  w.template store<DB>(acc, second ? (T*)p.dk : (T*)p.dv, second ? 0 : 1,
                       key0, second ? p.scale : 1.0f);
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
  const int rows = N * tiles;
  const int each = (rows + gridDim.y - 1) / gridDim.y;
  const int begin = blockIdx.y * each, end = min(rows, begin + each);
  float v = 0.0f;
  // 8 rows at a time, so that their loads are on the way together
  for (int r0 = begin + lane; r0 < end && b < buckets; r0 += 32) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = min(r0 + 4 * i, end - 1), n = r / tiles;
      w[i] = in[(((long)n * H + blockIdx.x) * tiles + r - n * tiles) *
                    buckets + b];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v += r0 + 4 * i < end ? w[i] : 0.0f;
  }
  sums[lane][b] = v;
  __syncthreads();
  if (lane == 0 && b < buckets)
    out[((long)blockIdx.x * gridDim.y + blockIdx.y) * buckets + b] =
        (T)((sums[0][b] + sums[1][b]) + (sums[2][b] + sums[3][b]));
}

std::vector<at::Tensor> backward(const Call& c, const at::Tensor& out,
                                 const at::Tensor& lse,
                                 const at::Tensor& dout, bool kv,
                                 bool table) {
  Args p = args_of(c);
  const c10::DeviceGuard guard(c.q.device());
  const auto f32 = c.q.options().dtype(at::kFloat);
  auto dq = at::empty(c.q.sizes(), c.q.options());
  at::Tensor dk, dv, dt;
  if (kv) {
    dk = at::empty(c.k.sizes(), c.q.options());
    dv = at::empty(c.k.sizes(), c.q.options());
  }
  if (table) dt = at::empty(c.table.sizes(), c.q.options());
  if (c.q.numel() == 0 || c.k.numel() == 0) {
    for (auto* t : {&dq, &dk, &dv, &dt})
      if (t->defined()) t->zero_();
    return {dq, dk, dv, dt};
  }
  const auto stream = at::hip::getCurrentHIPStream().stream();
  auto delta = at::empty({p.N, p.H, p.Lq}, f32);
  p.o = sa::memory_of(out);
  p.lse = sa::memory_of<float>(lse);
  p.delta = sa::memory_of<float>(delta);
  p.dout = sa::memory_of(dout);
  p.dn = dout.stride(0), p.dh = dout.stride(1), p.de = dout.stride(2);
  const long pairs = (long)p.N * p.Hkv;

  p.out = sa::memory_of(dq);
  // with a bias, a workgroup's rows are one head's
  p.pad = round_up(p.Lq, p.bias.table ? 128 : 32);
  p.tiles = sa::ceil_div((long)p.G * p.pad, 128);
  p.splits = cut(pairs * p.tiles, p.Lk, 128, &p.per_split);
  const bool walked = table || (c.q.scalar_type() == at::kBFloat16 &&
                                p.E <= 32 && p.splits > 1);
  at::Tensor part, sums, deltas;
  if (p.splits > 1) {
    part = at::empty({p.splits, c.q.numel()}, f32);
    p.part = sa::memory_of<float>(part);
  }
  if (walked) {
    deltas = at::empty({p.splits, 2, p.N, p.H, p.Lq}, f32);
    p.deltas = sa::memory_of<float>(deltas);
  }
  if (table) {
    sums = at::empty({p.N * p.splits, p.H, p.pad / 128, p.bias.buckets}, f32);
    p.dbias = sa::memory_of<float>(sums);
  }
  const size_t line = (2 * p.bias.max_distance + 1) * 4;
  with_type(c.q.scalar_type(), [&](auto zero) {
    using T = decltype(zero);
    with_depth(p.E, [&](auto depth) {
      constexpr int ED = decltype(depth)::value;
      constexpr int POS = tile_positions<T, ED>();
      const long blocks = pairs * p.splits * p.tiles;
      if (walked && p.bias.table) {
        launch(attend_dq_kernel<T, ED, POS, true, DELTA>, blocks, 256,
               backward_lds<T, ED>(line), p, stream);
      } else if (walked) {
        if constexpr (sizeof(T) == 2 && ED <= 32)
          launch(attend_dq_kernel<T, ED, POS, false, DELTA>, blocks, 256,
                 backward_lds<T, ED>(0), p, stream);
      }
      if (table) {
        launch(attend_dq_kernel<T, ED, POS, true, TABLE>, blocks, 256,
               backward_lds<T, ED>(5 * line + 32 + 4 * 32 * 33 * 4), p,
               stream);
      } else if (p.bias.table) {
        launch(attend_dq_kernel<T, ED, POS, true, DQ>, blocks, 256,
               backward_lds<T, ED>(line), p, stream);
      } else {
        launch(attend_dq_kernel<T, ED, POS, false, DQ>, blocks, 256,
               backward_lds<T, ED>(0), p, stream);
      }
    });
    if (p.splits > 1) {
      sum_splits_kernel<T><<<sa::ceil_div(c.q.numel(), 256), 256, 0, stream>>>(
          p.part, sa::memory_of<T>(dq), c.q.numel(), p.splits);
      SA_CHECK_HIP(hipGetLastError());
    }
    if (table) {
      const int of = p.N * p.splits, tiles = p.pad / 128;
      const int pieces =
          (int)std::min<long>(((long)of * tiles + 511) / 512, 256);
      const dim3 grid(p.H, pieces);
      if (pieces == 1) {
        sum_table_kernel<T><<<grid, 256, 0, stream>>>(
            p.dbias, sa::memory_of<T>(dt), of, p.H, tiles, p.bias.buckets);
      } else {
        auto some = at::empty({p.H, pieces, p.bias.buckets}, f32);
        sum_table_kernel<float><<<grid, 256, 0, stream>>>(
            p.dbias, sa::memory_of<float>(some), of, p.H, tiles,
            p.bias.buckets);
        sum_table_kernel<T><<<dim3(p.H, 1), 256, 0, stream>>>(
            sa::memory_of<float>(some), sa::memory_of<T>(dt), 1, p.H, pieces,
            p.bias.buckets);
      }
      SA_CHECK_HIP(hipGetLastError());
    }
  });
  if (!kv) return {dq, dk, dv, dt};

  p.dk = sa::memory_of(dk);
  p.dv = sa::memory_of(dv);
  p.tiles = sa::ceil_div(p.Lk, 128);
  with_type(c.q.scalar_type(), [&](auto zero) {
    using T = decltype(zero);
    with_depth(p.E, [&](auto depth) {
      constexpr int ED = decltype(depth)::value;
      constexpr int POS = tile_positions<T, ED>();
      p.pad = round_up(p.Lq, POS);
      p.splits = cut(pairs * p.tiles, (long)p.G * p.pad, POS, &p.per_split);
      if (p.splits > 1) {
        part = at::empty({2, p.splits, c.k.numel()}, f32);
        p.part = sa::memory_of<float>(part);
      }
      const long blocks = pairs * p.splits * p.tiles;
      const size_t lines =
          p.bias.table ? line_floats(p.bias.max_distance, true) : 0;
      if constexpr (ED * sizeof(T) > 128) {
        const size_t lds = deep_lds<T, ED>(lines);
        if (p.bias.table)
          launch(attend_dkv_pair_kernel<T, ED, POS, true>, blocks, 512, lds,
                 p, stream);
        else
          launch(attend_dkv_pair_kernel<T, ED, POS, false>, blocks, 512, lds,
                 p, stream);
      } else {
        const size_t lds = backward_lds<T, ED>(16 * POS + 4 * lines);
        if (p.bias.table)
          launch(attend_dkv_kernel<T, ED, POS, true>, blocks, 256, lds, p,
                 stream);
        else
          launch(attend_dkv_kernel<T, ED, POS, false>, blocks, 256, lds, p,
                 stream);
      }
    });
    if (p.splits > 1) {
      const int grid = sa::ceil_div(c.k.numel(), 256);
      sum_splits_kernel<T><<<grid, 256, 0, stream>>>(
          p.part, sa::memory_of<T>(dk), c.k.numel(), p.splits);
      sum_splits_kernel<T><<<grid, 256, 0, stream>>>(
          p.part + p.splits * c.k.numel(), sa::memory_of<T>(dv), c.k.numel(),
          p.splits);
      SA_CHECK_HIP(hipGetLastError());
    }
  });
  return {dq, dk, dv, dt};
}

}  // namespace attend
