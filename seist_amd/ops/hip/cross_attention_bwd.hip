// Backward kernels of the attention in cross_attention.hip, which has the
// formulas.

#include "cross_attention.h"

namespace attend {

__device__ __forceinline__ int clamped(int d, int most) {
  return max(-most, min(d, most)) + most;
}

// --- backward: dq, delta, dtable -------------------------------------------

// LDS of a workgroup: two staged tiles and what stands behind them, where
// the four waves' own columns pass through beforehand
template <typename T, int ED>
size_t backward_lds(size_t behind) {
  const size_t staged =
      2 * Tile<T, ED, tile_positions<T, ED>(), 256>::kBytes + behind;
  return std::max<size_t>(staged, 4 * Columns<T, ED>::kBytes);
}

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
__global__ __launch_bounds__(
    NW * 64, ED * (TABLE ? 2 : 1) * (sizeof(T) == 2 ? 2 : 8) <= 256 ? 2 : 1)
void attend_dq_kernel(Args p) {
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

  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
  typename M::Op q[ED / M::kDepth], go[ED / M::kDepth];
  const int i0 = __builtin_amdgcn_readfirstlane(i);
  const int head0 = __builtin_amdgcn_readfirstlane(head);
  T* own = (T*)shared + wave * (Columns<T, ED>::kBytes / sizeof(T));
  own_columns<T, ED>(q, own, (const T*)p.q + n * p.qn + head0 * p.qh, p.qe,
                     p.E, i0, p.Lq);
  own_columns<T, ED>(go, own, (const T*)p.dout + n * p.dn + head0 * p.dh,
                     p.de, p.E, i0, p.Lq);
  const long stat = ((long)n * p.H + head) * p.Lq + i;
  const float lse = live ? p.lse[stat] : INFINITY;
  float delta = 0.0f;
  if (!TWICE) {
    typename M::Op o[ED / M::kDepth];
    own_columns<T, ED>(o, own,
                       (const T*)p.o + ((long)n * p.H + head0) * p.E * p.Lq,
                       p.Lq, p.E, i0, p.Lq);
#pragma unroll
    for (int kk = 0; kk < ED / M::kDepth; ++kk)
#pragma unroll
      for (int j = 0; j < M::kDepth / 2; ++j)
        delta = fmaf(M::get(go[kk], j), M::get(o[kk], j), delta);
    delta = both_sum(delta);
  }
  __syncthreads();
  if (LINED) {
    line = (float*)(shared + 2 * Staged::kBytes) + wave * (TABLE ? 3 : 1) * wide;
    spread_bias<T>(p.bias, __builtin_amdgcn_readfirstlane(head), line, lane,
                   64);
    if (TABLE) {
      for (int d = lane; d < 2 * wide; d += 64) line[wide + d] = 0.0f;
      sums = line + (1 + h) * wide;
    }
  }

  f32x16 acc[DB] = {};
  const float scale = p.scale * kLog2e;
  const T* kb = (const T*)p.k + n * p.kn + hk * p.kh;
  const T* vb = (const T*)p.v + n * p.vn + hk * p.vh;

#pragma unroll 1
  for (int walk = TWICE ? 0 : 1; walk < 2; ++walk) {
    Staged ks, vs;
    ks.place(p.ke, p.E, threadIdx.x);
    vs.place(p.ve, p.E, threadIdx.x);
    if (begin < end) {
      Staged::blank(kt, p.E, threadIdx.x);
      Staged::blank(vt, p.E, threadIdx.x);
      ks.load(kb, begin, end, threadIdx.x);
      vs.load(vb, begin, end, threadIdx.x);
    }
    for (int at = begin; at < end; at += POS) {
      __syncthreads();
      ks.store(kt, p.E, threadIdx.x);
      vs.store(vt, p.E, threadIdx.x);
      __syncthreads();
      if (at + POS < end) {
        ks.load(kb, at + POS, end, threadIdx.x);
        vs.load(vb, at + POS, end, threadIdx.x);
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
          acc[d] = M::mul(M::template second<Staged::kStride, ED>(kt, 32 * d, 32 * b),
                       pr, acc[d]);
      }
    }
    if (TWICE && walk == 0) delta = both_sum(delta);
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
__global__ __launch_bounds__(NW * 64, ED * sizeof(T) <= 128 ? 2 : 1) void
attend_dkv_kernel(Args p) {
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

  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int key = (tile * NW + wave) * 32 + (lane & 31);
  const int total = key_count(p, n);
  const bool live = key < total;

  const int all = p.G * p.pad;
  const int begin = split * p.per_split;
  const int end = tile * NW * 32 < total ? min(all, begin + p.per_split) : 0;

  typename M::Op k[ED / M::kDepth], v[ED / M::kDepth];
  const int key0 = (tile * NW + wave) * 32;
  if (begin < end) {
    T* own = (T*)shared + wave * (Columns<T, ED>::kBytes / sizeof(T));
    own_columns<T, ED>(k, own, (const T*)p.k + n * p.kn + hk * p.kh, p.ke,
                       p.E, key0, total);
    own_columns<T, ED>(v, own, (const T*)p.v + n * p.vn + hk * p.vh, p.ve,
                       p.E, key0, total);
    __syncthreads();
  }

  f32x16 dk[DB] = {}, dv[DB] = {};
  const float scale = p.scale * kLog2e;
  Staged qs, os;
  qs.place(p.qe, p.E, threadIdx.x);
  os.place(p.de, p.E, threadIdx.x);
  float lse = INFINITY, delta = 0.0f;
  auto fetch = [&](int row) {
    const int g = row / p.pad, i = row - g * p.pad, head = hk * p.G + g;
    qs.load((const T*)p.q + n * p.qn + head * p.qh, i, p.Lq, threadIdx.x);
    os.load((const T*)p.dout + n * p.dn + head * p.dh, i, p.Lq, threadIdx.x);
    lse = INFINITY;
    delta = 0.0f;
    if (threadIdx.x < POS && i + (int)threadIdx.x < p.Lq) {
      const long at = ((long)n * p.H + head) * p.Lq + i + threadIdx.x;
      lse = p.lse[at];
      delta = p.delta[at];
    }
  };
  if (begin < end) {
    fetch(begin);
    Staged::blank(qt, p.E, threadIdx.x);
    Staged::blank(dt, p.E, threadIdx.x);
  }
  int lined = -1;
  for (int row = begin; row < end; row += POS) {
    const int g = row / p.pad, i = row - g * p.pad;
    __syncthreads();
    qs.store(qt, p.E, threadIdx.x);
    os.store(dt, p.E, threadIdx.x);
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
        dv[d] = M::mul(M::template second<Staged::kStride, ED>(dt, 32 * d, 32 * b),
                       pr, dv[d]);
        dk[d] = M::mul(M::template second<Staged::kStride, ED>(qt, 32 * d, 32 * b),
                       dr, dk[d]);
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

}  // namespace attend

using namespace attend;

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
                  dout.stride(2) >= 0 &&
                  (dout.stride(2) * (p.E - 1) + p.Lq) *
                          (long)q.element_size() < (1L << 32) &&
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
      const long blocks = pairs * p.splits * p.tiles;
      if (dtable)
        launch(attend_dq_kernel<T, ED, 4, POS, true, true>, blocks, 256,
               backward_lds<T, ED>(12 * line), p, stream);
      else if (p.bias.table)
        launch(attend_dq_kernel<T, ED, 4, POS, true, false>, blocks, 256,
               backward_lds<T, ED>(4 * line), p, stream);
      else
        launch(attend_dq_kernel<T, ED, 4, POS, false, false>, blocks, 256,
               backward_lds<T, ED>(0), p, stream);
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
      const long blocks = pairs * p.splits * p.tiles;
      if (p.bias.table)
        launch(attend_dkv_kernel<T, ED, 4, POS, true>, blocks, 256,
               backward_lds<T, ED>(8 * POS + line), p, stream);
      else
        launch(attend_dkv_kernel<T, ED, 4, POS, false>, blocks, 256,
               backward_lds<T, ED>(8 * POS), p, stream);
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
