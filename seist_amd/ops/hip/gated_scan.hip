// Gated linear recurrence over the last axis of (N, C, L):
//
//   a_t = sigmoid(gate_t),  h_t = a_t * h_{t-1} + (1 - a_t) * x_t
//
// A step is the map h -> A*h + B, and maps compose:
// (A2, B2) after (A1, B1) is (A2*A1, A2*B1 + B2). A lane composes 8
// neighbouring samples (4 in fp32) in registers, a row's lanes join their
// maps with log2 exchanges, waves join theirs through LDS, and the state
// carries from chunk to chunk, so a sample is read once and written once:
// memory bounds it. The gradient runs the other way: with u_t = a_t * G_t, G_t = dh_t + u_{t+1},
//
//   dx_t = (1-a_t)*G_t,  dgate_t = G_t*(h_{t-1}-x_t)*a_t*(1-a_t),
//
// which is the same kind of map in u. The backward pass needs h_{t-1} in
// full precision: it composes it again from x and gate (which it reads
// anyway) and the fp32 state that the forward pass left at each chunk's
// start, and never reads h.
//
// Everything between the loads and the stores is fp32; h, dx and dgate are
// rounded once, at the store. States are fp32 throughout.
//
// Few long rows do not fill the card: their chunks are then dealt to
// segments. A first kernel composes each segment's map, the second starts
// every segment from the maps before it. That reads the inputs of the map
// twice, so it is used only where the rows alone give too few waves.
//
// Measured: (100, 64, 8192) bf16 67 us (4.7 TB/s) and 97 us backward (5.4
// TB/s; a large copy reaches 5.2); one record of (24, 1000003) fp32 38 + 49
// us in two kernels (288 MB), 37 + 91 backward (480 MB). One sample of 64 x
// 96 states, a launch and no more, 3.7 us.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "sa_common.h"
#include "sa_tensor.h"

namespace gated_scan {
namespace {

// samples a lane holds: 16 bytes, so that a wave reads 1 KB in one piece
template <typename T>
constexpr int kItems = 16 / sizeof(T);

struct ScanArgs {
  const void* x;
  const void* gate;
  const void* dh;          // backward, may be null
  const float* state;      // (R) entering the first sample, may be null
  const float* dstate;     // (R) gradient of the last state, may be null
  const int* lengths;      // (N) or null
  float* marks;            // (R, chunks) state entering each chunk
  const float* maps;       // (R, segments, 2)
  float* maps_out;
  void* out;               // h, or dx
  void* out2;              // dgate
  float* last;             // (R) state after the last sample, or d(state)
  long xn, xc, gn, gc;     // strides of x and gate, in elements
  long rows;
  int C, L, chunks, segments, per_segment;
};

struct Map {
  float a, b;
};

__device__ __forceinline__ Map after(Map second, Map first) {
  return {second.a * first.a, fmaf(second.a, first.b, second.b)};
}

// sigmoid(g) and 1 - sigmoid(g), both to a few ulp: exp2's argument is
// rounded, so what the rounding left of g*log2(e) is put back to first order
__device__ __forceinline__ void gates(float g, float& a, float& keep) {
  const float kHi = 1.44269502162933349609375f;
  const float kLo = 1.92596299112661746887e-8f;
  const float m = -fabsf(g);
  const float hi = m * kHi;
  const float lo = fmaf(m, kLo, fmaf(m, kHi, -hi));
  float e = __builtin_amdgcn_exp2f(hi);
  if (e > 0.0f) e = fmaf(e, lo * 0.693147180559945f, e);
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  const float s = e * r;
  a = g < 0.0f ? s : r;
  keep = g < 0.0f ? r : s;
}

// a lane's samples of scan index s0.., in the words that they fill in
// memory, so that a load is not waited for before its samples are used; rows
// start anywhere, so the 16-byte accesses are not aligned. Rows of 16 bytes at
// most (SHORT), a lane each, go by samples. In others a lane that passes the
// row's end reads the last 16 bytes before it, which settle() moves to their
// places when they are used, and the one lane that the end falls into writes
// by samples. 52 million samples in bf16 in rows of 8192, 6000, 1500, 300 and
// 100 take 67, 69, 93, 122 and 102 us (98, 99, 142, 184 and 141 backward);
// with a row's last chunk by samples, 67, 84, 170, 166 and 174 (97, 139, 285,
// 282 and 285).
template <typename T>
struct Items {
  static constexpr int kEach = 4 / sizeof(T);  // samples of a word
  unsigned w[kItems<T> / kEach];
  template <bool REV, bool SHORT>
  __device__ __forceinline__ void load(const T* row, int s0, int L) {
    if (!SHORT || L == kItems<T>) {
      __builtin_memcpy(
          w, row + (REV ? max(L - kItems<T> - s0, 0) : min(s0, L - kItems<T>)),
          sizeof(w));
    } else {
#pragma unroll
      for (int k = 0; k < kItems<T>; ++k) {  // as they come in memory
        const int s = min(s0 + (REV ? kItems<T> - 1 - k : k), L - 1);
        unsigned v = 0;
        __builtin_memcpy(&v, row + (REV ? L - 1 - s : s), sizeof(T));
        if (k % kEach == 0) w[k / kEach] = v;
        else w[k / kEach] |= v << 16;
      }
    }
  }
  // in steps of 2 words, 1 word, half a word; what has no sample is any
  template <bool REV>
  __device__ __forceinline__ void settle(int s0, int L) {
    const int over = max(s0 + kItems<T> - L, 0);
    const bool two = over & (2 * kEach), one = over & kEach;
    const bool half = kEach == 2 && (over & 1);
    unsigned v[5];  // in scan order; values, as a choice of places is an address
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = w[REV ? 3 - k : k];
    v[4] = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const unsigned here = v[k], there = v[k + 2];
      v[k] = two ? there : here;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const unsigned here = v[k], there = v[k + 1];
      v[k] = one ? there : here;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const unsigned here = v[k], next = v[k + 1];
      const unsigned moved =
          REV ? here << 16 | next >> 16 : here >> 16 | next << 16;
      w[REV ? 3 - k : k] = half ? moved : here;
    }
  }
  template <bool REV>
  __device__ __forceinline__ float at(int i) const {
    const int k = REV ? kItems<T> - 1 - i : i;
    const unsigned v = w[k / kEach];
    if (kEach == 1) return __uint_as_float(v);
    return __uint_as_float(k % kEach == 0 ? v << 16 : v & 0xffff0000u);
  }
  template <bool REV>
  __device__ __forceinline__ void set(const float (&x)[kItems<T>]) {
    T v[kItems<T>];
#pragma unroll
    for (int k = 0; k < kItems<T>; ++k) v[k] = (T)x[REV ? kItems<T> - 1 - k : k];
    __builtin_memcpy(w, v, sizeof(w));
  }
  template <bool REV>
  __device__ __forceinline__ void store(T* row, int s0, int L,
                                        bool whole) const {
    if (whole || s0 + kItems<T> <= L) {
      __builtin_memcpy(row + (REV ? L - kItems<T> - s0 : s0), w, sizeof(w));
    } else {
#pragma unroll
      for (int k = 0; k < kItems<T>; ++k) {
        const int s = s0 + (REV ? kItems<T> - 1 - k : k);
        const unsigned v = w[k / kEach] >> (k % kEach * 16);
        if (s < L)
          __builtin_memcpy(row + (REV ? L - 1 - s : s), &v, sizeof(T));
      }
    }
  }
};

// one step of a scan over a wave's lanes: composes with the map CTRL away
template <int CTRL, int ROWS>
__device__ __forceinline__ Map dpp_after(Map m) {
  const Map o = {
      __int_as_float(__builtin_amdgcn_update_dpp(
          __float_as_int(1.0f), __float_as_int(m.a), CTRL, ROWS, 0xf, false)),
      __int_as_float(__builtin_amdgcn_update_dpp(
          0, __float_as_int(m.b), CTRL, ROWS, 0xf, false))};
  return after(m, o);
}

// each lane's map after those of the lanes below it, over 16 lanes or 64:
// shifts by 1, 2, 4, 8 within 16 lanes, then the last of 16 lanes to the
// next 16, then the last of 32 to the upper half
template <int LANES>
__device__ __forceinline__ Map scan_lanes(Map m) {
  m = dpp_after<0x111, 0xf>(m);
  m = dpp_after<0x112, 0xf>(m);
  m = dpp_after<0x114, 0xf>(m);
  m = dpp_after<0x118, 0xf>(m);
  if (LANES == 64) {
    m = dpp_after<0x142, 0xa>(m);
    m = dpp_after<0x143, 0xc>(m);
  }
  return m;
}

__device__ __forceinline__ Map of_lane(Map m, int lane) {
  return {__int_as_float(
              __builtin_amdgcn_readlane(__float_as_int(m.a), lane)),
          __int_as_float(
              __builtin_amdgcn_readlane(__float_as_int(m.b), lane))};
}

// What stands before (UP) or behind (!UP) each lane of its row's lanes, and
// the whole, all in scan order. A row has LPR lanes of one wave and W waves.
struct Joined {
  Map before, whole;
};

template <int LPR, int W, bool UP>
__device__ __forceinline__ Joined join(Map m, Map* lds) {
  Joined j;
  if constexpr (LPR == 64) {
    const int lane = threadIdx.x & 63;
    if (!UP) m = {__shfl(m.a, 63 - lane), __shfl(m.b, 63 - lane)};
    m = scan_lanes<64>(m);
    j.whole = of_lane(m, 63);
    j.before = {__shfl_up(m.a, 1), __shfl_up(m.b, 1)};
    if (lane == 0) j.before = {1.0f, 0.0f};
    if constexpr (W > 1) {
      const int wave =
          __builtin_amdgcn_readfirstlane(threadIdx.x / sa::kWave);
      if (lane == 0) lds[UP ? wave : W - 1 - wave] = j.whole;
      __syncthreads();
      Map all = {1.0f, 0.0f};
      if (lane < W) all = lds[lane];
      all = scan_lanes<16>(all);
      const int at = UP ? wave : W - 1 - wave;
      if (at > 0) j.before = after(j.before, of_lane(all, at - 1));
      j.whole = of_lane(all, W - 1);
    }
    if (!UP)
      j.before = {__shfl(j.before.a, 63 - lane),
                  __shfl(j.before.b, 63 - lane)};
  } else {
    const int lane = threadIdx.x & (LPR - 1);
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) {
      Map o;
      o.a = UP ? __shfl_up(m.a, d, LPR) : __shfl_down(m.a, d, LPR);
      o.b = UP ? __shfl_up(m.b, d, LPR) : __shfl_down(m.b, d, LPR);
      if (UP ? lane >= d : lane + d < LPR) m = after(m, o);
    }
    j.whole.a = __shfl(m.a, UP ? LPR - 1 : 0, LPR);
    j.whole.b = __shfl(m.b, UP ? LPR - 1 : 0, LPR);
    j.before.a = UP ? __shfl_up(m.a, 1, LPR) : __shfl_down(m.a, 1, LPR);
    j.before.b = UP ? __shfl_up(m.b, 1, LPR) : __shfl_down(m.b, 1, LPR);
    if (lane == (UP ? 0 : LPR - 1)) j.before = {1.0f, 0.0f};
  }
  return j;
}

// The state that reaches segment `seg` of a row from its neighbours: the
// maps of the segments before it (UP) or behind it, 64 at a time.
template <bool UP>
__device__ __forceinline__ float through(const float* maps, int segments,
                                         int seg, float state) {
  const int lane = threadIdx.x & (sa::kWave - 1);
  const int count = UP ? seg : segments - 1 - seg;
  for (int c = 0; c < count; c += sa::kWave) {
    Map m = {1.0f, 0.0f};
    const int k = c + lane;
    if (k < count) {
      const int at = UP ? k : segments - 1 - k;
      m = {maps[2 * at], maps[2 * at + 1]};
    }
    m = of_lane(scan_lanes<64>(m), 63);
    state = fmaf(m.a, state, m.b);
  }
  return state;
}

// A lane's place: its row, and the chunks of the row that it walks. Only
// chunks that hold a valid sample are walked; first..begin and end..last
// have none.
template <typename T, int LPR, int W, bool REV>
struct Place {
  static constexpr int kChunk = LPR * W * kItems<T>;
  static constexpr bool kShort = LPR == 1;
  const ScanArgs& p;
  long row, n, c;
  int lane, seg, first, last, begin, end, len;
  bool live;
  __device__ __forceinline__ Place(const ScanArgs& args) : p(args) {
    lane = W > 1 ? threadIdx.x : threadIdx.x & (LPR - 1);
    seg = blockIdx.y;
    row = W > 1 ? (long)blockIdx.x
                : ((long)blockIdx.x * blockDim.x + threadIdx.x) / LPR;
    if (LPR == 64 && W == 1)  // a wave's own, so that it stays scalar
      row = __builtin_amdgcn_readfirstlane((int)row);
    live = row < p.rows;
    if (!live) row = p.rows - 1;  // reads in bounds, writes nothing
    n = row / p.C;
    c = row % p.C;
    len = p.lengths == nullptr ? p.L : max(0, min(p.lengths[n], p.L));
    first = seg * p.per_segment;
    last = min(first + p.per_segment, p.chunks);
    begin = first;
    end = last;
    if (LPR == 64) {
      const int from = REV ? (p.L - len) / kChunk : 0;
      const int to = REV ? p.chunks : sa_ceil(len, kChunk);
      begin = min(max(begin, from), last);
      end = max(min(end, to), begin);
      if (len == 0) end = begin;
    }
  }
  __device__ static int sa_ceil(int a, int b) { return (a + b - 1) / b; }
  __device__ __forceinline__ int start(int chunk) const {
    return chunk * kChunk + lane * kItems<T>;  // under 2^30 + 2^13
  }
  // every sample of the chunk (of the row) in bounds; and valid
  __device__ __forceinline__ bool whole(int chunk) const {
    return (chunk + 1) * kChunk <= p.L;
  }
  __device__ __forceinline__ bool full(int chunk) const {
    return whole(chunk) && (REV ? chunk * kChunk >= p.L - len
                                : (chunk + 1) * kChunk <= len);
  }
  __device__ __forceinline__ bool valid(int s) const {
    return s < p.L && (REV ? p.L - 1 - s : s) < len;
  }
  __device__ __forceinline__ const T* x() const {
    return (const T*)p.x + n * p.xn + c * p.xc;
  }
  __device__ __forceinline__ const T* gate() const {
    return (const T*)p.gate + n * p.gn + c * p.gc;
  }
  __device__ __forceinline__ const T* dh() const {
    return p.dh ? (const T*)p.dh + row * p.L : nullptr;
  }
  // zeros where no sample is valid
  __device__ __forceinline__ void blank(T* out) const {
    if (!live) return;
    Items<T> zero;
#pragma unroll
    for (unsigned& w : zero.w) w = 0;
    for (int chunk = first; chunk < last; ++chunk)
      if (chunk < begin || chunk >= end)
        zero.template store<REV>(out, start(chunk), p.L, whole(chunk));
  }
};

// a, keep and one more of a lane's samples; outside the valid length a
// sample passes the state on
template <bool REV, bool FULL, typename T, typename P>
__device__ __forceinline__ void take(const P& at, int chunk,
                                     Items<T> gate, Items<T> more,
                                     bool given,
                                     float (&a)[kItems<T>],
                                     float (&keep)[kItems<T>],
                                     float (&m)[kItems<T>]) {
  if (!FULL && !P::kShort) {
    gate.template settle<REV>(at.start(chunk), at.p.L);
    more.template settle<REV>(at.start(chunk), at.p.L);
  }
#pragma unroll
  for (int i = 0; i < kItems<T>; ++i) {
    gates(gate.template at<REV>(i), a[i], keep[i]);
    m[i] = given ? more.template at<REV>(i) : 0.0f;
  }
  if (!FULL) {
    const int s0 = at.start(chunk);
#pragma unroll
    for (int i = 0; i < kItems<T>; ++i)
      if (!at.valid(s0 + i)) {
        a[i] = 1.0f;
        keep[i] = 0.0f;
        m[i] = 0.0f;
      }
  }
}

// Whether a chunk has only valid samples is the same for all of its lanes;
// those chunks go without a comparison.
template <typename P, typename F>
__device__ __forceinline__ void for_chunk(const P& at, int chunk, F f) {
  if (at.full(chunk)) f(std::true_type());
  else f(std::false_type());
}

#define SCAN_KERNEL \
  template <typename T, int LPR, int W, bool REV> \
  __global__ __launch_bounds__(W > 1 ? W * 64 : 256) void

// a segment's map
SCAN_KERNEL scan_map_kernel(ScanArgs p) {
  __shared__ Map lds[2][W];
  const Place<T, LPR, W, REV> at(p);
  const T *x = at.x(), *gate = at.gate();
  Items<T> xi, gi;
  auto fetch = [&](int chunk) {
    const int s0 = at.start(chunk);
    gi.template load<REV, at.kShort>(gate, s0, p.L);
    xi.template load<REV, at.kShort>(x, s0, p.L);
  };
  if (at.begin < at.end) fetch(at.begin);
  Map m = {1.0f, 0.0f};
  for (int chunk = at.begin; chunk < at.end; ++chunk) {
    for_chunk(at, chunk, [&](auto is_full) {
      constexpr bool FULL = decltype(is_full)::value;
      float xs[kItems<T>], a[kItems<T>], keep[kItems<T>];
      const Items<T> gn = gi, xn = xi;
      if (chunk + 1 < at.end) fetch(chunk + 1);
      take<REV, FULL>(at, chunk, gn, xn, true, a, keep, xs);
      Map own = {1.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kItems<T>; ++i)
        own = {own.a * a[i], fmaf(a[i], own.b, keep[i] * xs[i])};
      m = after(join<LPR, W, true>(own, lds[chunk & 1]).whole, m);
    });
  }
  if (at.live && at.lane == 0) {
    float* o = p.maps_out + (at.row * p.segments + at.seg) * 2;
    o[0] = m.a;
    o[1] = m.b;
  }
}

// the same for u_t = a_t * (dh_t + u_{t+1})
SCAN_KERNEL scan_map_back_kernel(ScanArgs p) {
  __shared__ Map lds[2][W];
  const Place<T, LPR, W, REV> at(p);
  const T *dh = at.dh(), *gate = at.gate();
  Items<T> di, gi;
  auto fetch = [&](int chunk) {
    const int s0 = at.start(chunk);
    gi.template load<REV, at.kShort>(gate, s0, p.L);
    if (dh) di.template load<REV, at.kShort>(dh, s0, p.L);
  };
  if (at.begin < at.end) fetch(at.end - 1);
  Map m = {1.0f, 0.0f};
  for (int chunk = at.end - 1; chunk >= at.begin; --chunk) {
    for_chunk(at, chunk, [&](auto is_full) {
      constexpr bool FULL = decltype(is_full)::value;
      float d[kItems<T>], a[kItems<T>], keep[kItems<T>];
      const Items<T> gn = gi, dn = di;
      if (chunk > at.begin) fetch(chunk - 1);
      take<REV, FULL>(at, chunk, gn, dn, dh != nullptr, a, keep, d);
      Map own = {1.0f, 0.0f};
#pragma unroll
      for (int i = kItems<T> - 1; i >= 0; --i)
        own = {own.a * a[i], a[i] * (d[i] + own.b)};
      m = after(join<LPR, W, false>(own, lds[chunk & 1]).whole, m);
    });
  }
  if (at.live && at.lane == 0) {
    float* o = p.maps_out + (at.row * p.segments + at.seg) * 2;
    o[0] = m.a;
    o[1] = m.b;
  }
}

SCAN_KERNEL scan_kernel(ScanArgs p) {
  __shared__ Map lds[2][W];
  const Place<T, LPR, W, REV> at(p);
  const T *x = at.x(), *gate = at.gate();
  T* out = (T*)p.out + at.row * p.L;
  Items<T> xi, gi;
  auto fetch = [&](int chunk) {
    const int s0 = at.start(chunk);
    gi.template load<REV, at.kShort>(gate, s0, p.L);
    xi.template load<REV, at.kShort>(x, s0, p.L);
  };
  if (at.begin < at.end) fetch(at.begin);
  float state = p.state ? p.state[at.row] : 0.0f;
  if (p.segments > 1)
    state = through<true>(p.maps + at.row * p.segments * 2, p.segments,
                          at.seg, state);
  for (int chunk = at.begin; chunk < at.end; ++chunk) {
    for_chunk(at, chunk, [&](auto is_full) {
      constexpr bool FULL = decltype(is_full)::value;
      if (p.marks && at.live && at.lane == 0)
        p.marks[at.row * p.chunks + chunk] = state;
      float xs[kItems<T>], a[kItems<T>], keep[kItems<T>];
      const Items<T> gn = gi, xn = xi;
      if (chunk + 1 < at.end) fetch(chunk + 1);
      take<REV, FULL>(at, chunk, gn, xn, true, a, keep, xs);
      Map own = {1.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kItems<T>; ++i) {
        xs[i] *= keep[i];
        own = {own.a * a[i], fmaf(a[i], own.b, xs[i])};
      }
      const Joined j = join<LPR, W, true>(own, lds[chunk & 1]);
      float h = fmaf(j.before.a, state, j.before.b);
      state = fmaf(j.whole.a, state, j.whole.b);
      const int s0 = at.start(chunk);
      float hs[kItems<T>];
#pragma unroll
      for (int i = 0; i < kItems<T>; ++i) {
        h = fmaf(a[i], h, xs[i]);
        hs[i] = FULL || at.valid(s0 + i) ? h : 0.0f;
      }
      Items<T> v;
      v.template set<REV>(hs);
      if (at.live) v.template store<REV>(out, s0, p.L, FULL || at.whole(chunk));
    });
  }
  at.blank(out);
  if (at.live && at.lane == 0 && at.seg == p.segments - 1)
    p.last[at.row] = state;
}

SCAN_KERNEL scan_back_kernel(ScanArgs p) {
  __shared__ Map lds[4][W];
  const Place<T, LPR, W, REV> at(p);
  const T *x = at.x(), *gate = at.gate(), *dh = at.dh();
  T* dx = (T*)p.out + at.row * p.L;
  T* dgate = (T*)p.out2 + at.row * p.L;
  const float* marks = p.marks + at.row * p.chunks;
  Items<T> xi, gi, di;
  float mark = 0.0f;
  auto fetch = [&](int chunk) {
    const int s0 = at.start(chunk);
    gi.template load<REV, at.kShort>(gate, s0, p.L);
    xi.template load<REV, at.kShort>(x, s0, p.L);
    if (dh) di.template load<REV, at.kShort>(dh, s0, p.L);
    mark = marks[chunk];
  };
  if (at.begin < at.end) fetch(at.end - 1);
  float u = p.dstate ? p.dstate[at.row] : 0.0f;
  if (p.segments > 1)
    u = through<false>(p.maps + at.row * p.segments * 2, p.segments, at.seg,
                       u);
  for (int chunk = at.end - 1; chunk >= at.begin; --chunk) {
    for_chunk(at, chunk, [&](auto is_full) {
      constexpr bool FULL = decltype(is_full)::value;
      const float state = mark;
      float xs[kItems<T>], a[kItems<T>], keep[kItems<T>], d[kItems<T>];
      const Items<T> gn = gi, xn = xi;
      if (!FULL && !at.kShort)
        di.template settle<REV>(at.start(chunk), p.L);
#pragma unroll
      for (int i = 0; i < kItems<T>; ++i)
        d[i] = dh ? di.template at<REV>(i) : 0.0f;
      if (chunk > at.begin) fetch(chunk - 1);
      take<REV, FULL>(at, chunk, gn, xn, true, a, keep, xs);
      const int s0 = at.start(chunk);
      Map own = {1.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kItems<T>; ++i) {
        if (!FULL && !at.valid(s0 + i)) d[i] = 0.0f;
        own = {own.a * a[i], fmaf(a[i], own.b, keep[i] * xs[i])};
      }
      const Joined jf = join<LPR, W, true>(own, lds[chunk & 1]);
      own.b = 0.0f;
#pragma unroll
      for (int i = kItems<T> - 1; i >= 0; --i) own.b = a[i] * (d[i] + own.b);
      const Joined jb = join<LPR, W, false>(own, lds[2 + (chunk & 1)]);
      float before[kItems<T>];
      float h = fmaf(jf.before.a, state, jf.before.b);
#pragma unroll
      for (int i = 0; i < kItems<T>; ++i) {
        before[i] = h;
        h = fmaf(a[i], h, keep[i] * xs[i]);
      }
      float w = fmaf(jb.before.a, u, jb.before.b);
      u = fmaf(jb.whole.a, u, jb.whole.b);
      Items<T> vx, vg;
#pragma unroll
      for (int i = kItems<T> - 1; i >= 0; --i) {
        const bool in = FULL || at.valid(s0 + i);
        const float g = d[i] + w;
        w = a[i] * g;
        d[i] = in ? keep[i] * g : 0.0f;
        xs[i] = in ? w * (before[i] - xs[i]) * keep[i] : 0.0f;
      }
      vx.template set<REV>(d);
      vg.template set<REV>(xs);
      if (at.live) {
        vx.template store<REV>(dx, s0, p.L, FULL || at.whole(chunk));
        vg.template store<REV>(dgate, s0, p.L, FULL || at.whole(chunk));
      }
    });
  }
  at.blank(dx);
  at.blank(dgate);
  if (at.live && at.lane == 0 && at.seg == 0) p.last[at.row] = u;
}

#undef SCAN_KERNEL

// How a problem is dealt out. A row gets as many lanes as its length fills.
// Rows over two waves' samples get 4 waves, which walk the row in longer
// contiguous pieces (training of (100, 64, 8192) bf16: 71 + 111 us with one
// wave, 68 + 98 with 4, 66 + 129 with 16, whose waits at the barriers show).
// Few rows get 16, and are cut into segments until the card has waves enough,
// two rounds of them (one row set of 24 x 1000003 fp32 in 11, 22 and 43
// segments: 333, 291 and 300 us).
struct Deal {
  int lpr, w, chunks, segments, per_segment;
  Deal(long rows, int L, int items) {
    lpr = L <= items ? 1 : L <= 16 * items ? 16 : 64;
    w = 1;
    const int wave = 64 * items;
    const long enough = 4096;  // waves
    if (L > 2 * wave) w = 4;
    if (L > 16 * wave && rows * 4 < enough) w = 16;
    chunks = sa::ceil_div(L, lpr * w * items);
    segments = 1;
    per_segment = chunks;
    if (lpr == 64 && rows * w < enough && chunks >= 4) {
      const long most = std::min<long>(chunks / 2, sa::ceil_div(2 * enough,
                                                                rows * w));
      per_segment = sa::ceil_div(chunks, most);
      segments = sa::ceil_div(chunks, per_segment);
    }
  }
  dim3 grid(long rows) const {
    return dim3(w > 1 ? rows : sa::ceil_div(rows * lpr, 256), segments);
  }
  int block() const { return w > 1 ? w * 64 : 256; }
};

enum Which { MAP, MAP_BACK, SCAN, SCAN_BACK };

template <typename T, int LPR, int W, bool REV>
void launch_one(Which which, const ScanArgs& p, const Deal& deal,
                hipStream_t stream) {
  const dim3 grid = deal.grid(p.rows), block(deal.block());
  switch (which) {
    case MAP:
      scan_map_kernel<T, LPR, W, REV><<<grid, block, 0, stream>>>(p);
      break;
    case MAP_BACK:
      scan_map_back_kernel<T, LPR, W, REV><<<grid, block, 0, stream>>>(p);
      break;
    case SCAN:
      scan_kernel<T, LPR, W, REV><<<grid, block, 0, stream>>>(p);
      break;
    case SCAN_BACK:
      scan_back_kernel<T, LPR, W, REV><<<grid, block, 0, stream>>>(p);
      break;
  }
  SA_CHECK_HIP(hipGetLastError());
}

template <typename T, bool REV>
void launch_rev(Which which, const ScanArgs& p, const Deal& deal,
                hipStream_t stream) {
  if (deal.lpr == 1) launch_one<T, 1, 1, REV>(which, p, deal, stream);
  else if (deal.lpr == 16) launch_one<T, 16, 1, REV>(which, p, deal, stream);
  else if (deal.w == 1) launch_one<T, 64, 1, REV>(which, p, deal, stream);
  else if (deal.w == 4) launch_one<T, 64, 4, REV>(which, p, deal, stream);
  else launch_one<T, 64, 16, REV>(which, p, deal, stream);
}

void launch(Which which, at::ScalarType type, bool rev, const ScanArgs& p,
            const Deal& deal, hipStream_t stream) {
  if (type == at::kBFloat16) {
    if (rev) launch_rev<__bf16, true>(which, p, deal, stream);
    else launch_rev<__bf16, false>(which, p, deal, stream);
  } else {
    if (rev) launch_rev<float, true>(which, p, deal, stream);
    else launch_rev<float, false>(which, p, deal, stream);
  }
}

// A call's tensors, as checked by checked(): x and gate with unit stride
// along L, the rest contiguous; state and lengths may be undefined.
struct Call {
  at::Tensor x, gate, state, lengths;
  bool reverse;
};

ScanArgs args_of(const Call& c, const Deal& deal) {
  ScanArgs p = {};
  p.x = sa::memory_of(c.x);
  p.gate = sa::memory_of(c.gate);
  if (c.lengths.defined()) p.lengths = sa::memory_of<int>(c.lengths);
  p.xn = c.x.stride(0);
  p.xc = c.x.stride(1);
  p.gn = c.gate.stride(0);
  p.gc = c.gate.stride(1);
  p.rows = c.x.size(0) * c.x.size(1);
  p.C = c.x.size(1);
  p.L = c.x.size(2);
  p.chunks = deal.chunks;
  p.segments = deal.segments;
  p.per_segment = deal.per_segment;
  return p;
}

// {h, last state, marks}; marks only if `marked`
std::vector<at::Tensor> forward(const Call& c, bool marked) {
  const c10::DeviceGuard guard(c.x.device());
  const auto f32 = c.x.options().dtype(at::kFloat);
  auto h = at::empty(c.x.sizes(), c.x.options());
  auto last = at::empty({c.x.size(0), c.x.size(1)}, f32);
  const long rows = last.numel();
  at::Tensor marks, maps;
  if (rows == 0) return {h, last, marks};
  const Deal deal(rows, c.x.size(2), 16 / c.x.element_size());
  ScanArgs p = args_of(c, deal);
  if (marked) {
    marks = at::empty({rows, deal.chunks}, f32);
    p.marks = sa::memory_of<float>(marks);
  }
  if (c.state.defined()) p.state = sa::memory_of<float>(c.state);
  p.out = sa::memory_of(h);
  p.last = sa::memory_of<float>(last);
  const auto stream = at::hip::getCurrentHIPStream().stream();
  const auto type = c.x.scalar_type();
  if (deal.segments > 1) {
    maps = at::empty({rows, deal.segments, 2}, f32);
    p.maps = p.maps_out = sa::memory_of<float>(maps);
    launch(MAP, type, c.reverse, p, deal, stream);
  }
  launch(SCAN, type, c.reverse, p, deal, stream);
  return {h, last, marks};
}

// {dx, dgate, d(first state)} of dh and d(last state), each maybe undefined
std::vector<at::Tensor> backward(const Call& c, const at::Tensor& marks,
                                 const at::Tensor& dh,
                                 const at::Tensor& dstate) {
  const c10::DeviceGuard guard(c.x.device());
  const auto f32 = c.x.options().dtype(at::kFloat);
  auto dx = at::empty(c.x.sizes(), c.x.options());
  auto dgate = at::empty(c.x.sizes(), c.x.options());
  auto first = at::empty({c.x.size(0), c.x.size(1)}, f32);
  const long rows = first.numel();
  if (rows == 0) return {dx, dgate, first};
  const Deal deal(rows, c.x.size(2), 16 / c.x.element_size());
  ScanArgs p = args_of(c, deal);
  if (dh.defined()) p.dh = sa::memory_of(dh);
  if (dstate.defined()) p.dstate = sa::memory_of<float>(dstate);
  p.marks = sa::memory_of<float>(marks);
  p.out = sa::memory_of(dx);
  p.out2 = sa::memory_of(dgate);
  p.last = sa::memory_of<float>(first);
  const auto stream = at::hip::getCurrentHIPStream().stream();
  const auto type = c.x.scalar_type();
  at::Tensor maps;
  if (deal.segments > 1) {
    maps = at::empty({rows, deal.segments, 2}, f32);
    p.maps = p.maps_out = sa::memory_of<float>(maps);
    launch(MAP_BACK, type, c.reverse, p, deal, stream);
  }
  launch(SCAN_BACK, type, c.reverse, p, deal, stream);
  return {dx, dgate, first};
}

std::string shape_of(const at::Tensor& t) {
  return c10::str(t.sizes(), " ", t.scalar_type(), " on ", t.device());
}

at::Tensor along_samples(const at::Tensor& t) {
  return t.stride(2) == 1 ? t : t.contiguous();
}

// What the kernels take for granted. Lengths outside 0..L are held to it by
// the kernels.
Call checked(const at::Tensor& x, const at::Tensor& gate,
             const c10::optional<at::Tensor>& state,
             const c10::optional<at::Tensor>& lengths, bool reverse) {
  TORCH_CHECK_VALUE(
      x.dim() == 3 && gate.sizes() == x.sizes() && x.size(2) >= 1,
      "gated_scan: x and gate of one shape (N, C, L), L at least 1, are "
      "needed, got ", shape_of(x), " and ", shape_of(gate));
  const auto type = x.scalar_type();
  TORCH_CHECK_VALUE(
      (type == at::kBFloat16 || type == at::kFloat) &&
          gate.scalar_type() == type,
      "gated_scan: x and gate have to be both float32 or both bfloat16, got ",
      type, " and ", gate.scalar_type());
  TORCH_CHECK_VALUE(x.is_cuda() && gate.device() == x.device(),
                    "gated_scan: x and gate have to be on one device");
  TORCH_CHECK(!sa::has_tangent(x) && !sa::has_tangent(gate) &&
                  !(state.has_value() && sa::has_tangent(*state)),
              "gated_scan: forward-mode derivatives are not available");
  TORCH_CHECK_VALUE(x.size(2) < (1L << 30) &&
                        x.size(0) * x.size(1) < (1L << 24),
                    "gated_scan: under 2**30 samples and 2**24 rows are "
                    "needed, got ", shape_of(x));
  Call c = {along_samples(x), along_samples(gate), {}, {}, reverse};
  if (state.has_value()) {
    TORCH_CHECK_VALUE(
        state->sizes() == x.sizes().slice(0, 2) &&
            state->scalar_type() == at::kFloat &&
            state->device() == x.device(),
        "gated_scan: state has to be ", x.sizes().slice(0, 2),
        " float32 on ", x.device(), ", got ", shape_of(*state));
    c.state = state->contiguous();
  }
  if (lengths.has_value()) {
    const auto& l = *lengths;
    TORCH_CHECK_VALUE(
        l.dim() == 1 && l.size(0) == x.size(0) &&
            (l.scalar_type() == at::kInt || l.scalar_type() == at::kLong) &&
            l.device() == x.device(),
        "gated_scan: lengths has to be [", x.size(0),
        "] int32 or int64 on ", x.device(), ", got ", shape_of(l));
    c.lengths = l.scalar_type() == at::kInt
                    ? l.contiguous()
                    : l.clamp(0, x.size(2)).to(at::kInt).contiguous();
  }
  return c;
}

// The node keeps the inputs and the fp32 state at each chunk's start.
class GatedScan : public torch::autograd::Function<GatedScan> {
 public:
  static torch::autograd::variable_list forward(
      torch::autograd::AutogradContext* ctx, const at::Tensor& x,
      const at::Tensor& gate, const c10::optional<at::Tensor>& state,
      const Call& call) {
    auto r = gated_scan::forward(call, true);
    ctx->save_for_backward({x, gate, call.lengths, r[2]});
    ctx->saved_data["reverse"] = call.reverse;
    ctx->saved_data["state"] = state.has_value();
    ctx->set_materialize_grads(false);
    return {r[0], r[1]};
  }
  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "gated_scan: second derivatives are not available");
    for (const auto& g : grads)
      TORCH_CHECK(!sa::has_tangent(g),
                  "gated_scan: forward-mode derivatives are not available");
    const auto s = ctx->get_saved_variables();
    const Call call = {s[0], s[1], {}, s[2],
                       ctx->saved_data["reverse"].toBool()};
    for (auto& g : grads)
      if (g.defined()) g = g.contiguous();
    auto r = gated_scan::backward(call, s[3], grads[0], grads[1]);
    const bool state = ctx->saved_data["state"].toBool();
    return {r[0], r[1], state ? r[2] : at::Tensor(), at::Tensor()};
  }
};

}  // namespace
}  // namespace gated_scan

// {h, last state}, or nothing where a call is recorded or a tensor only stands
// for one
std::vector<at::Tensor> gated_scan_run(
    const at::Tensor& x, const at::Tensor& gate,
    const c10::optional<at::Tensor>& state,
    const c10::optional<at::Tensor>& lengths, bool reverse) {
  if (sa::recorded() || sa::stands_in(x) || sa::stands_in(gate) ||
      sa::stands_in(state) || sa::stands_in(lengths))
    return {};
  const auto call = gated_scan::checked(x, gate, state, lengths, reverse);
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || gate.requires_grad() ||
       (state.has_value() && state->requires_grad())))
    return gated_scan::GatedScan::apply(
        call.x, call.gate,
        call.state.defined() ? c10::optional<at::Tensor>(call.state)
                             : c10::nullopt,
        call);
  auto r = gated_scan::forward(call, false);
  return {r[0], r[1]};
}
