// Gated linear recurrence over the last axis of (N, C, L):
//
//   a_t = sigmoid(gate_t),  h_t = a_t * h_{t-1} + (1 - a_t) * x_t
//
// A step is the map h -> A*h + B, and maps compose:
// (A2, B2) after (A1, B1) is (A2*A1, A2*B1 + B2). A lane composes 8
// neighbouring samples in registers, a row's lanes join their maps with
// log2 exchanges, waves join theirs through LDS, and the state carries from
// chunk to chunk, so a sample is read once and written once. The gradient
// runs the other way: with u_t = a_t * G_t, G_t = dh_t + u_{t+1},
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

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "sa_common.h"

namespace gated_scan {
namespace {

constexpr int kItems = 8;  // samples a lane holds

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
  if (m > -100.0f) e = fmaf(e, lo * 0.693147180559945f, e);
  const float r = 1.0f / (1.0f + e);
  const float s = e * r;
  a = g < 0.0f ? s : r;
  keep = g < 0.0f ? r : s;
}

// 8 samples from p on; rows start anywhere, so the 16-byte accesses are not
// aligned
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[kItems]) {
  T t[kItems];
  __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
  for (int i = 0; i < kItems; ++i) v[i] = (float)t[i];
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[kItems]) {
  T t[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) t[i] = (T)v[i];
  __builtin_memcpy(p, t, sizeof(t));
}

// v[i] = sample of scan index s0+i, 0 outside the row
template <typename T, bool REV>
__device__ __forceinline__ void load_items(const T* row, long s0, int L,
                                           float (&v)[kItems]) {
  if (s0 + kItems <= L) {
    float t[kItems];
    load8(row + (REV ? L - kItems - s0 : s0), t);
#pragma unroll
    for (int i = 0; i < kItems; ++i) v[i] = REV ? t[kItems - 1 - i] : t[i];
  } else {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const long s = s0 + i;
      v[i] = s < L ? (float)row[REV ? L - 1 - s : s] : 0.0f;
    }
  }
}

template <typename T, bool REV>
__device__ __forceinline__ void store_items(T* row, long s0, int L,
                                            const float (&v)[kItems]) {
  if (s0 + kItems <= L) {
    float t[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) t[i] = REV ? v[kItems - 1 - i] : v[i];
    store8(row + (REV ? L - kItems - s0 : s0), t);
  } else {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const long s = s0 + i;
      if (s < L) row[REV ? L - 1 - s : s] = (T)v[i];
    }
  }
}

// What stands before (UP) or behind (!UP) each lane of its row's lanes, and
// the whole, all in scan order. A row has LPR lanes of one wave and W waves.
template <int LPR, int W, bool UP>
struct Joined {
  Map before, whole;
};

template <int LPR, int W, bool UP>
__device__ __forceinline__ Joined<LPR, W, UP> join(Map m, Map* lds) {
  const int lane = threadIdx.x & (LPR - 1);
#pragma unroll
  for (int d = 1; d < LPR; d <<= 1) {
    Map o;
    o.a = UP ? __shfl_up(m.a, d, LPR) : __shfl_down(m.a, d, LPR);
    o.b = UP ? __shfl_up(m.b, d, LPR) : __shfl_down(m.b, d, LPR);
    if (UP ? lane >= d : lane + d < LPR) m = after(m, o);
  }
  Joined<LPR, W, UP> j;
  j.whole.a = __shfl(m.a, UP ? LPR - 1 : 0, LPR);
  j.whole.b = __shfl(m.b, UP ? LPR - 1 : 0, LPR);
  j.before.a = UP ? __shfl_up(m.a, 1, LPR) : __shfl_down(m.a, 1, LPR);
  j.before.b = UP ? __shfl_up(m.b, 1, LPR) : __shfl_down(m.b, 1, LPR);
  if (lane == (UP ? 0 : LPR - 1)) j.before = {1.0f, 0.0f};
  if constexpr (W > 1) {
    const int wave = threadIdx.x / sa::kWave;
    if (lane == 0) lds[wave] = j.whole;
    __syncthreads();
    Map all = {1.0f, 0.0f};
    Map head = all;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int w = UP ? i : W - 1 - i;
      if (w == wave) head = all;
      all = after(lds[w], all);
    }
    j.before = after(j.before, head);
    j.whole = all;
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
#pragma unroll
    for (int d = 1; d < sa::kWave; d <<= 1) {
      Map o = {__shfl_up(m.a, d), __shfl_up(m.b, d)};
      if (lane >= d) m = after(m, o);
    }
    state = fmaf(__shfl(m.a, sa::kWave - 1), state,
                 __shfl(m.b, sa::kWave - 1));
  }
  return state;
}

template <int LPR, int W>
struct Place {
  long row;
  int lane, seg, first, end;  // the chunks of this row that are walked
  bool live;
  __device__ __forceinline__ Place(const ScanArgs& p) {
    lane = threadIdx.x & (LPR * W - 1);
    if (W > 1) lane = threadIdx.x;
    seg = blockIdx.y;
    row = W > 1 ? (long)blockIdx.x
                : ((long)blockIdx.x * blockDim.x + threadIdx.x) / LPR;
    live = row < p.rows;
    if (!live) row = p.rows - 1;  // reads in bounds, writes nothing
    first = seg * p.per_segment;
    end = min(first + p.per_segment, p.chunks);
  }
};

__device__ __forceinline__ int valid_length(const ScanArgs& p, long n) {
  if (p.lengths == nullptr) return p.L;
  return max(0, min(p.lengths[n], p.L));
}

// a, keep and x of a lane's samples; outside the valid length a sample
// passes the state on
template <typename T, bool REV>
__device__ __forceinline__ void take(const T* x, const T* gate, long s0,
                                     int L, int len, float (&xs)[kItems],
                                     float (&a)[kItems],
                                     float (&keep)[kItems]) {
  float g[kItems];
  load_items<T, REV>(gate, s0, L, g);
  if (x != nullptr) load_items<T, REV>(x, s0, L, xs);
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    gates(g[i], a[i], keep[i]);
    const long s = s0 + i;
    const bool in = s < L && (REV ? L - 1 - s : s) < len;
    if (!in) {
      a[i] = 1.0f;
      keep[i] = 0.0f;
      xs[i] = 0.0f;
    }
  }
}

template <typename T, int LPR, int W, bool REV>
__global__ __launch_bounds__(W > 1 ? W * 64 : 256) void scan_map_kernel(
    ScanArgs p) {
  __shared__ Map lds[2][W];
  const Place<LPR, W> at(p);
  const long n = at.row / p.C, c = at.row % p.C;
  const int len = valid_length(p, n);
  const T* x = (const T*)p.x + n * p.xn + c * p.xc;
  const T* gate = (const T*)p.gate + n * p.gn + c * p.gc;
  Map m = {1.0f, 0.0f};
  for (int chunk = at.first; chunk < at.end; ++chunk) {
    const long s0 = ((long)chunk * LPR * W + at.lane) * kItems;
    float xs[kItems], a[kItems], keep[kItems];
    take<T, REV>(x, gate, s0, p.L, len, xs, a, keep);
    Map own = {1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      own = {own.a * a[i], fmaf(a[i], own.b, keep[i] * xs[i])};
    m = after(join<LPR, W, true>(own, lds[chunk & 1]).whole, m);
  }
  if (at.live && at.lane == 0) {
    float* o = p.maps_out + (at.row * p.segments + at.seg) * 2;
    o[0] = m.a;
    o[1] = m.b;
  }
}

// u_t = a_t * (dh_t + u_{t+1}) over a segment
template <typename T, int LPR, int W, bool REV>
__global__ __launch_bounds__(W > 1 ? W * 64 : 256) void scan_map_back_kernel(
    ScanArgs p) {
  __shared__ Map lds[2][W];
  const Place<LPR, W> at(p);
  const long n = at.row / p.C, c = at.row % p.C;
  const int len = valid_length(p, n);
  const T* gate = (const T*)p.gate + n * p.gn + c * p.gc;
  const T* dh = p.dh ? (const T*)p.dh + at.row * p.L : nullptr;
  Map m = {1.0f, 0.0f};
  for (int chunk = at.end - 1; chunk >= at.first; --chunk) {
    const long s0 = ((long)chunk * LPR * W + at.lane) * kItems;
    float d[kItems] = {}, a[kItems], keep[kItems];
    take<T, REV>(dh, gate, s0, p.L, len, d, a, keep);
    Map own = {1.0f, 0.0f};
#pragma unroll
    for (int i = kItems - 1; i >= 0; --i)
      own = {own.a * a[i], a[i] * (d[i] + own.b)};
    m = after(join<LPR, W, false>(own, lds[chunk & 1]).whole, m);
  }
  if (at.live && at.lane == 0) {
    float* o = p.maps_out + (at.row * p.segments + at.seg) * 2;
    o[0] = m.a;
    o[1] = m.b;
  }
}

template <typename T, int LPR, int W, bool REV>
__global__ __launch_bounds__(W > 1 ? W * 64 : 256) void scan_kernel(
    ScanArgs p) {
  __shared__ Map lds[2][W];
  const Place<LPR, W> at(p);
  const long n = at.row / p.C, c = at.row % p.C;
  const int len = valid_length(p, n);
  const T* x = (const T*)p.x + n * p.xn + c * p.xc;
  const T* gate = (const T*)p.gate + n * p.gn + c * p.gc;
  T* out = (T*)p.out + at.row * p.L;
  float state = p.state ? p.state[at.row] : 0.0f;
  if (p.segments > 1)
    state = through<true>(p.maps + at.row * p.segments * 2, p.segments,
                          at.seg, state);
  for (int chunk = at.first; chunk < at.end; ++chunk) {
    const long s0 = ((long)chunk * LPR * W + at.lane) * kItems;
    if (p.marks && at.live && at.lane == 0)
      p.marks[at.row * p.chunks + chunk] = state;
    float xs[kItems], a[kItems], keep[kItems];
    take<T, REV>(x, gate, s0, p.L, len, xs, a, keep);
    Map own = {1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      own = {own.a * a[i], fmaf(a[i], own.b, keep[i] * xs[i])};
    const auto j = join<LPR, W, true>(own, lds[chunk & 1]);
    float h = fmaf(j.before.a, state, j.before.b);
    state = fmaf(j.whole.a, state, j.whole.b);
    float v[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      h = fmaf(a[i], h, keep[i] * xs[i]);
      const long s = s0 + i;
      v[i] = (REV ? p.L - 1 - s : s) < len ? h : 0.0f;
    }
    if (at.live) store_items<T, REV>(out, s0, p.L, v);
  }
  if (at.live && at.lane == 0 && at.seg == p.segments - 1)
    p.last[at.row] = state;
}

template <typename T, int LPR, int W, bool REV>
__global__ __launch_bounds__(W > 1 ? W * 64 : 256) void scan_back_kernel(
    ScanArgs p) {
  __shared__ Map lds[4][W];
  const Place<LPR, W> at(p);
  const long n = at.row / p.C, c = at.row % p.C;
  const int len = valid_length(p, n);
  const T* x = (const T*)p.x + n * p.xn + c * p.xc;
  const T* gate = (const T*)p.gate + n * p.gn + c * p.gc;
  const T* dh = p.dh ? (const T*)p.dh + at.row * p.L : nullptr;
  T* dx = (T*)p.out + at.row * p.L;
  T* dgate = (T*)p.out2 + at.row * p.L;
  float u = p.dstate ? p.dstate[at.row] : 0.0f;
  if (p.segments > 1)
    u = through<false>(p.maps + at.row * p.segments * 2, p.segments, at.seg,
                       u);
  for (int chunk = at.end - 1; chunk >= at.first; --chunk) {
    const long s0 = ((long)chunk * LPR * W + at.lane) * kItems;
    const float state = p.marks[at.row * p.chunks + chunk];
    float xs[kItems], a[kItems], keep[kItems], d[kItems] = {};
    if (dh) load_items<T, REV>(dh, s0, p.L, d);
    take<T, REV>(x, gate, s0, p.L, len, xs, a, keep);
    Map own = {1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      own = {own.a * a[i], fmaf(a[i], own.b, keep[i] * xs[i])};
    const auto jf = join<LPR, W, true>(own, lds[chunk & 1]);
    own = {own.a, 0.0f};
#pragma unroll
    for (int i = kItems - 1; i >= 0; --i) {
      const long s = s0 + i;
      if ((REV ? p.L - 1 - s : s) >= len) d[i] = 0.0f;
      own.b = a[i] * (d[i] + own.b);
    }
    const auto jb = join<LPR, W, false>(own, lds[2 + (chunk & 1)]);
    float before[kItems];
    float h = fmaf(jf.before.a, state, jf.before.b);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      before[i] = h;
      h = fmaf(a[i], h, keep[i] * xs[i]);
    }
    float w = fmaf(jb.before.a, u, jb.before.b);
    u = fmaf(jb.whole.a, u, jb.whole.b);
    float vx[kItems], vg[kItems];
#pragma unroll
    for (int i = kItems - 1; i >= 0; --i) {
      const long s = s0 + i;
      const bool in = (REV ? p.L - 1 - s : s) < len;
      const float g = d[i] + w;
      vx[i] = in ? keep[i] * g : 0.0f;
      vg[i] = in ? g * (before[i] - xs[i]) * (a[i] * keep[i]) : 0.0f;
      w = a[i] * g;
    }
    if (at.live) {
      store_items<T, REV>(dx, s0, p.L, vx);
      store_items<T, REV>(dgate, s0, p.L, vg);
    }
  }
  if (p.last && at.live && at.lane == 0 && at.seg == 0) p.last[at.row] = u;
}

// How a problem is dealt out. A row gets as many lanes as its length fills;
// rows longer than a wave's 512 samples get 4 or 16 waves where the rows
// alone would leave the card short of waves, and segments beyond that.
struct Deal {
  int lpr, w, chunks, segments, per_segment;
  Deal(long rows, int L) {
    lpr = L <= kItems ? 1 : L <= 8 * kItems ? 8 : 64;
    w = 1;
    const long enough = 4096;  // waves
    if (lpr == 64) {
      while (w < 16 && rows * w < enough && 64L * kItems * w < L) w *= 4;
    }
    chunks = sa::ceil_div(L, lpr * w * kItems);
    segments = 1;
    per_segment = chunks;
    if (lpr == 64 && rows * w < enough / 2 && chunks >= 4) {
      const long most = std::min<long>(chunks / 2,
                                       (enough + rows * w - 1) / (rows * w));
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
  else if (deal.lpr == 8) launch_one<T, 8, 1, REV>(which, p, deal, stream);
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
  p.x = c.x.data_ptr();
  p.gate = c.gate.data_ptr();
  if (c.lengths.defined()) p.lengths = c.lengths.data_ptr<int>();
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
  const Deal deal(rows, c.x.size(2));
  ScanArgs p = args_of(c, deal);
  if (marked) {
    marks = at::empty({rows, deal.chunks}, f32);
    p.marks = marks.data_ptr<float>();
  }
  if (c.state.defined()) p.state = c.state.data_ptr<float>();
  p.out = h.data_ptr();
  p.last = last.data_ptr<float>();
  const auto stream = at::hip::getCurrentHIPStream().stream();
  const auto type = c.x.scalar_type();
  if (deal.segments > 1) {
    maps = at::empty({rows, deal.segments, 2}, f32);
    p.maps = p.maps_out = maps.data_ptr<float>();
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
  const Deal deal(rows, c.x.size(2));
  ScanArgs p = args_of(c, deal);
  if (dh.defined()) p.dh = dh.data_ptr();
  if (dstate.defined()) p.dstate = dstate.data_ptr<float>();
  p.marks = marks.data_ptr<float>();
  p.out = dx.data_ptr();
  p.out2 = dgate.data_ptr();
  p.last = first.data_ptr<float>();
  const auto stream = at::hip::getCurrentHIPStream().stream();
  const auto type = c.x.scalar_type();
  at::Tensor maps;
  if (deal.segments > 1) {
    maps = at::empty({rows, deal.segments, 2}, f32);
    p.maps = p.maps_out = maps.data_ptr<float>();
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

// {h, last state}
std::vector<at::Tensor> gated_scan_run(
    const at::Tensor& x, const at::Tensor& gate,
    const c10::optional<at::Tensor>& state,
    const c10::optional<at::Tensor>& lengths, bool reverse) {
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
