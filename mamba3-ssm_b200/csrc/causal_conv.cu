// Short depthwise causal convolution over (batch, length, channels), forward, backward, one step:
//   pre[t] = bias + sum_k w[k] x[t - K + 1 + k],   y = pre or silu(pre)
//   d = dy act'(pre),  dx[t] = sum_k w[k] d[t + K - 1 - k],  dw[k] = sum d[t] x[t - K + 1 + k],  dbias = sum d
// Bound by the memory's latency: the rows that 24 (forward) or 16 (backward) warps an SM have on their way. A lane holds
// one or two pairs of neighbouring channels (vector loads where the rows allow it) and walks a run of rows with the last K
// rows in registers, so each element is read once but for the K - 1 rows between runs; the next four rows are
// loaded while four are worked on, a multiple of the window so that it turns without moves. The backward forms
// pre again from x. 8 x 2048 x 2048 of bf16 with four taps, us: forward 36 (134 MB, 3.7 TB/s), backward 57 (201 MB, 3.5 TB/s)
// and 3 to join. Before, with a look at each row of the backward 74; with one pair a lane 45 and 103; weights read four at a time,
// which takes registers, 40 and 96; two or three rows ahead in the backward 155, 157.
#include <algorithm>
#include <type_traits>

#include "causal_conv.cuh"
#include "m3_common.cuh"
#include "pairs.cuh"

namespace m3 {
namespace {

constexpr int kWarps = 8;

// A row's 2 NV neighbouring channels of a lane as they lie in memory; converted when they are used, so that loads
// stay in flight.
template <typename T, int NV> struct RawRow;
template <> struct RawRow<float, 2> { float4 v; };
template <> struct RawRow<__nv_bfloat16, 2> { uint2 v; };
template <> struct RawRow<__half, 2> { uint2 v; };
template <typename T> struct RawRow<T, 1> { Raw2<T> v; };

template <typename T, int NV>
struct Chan {  // how a lane reaches its channels: all at once, or (NV = 1) one by one, the second one `second` further
  bool vec;
  int second;
  __device__ __forceinline__ RawRow<T, NV> load(const T* p) const {
    RawRow<T, NV> r;
    if constexpr (NV == 2) r = *reinterpret_cast<const RawRow<T, 2>*>(p);
    else r.v = load2<T>(p, vec, second);
    return r;
  }
  __device__ __forceinline__ void store(T* p, const f2 (&v)[NV]) const {
    float a[2 * NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) unpack2(v[i], a[2 * i], a[2 * i + 1]);
    if constexpr (NV == 2) {
      alignas(16) T o[4] = {from_f32<T>(a[0]), from_f32<T>(a[1]), from_f32<T>(a[2]), from_f32<T>(a[3])};
      *reinterpret_cast<RawRow<T, 2>*>(p) = *reinterpret_cast<const RawRow<T, 2>*>(o);
    } else {
      store2<T>(p, vec, second, a[0], a[1]);
    }
  }
};

template <typename T, int NV>
__device__ __forceinline__ void values(const RawRow<T, NV>& r, f2 (&v)[NV]) {
  if constexpr (NV == 1) {
    const float2 x = value2(r.v);
    v[0] = pack2(x.x, x.y);
  } else if constexpr (sizeof(T) == 4) {
    v[0] = pack2(r.v.x, r.v.y);
    v[1] = pack2(r.v.z, r.v.w);
  } else {
    const float2 x = value2(Raw2<T>{r.v.x}), y = value2(Raw2<T>{r.v.y});
    v[0] = pack2(x.x, x.y);
    v[1] = pack2(y.x, y.y);
  }
}

template <int NV>
__device__ __forceinline__ void zero(f2 (&v)[NV]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = 0;
}

template <typename T>
__device__ __forceinline__ float weight(const void* p, bool f32, int64_t i) {
  return f32 ? static_cast<const float*>(p)[i] : to_f32(static_cast<const T*>(p)[i]);
}

__device__ __forceinline__ int row_count(const int64_t* lengths, int b, int L) {
  if (lengths == nullptr) return L;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : n > L ? L : (int)n;
}

template <typename T, int NV, int K>
struct Lane {  // a lane's channels of one sequence
  const ConvParams& p;
  Chan<T, NV> ch;
  const T* x;
  const T* init;
  f2 w[K][NV], bias[NV];

  __device__ __forceinline__ Lane(const ConvParams& q, int b, int e) : p(q), ch{q.vec, e + 1 < q.E ? 1 : 0} {
    x = static_cast<const T*>(p.x) + (int64_t)b * p.xb + e;
    init = p.init != nullptr ? static_cast<const T*>(p.init) + (int64_t)b * p.ib + e : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e0 = e + 2 * i, e1 = e0 + ch.second;
#pragma unroll
      for (int k = 0; k < K; ++k)
        w[k][i] = pack2(weight<T>(p.w, p.w_f32, (int64_t)e0 * p.we + k), weight<T>(p.w, p.w_f32, (int64_t)e1 * p.we + k));
      bias[i] = p.bias != nullptr ? pack2(weight<T>(p.bias, p.w_f32, e0), weight<T>(p.bias, p.w_f32, e1)) : 0;
    }
  }
  // row t of the sequence with its state in front of it, -(K - 1) <= t < count
  __device__ __forceinline__ void row(int t, f2 (&v)[NV]) const {
    if (t >= 0) values<T, NV>(ch.load(x + (int64_t)t * p.xl), v);
    else if (init != nullptr) values<T, NV>(ch.load(init + (int64_t)(t + K - 1) * p.il), v);
    else zero(v);
  }
  __device__ __forceinline__ void pre(const f2 (&win)[K][NV], f2 (&v)[NV]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = bias[i];
#pragma unroll
      for (int k = 0; k < K; ++k) v[i] = fma2(w[k][i], win[k][i], v[i]);
    }
  }
};

template <int K, int NV>
__device__ __forceinline__ void shift(f2 (&win)[K][NV]) {
#pragma unroll
  for (int k = 0; k + 1 < K; ++k)
#pragma unroll
    for (int i = 0; i < NV; ++i) win[k][i] = win[k + 1][i];
}

template <typename T, int NV, int K>
__global__ void __launch_bounds__(32 * kWarps) conv_fwd_kernel(const ConvParams p) {
  const int e = (blockIdx.x * 32 + threadIdx.x) * 2 * NV, b = blockIdx.z;
  const int t0 = (blockIdx.y * kWarps + threadIdx.y) * p.run;
  if (e >= p.E) return;
  const int n = row_count(p.lengths, b, p.L);
  const int t1 = min(t0 + p.run, p.L), end = min(t1, n);
  constexpr int U = 4;
  RawRow<T, NV> in[U];  // the next rows, on their way while those before them are worked on
  const T* next = static_cast<const T*>(p.x) + (int64_t)b * p.xb + (int64_t)t0 * p.xl + e;
  auto fetch = [&](int t) {
    const Chan<T, NV> ch{p.vec, e + 1 < p.E ? 1 : 0};
    if (t + U <= end) {
#pragma unroll
      for (int u = 0; u < U; ++u) in[u] = ch.load(next + u * p.xl);
    } else {  // rows behind the end read the last one; nothing is made of them
#pragma unroll
      for (int u = 0; u < U; ++u) in[u] = ch.load(next + min(u, end - 1 - t) * p.xl);
    }
    next += U * p.xl;
  };
  if (t0 < end) fetch(t0);
  const Lane<T, NV, K> ln(p, b, e);
  if (t0 == 0 && p.last != nullptr) {
    T* last = static_cast<T*>(p.last) + (int64_t)b * (K - 1) * p.E + e;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      f2 v[NV];
      ln.row(n - (K - 1) + k, v);
      ln.ch.store(last + (int64_t)k * p.E, v);
    }
  }
  if (t0 >= t1) return;
  T* y = static_cast<T*>(p.y) + (int64_t)b * p.yb + e;
  f2 win[K][NV];
#pragma unroll
  for (int k = 0; k < K; ++k) zero(win[k]);
  if (t0 < n) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) ln.row(t0 - (K - 1) + k, win[k + 1]);
  }
  T* to = y + (int64_t)t0 * p.yl;
#pragma unroll 1
  for (int t = t0; t < end; t += U) {
    RawRow<T, NV> now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = in[u];
    if (t + U < end) fetch(t + U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // (the window turns whatever is stored: within a branch its registers would have to be moved back)
      f2 v[NV];
      shift(win);
      values<T, NV>(now[u], win[K - 1]);
      ln.pre(win, v);
      if (p.silu) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = mul2(v[i], sigmoid2(v[i]));
      }
      if (t + u < end) ln.ch.store(to + u * p.yl, v);
    }
    to += U * p.yl;
  }
  f2 none[NV];
  zero(none);
  for (int t = max(t0, n); t < t1; ++t) ln.ch.store(y + (int64_t)t * p.yl, none);  // padding
}

// d[t] from the window that ends at t
template <typename T, int NV, int K>
__device__ __forceinline__ void slope(const Lane<T, NV, K>& ln, const f2 (&win)[K][NV], f2 (&d)[NV]) {
  if (!ln.p.silu) return;
  f2 v[NV];
  ln.pre(win, v);
  const f2 one = pack2(1.f, 1.f), minus = pack2(-1.f, -1.f);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const f2 s = sigmoid2(v[i]);
    d[i] = mul2(d[i], mul2(s, fma2(v[i], fma2(s, minus, one), one)));
  }
}

// Gradient of the last rows that falls on row t (of the sequence with its state in front of it).
template <typename T, int NV, int K>
__device__ __forceinline__ void add_last(const Lane<T, NV, K>& ln, const ConvGrads& g, int b, int e, int n, int t, f2 (&v)[NV]) {
  const int i = t - n + K - 1;
  if (g.dlast == nullptr || i < 0 || i >= K - 1) return;
  f2 d[NV];
  values<T, NV>(ln.ch.load(static_cast<const T*>(g.dlast) + (int64_t)b * g.dlb + (int64_t)i * g.dll + e), d);
#pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = add2(v[j], d[j]);
}

template <typename T, int NV, int K>
__global__ void __launch_bounds__(32 * kWarps, 2) conv_bwd_kernel(const ConvParams p, const ConvGrads g) {
  __shared__ f2 sums[kWarps][K + 1][32 * NV];
  const int e = (blockIdx.x * 32 + threadIdx.x) * 2 * NV, b = blockIdx.z;
  const int t0 = (blockIdx.y * kWarps + threadIdx.y) * p.run, t1 = min(t0 + p.run, p.L);
  const bool live = e < p.E;
  f2 dw[K + 1][NV];  // dw, then dbias
#pragma unroll
  for (int k = 0; k <= K; ++k) zero(dw[k]);
  if (live) {
    const int n = row_count(p.lengths, b, p.L);
    const Lane<T, NV, K> ln(p, b, e);
    const T* dy = static_cast<const T*>(g.dy) + (int64_t)b * g.dyb + e;
    T* dx = static_cast<T*>(g.dx) + (int64_t)b * g.dxb + e;
    f2 win[K][NV], dwin[K][NV];  // rows t - K + 1 .. t of x, and of d
#pragma unroll
    for (int k = 0; k < K; ++k) { zero(win[k]); zero(dwin[k]); }
    if (t0 == 0 && g.dinit != nullptr) {
      // the rows in front of the first take part in the first K - 1 outputs only
      T* di = static_cast<T*>(g.dinit) + (int64_t)b * (K - 1) * p.E + e;
      f2 out[K][NV];
#pragma unroll
      for (int k = 0; k < K; ++k) zero(out[k]);
#pragma unroll
      for (int k = 0; k < K - 1; ++k) ln.row(k - (K - 1), win[k + 1]);
#pragma unroll
      for (int t = 0; t < K - 1; ++t) {
        if (t < n) {
          f2 d[NV];
          shift(win);
          ln.row(t, win[K - 1]);
          values<T, NV>(ln.ch.load(dy + (int64_t)t * g.dyl), d);
          slope(ln, win, d);
          // row t - K + 1 + k has index t + k among the state's rows
#pragma unroll
          for (int k = 0; k < K - 1 - t; ++k)
#pragma unroll
            for (int i = 0; i < NV; ++i) out[t + k][i] = fma2(ln.w[k][i], d[i], out[t + k][i]);
        }
      }
#pragma unroll
      for (int k = 0; k < K - 1; ++k) {
        add_last<T, NV, K>(ln, g, b, e, n, k - (K - 1), out[k]);
        ln.ch.store(di + (int64_t)k * p.E, out[k]);
      }
    }
    const int end = min(t1, n);  // rows of this run that count
    if (t0 < end) {
#pragma unroll
      for (int k = 0; k < K - 1; ++k) ln.row(t0 - (K - 1) + k, win[k + 1]);
      constexpr int U = 4;
      const int ahead = min(end + K - 1, n);  // rows whose d this run needs
      RawRow<T, NV> xn[U], dn[U];             // the next rows, on their way while those before them are worked on
      const T *xr = ln.x + (int64_t)t0 * p.xl, *dr = dy + (int64_t)t0 * g.dyl;
      auto fetch = [&](int t) {
        if (t + U <= ahead) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            xn[u] = ln.ch.load(xr + u * p.xl);
            dn[u] = ln.ch.load(dr + u * g.dyl);
          }
        } else {  // rows behind the end read the last one; nothing is made of them
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int64_t r = min(u, ahead - 1 - t);
            xn[u] = ln.ch.load(xr + r * p.xl);
            dn[u] = ln.ch.load(dr + r * g.dyl);
          }
        }
        xr += U * p.xl;
        dr += U * g.dyl;
      };
      fetch(t0);
      T* to = dx + (int64_t)(t0 - (K - 1)) * g.dxl;
      // U rows, all of which count and complete the gradient of a row of this run (ALL; the last rows' gradient falls on none
      // of those: t - K + 1 < n - K + 1), or each looked at
      auto rows = [&](auto all, int t, const RawRow<T, NV> (&in)[U], const RawRow<T, NV> (&din)[U]) {
        constexpr bool ALL = decltype(all)::value;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          shift(win);
          shift(dwin);
          values<T, NV>(in[u], win[K - 1]);
          values<T, NV>(din[u], dwin[K - 1]);
          slope(ln, win, dwin[K - 1]);
          if (!ALL && t + u >= ahead) zero(dwin[K - 1]);
          if (ALL || t + u < end) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
              for (int k = 0; k < K; ++k) dw[k][i] = fma2(dwin[K - 1][i], win[k][i], dw[k][i]);
              dw[K][i] = add2(dw[K][i], dwin[K - 1][i]);
            }
          }
          const int at = t + u - (K - 1);  // all of d[at ..  at + K - 1] is at hand
          if (ALL || (at >= t0 && at < end)) {
            f2 v[NV];
            zero(v);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
              for (int k = 0; k < K; ++k) v[i] = fma2(ln.w[k][i], dwin[K - 1 - k][i], v[i]);
            if (!ALL) add_last<T, NV, K>(ln, g, b, e, n, at, v);
            ln.ch.store(to + u * g.dxl, v);
          }
        }
        to += U * g.dxl;
      };
#pragma unroll 1
      for (int t = t0; t < end + K - 1; t += U) {
        RawRow<T, NV> in[U], din[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          in[u] = xn[u];
          din[u] = dn[u];
        }
        if (t + U < ahead) fetch(t + U);
        if (t >= t0 + K - 1 && t + U <= end) rows(std::true_type{}, t, in, din);
        else rows(std::false_type{}, t, in, din);
      }
    }
    f2 none[NV];
    zero(none);
    for (int t = max(t0, n); t < t1; ++t) ln.ch.store(dx + (int64_t)t * g.dxl, none);  // padding
  }
#pragma unroll
  for (int k = 0; k <= K; ++k)
#pragma unroll
    for (int i = 0; i < NV; ++i) sums[threadIdx.y][k][threadIdx.x * NV + i] = dw[k][i];
  __syncthreads();
  const int64_t part = (int64_t)blockIdx.z * gridDim.y + blockIdx.y;
  for (int i = threadIdx.y * 32 + threadIdx.x; i < (K + 1) * 32 * NV; i += 32 * kWarps) {
    const int k = i / (32 * NV), c = i % (32 * NV), to = (blockIdx.x * 32 * NV + c) * 2;
    if (to < p.E) {
      f2 v = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v = add2(v, sums[w][k][c]);
      float a, d;
      unpack2(v, a, d);
      float* out = g.part + (part * (K + 1) + k) * p.E + to;
      out[0] = a;
      if (to + 1 < p.E) out[1] = d;
    }
  }
}

// dw and dbias from the CTAs' parts, in two floats and a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) conv_bwd_join_kernel(const float* part, int64_t parts, int E, int taps, void* dw,
                                                          void* dbias, bool f32) {
  __shared__ Two sums[8][32];
  const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x, per = (int64_t)E * (taps + 1);
  Two v{0.f, 0.f};
  if (i < per) {
#pragma unroll 8
    for (int64_t j = threadIdx.y; j < parts; j += 8) v.add(part[j * per + i]);
  }
  sums[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y != 0 || i >= per) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) v.add(sums[w][threadIdx.x]);
  const int k = (int)(i / E), e = (int)(i % E);
  void* out = k < taps ? dw : dbias;
  if (out == nullptr) return;
  const int64_t at = k < taps ? (int64_t)e * taps + k : e;
  if (f32) static_cast<float*>(out)[at] = v.value();
  else st(static_cast<T*>(out) + at, v.value());
}

// One step: the window moves on by one row, in place.
template <typename T, int NV, int K>
__global__ void __launch_bounds__(128) conv_step_kernel(const ConvStepParams p) {
  const int per = (p.E + 2 * NV - 1) / (2 * NV);
  const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
  if (i >= p.batch * per) return;
  const int64_t b = i / per;
  const int e = (int)(i % per) * 2 * NV;
  const Chan<T, NV> ch{p.vec, e + 1 < p.E ? 1 : 0};
  T* state = static_cast<T*>(p.state) + b * p.sb + e;
  RawRow<T, NV> raw[K];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) raw[k] = ch.load(state + k * p.sl);
  raw[K - 1] = ch.load(static_cast<const T*>(p.x) + b * p.xb + e);
  f2 v[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e0 = e + 2 * j, e1 = e0 + ch.second;
    v[j] = p.bias != nullptr ? pack2(weight<T>(p.bias, p.w_f32, e0), weight<T>(p.bias, p.w_f32, e1)) : 0;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    f2 x[NV];
    values<T, NV>(raw[k], x);
    if (k > 0) ch.store(state + (k - 1) * p.sl, x);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e0 = e + 2 * j, e1 = e0 + ch.second;
      v[j] = fma2(pack2(weight<T>(p.w, p.w_f32, (int64_t)e0 * p.we + k), weight<T>(p.w, p.w_f32, (int64_t)e1 * p.we + k)), x[j], v[j]);
    }
  }
  if (p.silu) {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = mul2(v[j], sigmoid2(v[j]));
  }
  ch.store(static_cast<T*>(p.y) + b * p.E + e, v);
}

bool fits(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Whether rows of these pitches (in elements) hold whole vectors of v elements from p on.
bool rows_fit(const void* p, int64_t s0, int64_t s1, int v, int es) {
  return p == nullptr || (fits(p, (int64_t)v * es) && s0 % v == 0 && s1 % v == 0);
}

// f(pairs of channels that a lane takes): two where addresses and pitches let a row's four be moved at once, else one, whose two
// channels go at once or one by one (*vec).
template <typename Fits, typename F>
int by_vector(Fits&& ok, bool* vec, F&& f) {
  *vec = true;
  if (ok(4)) return f(std::integral_constant<int, 2>{});
  *vec = ok(2);
  return f(std::integral_constant<int, 1>{});
}

template <typename F>
int by_taps(int taps, F&& f) {
  if (taps == 2) return f(std::integral_constant<int, 2>{});
  if (taps == 3) return f(std::integral_constant<int, 3>{});
  return f(std::integral_constant<int, 4>{});
}

template <typename F>
int by_type(int dtype, F&& f) {
  if (dtype == M3_FLOAT32) return f(float{});
  if (dtype == M3_BFLOAT16) return f(__nv_bfloat16{});
  return f(__half{});
}

// Rows that a warp walks, `most` or fewer where that leaves less than about two CTAs an SM (rows between two runs are read twice;
// 4 x 777 x 2048 forward: 9.2 us, in runs of 32 a fifth more).
constexpr int kFwdRun = 32, kBwdRun = 64;  // (8 x 2048 x 2048, us: forward 36, with 64 37; backward 57, with 32 62)
int run_rows(int64_t batch, int64_t L, int64_t E, int most) {
  int run = most;
  while (run > 8 && batch * ((E + 127) / 128) * ((L + run * kWarps - 1) / (run * kWarps)) < 296) run /= 2;
  while (L > (int64_t)run * kWarps * 65535) run *= 2;  // of a grid's rows there are no more
  return run;
}
unsigned runs(int64_t L, int run) { return (unsigned)std::max<int64_t>(1, (L + run * kWarps - 1) / (run * kWarps)); }

}  // namespace

int launch_conv_fwd(ConvParams p, int taps, int dtype, cudaStream_t s) {
  p.run = run_rows(p.batch, p.L, p.E, kFwdRun);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto ok = [&](int v) {
      return p.E % v == 0 && rows_fit(p.x, p.xb, p.xl, v, sizeof(T)) && rows_fit(p.y, p.yb, p.yl, v, sizeof(T)) &&
             rows_fit(p.init, p.ib, p.il, v, sizeof(T)) && fits(p.last, v * sizeof(T));
    };
    return by_vector(ok, &p.vec, [&](auto nv) {
      return by_taps(taps, [&](auto k) {
        const int per = 64 * nv;
        const dim3 grid((unsigned)((p.E + per - 1) / per), runs(p.L, p.run), (unsigned)p.batch);
        conv_fwd_kernel<T, decltype(nv)::value, decltype(k)::value><<<grid, dim3(32, kWarps), 0, s>>>(p);
        return check_launch("conv_fwd_kernel");
      });
    });
  });
}

size_t conv_bwd_workspace(int64_t batch, int64_t L, int64_t E, int taps) {
  return (size_t)batch * runs(L, run_rows(batch, L, E, kBwdRun)) * E * (taps + 1) * sizeof(float);
}

int launch_conv_bwd(ConvParams p, ConvGrads g, int taps, int dtype, void* ws, cudaStream_t s) {
  g.part = static_cast<float*>(ws);
  p.run = run_rows(p.batch, p.L, p.E, kBwdRun);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int es = sizeof(T);
    auto ok = [&](int v) {
      return p.E % v == 0 && rows_fit(p.x, p.xb, p.xl, v, es) && rows_fit(g.dy, g.dyb, g.dyl, v, es) &&
             rows_fit(g.dx, g.dxb, g.dxl, v, es) && rows_fit(p.init, p.ib, p.il, v, es) &&
             rows_fit(g.dlast, g.dlb, g.dll, v, es) && fits(g.dinit, v * es);
    };
    const unsigned ny = runs(p.L, p.run);
    if (p.batch > 0) M3_TRY((by_vector(ok, &p.vec, [&](auto nv) {
      return by_taps(taps, [&](auto k) {
        const int per = 64 * nv;
        const dim3 grid((unsigned)((p.E + per - 1) / per), ny, (unsigned)p.batch);
        conv_bwd_kernel<T, decltype(nv)::value, decltype(k)::value><<<grid, dim3(32, kWarps), 0, s>>>(p, g);
        return check_launch("conv_bwd_kernel");
      });
    })));
    const int64_t per = (int64_t)p.E * (taps + 1);
    conv_bwd_join_kernel<T><<<(unsigned)((per + 31) / 32), dim3(32, 8), 0, s>>>(g.part, (int64_t)ny * p.batch, p.E, taps, g.dw,
                                                                              g.dbias, p.w_f32);
    return check_launch("conv_bwd_join_kernel");
  });
}

int launch_conv_step(ConvStepParams p, int taps, int dtype, cudaStream_t s) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int es = sizeof(T);
    auto ok = [&](int v) {
      return p.E % v == 0 && rows_fit(p.state, p.sb, p.sl, v, es) && rows_fit(p.x, p.xb, 0, v, es) && fits(p.y, v * es);
    };
    return by_vector(ok, &p.vec, [&](auto nv) {
      return by_taps(taps, [&](auto k) {
        const int64_t n = p.batch * ((p.E + 2 * nv - 1) / (2 * nv));
        conv_step_kernel<T, decltype(nv)::value, decltype(k)::value><<<(unsigned)((n + 127) / 128), 128, 0, s>>>(p);
        return check_launch("conv_step_kernel");
      });
    });
  });
}

}  // namespace m3
