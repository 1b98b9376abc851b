// Short depthwise causal convolution over (batch, length, channels), forward, backward, one step:
//   pre[t] = bias + sum_k w[k] x[t - K + 1 + k],   y = pre or silu(pre)
//   d = dy act'(pre),  dx[t] = sum_k w[k] d[t + K - 1 - k],  dw[k] = sum d[t] x[t - K + 1 + k],  dbias = sum d
// Bound by the memory. A lane holds V neighbouring channels (a vector load where the rows allow it),
// a warp 32 V of them, and walks a run of rows with the last K rows in registers, so each element is
// read once but for the K - 1 rows between runs. The backward forms pre again from x.
#include <algorithm>

#include "causal_conv.cuh"
#include "m3_common.cuh"

namespace m3 {
namespace {

constexpr int kRun = 16;        // rows that a warp walks
constexpr int kWarps = 8;

template <typename T, int V>
struct alignas(V * sizeof(T)) Pack { T e[V]; };

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&v)[V]) {
  const Pack<T, V> x = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_f32(x.e[i]);
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&v)[V]) {
  Pack<T, V> x;
#pragma unroll
  for (int i = 0; i < V; ++i) x.e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = x;
}

template <int V>
__device__ __forceinline__ void zero(float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = 0.f;
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

template <typename T, int V, int K>
struct Lane {  // a lane's channels of one sequence
  const ConvParams& p;
  const T* x;
  const T* init;
  int e;
  float w[K][V], bias[V];

  __device__ __forceinline__ Lane(const ConvParams& q, int b, int e_) : p(q), e(e_) {
    x = static_cast<const T*>(p.x) + (int64_t)b * p.xb + e;
    init = p.init != nullptr ? static_cast<const T*>(p.init) + (int64_t)b * p.ib + e : nullptr;
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][i] = weight<T>(p.w, p.w_f32, (int64_t)(e + i) * p.we + k);
      bias[i] = p.bias != nullptr ? weight<T>(p.bias, p.w_f32, e + i) : 0.f;
    }
  }
  // row t of the sequence with its state in front of it, -(K - 1) <= t < count
  __device__ __forceinline__ void row(int t, float (&v)[V]) const {
    if (t >= 0) load<T, V>(x + (int64_t)t * p.xl, v);
    else if (init != nullptr) load<T, V>(init + (int64_t)(t + K - 1) * p.il, v);
    else zero(v);
  }
  __device__ __forceinline__ void pre(const float (&win)[K][V], float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i] = bias[i];
#pragma unroll
      for (int k = 0; k < K; ++k) v[i] = fmaf(w[k][i], win[k][i], v[i]);
    }
  }
};

template <int K, int V>
__device__ __forceinline__ void shift(float (&win)[K][V]) {
#pragma unroll
  for (int k = 0; k + 1 < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) win[k][i] = win[k + 1][i];
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(32 * kWarps) conv_fwd_kernel(const ConvParams p) {
  const int e = (blockIdx.x * 32 + threadIdx.x) * V, b = blockIdx.z;
  const int t0 = (blockIdx.y * kWarps + threadIdx.y) * kRun;
  if (e >= p.E) return;
  const int n = row_count(p.lengths, b, p.L);
  const Lane<T, V, K> ln(p, b, e);
  if (t0 == 0 && p.last != nullptr) {
    T* last = static_cast<T*>(p.last) + (int64_t)b * (K - 1) * p.E + e;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      float v[V];
      ln.row(n - (K - 1) + k, v);
      store<T, V>(last + (int64_t)k * p.E, v);
    }
  }
  const int t1 = min(t0 + kRun, p.L);
  if (t0 >= t1) return;
  T* y = static_cast<T*>(p.y) + (int64_t)b * p.yb + e;
  float win[K][V];
  if (t0 < n) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) ln.row(t0 - (K - 1) + k, win[k + 1]);
  }
  constexpr int U = 8;
#pragma unroll 1
  for (int t = t0; t < t1; t += U) {
    float in[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u < min(t1, n)) load<T, V>(ln.x + (int64_t)(t + u) * p.xl, in[u]);
      else zero(in[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[V];
      shift(win);
#pragma unroll
      for (int i = 0; i < V; ++i) win[K - 1][i] = in[u][i];
      ln.pre(win, v);
      if (t + u < t1) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (p.silu) v[i] *= fast_sigmoid(v[i]);
          if (t + u >= n) v[i] = 0.f;
        }
        store<T, V>(y + (int64_t)(t + u) * p.yl, v);
      }
    }
  }
}

// d[t] from the window that ends at t
template <typename T, int V, int K>
__device__ __forceinline__ void slope(const Lane<T, V, K>& ln, const float (&win)[K][V], float (&d)[V]) {
  if (!ln.p.silu) return;
  float v[V];
  ln.pre(win, v);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float s = fast_sigmoid(v[i]);
    d[i] *= s * fmaf(v[i], 1.f - s, 1.f);
  }
}

// Gradient of the last rows that falls on row t (of the sequence with its state in front of it).
template <typename T, int V, int K>
__device__ __forceinline__ void add_last(const ConvParams& p, const ConvGrads& g, int b, int e, int n, int t, float (&v)[V]) {
  const int i = t - n + K - 1;
  if (g.dlast == nullptr || i < 0 || i >= K - 1) return;
  float d[V];
  load<T, V>(static_cast<const T*>(g.dlast) + (int64_t)b * g.dlb + (int64_t)i * g.dll + e, d);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] += d[j];
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(32 * kWarps) conv_bwd_kernel(const ConvParams p, const ConvGrads g) {
  __shared__ float sums[kWarps][K + 1][32 * V];
  const int e = (blockIdx.x * 32 + threadIdx.x) * V, b = blockIdx.z;
  const int t0 = (blockIdx.y * kWarps + threadIdx.y) * kRun, t1 = min(t0 + kRun, p.L);
  const bool live = e < p.E;
  float dw[K + 1][V];  // dw, then dbias
#pragma unroll
  for (int k = 0; k <= K; ++k) zero(dw[k]);
  if (live) {
    const int n = row_count(p.lengths, b, p.L);
    const Lane<T, V, K> ln(p, b, e);
    const T* dy = static_cast<const T*>(g.dy) + (int64_t)b * g.dyb + e;
    T* dx = static_cast<T*>(g.dx) + (int64_t)b * g.dxb + e;
    float win[K][V], dwin[K][V];  // rows t - K + 1 .. t of x, and of d
    if (t0 == 0 && g.dinit != nullptr) {
      // the rows in front of the first take part in the first K - 1 outputs only
      T* di = static_cast<T*>(g.dinit) + (int64_t)b * (K - 1) * p.E + e;
      float out[K][V];
#pragma unroll
      for (int k = 0; k < K; ++k) zero(out[k]);
#pragma unroll
      for (int k = 0; k < K - 1; ++k) ln.row(k - (K - 1), win[k + 1]);
#pragma unroll
      for (int t = 0; t < K - 1; ++t) {
        if (t < n) {
          float d[V];
          shift(win);
          ln.row(t, win[K - 1]);
          load<T, V>(dy + (int64_t)t * g.dyl, d);
          slope(ln, win, d);
          // row t - K + 1 + k has index t + k among the state's rows
#pragma unroll
          for (int k = 0; k < K - 1 - t; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) out[t + k][i] = fmaf(ln.w[k][i], d[i], out[t + k][i]);
        }
      }
#pragma unroll
      for (int k = 0; k < K - 1; ++k) {
        add_last<T, V, K>(p, g, b, e, n, k - (K - 1), out[k]);
        store<T, V>(di + (int64_t)k * p.E, out[k]);
      }
    }
    if (t0 < t1) {
#pragma unroll
      for (int k = 0; k < K; ++k) { zero(win[k]); zero(dwin[k]); }
      if (t0 < n) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) ln.row(t0 - (K - 1) + k, win[k + 1]);
      }
      constexpr int U = 4;
#pragma unroll 1
      for (int t = t0; t < t1 + K - 1; t += U) {
        float in[U][V], din[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (t + u < min(t1 + K - 1, n)) {
            load<T, V>(ln.x + (int64_t)(t + u) * p.xl, in[u]);
            load<T, V>(dy + (int64_t)(t + u) * g.dyl, din[u]);
          } else {
            zero(in[u]);
            zero(din[u]);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          shift(win);
          shift(dwin);
#pragma unroll
          for (int i = 0; i < V; ++i) { win[K - 1][i] = in[u][i]; dwin[K - 1][i] = din[u][i]; }
          if (t + u < n) slope(ln, win, dwin[K - 1]);
          if (t + u < min(t1, n)) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
#pragma unroll
              for (int k = 0; k < K; ++k) dw[k][i] = fmaf(dwin[K - 1][i], win[k][i], dw[k][i]);
              dw[K][i] += dwin[K - 1][i];
            }
          }
          const int at = t + u - (K - 1);  // all of d[at ..  at + K - 1] is at hand
          if (at >= t0 && at < t1) {
            float v[V];
            zero(v);
            if (at < n) {
#pragma unroll
              for (int i = 0; i < V; ++i)
#pragma unroll
                for (int k = 0; k < K; ++k) v[i] = fmaf(ln.w[k][i], dwin[K - 1 - k][i], v[i]);
              add_last<T, V, K>(p, g, b, e, n, at, v);
            }
            store<T, V>(dx + (int64_t)at * g.dxl, v);
          }
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k <= K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) sums[threadIdx.y][k][threadIdx.x * V + i] = dw[k][i];
  __syncthreads();
  const int64_t part = (int64_t)blockIdx.z * gridDim.y + blockIdx.y;
  for (int i = threadIdx.y * 32 + threadIdx.x; i < (K + 1) * 32 * V; i += 32 * kWarps) {
    const int k = i / (32 * V), c = i % (32 * V), ch = blockIdx.x * 32 * V + c;
    if (ch < p.E) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += sums[w][k][c];
      g.part[(part * (K + 1) + k) * p.E + ch] = v;
    }
  }
}

// dw and dbias from the CTAs' parts: a warp a value's column of parts in 64 bits, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) conv_bwd_join_kernel(const float* part, int64_t parts, int E, int taps, void* dw,
                                                          void* dbias, bool f32) {
  __shared__ double sums[8][32];
  const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x, per = (int64_t)E * (taps + 1);
  double v = 0.0;
  if (i < per) {
#pragma unroll 8
    for (int64_t j = threadIdx.y; j < parts; j += 8) v += (double)part[j * per + i];
  }
  sums[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y != 0 || i >= per) return;
  v = 0.0;
#pragma unroll
  for (int w = 0; w < 8; ++w) v += sums[w][threadIdx.x];
  const int k = (int)(i / E), e = (int)(i % E);
  void* out = k < taps ? dw : dbias;
  if (out == nullptr) return;
  const int64_t at = k < taps ? (int64_t)e * taps + k : e;
  if (f32) static_cast<float*>(out)[at] = (float)v;
  else st(static_cast<T*>(out) + at, (float)v);
}

// One step: the window moves on by one row, in place.
template <typename T, int V, int K>
__global__ void __launch_bounds__(128) conv_step_kernel(const ConvStepParams p) {
  const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const int per = p.E / V;
  if (i >= p.batch * per) return;
  const int64_t b = i / per;
  const int e = (int)(i % per) * V;
  T* state = static_cast<T*>(p.state) + b * p.sb + e;
  float win[K][V], v[V];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) load<T, V>(state + k * p.sl, win[k]);
  load<T, V>(static_cast<const T*>(p.x) + b * p.xb + e, win[K - 1]);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) store<T, V>(state + k * p.sl, win[k + 1]);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    v[j] = p.bias != nullptr ? weight<T>(p.bias, p.w_f32, e + j) : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) v[j] = fmaf(weight<T>(p.w, p.w_f32, (int64_t)(e + j) * p.we + k), win[k][j], v[j]);
    if (p.silu) v[j] *= fast_sigmoid(v[j]);
  }
  store<T, V>(static_cast<T*>(p.y) + b * p.E + e, v);
}

bool fits(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Whether rows of these pitches (in elements) hold whole vectors of v elements from p on.
bool rows_fit(const void* p, int64_t s0, int64_t s1, int v, int es) {
  return p == nullptr || (fits(p, (int64_t)v * es) && s0 % v == 0 && s1 % v == 0);
}

// f(V) with the channels that a lane takes: as many as fill `most` bytes, where base addresses and
// pitches allow it; else 4 bytes' worth; else one.
template <typename T, int MOST, typename Fits, typename F>
int by_vector(Fits&& ok, F&& f) {
  constexpr int es = sizeof(T), V0 = MOST / es, V1 = 4 / es;
  if (ok(V0)) return f(std::integral_constant<int, V0>{});
  if (V1 > 1 && ok(V1)) return f(std::integral_constant<int, V1>{});
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

unsigned runs(int64_t L) { return (unsigned)((L + kRun * kWarps - 1) / (kRun * kWarps)); }

}  // namespace

int launch_conv_fwd(const ConvParams& p, int taps, int dtype, cudaStream_t s) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto ok = [&](int v) {
      return p.E % v == 0 && rows_fit(p.x, p.xb, p.xl, v, sizeof(T)) && rows_fit(p.y, p.yb, p.yl, v, sizeof(T)) &&
             rows_fit(p.init, p.ib, p.il, v, sizeof(T)) && fits(p.last, v * sizeof(T));
    };
    return by_vector<T, 16>(ok, [&](auto v) {
      return by_taps(taps, [&](auto k) {
        const int per = 32 * v;
        const dim3 grid((unsigned)((p.E + per - 1) / per), std::max(1u, runs(p.L)), (unsigned)p.batch);
        conv_fwd_kernel<T, decltype(v)::value, decltype(k)::value><<<grid, dim3(32, kWarps), 0, s>>>(p);
        return check_launch("conv_fwd_kernel");
      });
    });
  });
}

size_t conv_bwd_workspace(int64_t batch, int64_t L, int64_t E, int taps) {
  return (size_t)batch * std::max(1u, runs(L)) * E * (taps + 1) * sizeof(float);
}

int launch_conv_bwd(const ConvParams& p, ConvGrads g, int taps, int dtype, void* ws, cudaStream_t s) {
  g.part = static_cast<float*>(ws);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int es = sizeof(T);
    auto ok = [&](int v) {
      return p.E % v == 0 && rows_fit(p.x, p.xb, p.xl, v, es) && rows_fit(g.dy, g.dyb, g.dyl, v, es) &&
             rows_fit(g.dx, g.dxb, g.dxl, v, es) && rows_fit(p.init, p.ib, p.il, v, es) &&
             rows_fit(g.dlast, g.dlb, g.dll, v, es) && fits(g.dinit, v * es);
    };
    const unsigned ny = std::max(1u, runs(p.L));
    if (p.batch > 0) M3_TRY((by_vector<T, es == 4 ? 16 : 8>(ok, [&](auto v) {
      return by_taps(taps, [&](auto k) {
        const int per = 32 * v;
        const dim3 grid((unsigned)((p.E + per - 1) / per), ny, (unsigned)p.batch);
        conv_bwd_kernel<T, decltype(v)::value, decltype(k)::value><<<grid, dim3(32, kWarps), 0, s>>>(p, g);
        return check_launch("conv_bwd_kernel");
      });
    })));
    const int64_t per = (int64_t)p.E * (taps + 1);
    conv_bwd_join_kernel<T><<<(unsigned)((per + 31) / 32), dim3(32, 8), 0, s>>>(g.part, (int64_t)ny * p.batch, p.E, taps, g.dw,
                                                                              g.dbias, p.w_f32);
    return check_launch("conv_bwd_join_kernel");
  });
}

int launch_conv_step(const ConvStepParams& p, int taps, int dtype, cudaStream_t s) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int es = sizeof(T);
    auto ok = [&](int v) {
      return p.E % v == 0 && rows_fit(p.state, p.sb, p.sl, v, es) && rows_fit(p.x, p.xb, 0, v, es) && fits(p.y, v * es);
    };
    return by_vector<T, es == 4 ? 16 : 8>(ok, [&](auto v) {
      return by_taps(taps, [&](auto k) {
        const int64_t n = p.batch * (p.E / v);
        conv_step_kernel<T, decltype(v)::value, decltype(k)::value><<<(unsigned)((n + 127) / 128), 128, 0, s>>>(p);
        return check_launch("conv_step_kernel");
      });
    });
  });
}

}  // namespace m3
