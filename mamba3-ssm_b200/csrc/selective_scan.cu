// Selective state space scan, forward and single step: per channel e and state n
//   dt = softplus(delta + bias),  h_t = exp(dt A) h_{t-1} + dt u B_t,  y = (sum_n C_t h_t + D u) silu(z)
// P lanes share a channel and hold K states each in registers (n = q K + k). A CTA walks the
// sequence in tiles of 32 steps: u and delta of its channels and B, C are brought into shared
// memory as (row, step), so that a lane reads four steps of one operand at once; the sums over a
// channel's lanes are formed for several steps together by halving exchanges, and y leaves
// through shared memory in whole rows. The next tile's operands are loaded while this one is scanned.
#include <algorithm>

#include "selective_scan.cuh"

namespace m3 {
namespace {

constexpr int TT = kSelTile;
constexpr int TS = TT + 4;  // row pitch: rows that a warp reads together start on different banks

// steps whose sums over the lanes are formed together
template <int P> constexpr int group_steps() { return P < 4 ? 4 : P; }

template <int K, int P, int NT>
struct FwdSmem {
  static constexpr int NP = K * P, EC = NT / P;
  float dt[EC][TS], dx[EC][TS];
  float B[NP][TS], C[NP][TS];
  float y[TT][EC + 8];
};

// OUT: the scan proper. Else only the state that a piece of the sequence leaves, from zero, and
// the sum of its step sizes.
template <typename T, int K, int P, int NT, bool OUT>
__global__ void __launch_bounds__(NT) sel_scan_kernel(const SelScanParams p) {
  using S = FwdSmem<K, P, NT>;
  constexpr int NP = S::NP, EC = S::EC, JN = TT * EC / NT, JB = (TT * NP + NT - 1) / NT, GS = group_steps<P>();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& sh = *reinterpret_cast<S*>(smem_raw);
  const int tid = threadIdx.x, q = tid % P, el = tid / P;
  const int Eg = p.E / p.G, tiles = (Eg + EC - 1) / EC;
  const int g = blockIdx.x / tiles, e_first = g * Eg + (blockIdx.x % tiles) * EC, e_end = (g + 1) * Eg;
  const int b = blockIdx.z, c = blockIdx.y;
  const int beg = c * p.chunk, end = min(p.L, beg + p.chunk);
  const int len = seq_len(p.lengths, b, p.L);
  const int e = e_first + el;
  const bool live = e < e_end;
  const int ec = live ? e : e_end - 1;
  // element (t, le) of a tile that this thread brings and stores
  const int le = tid % EC, lt = tid / EC;
  const int lec = min(e_first + le, e_end - 1);
  const bool lelive = e_first + le < e_end;

  float A2[K], h[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int n = q * K + k;
    A2[k] = n < p.N ? p.A[(int64_t)ec * p.N + n] * kLog2e : 0.f;
    h[k] = 0.f;
    if (OUT) {
      if (p.nchunk > 1) h[k] = p.states[(((int64_t)b * p.nchunk + c) * p.E + ec) * NP + n];
      else if (p.h0 != nullptr && n < p.N) h[k] = p.h0[((int64_t)b * p.E + ec) * p.N + n];
    }
  }
  const float bias = p.bias != nullptr ? p.bias[lec] : 0.f;
  const float Dv = OUT && p.D != nullptr ? p.D[lec] : 0.f;
  float dts = 0.f;

  const T* up = static_cast<const T*>(p.u.p) + (int64_t)b * p.u.sb + lec;
  const T* zp = OUT && p.z.p != nullptr ? static_cast<const T*>(p.z.p) + (int64_t)b * p.z.sb + lec : nullptr;
  T* yp = OUT ? static_cast<T*>(const_cast<void*>(p.y.p)) + (int64_t)b * p.y.sb + lec : nullptr;
  const int64_t doff = (int64_t)b * p.delta.sb + lec;
  const int64_t boff = (int64_t)b * p.B.sb + g * p.Bg, coff = (int64_t)b * p.C.sb + g * p.Cg;

  float ru[JN], rd[JN];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int j = 0; j < JN; ++j) {
      const int t = t0 + lt + j * (NT / EC);
      ru[j] = rd[j] = 0.f;
      if (t < len) {
        ru[j] = ld(up + (int64_t)t * p.u.sl);
        rd[j] = ld_any<T>(p.delta.p, p.delta_f32, doff + (int64_t)t * p.delta.sl);
      }
    }
  };
  if (beg < len) fetch(beg);
  int t0 = beg;
  for (; t0 < end && t0 < len; t0 += TT) {
#pragma unroll
    for (int j = 0; j < JN; ++j) {
      const int t = lt + j * (NT / EC);
      const float dt = t0 + t < len ? step_size(rd[j] + bias, p.softplus) : 0.f;
      sh.dt[le][t] = dt;
      sh.dx[le][t] = dt * ru[j];
    }
#pragma unroll 4
    for (int j = 0; j < JB; ++j) {
      const int i = tid + j * NT, n = i % NP, t = i / NP;
      if (t < TT) {
        const bool in = n < p.N && t0 + t < len;
        const int row = (n % K) * P + n / K;
        sh.B[row][t] = in ? ld_any<T>(p.B.p, p.bc_f32, boff + (int64_t)(t0 + t) * p.B.sl + n) : 0.f;
        if (OUT) sh.C[row][t] = in ? ld_any<T>(p.C.p, p.bc_f32, coff + (int64_t)(t0 + t) * p.C.sl + n) : 0.f;
      }
    }
    __syncthreads();
    float zu[JN], zz[JN];
    if (OUT) {
#pragma unroll
      for (int j = 0; j < JN; ++j) {
        const int t = t0 + lt + j * (NT / EC);
        zu[j] = ru[j];
        zz[j] = zp != nullptr && t < len ? ld(zp + (int64_t)t * p.z.sl) : 0.f;
      }
    }
    if (t0 + TT < end && t0 + TT < len) fetch(t0 + TT);
#pragma unroll 1
    for (int tg = 0; tg < TT; tg += GS) {
      float yv[GS];
#pragma unroll
      for (int i = 0; i < GS; ++i) yv[i] = 0.f;
#pragma unroll
      for (int i4 = 0; i4 < GS; i4 += 4) {
        if (OUT && p.save != nullptr && (tg + i4) % kSelSub == 0 && live && t0 + tg + i4 < len) {
          float* sv = p.save + (((int64_t)b * ((p.L + kSelSub - 1) / kSelSub) + (t0 + tg + i4) / kSelSub) * p.E + e) * NP + q * K;
#pragma unroll
          for (int k = 0; k < K; ++k) sv[k] = h[k];
        }
        const float4 d4 = *reinterpret_cast<const float4*>(&sh.dt[el][tg + i4]);
        const float4 x4 = *reinterpret_cast<const float4*>(&sh.dx[el][tg + i4]);
        const float dv[4] = {d4.x, d4.y, d4.z, d4.w}, xv[4] = {x4.x, x4.y, x4.z, x4.w};
        if (!OUT) dts += (dv[0] + dv[1]) + (dv[2] + dv[3]);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float4 b4 = *reinterpret_cast<const float4*>(&sh.B[k * P + q][tg + i4]);
          const float bv[4] = {b4.x, b4.y, b4.z, b4.w};
          float cv[4];
          if (OUT) {
            const float4 c4 = *reinterpret_cast<const float4*>(&sh.C[k * P + q][tg + i4]);
            cv[0] = c4.x; cv[1] = c4.y; cv[2] = c4.z; cv[3] = c4.w;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            h[k] = fmaf(ex2(dv[i] * A2[k]), h[k], xv[i] * bv[i]);
            if (OUT) yv[i4 + i] = fmaf(h[k], cv[i], yv[i4 + i]);
          }
        }
      }
      if (OUT) {
        const int at = spread_sum<GS, P>(yv, q);
#pragma unroll
        for (int j = 0; j < GS / P; ++j) sh.y[tg + at + j][el] = yv[j];
      }
    }
    __syncthreads();
    if (OUT) {
#pragma unroll
      for (int j = 0; j < JN; ++j) {
        const int t = lt + j * (NT / EC);
        if (lelive && t0 + t < end) {
          float v = fmaf(Dv, zu[j], sh.y[t][le]);
          if (zp != nullptr) v *= zz[j] * fast_sigmoid(zz[j]);
          st(yp + (int64_t)(t0 + t) * p.y.sl, t0 + t < len ? v : 0.f);
        }
      }
    }
  }
  if (OUT) {
    for (int t = t0 + lt; t < end; t += NT / EC)  // padding
      if (lelive) st(yp + (int64_t)t * p.y.sl, 0.f);
    if (p.h_last != nullptr && c == p.nchunk - 1 && live) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (q * K + k < p.N) p.h_last[((int64_t)b * p.E + e) * p.N + q * K + k] = h[k];
    }
  } else if (live) {
    const int64_t at = ((int64_t)b * p.nchunk + c) * p.E + e;
#pragma unroll
    for (int k = 0; k < K; ++k) p.states[at * NP + q * K + k] = h[k];
    if (q == 0) p.dtsum[at] = dts;
  }
}

// The states that enter the pieces, from those that each leaves by itself: h <- exp(A sum dt) h + local.
__global__ void __launch_bounds__(256) sel_carry_kernel(const SelScanParams p, int NP) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (int64_t)p.E * NP) return;
  const int e = (int)(i / NP), n = (int)(i % NP), b = blockIdx.y;
  const float A2 = n < p.N ? p.A[(int64_t)e * p.N + n] * kLog2e : 0.f;
  float h = p.h0 != nullptr && n < p.N ? p.h0[((int64_t)b * p.E + e) * p.N + n] : 0.f;
  const int64_t pitch = (int64_t)p.E * NP;
  float* st = p.states + (int64_t)b * p.nchunk * pitch + i;
  const float* ds = p.dtsum + (int64_t)b * p.nchunk * p.E + e;
#pragma unroll 4
  for (int c = 0; c < p.nchunk; ++c) {
    const float local = st[c * pitch], a = ex2(A2 * ds[(int64_t)c * p.E]);
    st[c * pitch] = h;
    h = fmaf(a, h, local);
  }
}

// One step: y and the state in place. P lanes a channel, K states each.
template <typename T, int K, int P>
__global__ void __launch_bounds__(256) sel_step_kernel(const SelStepParams p, bool vec) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t ch = i / P;
  const int q = (int)(i % P);
  const bool live = ch < p.batch * p.E;
  const int64_t b = live ? ch / p.E : 0;
  const int e = live ? (int)(ch % p.E) : 0;
  const int g = e / (p.E / p.G);
  float raw = ld_any<T>(p.delta, p.delta_f32, b * p.sd + e);
  const float u = ld(static_cast<const T*>(p.u) + b * p.su + e);
  if (p.bias != nullptr) raw += p.bias[e];
  float* st_ = p.state + b * p.sstate + (int64_t)e * p.N;
  float h[K], y = 0.f;
  if (vec) {
#pragma unroll
    for (int k = 0; k < K; k += 4) {
      const int n = q * K + k;
      const float4 v = live && n < p.N ? *reinterpret_cast<const float4*>(st_ + n) : make_float4(0.f, 0.f, 0.f, 0.f);
      h[k] = v.x; h[k + 1] = v.y; h[k + 2] = v.z; h[k + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) h[k] = live && q * K + k < p.N ? st_[q * K + k] : 0.f;
  }
  const float dt = step_size(raw, p.softplus), dx = dt * u;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int n = q * K + k;
    if (n < p.N) {
      const float a = ex2(dt * (p.A[(int64_t)e * p.N + n] * kLog2e));
      h[k] = fmaf(a, h[k], dx * ld_any<T>(p.B, p.bc_f32, b * p.sB + g * p.sBg + n));
      y = fmaf(h[k], ld_any<T>(p.C, p.bc_f32, b * p.sC + g * p.sCg + n), y);
    }
  }
#pragma unroll
  for (int m = P / 2; m >= 1; m /= 2) y += __shfl_xor_sync(0xffffffffu, y, m);
  if (!live) return;
  if (vec) {
#pragma unroll
    for (int k = 0; k < K; k += 4)
      if (q * K + k < p.N) *reinterpret_cast<float4*>(st_ + q * K + k) = make_float4(h[k], h[k + 1], h[k + 2], h[k + 3]);
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (q * K + k < p.N) st_[q * K + k] = h[k];
  }
  if (q == 0) {
    if (p.D != nullptr) y = fmaf(p.D[e], u, y);
    if (p.z != nullptr) {
      const float z = ld(static_cast<const T*>(p.z) + b * p.sz + e);
      y *= z * fast_sigmoid(z);
    }
    st(static_cast<T*>(p.y) + b * p.sy + e, y);
  }
}

template <typename F>
int by_type(int dtype, F&& f) {
  if (dtype == M3_FLOAT32) return f(float{});
  if (dtype == M3_BFLOAT16) return f(__nv_bfloat16{});
  return f(__half{});
}

template <typename T, int K, int P, bool OUT>
int launch_pass(const SelScanParams& p, cudaStream_t s) {
  constexpr int NT = 128;
  using S = FwdSmem<K, P, NT>;
  static std::atomic<bool> done[kMaxDevices];
  const void* kernel = reinterpret_cast<const void*>(&sel_scan_kernel<T, K, P, NT, OUT>);
  M3_TRY(ensure_dynamic_smem(kernel, sizeof(S), done));
  const int Eg = p.E / p.G;
  const dim3 grid((unsigned)(p.G * ((Eg + S::EC - 1) / S::EC)), (unsigned)p.nchunk, (unsigned)p.batch);
  sel_scan_kernel<T, K, P, NT, OUT><<<grid, NT, sizeof(S), s>>>(p);
  return check_launch("sel_scan_kernel");
}

// f(K, P) as types: lanes and states a lane by the padded number of states
template <int K, int P> struct KP { static constexpr int k = K, p = P; };
template <typename F>
int by_states(int n, F&& f) {
  switch (sel_padded_states(n)) {
    case 4: return f(KP<4, 1>{});
    case 8: return f(KP<4, 2>{});
    case 16: return f(KP<4, 4>{});
    case 32: return f(KP<4, 8>{});
    case 64: return f(KP<4, 16>{});
    default: return f(KP<4, 32>{});
  }
}

}  // namespace

// Pieces that the sequence is cut into: one, unless the channels alone leave most of the GPU idle. A
// piece's state has to be formed ahead (about as much work again), so cutting begins where
// there are less than a quarter of the warps that keep an SM busy.
int sel_pieces(const SelScanParams& p, int lanes, int sms, int* chunk) {
  const int64_t warps = (int64_t)p.batch * p.E * lanes / 32 + 1, want = (int64_t)sms * 16;
  int n = 1;
  if (warps * 4 <= want) n = (int)std::min<int64_t>(want / warps, (p.L + 4 * kSelTile - 1) / (4 * kSelTile));
  n = std::max(1, std::min(n, 4096));
  int64_t len = (p.L + n - 1) / n;
  len = (len + kSelTile - 1) / kSelTile * kSelTile;
  *chunk = (int)std::max<int64_t>(len, kSelTile);
  return std::max<int>(1, (int)((p.L + *chunk - 1) / *chunk));
}

size_t sel_scan_save_bytes(int64_t batch, int64_t L, int64_t E, int N) {
  return (size_t)batch * ((L + kSelSub - 1) / kSelSub) * E * sel_padded_states(N) * sizeof(float);
}

size_t sel_scan_fwd_workspace(const SelScanParams& p, int sms) {
  int chunk = 0;
  const int np = sel_padded_states(p.N), n = sel_pieces(p, np / 4, sms, &chunk);
  return n == 1 ? 0 : (size_t)p.batch * n * p.E * (np + 1) * sizeof(float);
}

int launch_sel_scan_fwd(SelScanParams p, int dtype, void* ws, cudaStream_t s) {
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  const int np = sel_padded_states(p.N);
  p.nchunk = sel_pieces(p, np / 4, sms, &p.chunk);
  if (p.nchunk > 1) {
    p.states = static_cast<float*>(ws);
    p.dtsum = p.states + (int64_t)p.batch * p.nchunk * p.E * np;
  }
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    return by_states(p.N, [&](auto kp) {
      using L_ = decltype(kp);
      if (p.nchunk > 1) {
        M3_TRY((launch_pass<T, L_::k, L_::p, false>(p, s)));
        const dim3 grid((unsigned)(((int64_t)p.E * np + 255) / 256), (unsigned)p.batch);
        sel_carry_kernel<<<grid, 256, 0, s>>>(p, np);
        M3_TRY(check_launch("sel_carry_kernel"));
      }
      return launch_pass<T, L_::k, L_::p, true>(p, s);
    });
  });
}

int launch_sel_step(const SelStepParams& p, int dtype, cudaStream_t s) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    return by_states(p.N, [&](auto kp) {
      using L_ = decltype(kp);
      const int64_t threads = p.batch * p.E * L_::p;
      const bool vec = p.N % 4 == 0 && p.sstate % 4 == 0 && (reinterpret_cast<uintptr_t>(p.state) & 15) == 0;
      sel_step_kernel<T, L_::k, L_::p><<<(unsigned)((threads + 255) / 256), 256, 0, s>>>(p, vec);
      return check_launch("sel_step_kernel");
    });
  });
}

}  // namespace m3
