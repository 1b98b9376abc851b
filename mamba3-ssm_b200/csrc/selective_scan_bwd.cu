// Selective state space scan, backward. With g_t the gradient of h_t and dy that of y before the gate,
//   g_t = C_t dy_t + exp(dt_{t+1} A) g_{t+1},   w_t = g_t exp(dt_t A) h_{t-1}
//   dB_t = sum_e g_t dt u,  dC_t = sum_e dy h_t,  dA = sum_t w_t dt
//   du = dt sum_n g B + D dy,  d(dt) = u sum_n g B + sum_n A w,  dz = dout y silu'(z),  dD = sum dy u
// The forward keeps the state in front of every eighth step, so eight steps at a time are done
// again and then walked backwards, all in registers: P lanes share a channel and hold K states each,
// M channels follow one another in a lane. Sums over the states of a channel (three a step and channel)
// and over the channels (dB, dC) are formed for eight steps together by halving exchanges; M and K set
// how many there are of each. Sums over channels of other warps go through shared memory, those of
// other CTAs through the workspace and a second kernel, in a fixed order.
#include <algorithm>

#include "selective_scan.cuh"

namespace m3 {
namespace {

constexpr int TT = kSelTile, TS = TT + 4, SUB = kSelSub;

template <int K, int P, int M, int NT>
struct BwdSmem {
  static constexpr int NP = K * P, EC = NT / P * M, W = NT / 32;
  float dt[EC][TS], dx[EC][TS], dy[EC][TS];
  float B[NP][TS], C[NP][TS];
  float s0[TT][EC + 1], s1[TT][EC + 1], s2[TT][EC + 1];  // sums over the states: C h, g B, A w
  float red[W][2 * SUB * NP];
  double ends[2][NT];
};

template <typename T, int K, int P, int M, int NT>
__global__ void __launch_bounds__(NT) sel_bwd_kernel(const SelScanParams p, const SelScanGrads g) {
  using S = BwdSmem<K, P, M, NT>;
  constexpr int NP = S::NP, EC = S::EC, W = S::W, Q = 32 / P;
  constexpr int JN = TT * EC / NT, JB = (TT * NP + NT - 1) / NT;
  static_assert(NT % EC == 0, "a thread brings and stores one channel");
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& sh = *reinterpret_cast<S*>(smem_raw);
  const int tid = threadIdx.x, q = tid % P, lane = tid & 31, warp = tid >> 5;
  const int Eg = p.E / p.G, tiles = (Eg + EC - 1) / EC;
  const int gr = blockIdx.x / tiles, tile = blockIdx.x % tiles;
  const int e_first = gr * Eg + tile * EC, e_end = (gr + 1) * Eg;
  const int b = blockIdx.z, c = blockIdx.y;
  const int beg = c * p.chunk, end = min(p.L, beg + p.chunk);
  const int len = seq_len(p.lengths, b, p.L);
  const int nsave = (p.L + SUB - 1) / SUB;
  const int le = tid % EC, lt = tid / EC;
  const int lec = min(e_first + le, e_end - 1);
  const bool lelive = e_first + le < e_end;

  int el[M], ec[M];
  float A[M][K], gv[M][K];
  double dA[M][K];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    el[m] = m * (NT / P) + tid / P;
    ec[m] = min(e_first + el[m], e_end - 1);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int n = q * K + k;
      A[m][k] = n < p.N ? p.A[(int64_t)ec[m] * p.N + n] : 0.f;
      dA[m][k] = 0.0;
      gv[m][k] = 0.f;
      if (p.nchunk > 1) gv[m][k] = p.states[(((int64_t)b * p.nchunk + c) * p.E + ec[m]) * NP + n];
      else if (g.dstate != nullptr && n < p.N) gv[m][k] = g.dstate[((int64_t)b * p.E + ec[m]) * p.N + n];
      if (e_first + el[m] >= e_end) gv[m][k] = 0.f;
    }
  }
  const float bias = p.bias != nullptr ? p.bias[lec] : 0.f;
  const float Dv = p.D != nullptr ? p.D[lec] : 0.f;
  double sumD = 0.0, sumbias = 0.0;

  const T* up = static_cast<const T*>(p.u.p) + (int64_t)b * p.u.sb + lec;
  const T* zp = p.z.p != nullptr ? static_cast<const T*>(p.z.p) + (int64_t)b * p.z.sb + lec : nullptr;
  const T* yp = static_cast<const T*>(g.dy.p) + (int64_t)b * g.dy.sb + lec;
  T* dup = static_cast<T*>(const_cast<void*>(g.du.p)) + (int64_t)b * g.du.sb + lec;
  T* dzp = zp != nullptr ? static_cast<T*>(const_cast<void*>(g.dz.p)) + (int64_t)b * g.dz.sb + lec : nullptr;
  const int64_t doff = (int64_t)b * p.delta.sb + lec, ddoff = (int64_t)b * g.ddelta.sb + lec;
  const int64_t boff = (int64_t)b * p.B.sb + gr * p.Bg, coff = (int64_t)b * p.C.sb + gr * p.Cg;
  auto put_ddelta = [&](int t, float v) {
    const int64_t i = ddoff + (int64_t)t * g.ddelta.sl;
    void* d = const_cast<void*>(g.ddelta.p);
    if (p.delta_f32) static_cast<float*>(d)[i] = v;
    else st(static_cast<T*>(d) + i, v);
  };

  // padding behind the sequence: gradients of zero
  const int first_pad = max(beg, len);
  for (int t = first_pad + lt; t < end; t += NT / EC)
    if (lelive) {
      st(dup + (int64_t)t * g.du.sl, 0.f);
      put_ddelta(t, 0.f);
      if (zp != nullptr) st(dzp + (int64_t)t * g.dz.sl, 0.f);
    }

  const int last = min(end, len);
  for (int t0 = last > beg ? beg + (last - 1 - beg) / TT * TT : beg - TT; t0 >= beg; t0 -= TT) {
#pragma unroll
    for (int j = 0; j < JN; ++j) {
      const int t = lt + j * (NT / EC);
      float dt = 0.f, u = 0.f, dy = 0.f;
      if (t0 + t < len && lelive) {
        u = ld(up + (int64_t)(t0 + t) * p.u.sl);
        dt = step_size(ld_any<T>(p.delta.p, p.delta_f32, doff + (int64_t)(t0 + t) * p.delta.sl) + bias, p.softplus);
        dy = ld(yp + (int64_t)(t0 + t) * g.dy.sl);
        if (zp != nullptr) {
          const float z = ld(zp + (int64_t)(t0 + t) * p.z.sl);
          dy *= z * fast_sigmoid(z);
        }
      }
      sh.dt[le][t] = dt;
      sh.dx[le][t] = dt * u;
      sh.dy[le][t] = dy;
    }
#pragma unroll 4
    for (int j = 0; j < JB; ++j) {
      const int i = tid + j * NT, n = i % NP, t = i / NP;
      if (t < TT) {
        const bool in = n < p.N && t0 + t < len;
        const int row = (n % K) * P + n / K;
        sh.B[row][t] = in ? ld_any<T>(p.B.p, p.bc_f32, boff + (int64_t)(t0 + t) * p.B.sl + n) : 0.f;
        sh.C[row][t] = in ? ld_any<T>(p.C.p, p.bc_f32, coff + (int64_t)(t0 + t) * p.C.sl + n) : 0.f;
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int ts = TT - SUB; ts >= 0; ts -= SUB) {
      if (t0 + ts >= len) continue;  // the same for the whole CTA
      float acc[2 * SUB * K];  // dB, then dC: (step, k)
#pragma unroll
      for (int i = 0; i < 2 * SUB * K; ++i) acc[i] = 0.f;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        float dt[SUB], dx[SUB], dy[SUB], S0[SUB], S1[SUB], S2[SUB];
#pragma unroll
        for (int i = 0; i < SUB; i += 4) {
          const float4 a = *reinterpret_cast<const float4*>(&sh.dt[el[m]][ts + i]);
          const float4 x = *reinterpret_cast<const float4*>(&sh.dx[el[m]][ts + i]);
          const float4 y = *reinterpret_cast<const float4*>(&sh.dy[el[m]][ts + i]);
          dt[i] = a.x; dt[i + 1] = a.y; dt[i + 2] = a.z; dt[i + 3] = a.w;
          dx[i] = x.x; dx[i + 1] = x.y; dx[i + 2] = x.z; dx[i + 3] = x.w;
          dy[i] = y.x; dy[i + 1] = y.y; dy[i + 2] = y.z; dy[i + 3] = y.w;
        }
#pragma unroll
        for (int i = 0; i < SUB; ++i) S0[i] = S1[i] = S2[i] = 0.f;
        const float* sv = p.save + (((int64_t)b * nsave + (t0 + ts) / SUB) * p.E + ec[m]) * NP + q * K;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float h_in = sv[k], A2 = A[m][k] * kLog2e;
          float bv[SUB], cv[SUB], av[SUB], hv[SUB];
#pragma unroll
          for (int i = 0; i < SUB; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(&sh.B[k * P + q][ts + i]);
            const float4 y = *reinterpret_cast<const float4*>(&sh.C[k * P + q][ts + i]);
            bv[i] = x.x; bv[i + 1] = x.y; bv[i + 2] = x.z; bv[i + 3] = x.w;
            cv[i] = y.x; cv[i + 1] = y.y; cv[i + 2] = y.z; cv[i + 3] = y.w;
          }
          float h = h_in;
#pragma unroll
          for (int i = 0; i < SUB; ++i) {
            av[i] = ex2(dt[i] * A2);
            h = fmaf(av[i], h, dx[i] * bv[i]);
            hv[i] = h;
            S0[i] = fmaf(cv[i], h, S0[i]);
          }
          float gk = gv[m][k], da = 0.f;
#pragma unroll
          for (int i = SUB - 1; i >= 0; --i) {
            gk = fmaf(cv[i], dy[i], gk);
            acc[i * K + k] = fmaf(gk, dx[i], acc[i * K + k]);
            acc[(SUB + i) * K + k] = fmaf(dy[i], hv[i], acc[(SUB + i) * K + k]);
            S1[i] = fmaf(gk, bv[i], S1[i]);
            gk *= av[i];
            const float w = gk * (i > 0 ? hv[i - 1] : h_in);
            S2[i] = fmaf(A[m][k], w, S2[i]);
            da = fmaf(dt[i], w, da);
          }
          gv[m][k] = gk;
          dA[m][k] += (double)da;
        }
        int at = spread_sum<SUB, P>(S0, q);
        spread_sum<SUB, P>(S1, q);
        spread_sum<SUB, P>(S2, q);
#pragma unroll
        for (int j = 0; j < (SUB > P ? SUB / P : 1); ++j) {
          sh.s0[ts + at + j][el[m]] = S0[j];
          sh.s1[ts + at + j][el[m]] = S1[j];
          sh.s2[ts + at + j][el[m]] = S2[j];
        }
      }
      // over the warp's channels: lanes q, q + P, ... ; then over the warps
      const int at = spread_sum<2 * SUB * K, Q, P>(acc, lane / P);
#pragma unroll
      for (int j = 0; j < 2 * SUB * K / Q; ++j) {
        const int i = at + j, w = i / (SUB * K), t = i / K % SUB, k = i % K;
        sh.red[warp][(t * 2 + w) * NP + q * K + k] = acc[j];
      }
      __syncthreads();
      for (int i = tid; i < 2 * SUB * NP; i += NT) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += sh.red[w][i];
        const int t = t0 + ts + i / (2 * NP);
        if (t < len) g.part_bc[((((int64_t)b * p.L + t) * p.G + gr) * tiles + tile) * 2 * NP + i % (2 * NP)] = v;
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < JN; ++j) {
      const int t = lt + j * (NT / EC);
      if (t0 + t < len && lelive) {
        const float u = ld(up + (int64_t)(t0 + t) * p.u.sl);
        const float dt = sh.dt[le][t], dy = sh.dy[le][t], s1 = sh.s1[t][le];
        st(dup + (int64_t)(t0 + t) * g.du.sl, fmaf(dt, s1, Dv * dy));
        float dd = fmaf(u, s1, sh.s2[t][le]);
        if (p.softplus)
          dd *= fast_sigmoid(ld_any<T>(p.delta.p, p.delta_f32, doff + (int64_t)(t0 + t) * p.delta.sl) + bias);
        put_ddelta(t0 + t, dd);
        sumbias += (double)dd;
        sumD += (double)(dy * u);
        if (zp != nullptr) {
          const float z = ld(zp + (int64_t)(t0 + t) * p.z.sl), dout = ld(yp + (int64_t)(t0 + t) * g.dy.sl);
          const float sg = fast_sigmoid(z);
          st(dzp + (int64_t)(t0 + t) * g.dz.sl, dout * fmaf(Dv, u, sh.s0[t][le]) * (sg * fmaf(z, 1.f - sg, 1.f)));
        }
      }
    }
    __syncthreads();
  }
  // this piece's part of dA, dD, dbias; the gradient of the first state
  float* pa = g.part_a + ((int64_t)b * p.nchunk + c) * p.E * (NP + 2);
#pragma unroll
  for (int m = 0; m < M; ++m) {
    if (e_first + el[m] < e_end) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        pa[(int64_t)ec[m] * (NP + 2) + q * K + k] = (float)dA[m][k];
        if (g.dh0 != nullptr && c == 0 && q * K + k < p.N) g.dh0[((int64_t)b * p.E + ec[m]) * p.N + q * K + k] = gv[m][k];
      }
    }
  }
  sh.ends[0][tid] = sumD;
  sh.ends[1][tid] = sumbias;
  __syncthreads();
  if (tid < EC && lelive) {
    double sd = 0.0, sb = 0.0;
#pragma unroll
    for (int j = 0; j < NT / EC; ++j) { sd += sh.ends[0][tid + j * EC]; sb += sh.ends[1][tid + j * EC]; }
    pa[(int64_t)lec * (NP + 2) + NP] = (float)sd;
    pa[(int64_t)lec * (NP + 2) + NP + 1] = (float)sb;
  }
}

// The gradient of the state that each piece of the sequence passes to the piece in front of it,
// for a gradient of zero from behind, and the sum of its step sizes: g <- exp(dt A) (C dy + g).
template <typename T, int K, int P, int NT>
__global__ void __launch_bounds__(NT) sel_bwd_piece_kernel(const SelScanParams p, const SelScanGrads g) {
  constexpr int NP = K * P, EC = NT / P, JN = TT * EC / NT, JB = (TT * NP + NT - 1) / NT;
  __shared__ __align__(16) float sdt[EC][TS], sdy[EC][TS], sC[NP][TS];
  const int tid = threadIdx.x, q = tid % P, el = tid / P;
  const int Eg = p.E / p.G, tiles = (Eg + EC - 1) / EC;
  const int gr = blockIdx.x / tiles, e_first = gr * Eg + (blockIdx.x % tiles) * EC, e_end = (gr + 1) * Eg;
  const int b = blockIdx.z, c = blockIdx.y;
  const int beg = c * p.chunk, end = min(p.L, beg + p.chunk);
  const int len = seq_len(p.lengths, b, p.L);
  const int ec = min(e_first + el, e_end - 1);
  const int le = tid % EC, lt = tid / EC, lec = min(e_first + le, e_end - 1);
  float A2[K], gk[K], dts = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int n = q * K + k;
    A2[k] = n < p.N ? p.A[(int64_t)ec * p.N + n] * kLog2e : 0.f;
    gk[k] = 0.f;
  }
  const float bias = p.bias != nullptr ? p.bias[lec] : 0.f;
  const T* zp = p.z.p != nullptr ? static_cast<const T*>(p.z.p) + (int64_t)b * p.z.sb + lec : nullptr;
  const T* yp = static_cast<const T*>(g.dy.p) + (int64_t)b * g.dy.sb + lec;
  const int64_t doff = (int64_t)b * p.delta.sb + lec, coff = (int64_t)b * p.C.sb + gr * p.Cg;
  const int last = min(end, len);
  for (int t0 = last > beg ? beg + (last - 1 - beg) / TT * TT : beg - TT; t0 >= beg; t0 -= TT) {
#pragma unroll
    for (int j = 0; j < JN; ++j) {
      const int t = lt + j * (NT / EC);
      float dt = 0.f, dy = 0.f;
      if (t0 + t < len) {
        dt = step_size(ld_any<T>(p.delta.p, p.delta_f32, doff + (int64_t)(t0 + t) * p.delta.sl) + bias, p.softplus);
        dy = ld(yp + (int64_t)(t0 + t) * g.dy.sl);
        if (zp != nullptr) {
          const float z = ld(zp + (int64_t)(t0 + t) * p.z.sl);
          dy *= z * fast_sigmoid(z);
        }
      }
      sdt[le][t] = dt;
      sdy[le][t] = dy;
    }
#pragma unroll 4
    for (int j = 0; j < JB; ++j) {
      const int i = tid + j * NT, n = i % NP, t = i / NP;
      if (t < TT)
        sC[(n % K) * P + n / K][t] = n < p.N && t0 + t < len
            ? ld_any<T>(p.C.p, p.bc_f32, coff + (int64_t)(t0 + t) * p.C.sl + n) : 0.f;
    }
    __syncthreads();
#pragma unroll 2
    for (int t = TT - 4; t >= 0; t -= 4) {
      const float4 d4 = *reinterpret_cast<const float4*>(&sdt[el][t]);
      const float4 y4 = *reinterpret_cast<const float4*>(&sdy[el][t]);
      const float dv[4] = {d4.x, d4.y, d4.z, d4.w}, yv[4] = {y4.x, y4.y, y4.z, y4.w};
      dts += (dv[0] + dv[1]) + (dv[2] + dv[3]);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float4 c4 = *reinterpret_cast<const float4*>(&sC[k * P + q][t]);
        const float cv[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
        for (int i = 3; i >= 0; --i) gk[k] = ex2(dv[i] * A2[k]) * fmaf(cv[i], yv[i], gk[k]);
      }
    }
    __syncthreads();
  }
  if (e_first + el < e_end) {
    const int64_t at = ((int64_t)b * p.nchunk + c) * p.E + ec;
#pragma unroll
    for (int k = 0; k < K; ++k) p.states[at * NP + q * K + k] = gk[k];
    if (q == 0) p.dtsum[at] = dts;
  }
}

// The gradients that enter the pieces from behind, last piece first.
__global__ void __launch_bounds__(256) sel_bwd_carry_kernel(const SelScanParams p, const float* dstate, int NP) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (int64_t)p.E * NP) return;
  const int e = (int)(i / NP), n = (int)(i % NP), b = blockIdx.y;
  const float A2 = n < p.N ? p.A[(int64_t)e * p.N + n] * kLog2e : 0.f;
  float v = dstate != nullptr && n < p.N ? dstate[((int64_t)b * p.E + e) * p.N + n] : 0.f;
  const int64_t pitch = (int64_t)p.E * NP;
  float* st = p.states + (int64_t)b * p.nchunk * pitch + i;
  const float* ds = p.dtsum + (int64_t)b * p.nchunk * p.E + e;
#pragma unroll 4
  for (int c = p.nchunk - 1; c >= 0; --c) {
    const float local = st[c * pitch], a = ex2(A2 * ds[(int64_t)c * p.E]);
    st[c * pitch] = v;
    v = fmaf(a, v, local);
  }
}

// dB and dC from the channel tiles' parts, dA, dD and dbias from the pieces' and sequences', each in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) sel_bwd_join_kernel(const SelScanParams p, const SelScanGrads g, int NP, int tiles,
                                                         int64_t rows, unsigned bc_ctas) {
  if (blockIdx.x < bc_ctas) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * 2 * NP) return;
    const int64_t row = i / (2 * NP);
    const int c = (int)(i % (2 * NP)), n = c % NP;
    if (n >= p.N) return;
    const int64_t pos = row / p.G;
    float v = 0.f;
    if ((int)(pos % p.L) < seq_len(p.lengths, (int)(pos / p.L), p.L)) {
      const float* src = g.part_bc + row * tiles * 2 * NP + c;
#pragma unroll 8
      for (int j = 0; j < tiles; ++j) v += src[(int64_t)j * 2 * NP];
    }
    void* out = c < NP ? g.dB : g.dC;
    if (p.bc_f32) static_cast<float*>(out)[row * p.N + n] = v;
    else st(static_cast<T*>(out) + row * p.N + n, v);
    return;
  }
  const int64_t i = (int64_t)(blockIdx.x - bc_ctas) * 256 + threadIdx.x;
  if (i >= (int64_t)p.E * (NP + 2)) return;
  const int e = (int)(i / (NP + 2)), n = (int)(i % (NP + 2));
  double v = 0.0;
  for (int j = 0; j < p.batch * p.nchunk; ++j) v += (double)g.part_a[(int64_t)j * p.E * (NP + 2) + i];
  if (n < p.N) g.dA[(int64_t)e * p.N + n] = (float)v;
  else if (n == NP && g.dD != nullptr) g.dD[e] = (float)v;
  else if (n == NP + 1 && g.dbias != nullptr) g.dbias[e] = (float)v;
}

template <typename F>
int by_type(int dtype, F&& f) {
  if (dtype == M3_FLOAT32) return f(float{});
  if (dtype == M3_BFLOAT16) return f(__nv_bfloat16{});
  return f(__half{});
}

// states a lane, lanes, channels a lane by the padded number of states
template <int K, int P, int M> struct KPM { static constexpr int k = K, p = P, m = M; };
template <typename F>
int by_states(int n, F&& f) {
  switch (sel_padded_states(n)) {
    case 4: return f(KPM<2, 2, 2>{});
    case 8: return f(KPM<2, 4, 2>{});
    case 16: return f(KPM<2, 8, 2>{});
    case 32: return f(KPM<2, 16, 2>{});
    case 64: return f(KPM<2, 32, 2>{});
    default: return f(KPM<4, 32, 1>{});
  }
}

constexpr int kBwdThreads = 128;

struct BwdPlan {
  int np, tiles, nchunk, chunk;
  size_t bc, a, states, dtsum;  // floats
};

BwdPlan plan(const SelScanParams& p, int sms) {
  BwdPlan w;
  w.np = sel_padded_states(p.N);
  by_states(p.N, [&](auto l) {
    using L_ = decltype(l);
    const int ec = kBwdThreads / L_::p * L_::m, Eg = p.E / p.G;
    w.tiles = (Eg + ec - 1) / ec;
    w.nchunk = sel_pieces(p, std::max(1, L_::p / L_::m), sms, &w.chunk);
    return 0;
  });
  w.bc = (size_t)p.batch * p.L * p.G * w.tiles * 2 * w.np;
  w.a = (size_t)p.batch * w.nchunk * p.E * (w.np + 2);
  w.states = w.nchunk > 1 ? (size_t)p.batch * w.nchunk * p.E * w.np : 0;
  w.dtsum = w.nchunk > 1 ? (size_t)p.batch * w.nchunk * p.E : 0;
  return w;
}

}  // namespace

size_t sel_scan_bwd_workspace(const SelScanParams& p, int sms) {
  const BwdPlan w = plan(p, sms);
  return (w.bc + w.a + w.states + w.dtsum) * sizeof(float);
}

int launch_sel_scan_bwd(SelScanParams p, SelScanGrads g, int dtype, void* ws, cudaStream_t s) {
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  const BwdPlan w = plan(p, sms);
  g.part_bc = static_cast<float*>(ws);
  g.part_a = g.part_bc + w.bc;
  p.states = g.part_a + w.a;
  p.dtsum = p.states + w.states;
  p.nchunk = w.nchunk;
  p.chunk = w.chunk;
  const int Eg = p.E / p.G;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    M3_TRY(by_states(p.N, [&](auto l) {
      using L_ = decltype(l);
      constexpr int K = L_::k, P = L_::p, M = L_::m, NT = kBwdThreads;
      if (p.batch == 0) return (int)M3_OK;  // parameters' gradients of zero
      if (p.nchunk > 1) {
        constexpr int ec = NT / P;
        const dim3 grid((unsigned)(p.G * ((Eg + ec - 1) / ec)), (unsigned)p.nchunk, (unsigned)p.batch);
        sel_bwd_piece_kernel<T, K, P, NT><<<grid, NT, 0, s>>>(p, g);
        M3_TRY(check_launch("sel_bwd_piece_kernel"));
        const dim3 cgrid((unsigned)(((int64_t)p.E * w.np + 255) / 256), (unsigned)p.batch);
        sel_bwd_carry_kernel<<<cgrid, 256, 0, s>>>(p, g.dstate, w.np);
        M3_TRY(check_launch("sel_bwd_carry_kernel"));
      }
      using S = BwdSmem<K, P, M, NT>;
      static std::atomic<bool> done[kMaxDevices];
      M3_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(&sel_bwd_kernel<T, K, P, M, NT>), sizeof(S), done));
      const dim3 grid((unsigned)(p.G * w.tiles), (unsigned)p.nchunk, (unsigned)p.batch);
      sel_bwd_kernel<T, K, P, M, NT><<<grid, NT, sizeof(S), s>>>(p, g);
      return check_launch("sel_bwd_kernel");
    }));
    const int64_t rows = (int64_t)p.batch * p.L * p.G;
    const unsigned bc_ctas = (unsigned)((rows * 2 * w.np + 255) / 256);
    const unsigned a_ctas = (unsigned)(((int64_t)p.E * (w.np + 2) + 255) / 256);
    sel_bwd_join_kernel<T><<<bc_ctas + a_ctas, 256, 0, s>>>(p, g, w.np, w.tiles, rows, bc_ctas);
    return check_launch("sel_bwd_join_kernel");
  });
}

}  // namespace m3
