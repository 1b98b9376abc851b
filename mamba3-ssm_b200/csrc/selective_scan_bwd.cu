// Selective state space scan, backward. With g_t the gradient of h_t and dy that of y before the gate,
//   g_t = C_t dy_t + exp(dt_{t+1} A) g_{t+1},   w_t = g_t exp(dt_t A) h_{t-1}
//   dB_t = sum_e g_t dt u,  dC_t = sum_e dy h_t,  dA = sum_t w_t dt
//   du = dt sum_n g B + D dy,  d(dt) = u sum_n g B + sum_n A w,  dz = dout y silu'(z),  dD = sum dy u
// The forward keeps the state in front of every eighth step, so eight steps at a time are done
// again and then walked backwards, all in registers: P lanes share a channel and hold K states each,
// M channels follow one another in a lane. Sums over the states of a channel (three a step and channel)
// and over the channels (dB, dC) are formed for eight steps together by halving exchanges; K sets how many
// exchanges the first take, M K how many the second. Sums over channels of other warps go through shared
// memory, those of other CTAs through the workspace and a second kernel, in a fixed order.
//
// Bound by the issue of instructions and by shared memory's port together: about 24 instructions a step, channel and
// state, four of them reads of shared memory (dt, dx, dy, B, C, whose broadcasts cost as much as other reads), at 0.43 a clock
// with the two warps a scheduler that 255 registers leave. 8 x 2048 x 2048 x 16 of bf16 with a gate take 855 us and 18 to join
// (742 MB, the forward's too, would take 113); the same in other shapes, us: K = 2, P = 8, M = 2 with all sums by shuffles 2690;
// K = 4, P = 4, M = 1 1043; 64 threads 838 and 31 to join; 85 or 128 registers, which spill, 1320 to 1360; four steps at a time,
// with the upper four's first state formed again, 1008 at two CTAs an SM and 1077 at three.
#include <algorithm>

#include "selective_scan.cuh"

namespace m3 {
namespace {

constexpr int TT = kSelTile, TS = kSelPitch, SUB = kSelSub;

template <int K, int P, int M, int NT>
struct BwdSmem {
  static constexpr int NP = K * P, EC = NT / P * M, W = NT / 32;
  // (channel, step): dt, dy, u; and what becomes a gradient in its place: dt u -> du, the softplus's slope ->
  // ddelta, dout silu'(z) -> dz
  float dt[EC][TS], dy[EC][TS], u[EC][TS], du[EC][TS], dd[EC][TS], dz[EC][TS];
  float B[NP][TS], C[NP][TS];
  float red[W][2 * SUB * NP];
  float h[2][M][NT][K];  // the states in front of these eight steps and of the next eight (earlier) ones, by thread
  // sums over the tiles so far, by thread, in two floats: those of one tile are formed in one
  Two dA[M * K][NT], dD[M][NT], dbias[M][NT];
};

// Copies 16 bytes (or K floats) into shared memory without passing registers.
template <int K>
__device__ __forceinline__ void copy_ahead(float* to, const float* from) {
  const unsigned dst = (unsigned)__cvta_generic_to_shared(to);
  if constexpr (K == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from));
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(from), "n"(K * 4));
}
__device__ __forceinline__ void copies_sent() { asm volatile("cp.async.commit_group;"); }
template <int LEFT>
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

__device__ __forceinline__ void lds4(const float* p, f2& a, f2& b) {
  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p);
  a = v.x;
  b = v.y;
}

template <typename T, int K, int P, int M, int NT, bool FAST>
__global__ void __launch_bounds__(NT) sel_bwd_kernel(const SelScanParams p, const SelScanGrads g) {
  using S = BwdSmem<K, P, M, NT>;
  constexpr int NP = S::NP, EC = S::EC, W = S::W, Q = 32 / P;
  constexpr int R = TT * EC / 2 / NT > 0 ? TT * EC / 2 / NT : 1;  // steps of a pair of channels that a thread brings and stores
  constexpr int RR = R < 4 ? R : 4;                               // of them at a time
  constexpr int SP = SUB / P > 0 ? SUB / P : 1;                   // steps of a channel whose sums a lane ends up with
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& sh = *reinterpret_cast<S*>(smem_raw);
  const int tid = threadIdx.x, q = tid % P, lane = tid & 31, warp = tid >> 5;
  // register k of a lane holds state q K + (k ^ flip): neighbouring channels of a warp hold them in orders in which
  // what one gives to the other when dB and dC are summed stands in the same registers, without selecting
  constexpr int FLIP = K < Q ? K : Q;  // orders
  const int flip = lane / P % FLIP;
  const int Eg = p.E / p.G, tiles = (Eg + EC - 1) / EC;
  const int gr = blockIdx.x / tiles, tile = blockIdx.x % tiles;
  const int e_first = gr * Eg + tile * EC, e_end = (gr + 1) * Eg;
  const int b = blockIdx.z, c = blockIdx.y;
  const int beg = c * p.chunk, end = min(p.L, beg + p.chunk);
  const int len = seq_len(p.lengths, b, p.L);
  const int nsave = (p.L + SUB - 1) / SUB;
  const int le = tid % (EC / 2) * 2, lt = tid / (EC / 2) * R;
  const bool brings = TT * EC / 2 >= NT * R || lt < TT;
  const int l0 = e_first + le < e_end ? e_first + le : e_first, second = l0 + 1 < e_end ? 1 : 0;
  const bool lelive = brings && e_first + le < e_end, lelive1 = brings && e_first + le + 1 < e_end;
  const bool vu = FAST || p.vec_u, vd = FAST || p.vec_d, vz = FAST || p.vec_z, vy = FAST || p.vec_y;

  int nk[K], row[K];  // states, and their rows among B and C
#pragma unroll
  for (int k = 0; k < K; ++k) {
    nk[k] = q * K + (k ^ flip);
    row[k] = (k ^ flip) * P + q;
  }
  float A2[M][K], gv[M][K];
  const float* save[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const int e = e_first + m * (NT / P) + tid / P, ec = min(e, e_end - 1);
    save[m] = p.save + ((int64_t)b * nsave * p.E + ec) * NP + q * K;
    sh.dD[m][tid] = sh.dbias[m][tid] = Two{0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int n = nk[k];
      A2[m][k] = n < p.N ? p.A[(int64_t)ec * p.N + n] * kLog2e : 0.f;
      sh.dA[m * K + k][tid] = Two{0.f, 0.f};
      gv[m][k] = 0.f;
      if (e < e_end) {
        if (p.nchunk > 1) gv[m][k] = p.states[(((int64_t)b * p.nchunk + c) * p.E + ec) * NP + n];
        else if (g.dstate != nullptr && n < p.N) gv[m][k] = g.dstate[((int64_t)b * p.E + ec) * p.N + n];
      }
    }
  }
  const float bias0 = p.bias != nullptr ? p.bias[l0] : 0.f, bias1 = p.bias != nullptr ? p.bias[l0 + second] : 0.f;
  float Dv[M];
#pragma unroll
  for (int m = 0; m < M; ++m) Dv[m] = p.D != nullptr ? p.D[min(e_first + m * (NT / P) + tid / P, e_end - 1)] : 0.f;

  const bool has_z = p.z.p != nullptr;
  const T* up = static_cast<const T*>(p.u.p) + (int64_t)b * p.u.sb + l0;
  const T* zp = has_z ? static_cast<const T*>(p.z.p) + (int64_t)b * p.z.sb + l0 : nullptr;
  const T* yp = static_cast<const T*>(g.dy.p) + (int64_t)b * g.dy.sb + l0;
  T* dup = static_cast<T*>(const_cast<void*>(g.du.p)) + (int64_t)b * g.du.sb + l0;
  T* dzp = has_z ? static_cast<T*>(const_cast<void*>(g.dz.p)) + (int64_t)b * g.dz.sb + l0 : nullptr;
  const int64_t doff = (int64_t)b * p.delta.sb + l0, ddoff = (int64_t)b * g.ddelta.sb + l0;
  const int64_t boff = (int64_t)b * p.B.sb + gr * p.Bg, coff = (int64_t)b * p.C.sb + gr * p.Cg;
  auto put_ddelta = [&](int t, float v0, float v1) {
    const int64_t i = ddoff + (int64_t)t * g.ddelta.sl;
    void* d = const_cast<void*>(g.ddelta.p);
    if (!FAST && p.delta_f32) store2<float>(static_cast<float*>(d) + i, g.vec_dd, second, v0, v1);
    else store2<T>(static_cast<T*>(d) + i, FAST || g.vec_dd, second, v0, v1);
  };

  // padding behind the sequence: gradients of zero, by all threads of a pair of channels (also those that bring nothing)
  if (e_first + le < e_end)
    for (int t = max(beg, len) + tid / (EC / 2); t < end; t += NT / (EC / 2)) {
      store2<T>(dup + (int64_t)t * g.du.sl, FAST || g.vec_du, second, 0.f, 0.f);
      put_ddelta(t, 0.f, 0.f);
      if (has_z) store2<T>(dzp + (int64_t)t * g.dz.sl, FAST || g.vec_dz, second, 0.f, 0.f);
    }

  const int last = min(end, len);
  // the states in front of the eight steps that begin at 8 s, or nothing in front of this piece; a thread reads what it copied itself
  auto copy_states = [&](int s, int half) {
    if (s * SUB >= beg) {
#pragma unroll
      for (int m = 0; m < M; ++m) copy_ahead<K>(sh.h[half][m][tid], save[m] + (int64_t)s * p.E * NP);
    }
    copies_sent();
  };
  int half = 0;
  if (last > beg) copy_states((last - 1) / SUB, 0);
  for (int t0 = last > beg ? beg + (last - 1 - beg) / TT * TT : beg - TT; t0 >= beg; t0 -= TT) {
    const int top = min(TT, last - t0);  // steps of the tile that count
    float dA[M][K], sumD[M], sumbias[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
      sumD[m] = sumbias[m] = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) dA[m][k] = 0.f;
    }
    if (brings) {
#pragma unroll 1
      for (int j0 = 0; j0 < R; j0 += RR) {
        Raw2<T> ru[RR], rz[RR], ry[RR];
        std::conditional_t<FAST, Raw2<T>, RawAny<T>> rd[RR];
#pragma unroll
        for (int j = 0; j < RR; ++j) {  // rows behind the end read the last one; nothing is made of them
          const int64_t t = min(t0 + lt + j0 + j, len - 1);
          ru[j] = load2<T>(up + t * p.u.sl, vu, second);
          load2_any<T>(rd[j], p.delta.p, p.delta_f32, doff + t * p.delta.sl, vd, second);
          ry[j] = load2<T>(yp + t * g.dy.sl, vy, second);
          if (has_z) rz[j] = load2<T>(zp + t * p.z.sl, vz, second);
        }
        float v[6][2][RR];
#pragma unroll
        for (int j = 0; j < RR; ++j) {
          const float2 r = value2<T>(rd[j], p.delta_f32), raw = make_float2(r.x + bias0, r.y + bias1);
          float2 dt = step_size2(raw, p.softplus), sl = p.softplus ? sigmoid2(raw) : make_float2(1.f, 1.f);
          float2 u = value2(ru[j]), dy = value2(ry[j]), zf = make_float2(0.f, 0.f);
          if (has_z) {
            const float2 z = value2(rz[j]), sg = sigmoid2(z);
            zf.x = dy.x * (sg.x * fmaf(z.x, 1.f - sg.x, 1.f));
            zf.y = dy.y * (sg.y * fmaf(z.y, 1.f - sg.y, 1.f));
            dy.x *= z.x * sg.x;
            dy.y *= z.y * sg.y;
          }
          const bool in0 = t0 + lt + j0 + j < len && lelive, in1 = in0 && lelive1;
          v[0][0][j] = in0 ? dt.x : 0.f; v[0][1][j] = in1 ? dt.y : 0.f;
          v[1][0][j] = in0 ? dy.x : 0.f; v[1][1][j] = in1 ? dy.y : 0.f;
          v[2][0][j] = in0 ? u.x : 0.f; v[2][1][j] = in1 ? u.y : 0.f;
          v[3][0][j] = v[0][0][j] * v[2][0][j]; v[3][1][j] = v[0][1][j] * v[2][1][j];
          v[4][0][j] = in0 ? sl.x : 0.f; v[4][1][j] = in1 ? sl.y : 0.f;
          v[5][0][j] = zf.x; v[5][1][j] = zf.y;
        }
        const int t = lt + j0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          put_steps<RR>(&sh.dt[le + i][t], v[0][i]);
          put_steps<RR>(&sh.dy[le + i][t], v[1][i]);
          put_steps<RR>(&sh.u[le + i][t], v[2][i]);
          put_steps<RR>(&sh.du[le + i][t], v[3][i]);
          put_steps<RR>(&sh.dd[le + i][t], v[4][i]);
          if (has_z) put_steps<RR>(&sh.dz[le + i][t], v[5][i]);
        }
      }
    }
    {
      BcTile<T, K, P, NT, FAST> tb;
      tb.fetch(p.B.p, p.bc_f32, boff, p.B.sl, p.vec_B, p.N, t0, len, tid);
      tb.put(sh.B, p.bc_f32, p.N, t0, len, tid);
      tb.fetch(p.C.p, p.bc_f32, coff, p.C.sl, p.vec_C, p.N, t0, len, tid);
      tb.put(sh.C, p.bc_f32, p.N, t0, len, tid);
    }
    __syncthreads();
#pragma unroll 1
    for (int ts = (top - 1) / SUB * SUB; ts >= 0; ts -= SUB) {
      copy_states((t0 + ts) / SUB - 1, half ^ 1);
      copies_done<1>();
      f2 acc[2][K][SUB / 2];  // dB, dC
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < SUB / 2; ++j) acc[i][k][j] = 0;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const int el = m * (NT / P) + tid / P;
        f2 dt[SUB / 2], dx[SUB / 2], dy[SUB / 2], S0[SUB / 2], S1[SUB / 2], S2[SUB / 2];
#pragma unroll
        for (int j = 0; j < SUB / 2; j += 2) {
          lds4(&sh.dt[el][ts + 2 * j], dt[j], dt[j + 1]);
          lds4(&sh.du[el][ts + 2 * j], dx[j], dx[j + 1]);
          lds4(&sh.dy[el][ts + 2 * j], dy[j], dy[j + 1]);
        }
#pragma unroll
        for (int j = 0; j < SUB / 2; ++j) S0[j] = S1[j] = S2[j] = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float h_in = sh.h[half][m][tid][k ^ flip];
          const f2 A2k = pack2(A2[m][k], A2[m][k]), mean = pack2(kEx2Mean, kEx2Mean);
          f2 bv[SUB / 2], cv[SUB / 2];
          float av[SUB], hv[SUB];
#pragma unroll
          for (int j = 0; j < SUB / 2; j += 2) {
            lds4(&sh.B[row[k]][ts + 2 * j], bv[j], bv[j + 1]);
            lds4(&sh.C[row[k]][ts + 2 * j], cv[j], cv[j + 1]);
          }
          float h = h_in;
#pragma unroll
          for (int j = 0; j < SUB / 2; ++j) {
            float x0, x1;
            unpack2(fma2(dt[j], A2k, mean), av[2 * j], av[2 * j + 1]);
            av[2 * j] = ex2(av[2 * j]);
            av[2 * j + 1] = ex2(av[2 * j + 1]);
            unpack2(mul2(dx[j], bv[j]), x0, x1);
            hv[2 * j] = fmaf(av[2 * j], h, x0);
            h = hv[2 * j + 1] = fmaf(av[2 * j + 1], hv[2 * j], x1);
            const f2 hh = pack2(hv[2 * j], hv[2 * j + 1]);
            S0[j] = fma2(cv[j], hh, S0[j]);
            acc[1][k][j] = fma2(dy[j], hh, acc[1][k][j]);
          }
          float gk = gv[m][k];
          f2 da = 0;
#pragma unroll
          for (int j = SUB / 2 - 1; j >= 0; --j) {
            float c0, c1, y0, y1;
            unpack2(cv[j], c0, c1);
            unpack2(dy[j], y0, y1);
            const float g1 = fmaf(c1, y1, gk), a1 = g1 * av[2 * j + 1];
            const float g0 = fmaf(c0, y0, a1);
            gk = g0 * av[2 * j];
            const f2 gg = pack2(g0, g1);
            const f2 w = pack2(gk * (j > 0 ? hv[2 * j - 1] : h_in), a1 * hv[2 * j]);
            acc[0][k][j] = fma2(gg, dx[j], acc[0][k][j]);
            S1[j] = fma2(gg, bv[j], S1[j]);
            S2[j] = fma2(A2k, w, S2[j]);  // times log2(e)
            da = fma2(dt[j], w, da);
          }
          gv[m][k] = gk;
          float d0, d1;
          unpack2(da, d0, d1);
          dA[m][k] += d0 + d1;
        }
        float s0[SUB], s1[SUB], s2[SUB];
#pragma unroll
        for (int j = 0; j < SUB / 2; ++j) {
          unpack2(S0[j], s0[2 * j], s0[2 * j + 1]);
          unpack2(S1[j], s1[2 * j], s1[2 * j + 1]);
          unpack2(S2[j], s2[2 * j], s2[2 * j + 1]);
        }
        if (has_z) spread_sum<SUB, P>(s0, q);
        spread_sum<SUB, P>(s1, q);
        const int at = spread_sum<SUB, P>(s2, q);
        __syncwarp();  // the channel's lanes have read dt u
        if (P <= SUB || q % (P > SUB ? P / SUB : 1) == 0) {
          const int t = ts + at;
          float u[SP], d[SP], y[SP], sl[SP], zf[SP], du[SP];
          get_steps<SP>(&sh.u[el][t], u);
          get_steps<SP>(&sh.dt[el][t], d);
          get_steps<SP>(&sh.dy[el][t], y);
          get_steps<SP>(&sh.dd[el][t], sl);
          if (has_z) get_steps<SP>(&sh.dz[el][t], zf);
          float sD = 0.f, sb = 0.f;
#pragma unroll
          for (int j = 0; j < SP; ++j) {
            du[j] = fmaf(d[j], s1[j], Dv[m] * y[j]);
            sl[j] *= fmaf(u[j], s1[j], 0.6931471805599453f * s2[j]);
            if (has_z) zf[j] *= fmaf(Dv[m], u[j], s0[j]);
            sD = fmaf(y[j], u[j], sD);
            sb += sl[j];
          }
          put_steps<SP>(&sh.du[el][t], du);
          put_steps<SP>(&sh.dd[el][t], sl);
          if (has_z) put_steps<SP>(&sh.dz[el][t], zf);
          sumD[m] += sD;
          sumbias[m] += sb;
        }
      }
      // over the warp's channels: lanes q, q + P, ..; exchanges of registers k and k ^ o first, then of steps; then over the warps
      float v[K][2 * SUB];
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < SUB / 2; ++j) unpack2(acc[i][k][j], v[k][i * SUB + 2 * j], v[k][i * SUB + 2 * j + 1]);
      constexpr int KL = K / FLIP;  // registers k that are left
#pragma unroll
      for (int o = FLIP / 2; o >= 1; o /= 2)
#pragma unroll
        for (int k = 0; k < K; ++k)
          if ((k & (FLIP - 1)) < o) {
#pragma unroll
            for (int i = 0; i < 2 * SUB; ++i) v[k][i] += __shfl_xor_sync(0xffffffffu, v[k + o][i], o * P);
          }
#pragma unroll
      for (int kl = 0; kl < KL; ++kl) {
        const int k = kl * FLIP;
        const int at = spread_sum<2 * SUB, Q / FLIP, P * FLIP>(v[k], lane / (P * FLIP));
#pragma unroll
        for (int j = 0; j < 2 * SUB / (Q / FLIP); ++j) {
          const int i = at + j, w = i / SUB, t = i % SUB;
          sh.red[warp][(t * 2 + w) * NP + nk[k]] = v[k][j];
        }
      }
      __syncthreads();
      for (int i = tid; i < 2 * SUB * NP; i += NT) {
        float r = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) r += sh.red[w][i];
        const int t = t0 + ts + i / (2 * NP);
        if (t < len) g.part_bc[((((int64_t)b * p.L + t) * p.G + gr) * tiles + tile) * 2 * NP + i % (2 * NP)] = r;
      }
      __syncthreads();
      half ^= 1;
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
      sh.dD[m][tid].add(sumD[m]);
      sh.dbias[m][tid].add(sumbias[m]);
#pragma unroll
      for (int k = 0; k < K; ++k) sh.dA[m * K + k][tid].add(dA[m][k]);
    }
    if (lelive) {
#pragma unroll 1
      for (int j0 = 0; j0 < R; j0 += RR) {
        float v[3][2][RR];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          get_steps<RR>(&sh.du[le + i][lt + j0], v[0][i]);
          get_steps<RR>(&sh.dd[le + i][lt + j0], v[1][i]);
          if (has_z) get_steps<RR>(&sh.dz[le + i][lt + j0], v[2][i]);
        }
#pragma unroll
        for (int j = 0; j < RR; ++j) {
          const int t = t0 + lt + j0 + j;
          if (t < last) {
            store2<T>(dup + (int64_t)t * g.du.sl, FAST || g.vec_du, second, v[0][0][j], v[0][1][j]);
            put_ddelta(t, v[1][0][j], v[1][1][j]);
            if (has_z) store2<T>(dzp + (int64_t)t * g.dz.sl, FAST || g.vec_dz, second, v[2][0][j], v[2][1][j]);
          }
        }
      }
    }
    __syncthreads();
  }
  // this piece's part of dA, dD, dbias; the gradient of the first state
  float* pa = g.part_a + ((int64_t)b * p.nchunk + c) * p.E * (NP + 2);
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const int e = e_first + m * (NT / P) + tid / P;
    Two sumD = sh.dD[m][tid], sumbias = sh.dbias[m][tid];
#pragma unroll
    for (int o = P / 2; o >= 1; o /= 2) {
      sumD.add(sumD.shuffled(o));
      sumbias.add(sumbias.shuffled(o));
    }
    if (e < e_end) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        pa[(int64_t)e * (NP + 2) + nk[k]] = sh.dA[m * K + k][tid].value();
        if (g.dh0 != nullptr && c == 0 && nk[k] < p.N) g.dh0[((int64_t)b * p.E + e) * p.N + nk[k]] = gv[m][k];
      }
      if (q == 0) {
        pa[(int64_t)e * (NP + 2) + NP] = sumD.value();
        pa[(int64_t)e * (NP + 2) + NP + 1] = sumbias.value();
      }
    }
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
  Two sum{0.f, 0.f};
#pragma unroll 4
  for (int j = 0; j < p.batch * p.nchunk; ++j) sum.add(g.part_a[(int64_t)j * p.E * (NP + 2) + i]);
  const float v = sum.value();
  if (n < p.N) g.dA[(int64_t)e * p.N + n] = v;
  else if (n == NP && g.dD != nullptr) g.dD[e] = v;
  else if (n == NP + 1 && g.dbias != nullptr) g.dbias[e] = v;
}

template <typename F>
int by_type(int dtype, F&& f) {
  if (dtype == M3_FLOAT32) return f(float{});
  if (dtype == M3_BFLOAT16) return f(__nv_bfloat16{});
  return f(__half{});
}

constexpr int kBwdThreads = 128;

// f(K, P, M) as types: states a lane, lanes, channels a lane by the padded number of states. single: one channel a lane,
// for launches that leave SMs idle otherwise (3 x 341 x 507 x 16: 55 us, with two channels 96).
template <int K, int P, int M> struct KPM { static constexpr int k = K, p = P, m = M; };
template <typename F>
int by_states(int n, bool single, F&& f) {
  switch (sel_padded_states(n)) {
    case 4: return f(KPM<2, 2, 1>{});
    case 8: return f(KPM<4, 2, 1>{});
    case 16: return single ? f(KPM<4, 4, 1>{}) : f(KPM<4, 4, 2>{});
    case 32: return single ? f(KPM<4, 8, 1>{}) : f(KPM<4, 8, 2>{});
    case 64: return single ? f(KPM<4, 16, 1>{}) : f(KPM<4, 16, 2>{});
    default: return single ? f(KPM<4, 32, 1>{}) : f(KPM<4, 32, 2>{});
  }
}

struct BwdPlan {
  int np, tiles, nchunk, chunk;
  bool single;
  size_t bc, a, states, dtsum;  // floats
};

BwdPlan plan(const SelScanParams& p, int sms) {
  BwdPlan w;
  w.np = sel_padded_states(p.N);
  for (const bool single : {false, true}) {
    by_states(p.N, single, [&](auto l) {
      using L_ = decltype(l);
      const int ec = kBwdThreads / L_::p * L_::m, Eg = p.E / p.G;
      w.tiles = (Eg + ec - 1) / ec;
      if (!single) w.nchunk = sel_pieces(p, std::max(1, L_::p / L_::m), sms, &w.chunk);
      return 0;
    });
    w.single = single;
    if ((int64_t)p.batch * p.G * w.tiles * w.nchunk > sms) break;
  }
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
  p.y = g.dy;  // the flags of y are those of its gradient here
  sel_pair_flags(&p, dtype);
  SelScanParams o = p;
  o.u = g.du; o.delta = g.ddelta; o.z = g.dz;
  sel_pair_flags(&o, dtype);
  g.vec_du = o.vec_u; g.vec_dd = o.vec_d; g.vec_dz = o.vec_z;
  const int Eg = p.E / p.G;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    M3_TRY(by_states(p.N, w.single, [&](auto l) {
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
      const dim3 grid((unsigned)(p.G * w.tiles), (unsigned)p.nchunk, (unsigned)p.batch);
      auto go = [&](auto fast) {
        constexpr bool FAST = decltype(fast)::value;
        static std::atomic<bool> done[kMaxDevices];
        M3_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(&sel_bwd_kernel<T, K, P, M, NT, FAST>), sizeof(S), done));
        sel_bwd_kernel<T, K, P, M, NT, FAST><<<grid, NT, sizeof(S), s>>>(p, g);
        return check_launch("sel_bwd_kernel");
      };
      const bool fast = p.vec_u && p.vec_d && (p.vec_z || p.z.p == nullptr) && p.vec_y && p.vec_B && p.vec_C && g.vec_du &&
                        g.vec_dd && (g.vec_dz || p.z.p == nullptr) && (sizeof(T) == 4 || (!p.delta_f32 && !p.bc_f32));
      return fast ? go(std::true_type{}) : go(std::false_type{});
    }));
    const int64_t rows = (int64_t)p.batch * p.L * p.G;
    const unsigned bc_ctas = (unsigned)((rows * 2 * w.np + 255) / 256);
    const unsigned a_ctas = (unsigned)(((int64_t)p.E * (w.np + 2) + 255) / 256);
    sel_bwd_join_kernel<T><<<bc_ctas + a_ctas, 256, 0, s>>>(p, g, w.np, w.tiles, rows, bc_ctas);
    return check_launch("sel_bwd_join_kernel");
  });
}

}  // namespace m3
