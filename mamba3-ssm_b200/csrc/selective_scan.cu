// Selective state space scan, forward and single step: per channel e and state n
//   dt = softplus(delta + bias),  h_t = exp(dt A) h_{t-1} + dt u B_t,  y = (sum_n C_t h_t + D u) silu(z)
// P lanes share a channel and hold K states each in registers (n = q K + k). A CTA walks the
// sequence in tiles of 32 steps: u and delta of its channels and B, C are brought into shared
// memory as (row, step), so that a lane reads four steps of one operand at once; the sums over a
// channel's lanes are formed for several steps together by halving exchanges, and y leaves
// through shared memory in whole rows. The next tile's operands are loaded while this one is scanned.
//
// Bound by the issue of instructions: about 10 a step, channel and state, of which the exponential alone holds its unit (16 a
// clock and SM) for as long as eight issues. 8 x 2048 x 2048 x 16 of bf16 with a gate take 309 us (268 MB and as much of states that
// the backward needs, 1.7 TB/s; the exponentials alone would take 120). In other shapes, us: 128 threads 327; 32 threads and
// two channels a lane 344, 64 and two 331 to 348; a quarter of the decays by a polynomial on the FMA pipe 323; without
// pairs, in its first form, 727.
#include <algorithm>
#include <type_traits>

#include "selective_scan.cuh"

namespace m3 {
namespace {

constexpr int TT = kSelTile;
constexpr int TS = kSelPitch;

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
// the sum of its step sizes. FAST: every operand is of u's type and read two elements at a time.
template <typename T, int K, int P, int NT, bool OUT, bool FAST>
__global__ void __launch_bounds__(NT) sel_scan_kernel(const SelScanParams p) {
  using S = FwdSmem<K, P, NT>;
  constexpr int NP = S::NP, EC = S::EC, GS = group_steps<P>();
  constexpr int R = TT / (2 * P) > 0 ? TT / (2 * P) : 1;  // steps of a pair of channels that a thread brings
  constexpr bool kAhead = BcTile<T, K, P, NT, FAST>::J <= 2;  // B and C of the next tile are loaded ahead too
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& sh = *reinterpret_cast<S*>(smem_raw);
  const int tid = threadIdx.x, q = tid % P, el = tid / P;
  const int Eg = p.E / p.G, tiles = (Eg + EC - 1) / EC;
  const int g = blockIdx.x / tiles, e_first = g * Eg + (blockIdx.x % tiles) * EC, e_end = (g + 1) * Eg;
  const int b = blockIdx.z, c = blockIdx.y;
  const int beg = c * p.chunk, end = min(p.L, beg + p.chunk);
  const int len = seq_len(p.lengths, b, p.L);
  // channels (le, le + 1) at steps lt .. lt + R - 1 of a tile: what this thread brings and stores. A pair
  // behind the last channel reads the tile's first one instead, which lies on a pair's boundary too.
  const int le = tid % (EC / 2) * 2, lt = tid / (EC / 2) * R;
  const bool brings = TT * EC / 2 >= NT * R || lt < TT;
  const int l0 = e_first + le < e_end ? e_first + le : e_first, second = l0 + 1 < e_end ? 1 : 0;
  const bool lelive = brings && e_first + le < e_end;
  const bool vu = FAST || p.vec_u, vd = FAST || p.vec_d, vz = FAST || p.vec_z, vy = FAST || p.vec_y;

  float A2[K], h[K], dts = 0.f;
  const int ec = min(e_first + el, e_end - 1);
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
  const float bias0 = p.bias != nullptr ? p.bias[l0] : 0.f, bias1 = p.bias != nullptr ? p.bias[l0 + second] : 0.f;
  const float D0 = OUT && p.D != nullptr ? p.D[l0] : 0.f, D1 = OUT && p.D != nullptr ? p.D[l0 + second] : 0.f;

  const T* up = static_cast<const T*>(p.u.p) + (int64_t)b * p.u.sb + l0;
  const T* zp = OUT && p.z.p != nullptr ? static_cast<const T*>(p.z.p) + (int64_t)b * p.z.sb + l0 : nullptr;
  T* yp = OUT ? static_cast<T*>(const_cast<void*>(p.y.p)) + (int64_t)b * p.y.sb + l0 : nullptr;
  const int64_t doff = (int64_t)b * p.delta.sb + l0;
  const int64_t boff = (int64_t)b * p.B.sb + g * p.Bg, coff = (int64_t)b * p.C.sb + g * p.Cg;

  // loads of rows behind the sequence's end read its last one; nothing is made of them
  Raw2<T> ru[R];
  std::conditional_t<FAST, Raw2<T>, RawAny<T>> rd[R];
  BcTile<T, K, P, NT, FAST> tb, tc;
  auto fetch = [&](int t0) {
    if (brings) {
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int64_t t = min(t0 + lt + j, len - 1);
        ru[j] = load2<T>(up + t * p.u.sl, vu, second);
        load2_any<T>(rd[j], p.delta.p, p.delta_f32, doff + t * p.delta.sl, vd, second);
      }
    }
  };
  auto fetch_bc = [&](int t0) {
    tb.fetch(p.B.p, p.bc_f32, boff, p.B.sl, p.vec_B, p.N, t0, len, tid);
    if (OUT) tc.fetch(p.C.p, p.bc_f32, coff, p.C.sl, p.vec_C, p.N, t0, len, tid);
  };
  if (beg < len) {
    fetch(beg);
    if (kAhead) fetch_bc(beg);
  }
  for (int t0 = beg; t0 < end && t0 < len; t0 += TT) {
    if (!kAhead) fetch_bc(t0);
    Raw2<T> zu[R], zz[R];
    if (brings) {
      float d0[R], d1[R], x0[R], x1[R];
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const float2 r = value2<T>(rd[j], p.delta_f32), u = value2(ru[j]);
        const float2 d = step_size2(make_float2(r.x + bias0, r.y + bias1), p.softplus);
        const bool in = t0 + lt + j < len;
        d0[j] = in ? d.x : 0.f;
        d1[j] = in ? d.y : 0.f;
        x0[j] = in ? d.x * u.x : 0.f;
        x1[j] = in ? d.y * u.y : 0.f;
        zu[j] = ru[j];
      }
      put_steps<R>(&sh.dt[le][lt], d0);
      put_steps<R>(&sh.dt[le + 1][lt], d1);
      put_steps<R>(&sh.dx[le][lt], x0);
      put_steps<R>(&sh.dx[le + 1][lt], x1);
    }
    tb.put(sh.B, p.bc_f32, p.N, t0, len, tid);
    if (OUT) tc.put(sh.C, p.bc_f32, p.N, t0, len, tid);
    __syncthreads();
    if (OUT && zp != nullptr && brings) {
#pragma unroll
      for (int j = 0; j < R; ++j) zz[j] = load2<T>(zp + (int64_t)min(t0 + lt + j, len - 1) * p.z.sl, vz, second);
    }
    if (t0 + TT < end && t0 + TT < len) {
      fetch(t0 + TT);
      if (kAhead) fetch_bc(t0 + TT);
    }
    constexpr int BS = GS < kSelSub ? kSelSub : GS;  // steps between two looks at whether states are kept
#pragma unroll 1
    for (int tb8 = 0; tb8 < TT; tb8 += BS)
#pragma unroll
      for (int tg = tb8; tg < tb8 + BS; tg += GS) {
        float yv[GS];
#pragma unroll
        for (int i4 = 0; i4 < GS; i4 += 4) {
          if (OUT && (GS < kSelSub ? tg == tb8 : i4 % kSelSub == 0) && p.save != nullptr && t0 + tg + i4 < len) {
            float* sv = p.save + (((int64_t)b * ((p.L + kSelSub - 1) / kSelSub) + (t0 + tg + i4) / kSelSub) * p.E + e_first + el) * NP + q * K;
            if (e_first + el < e_end) {
              if constexpr (K == 4) *reinterpret_cast<float4*>(sv) = make_float4(h[0], h[1], h[2], h[3]);
              else *reinterpret_cast<float2*>(sv) = make_float2(h[0], h[1]);
            }
          }
          const ulonglong2 d4 = *reinterpret_cast<const ulonglong2*>(&sh.dt[el][tg + i4]);
          const ulonglong2 x4 = *reinterpret_cast<const ulonglong2*>(&sh.dx[el][tg + i4]);
          f2 ya = 0, yb = 0;
          if (!OUT) {
            float s0, s1;
            unpack2(add2(d4.x, d4.y), s0, s1);
            dts += s0 + s1;
          }
#pragma unroll
          for (int k = 0; k < K; ++k) {
            const ulonglong2 b4 = *reinterpret_cast<const ulonglong2*>(&sh.B[k * P + q][tg + i4]);
            ulonglong2 c4{0, 0};
            if (OUT) c4 = *reinterpret_cast<const ulonglong2*>(&sh.C[k * P + q][tg + i4]);
            const f2 A2k = pack2(A2[k], A2[k]), mean = pack2(kEx2Mean, kEx2Mean);
            float a[4], x[4], hv[4];
            unpack2(fma2(d4.x, A2k, mean), a[0], a[1]);
            unpack2(fma2(d4.y, A2k, mean), a[2], a[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = ex2(a[i]);
            unpack2(mul2(x4.x, b4.x), x[0], x[1]);
            unpack2(mul2(x4.y, b4.y), x[2], x[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) hv[i] = h[k] = fmaf(a[i], h[k], x[i]);
            if (OUT) {
              ya = fma2(pack2(hv[0], hv[1]), c4.x, ya);
              yb = fma2(pack2(hv[2], hv[3]), c4.y, yb);
            }
          }
          unpack2(ya, yv[i4], yv[i4 + 1]);
          unpack2(yb, yv[i4 + 2], yv[i4 + 3]);
        }
        if (OUT) {
          const int at = spread_sum<GS, P>(yv, q);
#pragma unroll
          for (int j = 0; j < GS / P; ++j) sh.y[tg + at + j][el] = yv[j];
        }
      }
    __syncthreads();
    if (OUT && lelive) {
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int t = t0 + lt + j;
        if (t < end) {
          const float2 u = value2(zu[j]), y2 = *reinterpret_cast<const float2*>(&sh.y[lt + j][le]);
          float v0 = fmaf(D0, u.x, y2.x), v1 = fmaf(D1, u.y, y2.y);
          if (zp != nullptr) {
            const float2 z = value2(zz[j]);
            const float2 sg = sigmoid2(z);
            v0 *= z.x * sg.x;
            v1 *= z.y * sg.y;
          }
          store2<T>(yp + (int64_t)t * p.y.sl, vy, second, t < len ? v0 : 0.f, t < len ? v1 : 0.f);
        }
      }
    }
  }
  if (OUT) {
    // padding behind the last tile with a position that counts
    const int from = len > beg ? beg + (min(len, end) - beg + TT - 1) / TT * TT : beg;
    for (int t0 = from; t0 < end; t0 += TT) {
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (lelive && t0 + lt + j < end) store2<T>(yp + (int64_t)(t0 + lt + j) * p.y.sl, vy, second, 0.f, 0.f);
    }
  }
  const int e = e_first + el;
  if (e < e_end) {
    if (OUT) {
      if (p.h_last != nullptr && c == p.nchunk - 1) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (q * K + k < p.N) p.h_last[((int64_t)b * p.E + e) * p.N + q * K + k] = h[k];
      }
    } else {
      const int64_t at = ((int64_t)b * p.nchunk + c) * p.E + e;
#pragma unroll
      for (int k = 0; k < K; ++k) p.states[at * NP + q * K + k] = h[k];
      if (q == 0) p.dtsum[at] = dts;
    }
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
  for (int c = 0; c < p.nchunk - 1; ++c) {
    const float local = st[c * pitch], a = ex2(A2 * ds[(int64_t)c * p.E]);
    st[c * pitch] = h;
    h = fmaf(a, h, local);
  }
  st[(p.nchunk - 1) * pitch] = h;
}

// Four values of a row from element i on, as fp32; vec: the address is on a boundary of the four.
template <typename T>
__device__ __forceinline__ void load4(const void* p, bool f32, int64_t i, bool vec, int n, float (&v)[4]) {
  if (vec) {
    if (sizeof(T) == 4 || f32) {
      const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
      if constexpr (sizeof(T) == 2) {
        const float2 lo = value2(Raw2<T>{x.x}), hi = value2(Raw2<T>{x.y});
        v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = k < n ? ld_any<T>(p, f32, i + k) : 0.f;
  }
}

// One step: y and the state in place. P lanes share a channel with four states each and take RB sequences, so that
// A and the channel's parameters are loaded once, a step size is formed by one lane, and loads of RB states are in flight.
template <typename T, int P, int RB>
__global__ void __launch_bounds__(256) sel_step_kernel(const SelStepParams p, bool vec, bool vec_bc) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t ch = i / P;
  const int q = (int)(i % P), n = q * 4;
  const int64_t b0 = ch / p.E * RB;
  const bool live = b0 < p.batch;
  const int rows = live ? (int)min((int64_t)RB, p.batch - b0) : 0;
  const int e = live ? (int)(ch % p.E) : 0;
  const int g = e / (p.E / p.G), mine = p.N - n;  // states from this lane on
  float h[RB][4], A2[4], y[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    if (r < rows && mine > 0) load4<float>(p.state + (b0 + r) * p.sstate + (int64_t)e * p.N, true, n, vec, mine, h[r]);
    else h[r][0] = h[r][1] = h[r][2] = h[r][3] = 0.f;
  }
  // step size and input of the sequences: one a lane where there are lanes enough
  constexpr int OWN = P < RB ? RB : 1;
  float dt[OWN], u[OWN];
  const float bias = p.bias != nullptr ? p.bias[e] : 0.f;
#pragma unroll
  for (int r = 0; r < OWN; ++r) {
    const int64_t b = b0 + min(OWN == 1 ? q % RB : r, max(rows - 1, 0));
    dt[r] = live ? step_size(ld_any<T>(p.delta, p.delta_f32, b * p.sd + e) + bias, p.softplus) : 0.f;
    u[r] = live ? ld(static_cast<const T*>(p.u) + b * p.su + e) : 0.f;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) A2[k] = k < mine ? p.A[(int64_t)e * p.N + n + k] * kLog2e : 0.f;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const float d = OWN == 1 ? __shfl_sync(0xffffffffu, dt[0], r, P) : dt[OWN == 1 ? 0 : r];
    const float x = d * (OWN == 1 ? __shfl_sync(0xffffffffu, u[0], r, P) : u[OWN == 1 ? 0 : r]);
    y[r] = 0.f;
    if (r < rows && mine > 0) {
      float B[4], C[4];
      load4<T>(p.B, p.bc_f32, (b0 + r) * p.sB + g * p.sBg + n, vec_bc, mine, B);
      load4<T>(p.C, p.bc_f32, (b0 + r) * p.sC + g * p.sCg + n, vec_bc, mine, C);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        h[r][k] = fmaf(ex2(fmaf(d, A2[k], kEx2Mean)), h[r][k], x * B[k]);
        y[r] = fmaf(h[r][k], C[k], y[r]);
      }
      float* to = p.state + (b0 + r) * p.sstate + (int64_t)e * p.N + n;
      if (vec) *reinterpret_cast<float4*>(to) = make_float4(h[r][0], h[r][1], h[r][2], h[r][3]);
      else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < mine) to[k] = h[r][k];
      }
    }
  }
  const int at = spread_sum<RB, P>(y, q);
  constexpr int LEFT = RB / P > 0 ? RB / P : 1;
  if (P > RB && q % (P > RB ? P / RB : 1) != 0) return;  // lanes with the same sums
#pragma unroll
  for (int j = 0; j < LEFT; ++j) {
    const int r = at + j;
    if (r < rows) {
      const int64_t b = b0 + r;
      float v = y[j];
      if (p.D != nullptr) v = fmaf(p.D[e], ld(static_cast<const T*>(p.u) + b * p.su + e), v);
      if (p.z != nullptr) {
        const float z = ld(static_cast<const T*>(p.z) + b * p.sz + e);
        v *= z * fast_sigmoid(z);
      }
      st(static_cast<T*>(p.y) + b * p.sy + e, v);
    }
  }
}

template <typename F>
int by_type(int dtype, F&& f) {
  if (dtype == M3_FLOAT32) return f(float{});
  if (dtype == M3_BFLOAT16) return f(__nv_bfloat16{});
  return f(__half{});
}

// f(K, P) as types: lanes and states a lane by the padded number of states. wide: twice the lanes with half the
// states each, for the pass that forms the pieces' states, whose sums over lanes it has not to form (2048 channels x 16 states of 8192
// steps: 81 us, not wide 90), and for launches of no more CTAs than SMs, where a warp's own time counts (3 x 341 x 507 x 16: 34 us,
// not wide 46; 200 x 1024 of 16 and 32: 13, 12; 18, 17). In larger ones it costs more (8 x 2048 x 2048 x 16: 335, not wide 310).
template <int K, int P> struct KP { static constexpr int k = K, p = P; };
template <typename F>
int by_states(int n, bool wide, F&& f) {
  switch (sel_padded_states(n)) {
    case 4: return f(KP<2, 2>{});
    case 8: return f(KP<4, 2>{});
    case 16: return wide ? f(KP<2, 8>{}) : f(KP<4, 4>{});
    case 32: return wide ? f(KP<2, 16>{}) : f(KP<4, 8>{});
    case 64: return f(KP<4, 16>{});
    default: return f(KP<4, 32>{});
  }
}

// threads of a CTA, which has 32, 32, 16, 8, 8 and 4 channels with 4, 8, 16, 32, 64 and 128 states, and CTAs of one piece of one
// sequence
template <int K, int P> constexpr int pass_threads() { return P >= 16 || (K == 2 && P == 8) ? 128 : 64; }
template <int K, int P>
int64_t pass_tiles(const SelScanParams& p) {
  using S = FwdSmem<K, P, pass_threads<K, P>()>;
  const int Eg = p.E / p.G;
  return (int64_t)p.G * ((Eg + S::EC - 1) / S::EC);
}

template <typename T, int K, int P, bool OUT>
int launch_pass(const SelScanParams& p, cudaStream_t s) {
  constexpr int NT = pass_threads<K, P>();
  using S = FwdSmem<K, P, NT>;
  // what the last piece leaves enters no other
  const dim3 grid((unsigned)pass_tiles<K, P>(p), (unsigned)(OUT ? p.nchunk : p.nchunk - 1), (unsigned)p.batch);
  auto go = [&](auto fast) {
    static std::atomic<bool> done[kMaxDevices];
    constexpr bool FAST = decltype(fast)::value;
    M3_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(&sel_scan_kernel<T, K, P, NT, OUT, FAST>), sizeof(S), done));
    sel_scan_kernel<T, K, P, NT, OUT, FAST><<<grid, NT, sizeof(S), s>>>(p);
    return check_launch("sel_scan_kernel");
  };
  const bool f32 = sizeof(T) == 4;
  const bool fast = p.vec_u && p.vec_d && (p.vec_z || p.z.p == nullptr) && p.vec_y && p.vec_B && p.vec_C &&
                    (f32 || (!p.delta_f32 && !p.bc_f32));
  return fast ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace

static int sel_lanes(int np) { return std::max(2, np / 4); }

// Pieces that the sequence is cut into: one, unless the channels alone leave most of the GPU idle. A
// piece's state has to be formed ahead (about as much work again), so cutting begins where there are less than a quarter of
// the warps that keep an SM busy, and a piece has 256 steps at least. Steps x channels of 16 states, us cut and not:
// 8192 x 4096 447, 586; 8192 x 8192 793, 755.
int sel_pieces(const SelScanParams& p, int lanes, int sms, int* chunk) {
  const int64_t warps = (int64_t)p.batch * p.E * lanes / 32 + 1, want = (int64_t)sms * 16;
  int n = 1;
  if (warps * 4 <= want) n = (int)std::min<int64_t>(want / warps, p.L / (8 * kSelTile));
  n = std::max(1, std::min(n, 4096));
  int64_t len = (p.L + n - 1) / n;
  len = (len + kSelTile - 1) / kSelTile * kSelTile;
  *chunk = (int)std::max<int64_t>(len, kSelTile);
  return std::max<int>(1, (int)((p.L + *chunk - 1) / *chunk));
}

// Whether two neighbouring elements of the rows may be moved at once: pairs begin on even channels of each group.
static bool pairs(const Seq& s, int64_t inner, int es) {
  return s.p != nullptr && inner % 2 == 0 && s.sb % 2 == 0 && s.sl % 2 == 0 &&
         (reinterpret_cast<uintptr_t>(s.p) & (2 * es - 1)) == 0;
}

void sel_pair_flags(SelScanParams* p, int dtype) {
  const int es = (int)dtype_size(dtype), Eg = p->E / p->G;
  p->vec_u = pairs(p->u, Eg, es);
  p->vec_d = pairs(p->delta, Eg, p->delta_f32 ? 4 : es);
  p->vec_z = pairs(p->z, Eg, es);
  p->vec_y = pairs(p->y, Eg, es);
  p->vec_B = pairs(p->B, p->N, p->bc_f32 ? 4 : es) && p->Bg % 2 == 0;
  p->vec_C = pairs(p->C, p->N, p->bc_f32 ? 4 : es) && p->Cg % 2 == 0;
}

size_t sel_scan_save_bytes(int64_t batch, int64_t L, int64_t E, int N) {
  return (size_t)batch * ((L + kSelSub - 1) / kSelSub) * E * sel_padded_states(N) * sizeof(float);
}

size_t sel_scan_fwd_workspace(const SelScanParams& p, int sms) {
  int chunk = 0;
  const int np = sel_padded_states(p.N), n = sel_pieces(p, sel_lanes(np), sms, &chunk);
  return n == 1 ? 0 : (size_t)p.batch * n * p.E * (np + 1) * sizeof(float);
}

int launch_sel_scan_fwd(SelScanParams p, int dtype, void* ws, cudaStream_t s) {
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  const int np = sel_padded_states(p.N);
  sel_pair_flags(&p, dtype);
  p.nchunk = sel_pieces(p, sel_lanes(np), sms, &p.chunk);
  if (p.nchunk > 1) {
    p.states = static_cast<float*>(ws);
    p.dtsum = p.states + (int64_t)p.batch * p.nchunk * p.E * np;
  }
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (p.nchunk > 1) {
      M3_TRY(by_states(p.N, true, [&](auto kp) { return launch_pass<T, decltype(kp)::k, decltype(kp)::p, false>(p, s); }));
      const dim3 grid((unsigned)(((int64_t)p.E * np + 255) / 256), (unsigned)p.batch);
      sel_carry_kernel<<<grid, 256, 0, s>>>(p, np);
      M3_TRY(check_launch("sel_carry_kernel"));
    }
    bool few = false;
    by_states(p.N, false, [&](auto kp) {
      few = pass_tiles<decltype(kp)::k, decltype(kp)::p>(p) * p.nchunk * p.batch <= sms;
      return 0;
    });
    return by_states(p.N, few, [&](auto kp) { return launch_pass<T, decltype(kp)::k, decltype(kp)::p, true>(p, s); });
  });
}

int launch_sel_step(const SelStepParams& p, int dtype, cudaStream_t s) {
  const bool vec = p.N % 4 == 0 && p.sstate % 4 == 0 && (reinterpret_cast<uintptr_t>(p.state) & 15) == 0;
  auto go = [&](auto t, auto lanes) {
    using T = decltype(t);
    constexpr int P = decltype(lanes)::value;
    const int es = sizeof(T) == 4 || p.bc_f32 ? 4 : 2;
    const bool vec_bc = p.N % 4 == 0 && p.sB % 4 == 0 && p.sC % 4 == 0 && p.sBg % 4 == 0 && p.sCg % 4 == 0 &&
                        ((reinterpret_cast<uintptr_t>(p.B) | reinterpret_cast<uintptr_t>(p.C)) & (4 * es - 1)) == 0;
    // four sequences a thread where that leaves some warps for every SM: sequences of 5120 x 16, us, four a thread and one:
    // 8 5.5, 4.5; 16 5.7, 6.9; 32 8.0, 11.0; 256 46, 71 (179 MB: 3.9 TB/s)
    const bool four = p.batch >= 4 && p.batch * p.E * P >= 2 * 128 * 1024;
    const int64_t threads = (four ? (p.batch + 3) / 4 : p.batch) * p.E * P;
    const unsigned grid = (unsigned)((threads + 255) / 256);
    if (four) sel_step_kernel<T, P, 4><<<grid, 256, 0, s>>>(p, vec, vec_bc);
    else sel_step_kernel<T, P, 1><<<grid, 256, 0, s>>>(p, vec, vec_bc);
    return check_launch("sel_step_kernel");
  };
  return by_type(dtype, [&](auto t) {
    switch (sel_padded_states(p.N)) {
      case 4: return go(t, std::integral_constant<int, 1>{});
      case 8: return go(t, std::integral_constant<int, 2>{});
      case 16: return go(t, std::integral_constant<int, 4>{});
      case 32: return go(t, std::integral_constant<int, 8>{});
      case 64: return go(t, std::integral_constant<int, 16>{});
      default: return go(t, std::integral_constant<int, 32>{});
    }
  });
}

}  // namespace m3
