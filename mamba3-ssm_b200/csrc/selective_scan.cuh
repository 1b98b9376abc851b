// Selective state space scan with a decay per channel and state: parameters of the launches
// (selective_scan.cu: forward, state passes, single step; selective_scan_bwd.cu: backward) and
// the device functions they share.
#pragma once

#include <type_traits>

#include "m3_common.cuh"
#ifdef __CUDACC__
#include "pairs.cuh"
#endif

namespace m3 {

// (batch, length, .) view of u, delta, z, B, C or an output: strides in elements, innermost 1
struct Seq {
  const void* p;
  int64_t sb, sl;
};

struct SelScanParams {
  Seq u, delta, z, B, C, y;      // z.p may be null; B, C: (batch, length, G, N) with rows of G * N
  int64_t Bg, Cg;                // stride of the groups of B and C
  bool delta_f32, bc_f32;        // else u's type
  bool vec_u, vec_d, vec_z, vec_y, vec_B, vec_C;  // rows that may be read or written two elements at a time
  const float* A;                // (E, N) contiguous
  const float* D;                // (E), may be null
  const float* bias;             // (E), may be null
  bool softplus;
  const float* h0;               // (batch, E, N) contiguous, may be null
  float* h_last;                 // the same, may be null
  const int64_t* lengths;        // (batch), may be null
  int batch, L, E, N, G;
  // work split: the sequence in nchunk pieces of `chunk` steps (a multiple of the tile)
  int chunk, nchunk;
  float* states;                 // (batch, nchunk, E, NP): local end states, then the states that enter each piece
  float* dtsum;                  // (batch, nchunk, E): sum of the step sizes of each piece
  float* save;                   // (batch, ceil(L / 8), E, NP): the state in front of every eighth step, may be null
};

struct SelScanGrads {
  Seq dy, du, ddelta, dz;        // dy: gradient of the output (after the gate), u's type
  bool vec_du, vec_dd, vec_dz;   // rows that may be written two elements at a time
  const float* dstate;           // (batch, E, N): gradient of the last state, may be null
  float* dA;                     // (E, N)
  float* dD;                     // (E), may be null
  float* dbias;                  // (E), may be null
  void *dB, *dC;                 // (batch, length, G, N) contiguous, B's type
  float* dh0;                    // (batch, E, N), may be null
  float* part_bc;                // (batch, length, tiles, 2 NP): each channel tile's part of dB and dC
  float* part_a;                 // (batch, E, NP + 2): each sequence's part of dA, dD, dbias
};

struct SelStepParams {
  const void *u, *delta, *z, *B, *C;   // (batch, E) and (batch, G, N); z may be null
  void* y;
  int64_t su, sd, sz, sB, sC, sBg, sCg, sy;
  bool delta_f32, bc_f32;
  const float *A, *D, *bias;
  bool softplus;
  float* state; int64_t sstate;  // (batch, E, N), each sequence's part contiguous
  int64_t batch; int E, N, G;
};

constexpr int kSelMaxStates = 128;
constexpr int kSelTile = 32;   // steps that a CTA brings into shared memory at a time
constexpr int kSelSub = 8;     // steps between two saved states

// States that the lanes of a channel hold in all: N rounded up to the layouts that are compiled.
inline int sel_padded_states(int n) {
  int p = 4;
  while (p < n) p *= 2;
  return p;
}

size_t sel_scan_fwd_workspace(const SelScanParams& p, int sms);
int launch_sel_scan_fwd(SelScanParams p, int dtype, void* ws, cudaStream_t s);
size_t sel_scan_save_bytes(int64_t batch, int64_t L, int64_t E, int N);
size_t sel_scan_bwd_workspace(const SelScanParams& p, int sms);
int launch_sel_scan_bwd(SelScanParams p, SelScanGrads g, int dtype, void* ws, cudaStream_t s);
int launch_sel_step(const SelStepParams& p, int dtype, cudaStream_t s);
void sel_pair_flags(SelScanParams* p, int dtype);
// the piece-wise passes that the forward and the backward share
int sel_pieces(const SelScanParams& p, int lanes, int sms, int* chunk);

#ifdef __CUDACC__
// The hardware's 2^x is 2e-8 too small on average between -1/2 and -1/500 and 5e-9 closer to 0 (measured); a decay
// that is wrong by that in each of the many steps a slow state remembers shows in the state. Added to the
// exponent in the product's own rounding, this halves it where it is largest and keeps 2^0 = 1.
constexpr float kEx2Mean = 1.5e-8f;

// a row that is either T or fp32
template <typename T>
struct RawAny { uint32_t a, b; };
template <typename T>
__device__ __forceinline__ float2 value2(Raw2<T> r, bool) { return value2(r); }
template <typename T>
__device__ __forceinline__ float2 value2(RawAny<T> r, bool f32) {
  if (f32) return make_float2(__uint_as_float(r.a), __uint_as_float(r.b));
  if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(r.a), __uint_as_float(r.b));
  else return value2(Raw2<T>{r.a});
}
template <typename T>
__device__ __forceinline__ void load2_any(Raw2<T>& r, const void* p, bool, int64_t i, bool, int) {
  r = load2<T>(static_cast<const T*>(p) + i, true, 1);
}
template <typename T>
__device__ __forceinline__ void load2_any(RawAny<T>& r, const void* p, bool f32, int64_t i, bool vec, int second) {
  if (sizeof(T) == 4 || f32) {
    const float2 v = load2<float>(static_cast<const float*>(p) + i, vec, second).v;
    r.a = __float_as_uint(v.x);
    r.b = __float_as_uint(v.y);
  } else {
    if constexpr (sizeof(T) == 2) r.a = load2<T>(static_cast<const T*>(p) + i, vec, second).v;
    r.b = 0;
  }
}

// log(1 + e^x) = max(x, 0) + log1p(w), w = e^-|x| in [0, 1], log1p(w) / w by a polynomial of degree 8 that is 1 at 0, fitted
// here for the smallest relative error (3.3e-8; 1.1e-7 with its roundings), which also holds for the small
// step sizes that matter most, where a logarithm of 1 + w would lose their digits. Two numbers at once.
__device__ __forceinline__ f2 softplus2(float x0, float x1) {
  const f2 w = pack2(ex2(-fabsf(x0) * kLog2e), ex2(-fabsf(x1) * kLog2e));
  auto c = [](float v) { return pack2(v, v); };
  f2 r = fma2(w, c(0.005364825617334684f), c(-0.030065797599842133f));
  r = fma2(w, r, c(0.07920454444779973f));
  r = fma2(w, r, c(-0.1375380311293698f));
  r = fma2(w, r, c(0.19153655310223328f));
  r = fma2(w, r, c(-0.24857163763289894f));
  r = fma2(w, r, c(0.33321322629882966f));
  r = fma2(w, r, c(-0.49999647963987515f));
  r = fma2(w, r, c(1.f));
  return fma2(w, r, pack2(fmaxf(x0, 0.f), fmaxf(x1, 0.f)));
}

// dt of two raw step sizes
__device__ __forceinline__ float2 step_size2(float2 raw, bool softplus) {
  if (softplus) unpack2(softplus2(raw.x, raw.y), raw.x, raw.y);
  return raw;
}
__device__ __forceinline__ float step_size(float raw, bool softplus) { return step_size2(make_float2(raw, raw), softplus).x; }

template <typename T>
__device__ __forceinline__ float ld_any(const void* p, bool f32, int64_t i) {
  return f32 ? static_cast<const float*>(p)[i] : to_f32(static_cast<const T*>(p)[i]);
}

// Positions of a sequence that count.
__device__ __forceinline__ int seq_len(const int64_t* lengths, int b, int L) {
  if (lengths == nullptr) return L;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : n > L ? L : (int)n;
}

// Sums of V values over P lanes that lie STRIDE apart, spread over them (`lane`: the index among the P):
// after the call value j of the result (V / min(P, V) of them) is the sum of v[at + j], where `at`
// is returned. Halving: each exchange sends one half of the values and keeps the other,
// V (1 - 1 / P) shuffles in all; where P > V the last exchanges leave both partners with the same sum.
template <int V, int P, int STRIDE = 1>
__device__ __forceinline__ int spread_sum(float (&v)[V], int lane) {
  int at = 0, n = V;
#pragma unroll
  for (int m = P / 2; m >= 1; m /= 2) {
    if (n > 1) {
      n /= 2;
      const bool up = lane & m;
#pragma unroll
      for (int j = 0; j < V / 2; ++j)
        if (j < n) {
          const float give = up ? v[j] : v[j + n], keep = up ? v[j + n] : v[j];
          v[j] = keep + __shfl_xor_sync(0xffffffffu, give, m * STRIDE);
        }
      at += up ? n : 0;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], m * STRIDE);
    }
  }
  return at;
}

constexpr int kSelPitch = kSelTile + 4;  // of a tile's rows: those that a warp reads together start on different banks

// Four (or R < 4) steps of one row of a tile in shared memory.
template <int R>
__device__ __forceinline__ void put_steps(float* row, const float (&v)[R]) {
  if constexpr (R % 4 == 0) {
#pragma unroll
    for (int i = 0; i < R; i += 4) *reinterpret_cast<float4*>(row + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else if constexpr (R == 2) {
    *reinterpret_cast<float2*>(row) = make_float2(v[0], v[1]);
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) row[i] = v[i];
  }
}

template <int R>
__device__ __forceinline__ void get_steps(const float* row, float (&v)[R]) {
  if constexpr (R % 4 == 0) {
#pragma unroll
    for (int i = 0; i < R; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(row + i);
      v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
    }
  } else if constexpr (R == 2) {
    const float2 x = *reinterpret_cast<const float2*>(row);
    v[0] = x.x; v[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = row[i];
  }
}

// B or C of a tile: a task is two neighbouring states at four steps. Rows behind the sequence's end
// read its last one, and put() writes zeros in their place.
template <typename T, int K, int P, int NT, bool FAST>
struct BcTile {
  static constexpr int NP = K * P, TASKS = NP / 2 * (kSelTile / 4), J = (TASKS + NT - 1) / NT;
  std::conditional_t<FAST, Raw2<T>, RawAny<T>> r[J][4];
  __device__ __forceinline__ void fetch(const void* p, bool f32, int64_t off, int64_t sl, bool vec, int N, int t0, int len, int tid) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int i = tid + j * NT, n0 = i % (NP / 2) * 2, n = n0 < N ? n0 : 0, t = t0 + i / (NP / 2) * 4;
      if (TASKS % NT == 0 || i < TASKS) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          load2_any<T>(r[j][u], p, f32, off + (int64_t)min(t + u, len - 1) * sl + n, vec, n + 1 < N ? 1 : 0);
      }
    }
  }
  __device__ __forceinline__ void put(float (*rows)[kSelPitch], bool f32, int N, int t0, int len, int tid) const {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int i = tid + j * NT, n = i % (NP / 2) * 2, t = i / (NP / 2) * 4;
      if (TASKS % NT == 0 || i < TASKS) {
        float a[4], b[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float2 v = value2<T>(r[j][u], f32);
          const bool in = t0 + t + u < len;
          a[u] = in && n < N ? v.x : 0.f;
          b[u] = in && n + 1 < N ? v.y : 0.f;
        }
        put_steps<4>(&rows[n % K * P + n / K][t], a);
        put_steps<4>(&rows[(n + 1) % K * P + (n + 1) / K][t], b);
      }
    }
  }
};

#endif

}  // namespace m3
