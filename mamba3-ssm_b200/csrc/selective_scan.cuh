// Selective state space scan with a decay per channel and state: parameters of the launches
// (selective_scan.cu: forward, state passes, single step; selective_scan_bwd.cu: backward) and
// the device functions they share.
#pragma once

#include "m3_common.cuh"

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
// the piece-wise passes that the forward and the backward share
int sel_pieces(const SelScanParams& p, int lanes, int sms, int* chunk);

#ifdef __CUDACC__
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// log(1 + e^x) = max(x, 0) + log1p(w), w = e^-|x|, with log1p(w) = 2 atanh(s), s = w / (2 + w) <= 1/3,
// by its series up to s^13 (the rest is below 2e-8 of it): relative error a few 1e-7 everywhere, which
// a logarithm of 1 + w would not have for the small step sizes that matter most.
__device__ __forceinline__ float softplus_series(float x) {
  const float w = ex2(-fabsf(x) * kLog2e);
  const float s = __fdividef(w, 2.f + w), q = s * s;
  float r = fmaf(q, 1.f / 13, 1.f / 11);
  r = fmaf(q, r, 1.f / 9);
  r = fmaf(q, r, 1.f / 7);
  r = fmaf(q, r, 1.f / 5);
  r = fmaf(q, r, 1.f / 3);
  r = fmaf(q * r, s, s);
  return fmaxf(x, 0.f) + 2.f * r;
}

__device__ __forceinline__ float step_size(float raw, bool softplus) { return softplus ? softplus_series(raw) : raw; }

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
#endif

}  // namespace m3
