// Losses over the tokens of a language model's logits, forward and backward.
//
// A row is the V logits l of one position, s = 1 / temperature, c = s log2(e):
//   logp = s l[tok] - log sum_v exp(s l[v]) = ln 2 (c (l[tok] - m) - log2 S),
//   S = sum_v 2^(c (l[v] - m)),  m = max(l)
//   d logp / d l[v] = s (1[v = tok] - 2^(c (l[v] - m)) / S)
// The maximum comes off before the scaling, so that logits at a type's lowest value (masked
// entries) neither overflow nor, in a row that has no others, lose their differences. c is
// held in two floats: one float's rounding (up to 3e-8 of c) would move every log-probability
// of a sequence the same way, and the preference loss sums them.
// The element work runs in 32 bits, what happens once a row (the logarithm, the ratio, the
// losses) in 64 bits.
//
// Policy loss (r = exp(logp - old), A the advantage, d = ref - logp):
//   loss_t = -min(r A, clip(r, lo, hi) A) + k (exp(d) - d - 1)
//   d loss_t / d logp = -[r A is the minimum] r A + k (1 - exp(d))
// summed with weights 1 / (positions that count), or by sequence 1 / (positions of the
// sequence) / (sequences with any).
// Preference loss: reward_i = beta sum_t (logp - ref), z = chosen - rejected,
//   loss = mean -(1 - e) log sigma(z) - e log sigma(-z).
//
// Positions that do not count (mask 0 or the ignored token) are not read: their
// log-probability is 0 and their gradient row zeros, whatever the logits hold. A token id
// outside the vocabulary that is not the ignored one gives NaN.
#include <cooperative_groups.h>

#include <algorithm>

#include "m3_common.cuh"
#include "token_loss.cuh"

namespace cg = cooperative_groups;

namespace m3 {
namespace {

constexpr int kRowThreads = 512;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kUnroll = 4;  // 16-byte loads in flight per thread

constexpr double kLn2 = 0.693147180559945309417;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct alignas(16) Vec {
  static constexpr int N = 16 / sizeof(T);
  T e[N];
};

template <typename T>
__device__ __forceinline__ T map_at(const Map2<const T>& m, int64_t b, int64_t t) {
  return m.p[b * m.sb + t * m.st];
}

// How a row splits at its 16-byte boundaries: `head` single elements, `nv` vectors from
// there, and the rest single elements again.
struct RowCut {
  int head, nv, tail0;
};
template <typename T>
__device__ __forceinline__ RowCut cut_row(const T* row, int V) {
  constexpr int N = 16 / sizeof(T);
  RowCut c;
  c.head = (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T));
  if (c.head > V) c.head = V;
  c.nv = (V - c.head) / N;
  c.tail0 = c.head + c.nv * N;
  return c;
}

// The value that comes off a row's logits: its maximum, or 0 where there is none yet.
__device__ __forceinline__ float base_of(float mx) { return mx == -INFINITY ? 0.f : mx; }

// c (l - base) without losing c's lower half. c_lo is positive, so that l = -inf stays -inf.
__device__ __forceinline__ float exponent(float l, float base, float c_hi, float c_lo) {
  const float d = l - base;
  return fmaf(d, c_hi, d * c_lo);
}

// Running maximum of the logits and sum of 2^(c (l - base(maximum))).
struct MaxSum {
  float mx, s;
};
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c_hi, float c_lo) {
  MaxSum r;
  r.mx = fmaxf(a.mx, b.mx);
  const float base = base_of(r.mx);
  // a side without a value (sum 0) adds none, however far its base is
  const float fa = a.s == 0.f ? 0.f : a.s * exp2_approx(exponent(base_of(a.mx), base, c_hi, c_lo));
  const float fb = b.s == 0.f ? 0.f : b.s * exp2_approx(exponent(base_of(b.mx), base, c_hi, c_lo));
  r.s = fa + fb;
  return r;
}

template <int N>
__device__ __forceinline__ void take(MaxSum& a, const float (&l)[N], float c_hi, float c_lo) {
  float m = l[0];
#pragma unroll
  for (int k = 1; k < N; ++k) m = fmaxf(m, l[k]);
  if (m > a.mx) {
    if (a.s != 0.f) a.s *= exp2_approx(exponent(base_of(a.mx), m, c_hi, c_lo));
    a.mx = m;
  }
  const float base = base_of(a.mx);
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) s += exp2_approx(exponent(l[k], base, c_hi, c_lo));
  a.s += s;
}

// Whether a position counts, its token, and whether that token is one of the vocabulary.
struct Position {
  bool keep, known;
  int64_t tok;
};
__device__ __forceinline__ Position position(const TokenRows& p, int64_t b, int64_t t) {
  Position q;
  q.tok = map_at(p.tok, b, t);
  q.keep = q.tok != p.ignore && (p.mask.p == nullptr || map_at(p.mask, b, t) != 0);
  q.known = q.tok >= 0 && q.tok < p.V;
  return q;
}

// ------------------------------------------------------------------- policy workspace
// counts (batch) int32, then one PolicyHead, then per-row results and their partial sums
struct PolicyHead {
  double total, sequences;  // positions that count; sequences with any
  unsigned done;            // CTAs of the final sum that have finished
};
struct RowResult {
  float loss, kl, clipped;  // weighted loss; KL and 0 / 1, zero where the position does not count
};
constexpr int kSumRows = 2048;  // rows of one CTA of the final sum
struct SumPart {
  double loss, kl, clipped;
};
struct PolicyWs {
  PolicyHead* head;
  int* counts;
  RowResult* rows;
  SumPart* parts;
};
__host__ __device__ inline size_t up16(size_t n) { return (n + 15) & ~size_t(15); }
inline PolicyWs policy_ws(void* ws, int64_t batch, int64_t rows, size_t* bytes) {
  char* q = static_cast<char*>(ws);
  size_t at = 0;
  PolicyWs w;
  w.head = reinterpret_cast<PolicyHead*>(q + at);
  at += up16(sizeof(PolicyHead));
  w.parts = reinterpret_cast<SumPart*>(q + at);
  at += up16(sizeof(SumPart) * (size_t)((rows + kSumRows - 1) / kSumRows));
  w.counts = reinterpret_cast<int*>(q + at);
  at += up16(sizeof(int) * (size_t)batch);
  w.rows = reinterpret_cast<RowResult*>(q + at);
  at += up16(sizeof(RowResult) * (size_t)rows);
  *bytes = at;
  return w;
}

// Positions that count, by sequence and in all. One cluster of CTAs; a warp counts a segment
// of a sequence and adds its (whole) number, so the result does not depend on the order.
constexpr int kCountCluster = 8, kCountThreads = 1024, kCountSegment = 1024;
__global__ void __cluster_dims__(kCountCluster, 1, 1) __launch_bounds__(kCountThreads)
    policy_count_kernel(TokenRows p, int64_t batch, PolicyWs w) {
  cg::cluster_group cl = cg::this_cluster();
  const int64_t nthreads = (int64_t)gridDim.x * blockDim.x, me = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (int64_t b = me; b < batch; b += nthreads) w.counts[b] = 0;
  if (me == 0) w.head->done = 0;
  __threadfence();
  cl.sync();
  const int lane = threadIdx.x & 31;
  const int64_t segs = (p.T + kCountSegment - 1) / kCountSegment, units = batch * segs;
  for (int64_t u = me >> 5; u < units; u += nthreads >> 5) {
    const int64_t b = u / segs, t0 = (u % segs) * kCountSegment;
    const int64_t t1 = t0 + kCountSegment < p.T ? t0 + kCountSegment : p.T;
    int n = 0;
    for (int64_t t = t0 + lane; t < t1; t += 32) n += position(p, b, t).keep;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0 && n > 0) atomicAdd(&w.counts[b], n);
  }
  __threadfence();
  cl.sync();
  if (blockIdx.x != 0) return;
  __shared__ long long tot[kCountThreads / 32], seq[kCountThreads / 32];
  long long n = 0, m = 0;
  for (int64_t b = threadIdx.x; b < batch; b += blockDim.x) {
    const int k = *reinterpret_cast<volatile int*>(&w.counts[b]);
    n += k;
    m += k > 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    n += __shfl_xor_sync(0xffffffffu, n, o);
    m += __shfl_xor_sync(0xffffffffu, m, o);
  }
  if (lane == 0) { tot[threadIdx.x >> 5] = n; seq[threadIdx.x >> 5] = m; }
  __syncthreads();
  if (threadIdx.x == 0) {
    n = m = 0;
    for (int i = 0; i < kCountThreads / 32; ++i) { n += tot[i]; m += seq[i]; }
    w.head->total = (double)n;
    w.head->sequences = (double)m;
  }
}

struct TokenLoss {
  double loss, kl, dlogp;
  bool clipped;
};
__device__ __forceinline__ TokenLoss policy_token(const PolicyArgs& a, double logp, int64_t b, int64_t t) {
  TokenLoss o;
  const double A = map_at(a.adv, b, t), r = exp(logp - (double)map_at(a.old_logp, b, t));
  const double rc = fmin(fmax(r, a.clip_lo), a.clip_hi);
  o.clipped = (A > 0 && r > a.clip_hi) || (A < 0 && r < a.clip_lo);
  o.loss = o.clipped ? -rc * A : -r * A;
  o.dlogp = o.clipped ? 0.0 : -r * A;
  o.kl = 0.0;
  if (a.ref.p != nullptr) {
    const double d = (double)map_at(a.ref, b, t) - logp, e = expm1(d);
    o.kl = e - d;
    o.loss += a.kl_coef * o.kl;
    o.dlogp -= a.kl_coef * e;
  }
  return o;
}

// --------------------------------------------------------------------- the row kernels
struct RowOut {
  float* logp;
  double* logp64;  // unrounded, for sums over a sequence
  float2* stats;
  float* coef;
  void* dlogits;
  int64_t dsb, dst;
};

// g (one-hot - softmax) over the part [v0, v1) of a row's vectors (and, with `ends`, its
// single elements). tok < 0: no element is the token's.
template <typename T>
__device__ __forceinline__ void write_grad(const T* row, T* out, int V, RowCut c, int v0, int v1, bool ends, int tid,
                                           int nt, int tok, float g, float base, float inv, float c_hi, float c_lo) {
  constexpr int N = Vec<T>::N;
  const bool same = (reinterpret_cast<uintptr_t>(out + c.head) & 15) == 0;
  auto one = [&](float l, int i) {
    const float pr = exp2_approx(exponent(l, base, c_hi, c_lo)) * inv;
    return g * ((i == tok ? 1.f : 0.f) - pr);
  };
  const Vec<T>* rv = reinterpret_cast<const Vec<T>*>(row + c.head);
  for (int j = v0 + tid; j < v1; j += nt) {
    const Vec<T> v = rv[j];
    const int i0 = c.head + j * N;
    Vec<T> o;
#pragma unroll
    for (int k = 0; k < N; ++k) o.e[k] = from_f32<T>(one(to_f32(v.e[k]), i0 + k));
    if (same) {
      *reinterpret_cast<Vec<T>*>(out + i0) = o;
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) out[i0 + k] = o.e[k];
    }
  }
  if (ends) {
    for (int i = tid; i < c.head; i += nt) out[i] = from_f32<T>(one(to_f32(row[i]), i));
    for (int i = c.tail0 + tid; i < V; i += nt) out[i] = from_f32<T>(one(to_f32(row[i]), i));
  }
}

template <typename T>
__device__ __forceinline__ void fill_row(T* out, int V, int i0, int i1, int tid, int nt, T value) {
  // element bounds [i0, i1) of this CTA's part; vectors inside them
  constexpr int N = Vec<T>::N;
  const int h = min(i1, i0 + (int)(((16 - (reinterpret_cast<uintptr_t>(out + i0) & 15)) & 15) / sizeof(T)));
  const int nv = (i1 - h) / N;
  Vec<T> z;
#pragma unroll
  for (int k = 0; k < N; ++k) z.e[k] = value;
  for (int j = tid; j < nv; j += nt) *reinterpret_cast<Vec<T>*>(out + h + j * N) = z;
  for (int i = i0 + tid; i < h; i += nt) out[i] = value;
  for (int i = h + nv * N + tid; i < i1; i += nt) out[i] = value;
}

// One cluster of CTAs (of one CTA where there are rows enough) per row: every CTA reduces its
// part, the parts are joined through distributed shared memory, and with GRAD the gradient is
// written from a second look at the same part.
template <typename T, bool POLICY>
__global__ void __launch_bounds__(kRowThreads) token_rows_kernel(TokenRows p, PolicyArgs a, PolicyWs w, RowOut o) {
  constexpr int N = Vec<T>::N;
  __shared__ MaxSum wred[kRowWarps];
  __shared__ MaxSum cta_part;
  __shared__ float sh_g, sh_base, sh_inv;
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int64_t r = blockIdx.x / C;
  const int64_t b = r / p.T, t = r % p.T;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* row = static_cast<const T*>(p.logits) + b * p.sb + t * p.st;
  T* drow = nullptr;
  if constexpr (POLICY)
    if (o.dlogits) drow = static_cast<T*>(o.dlogits) + b * o.dsb + t * o.dst;
  const Position pos = position(p, b, t);
  if (!pos.keep) {  // the same for the whole cluster
    if (rank == 0 && tid == 0) {
      o.logp[r] = 0.f;
      if (o.logp64) o.logp64[r] = 0.0;
      if (o.stats) o.stats[r] = make_float2(0.f, 1.f);
      if constexpr (POLICY) {
        w.rows[r] = RowResult{0.f, 0.f, 0.f};
        if (o.coef) o.coef[r] = 0.f;
      }
    }
    if (drow) fill_row<T>(drow, p.V, (int)((int64_t)p.V * rank / C), (int)((int64_t)p.V * (rank + 1) / C), tid,
                          kRowThreads, from_f32<T>(0.f));
    return;
  }
  const RowCut c = cut_row(row, p.V);
  const int v0 = (int)((int64_t)c.nv * rank / C), v1 = (int)((int64_t)c.nv * (rank + 1) / C);
  const Vec<T>* rv = reinterpret_cast<const Vec<T>*>(row + c.head);
  MaxSum acc{-INFINITY, 0.f};
  int j = v0 + tid;
  for (; j + (kUnroll - 1) * kRowThreads < v1; j += kUnroll * kRowThreads) {
    Vec<T> v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = rv[j + u * kRowThreads];
    float l[kUnroll * N];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int k = 0; k < N; ++k) l[u * N + k] = to_f32(v[u].e[k]);
    take(acc, l, p.c_hi, p.c_lo);
  }
  for (; j < v1; j += kRowThreads) {
    const Vec<T> v = rv[j];
    float l[N];
#pragma unroll
    for (int k = 0; k < N; ++k) l[k] = to_f32(v.e[k]);
    take(acc, l, p.c_hi, p.c_lo);
  }
  if (rank == 0) {
    for (int i = tid; i < c.head; i += kRowThreads) { const float l[1] = {to_f32(row[i])}; take(acc, l, p.c_hi, p.c_lo); }
    for (int i = c.tail0 + tid; i < p.V; i += kRowThreads) {
      const float l[1] = {to_f32(row[i])};
      take(acc, l, p.c_hi, p.c_lo);
    }
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    MaxSum x;
    x.mx = __shfl_xor_sync(0xffffffffu, acc.mx, s);
    x.s = __shfl_xor_sync(0xffffffffu, acc.s, s);
    acc = join(acc, x, p.c_hi, p.c_lo);
  }
  if (lane == 0) wred[warp] = acc;
  __syncthreads();
  if (warp == 0) {
    acc = lane < kRowWarps ? wred[lane] : MaxSum{-INFINITY, 0.f};
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      MaxSum x;
      x.mx = __shfl_xor_sync(0xffffffffu, acc.mx, s);
      x.s = __shfl_xor_sync(0xffffffffu, acc.s, s);
      acc = join(acc, x, p.c_hi, p.c_lo);
    }
    if (lane == 0) cta_part = acc;
  }
  if (C > 1) cl.sync();
  if (tid == 0) {
    MaxSum all{-INFINITY, 0.f};
    if (C > 1) {
      for (int k = 0; k < C; ++k) all = join(all, *cl.map_shared_rank(&cta_part, k), p.c_hi, p.c_lo);
    } else {
      all = cta_part;
    }
    const float base = base_of(all.mx);
    const double c = p.scale * 1.44269504088896340736;
    const double logp = pos.known ? (((double)to_f32(row[pos.tok]) - (double)base) * c - log2((double)all.s)) * kLn2
                                  : (double)NAN;
    double coef = 0.0;
    RowResult res{0.f, 0.f, 0.f};
    if constexpr (POLICY) {
      const TokenLoss tl = policy_token(a, logp, b, t);
      const double weight = a.by_sequence ? 1.0 / ((double)w.counts[b] * w.head->sequences) : 1.0 / w.head->total;
      coef = weight * tl.dlogp;
      res = RowResult{(float)(weight * tl.loss), (float)tl.kl, tl.clipped ? 1.f : 0.f};
      sh_g = (float)(coef * p.scale);
      sh_base = base;
      sh_inv = 1.f / all.s;
    }
    if (rank == 0) {
      o.logp[r] = (float)logp;
      if (o.logp64) o.logp64[r] = logp;
      if (o.stats) o.stats[r] = make_float2(base, all.s);
      if constexpr (POLICY) {
        w.rows[r] = res;
        if (o.coef) o.coef[r] = (float)coef;
      }
    }
  }
  if constexpr (POLICY) {
    if (drow) {
      __syncthreads();
      const float g = sh_g;
      if (g == 0.f) {
        fill_row<T>(drow, p.V, (int)((int64_t)p.V * rank / C), (int)((int64_t)p.V * (rank + 1) / C), tid, kRowThreads,
                    from_f32<T>(0.f));
      } else {
        write_grad<T>(row, drow, p.V, c, v0, v1, rank == 0, tid, kRowThreads, pos.known ? (int)pos.tok : -1, g, sh_base,
                      sh_inv, p.c_hi, p.c_lo);
      }
    }
  }
  if (C > 1) cl.sync();  // no CTA leaves while another reads its part
}

// Sums of the rows' results. Every CTA sums a fixed range in a fixed order; the one that
// finishes last adds the ranges' sums in order.
__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += sh[i];
  return t;
}

constexpr int kSumThreads = 256;
__global__ void __launch_bounds__(kSumThreads) policy_sum_kernel(int64_t R, PolicyWs w, float* loss, float* kl,
                                                                  float* clipped) {
  __shared__ double sh[kSumThreads / 32];
  __shared__ bool last;
  const int64_t r0 = (int64_t)blockIdx.x * kSumRows, r1 = r0 + kSumRows < R ? r0 + kSumRows : R;
  SumPart s{0.0, 0.0, 0.0};
  for (int64_t r = r0 + threadIdx.x; r < r1; r += kSumThreads) {
    const RowResult x = w.rows[r];
    s.loss += x.loss;
    s.kl += x.kl;
    s.clipped += x.clipped;
  }
  s.loss = block_sum(s.loss, sh);
  s.kl = block_sum(s.kl, sh);
  s.clipped = block_sum(s.clipped, sh);
  if (threadIdx.x == 0) {
    w.parts[blockIdx.x] = s;
    __threadfence();
    last = atomicAdd(&w.head->done, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  s = SumPart{0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kSumThreads) {
    const volatile SumPart* q = &w.parts[i];
    s.loss += q->loss;
    s.kl += q->kl;
    s.clipped += q->clipped;
  }
  s.loss = block_sum(s.loss, sh);
  s.kl = block_sum(s.kl, sh);
  s.clipped = block_sum(s.clipped, sh);
  if (threadIdx.x == 0) {
    const double n = w.head->total > 0 ? w.head->total : 1.0;
    *loss = (float)s.loss;
    *kl = (float)(s.kl / n);
    *clipped = (float)(s.clipped / n);
  }
}

// Rewards of the answers, then (by the CTA that finishes last) the loss of the pairs and the
// derivative by each answer's log-probabilities. One CTA per answer.
struct PrefWs {
  unsigned* done;
  double* rewards;  // (2 N)
  double* logp;     // (2 N, T)
};
inline PrefWs pref_ws(void* ws, int64_t batch, int64_t rows, size_t* bytes) {
  PrefWs w;
  w.done = static_cast<unsigned*>(ws);
  w.rewards = reinterpret_cast<double*>(static_cast<char*>(ws) + 16);
  w.logp = w.rewards + batch;
  *bytes = 16 + sizeof(double) * (size_t)(batch + rows);
  return w;
}

__global__ void __launch_bounds__(kSumThreads)
    preference_pairs_kernel(TokenRows p, Map2<const float> ref, double beta, double smoothing, int pairs,
                            PrefWs w, float* loss, float* rewards, float* seq_coef) {
  __shared__ double sh[kSumThreads / 32];
  __shared__ bool last;
  const int64_t b = blockIdx.x;
  double s = 0.0;
  for (int t = threadIdx.x; t < p.T; t += kSumThreads)
    if (position(p, b, t).keep) s += w.logp[b * p.T + t] - (ref.p ? (double)map_at(ref, b, (int64_t)t) : 0.0);
  s = beta * block_sum(s, sh);
  if (threadIdx.x == 0) {
    rewards[b] = (float)s;
    w.rewards[b] = s;
    __threadfence();
    last = atomicAdd(w.done, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  const volatile double* rw = w.rewards;
  s = 0.0;
  for (int i = threadIdx.x; i < pairs; i += kSumThreads) {
    const double z = rw[i] - rw[pairs + i];
    const double l = log1p(exp(-fabs(z)));  // softplus(-|z|)
    s += (1.0 - smoothing) * (l + fmax(-z, 0.0)) + smoothing * (l + fmax(z, 0.0));
    const double dz = (1.0 / (1.0 + exp(-z)) - (1.0 - smoothing)) * beta / pairs;
    seq_coef[i] = (float)dz;
    seq_coef[pairs + i] = (float)-dz;
  }
  s = block_sum(s, sh);
  if (threadIdx.x == 0) *loss = (float)(s / pairs);
}

// The gradient of the logits from the rows' (m, S): a part of a row at a time, parts taken
// from the end (the forward read the end last, so some of it is still in the L2 cache).
constexpr int kGradThreads = 256;
constexpr int kGradPart = kGradThreads * 8;  // vectors of one part
template <typename T>
__global__ void __launch_bounds__(kGradThreads)
    token_grad_kernel(TokenRows p, const float2* stats, Map2<const float> coef, const float* up, bool keep_if_one,
                      T* dlogits, int64_t dsb, int64_t dst, int parts, int64_t units) {
  const float u = up ? *up : 1.f;
  if (keep_if_one && u == 1.f) return;
  for (int64_t i = blockIdx.x; i < units; i += gridDim.x) {
    const int64_t at = units - 1 - i, r = at / parts, b = r / p.T, t = r % p.T;
    const int part = (int)(at % parts);
    const T* row = static_cast<const T*>(p.logits) + b * p.sb + t * p.st;
    T* out = dlogits + b * dsb + t * dst;
    const Position pos = position(p, b, t);
    const RowCut c = cut_row(row, p.V);
    const int v0 = min(c.nv, part * kGradPart), v1 = min(c.nv, v0 + kGradPart);
    float g = 0.f;
    if (pos.keep) {
      g = (float)((double)u * (double)map_at(coef, b, t) * p.scale);
      if (!pos.known) g = NAN;
    }
    if (g == 0.f) {
      constexpr int N = Vec<T>::N;
      fill_row<T>(out, p.V, part == 0 ? 0 : c.head + v0 * N, part == parts - 1 ? p.V : c.head + v1 * N, threadIdx.x,
                  kGradThreads, from_f32<T>(0.f));
      continue;
    }
    const float2 st = stats[r];
    write_grad<T>(row, out, p.V, c, v0, v1, part == 0, threadIdx.x, kGradThreads, pos.known ? (int)pos.tok : -1, g,
                  st.x, 1.f / st.y, p.c_hi, p.c_lo);
  }
}

// CTAs of a row's cluster: with few rows a row is split so that the device is filled (up to
// the eight CTAs that every device can place as one cluster), down to parts of 16 KB.
int row_cluster(int64_t rows, int64_t row_bytes, int* C) {
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  int c = 1;
  while (c < 8 && rows * c * 2 <= 2 * (int64_t)sms && row_bytes / (2 * c) >= 16384) c *= 2;
  *C = c;
  return M3_OK;
}

template <typename T, bool POLICY>
int launch_rows(const TokenRows& p, const PolicyArgs& a, const PolicyWs& w, const RowOut& o, cudaStream_t s) {
  if (p.R == 0) return M3_OK;
  int C = 1;
  M3_TRY(row_cluster(p.R, (int64_t)p.V * (int64_t)sizeof(T), &C));
  if (p.R > INT32_MAX / C) return fail(M3_ERR_UNSUPPORTED, "token rows: too many positions");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.R * C));
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, token_rows_kernel<T, POLICY>, p, a, w, o);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(M3_ERR_CUDA, std::string("token_rows_kernel: ") + cudaGetErrorString(e));
  }
  return M3_OK;
}

template <bool POLICY>
int launch_rows_of(const TokenRows& p, int dtype, const PolicyArgs& a, const PolicyWs& w, const RowOut& o,
                   cudaStream_t s) {
  switch (dtype) {
    case M3_FLOAT32: return launch_rows<float, POLICY>(p, a, w, o, s);
    case M3_BFLOAT16: return launch_rows<__nv_bfloat16, POLICY>(p, a, w, o, s);
    case M3_FLOAT16: return launch_rows<__half, POLICY>(p, a, w, o, s);
  }
  return fail(M3_ERR_UNSUPPORTED, "token rows: unsupported dtype");
}

}  // namespace

size_t policy_workspace_bytes(int64_t batch, int64_t rows) {
  size_t n = 0;
  policy_ws(nullptr, batch, rows, &n);
  return n;
}

size_t preference_workspace_bytes(int64_t batch, int64_t rows) {
  size_t n = 0;
  pref_ws(nullptr, batch, rows, &n);
  return n;
}

int launch_token_logprobs(const TokenRows& p, int dtype, float* logp, float2* stats, cudaStream_t s) {
  return launch_rows_of<false>(p, dtype, PolicyArgs{}, PolicyWs{}, RowOut{logp, nullptr, stats, nullptr, nullptr, 0, 0}, s);
}

int launch_policy_loss(const TokenRows& p, int dtype, const PolicyArgs& a, int64_t batch, float* loss, float* kl,
                       float* clipped, float* logp, float2* stats, float* coef, void* dlogits, int64_t dsb, int64_t dst,
                       void* ws, cudaStream_t s) {
  size_t bytes = 0;
  const PolicyWs w = policy_ws(ws, batch, p.R, &bytes);
  policy_count_kernel<<<kCountCluster, kCountThreads, 0, s>>>(p, batch, w);
  M3_TRY(check_launch("policy_count_kernel"));
  M3_TRY(launch_rows_of<true>(p, dtype, a, w, RowOut{logp, nullptr, stats, coef, dlogits, dsb, dst}, s));
  policy_sum_kernel<<<(unsigned)((p.R + kSumRows - 1) / kSumRows), kSumThreads, 0, s>>>(p.R, w, loss, kl, clipped);
  return check_launch("policy_sum_kernel");
}

int launch_preference_loss(const TokenRows& p, int dtype, Map2<const float> ref, double beta, double smoothing,
                           int64_t pairs, float* loss, float* rewards, float* logp, float2* stats, float* seq_coef,
                           void* ws, cudaStream_t s) {
  size_t bytes = 0;
  const PrefWs w = pref_ws(ws, 2 * pairs, p.R, &bytes);
  cudaError_t e = cudaMemsetAsync(w.done, 0, sizeof(unsigned), s);
  if (e != cudaSuccess) return fail(M3_ERR_CUDA, std::string("preference loss: ") + cudaGetErrorString(e));
  M3_TRY(launch_rows_of<false>(p, dtype, PolicyArgs{}, PolicyWs{},
                               RowOut{logp, w.logp, stats, nullptr, nullptr, 0, 0}, s));
  preference_pairs_kernel<<<(unsigned)(2 * pairs), kSumThreads, 0, s>>>(p, ref, beta, smoothing, (int)pairs, w, loss,
                                                                       rewards, seq_coef);
  return check_launch("preference_pairs_kernel");
}

template <typename T>
static int launch_grad(const TokenRows& p, const float2* stats, Map2<const float> coef, const float* up,
                       bool keep_if_one, void* dlogits, int64_t dsb, int64_t dst, cudaStream_t s) {
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  const int N = 16 / (int)sizeof(T);
  const int parts = std::max(1, (p.V / N + kGradPart - 1) / kGradPart);
  const int64_t units = p.R * parts;
  const unsigned grid = (unsigned)std::min<int64_t>(units, (int64_t)sms * 8);
  token_grad_kernel<T><<<grid, kGradThreads, 0, s>>>(p, stats, coef, up, keep_if_one, static_cast<T*>(dlogits), dsb,
                                                    dst, parts, units);
  return check_launch("token_grad_kernel");
}

int launch_token_grad(const TokenRows& p, int dtype, const float2* stats, Map2<const float> coef, const float* up,
                      bool keep_if_one, void* dlogits, int64_t dsb, int64_t dst, cudaStream_t s) {
  switch (dtype) {
    case M3_FLOAT32: return launch_grad<float>(p, stats, coef, up, keep_if_one, dlogits, dsb, dst, s);
    case M3_BFLOAT16: return launch_grad<__nv_bfloat16>(p, stats, coef, up, keep_if_one, dlogits, dsb, dst, s);
    case M3_FLOAT16: return launch_grad<__half>(p, stats, coef, up, keep_if_one, dlogits, dsb, dst, s);
  }
  return fail(M3_ERR_UNSUPPORTED, "token gradient: unsupported dtype");
}

}  // namespace m3
