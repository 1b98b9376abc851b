// Losses over the tokens of a language model's logits, forward and backward.
//
// A row is the V logits l of one position, s = 1 / temperature, c = s log2(e):
//   logp = s l[tok] - log sum_v exp(s l[v]) = ln 2 (c (l[tok] - m) - log2 S),
//   S = sum_v 2^(c (l[v] - m)),  m any value near max(l)
//   d logp / d l[v] = s (1[v = tok] - 2^(c (l[v] - m)) / S)
// m is the largest of the row's first elements: every warp finds the same one by itself, sums
// of all warps (and CTAs) join by addition, and no element passes through a second rounding
// exponential. Where S then leaves 2^-60 .. 2^100 the row is done again with its true maximum.
// c is held in two floats: one float's rounding (up to 3e-8 of c) would move every
// log-probability of a sequence the same way, and the preference loss sums them.
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
#include <type_traits>

#include "m3_common.cuh"
#include "token_loss.cuh"

namespace cg = cooperative_groups;

namespace m3 {
namespace {

constexpr int kRowThreads = 512;  // at most, of one CTA of a row
constexpr int kRowWarps = kRowThreads / 32;

constexpr double kLn2 = 0.693147180559945309417;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sixteen bytes of a row, two elements of 16 bits to a word: element by element the compiler
// moves them through registers of their own (twice the registers of the gradient in bf16).
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  uint4 u;
};
__device__ __forceinline__ float2 two(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 two(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t word(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t word(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ void unpack(const Vec<T>& v, float (&f)[Vec<T>::N]) {
  const uint32_t w[4] = {v.u.x, v.u.y, v.u.z, v.u.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      f[k] = __uint_as_float(w[k]);
    } else {
      const float2 x = two(w[k], T{});
      f[2 * k] = x.x;
      f[2 * k + 1] = x.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ Vec<T> pack(const float (&f)[Vec<T>::N]) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(f[k]);
    else w[k] = word(f[2 * k], f[2 * k + 1], T{});
  }
  return Vec<T>{make_uint4(w[0], w[1], w[2], w[3])};
}

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

// What comes off a row's logits before the exponential. `far`: so large (masked entries at a
// type's lowest value in a row that has no others, or an infinity) that c * base could
// overflow; the difference is then formed first.
struct Base {
  float m, k;  // the base and -c_hi * base
  bool far;
};
__device__ __forceinline__ Base base_at(float m, float c_hi) {
  if (m == -INFINITY) m = 0.f;
  const bool far = !(fabsf(m) < 1e30f);
  return Base{m, far ? 0.f : -(m * c_hi), far};
}

// c (l - base) with c in two floats. c_lo is positive, so that l = -inf stays -inf.
template <bool FAR>
__device__ __forceinline__ float exponent(float l, const Base& b, float c_hi, float c_lo) {
  if constexpr (FAR) {
    const float d = l - b.m;
    return fmaf(d, c_hi, d * c_lo);
  }
  return fmaf(l, c_lo, fmaf(l, c_hi, b.k));
}

template <bool FAR, typename T>
__device__ __forceinline__ float vec_sum(const Vec<T>& v, const Base& b, float c_hi, float c_lo) {
  constexpr int N = Vec<T>::N;
  float l[N], s[2] = {0.f, 0.f};
  unpack(v, l);
#pragma unroll
  for (int k = 0; k < N; ++k) s[k & 1] += exp2_approx(exponent<FAR>(l[k], b, c_hi, c_lo));
  return s[0] + s[1];
}
template <typename T>
__device__ __forceinline__ float vec_max(const Vec<T>& v) {
  float l[Vec<T>::N];
  unpack(v, l);
  float m = l[0];
#pragma unroll
  for (int k = 1; k < Vec<T>::N; ++k) m = fmaxf(m, l[k]);
  return m;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, s));
  return v;
}

// log S. ex2.approx falls short by 5.1e-8 of its value on average (measured over its whole
// range of fractions); all terms but the base's own, which is exact, carry that. The integer
// part of the logarithm is scaled in 64 bits, so that the result is off by 3e-8 at most
// instead of half a step of a value near 10 (5e-7).
__device__ __forceinline__ double log_sum(float S) {
  if (!(S > 0.f && S < INFINITY)) return (double)NAN;
  int e;
  float m = frexpf(S, &e);  // 0.5 .. 1
  if (m < 0.75f) { m *= 2.f; --e; }
  return (double)e * kLn2 + (double)log1pf(m - 1.f) + (S > 1.f ? 5.1e-8 * (double)((S - 1.f) / S) : 0.0);
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

// A position's operands of the policy loss, loaded ahead of the row's sum.
struct TokenOps {
  float old_logp, adv, ref;
  double weight;
};
__device__ __forceinline__ TokenOps token_ops(const PolicyArgs& a, const PolicyWs& w, int64_t b, int64_t t) {
  TokenOps o;
  o.old_logp = map_at(a.old_logp, b, t);
  o.adv = map_at(a.adv, b, t);
  o.ref = a.ref.p ? map_at(a.ref, b, t) : 0.f;
  o.weight = a.by_sequence ? 1.0 / ((double)w.counts[b] * w.head->sequences) : 1.0 / w.head->total;
  return o;
}

// exp(d) - 1 - d without the cancellation of a small d: the series to d^9 below 1/2 (its
// remainder is 2^-30 of the result), the difference above.
__device__ __forceinline__ float kl_term(float d) {
  if (fabsf(d) >= 0.5f) return expm1f(d) - d;
  float q = 1.f / 362880.f;
  q = fmaf(q, d, 1.f / 40320.f);
  q = fmaf(q, d, 1.f / 5040.f);
  q = fmaf(q, d, 1.f / 720.f);
  q = fmaf(q, d, 1.f / 120.f);
  q = fmaf(q, d, 1.f / 24.f);
  q = fmaf(q, d, 1.f / 6.f);
  q = fmaf(q, d, 0.5f);
  return q * d * d;
}

// The differences of log-probabilities are formed in 64 bits; their exponentials, and what is
// linear in those, in 32.
struct TokenLoss {
  float loss, kl, dlogp;
  bool clipped;
};
__device__ __forceinline__ TokenLoss policy_token(const PolicyArgs& a, const TokenOps& x, double logp) {
  TokenLoss o;
  const float r = expf((float)(logp - (double)x.old_logp)), lo = (float)a.clip_lo, hi = (float)a.clip_hi;
  o.clipped = (x.adv > 0.f && r > hi) || (x.adv < 0.f && r < lo);
  o.loss = -x.adv * (o.clipped ? fminf(fmaxf(r, lo), hi) : r);
  o.dlogp = o.clipped ? 0.f : -r * x.adv;
  o.kl = 0.f;
  if (a.ref.p != nullptr) {
    const float d = (float)((double)x.ref - logp), k = (float)a.kl_coef;
    o.kl = kl_term(d);
    o.loss = fmaf(k, o.kl, o.loss);
    o.dlogp = fmaf(-k, expm1f(d), o.dlogp);
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

// The gradient of one row: g (one-hot - softmax). tok < 0: no element is the token's.
struct GradRow {
  Base base;
  float g, inv;  // inv = 1 / S
  int tok;
  float at;      // the token's logit
};
template <bool FAR, typename T>
__device__ __forceinline__ Vec<T> vec_grad(const Vec<T>& v, const GradRow& r, float c_hi, float c_lo) {
  float l[Vec<T>::N];
  unpack(v, l);
  const float q = -r.g * r.inv;
#pragma unroll
  for (int k = 0; k < Vec<T>::N; ++k) l[k] = q * exp2_approx(exponent<FAR>(l[k], r.base, c_hi, c_lo));
  return pack<T>(l);
}
template <typename T>
__device__ __forceinline__ T one_grad(float l, const GradRow& r, float hot, float c_hi, float c_lo) {
  const float e = r.base.far ? exponent<true>(l, r.base, c_hi, c_lo) : exponent<false>(l, r.base, c_hi, c_lo);
  return from_f32<T>(r.g * (hot - exp2_approx(e) * r.inv));
}
// Vector j of a row to its place; whoever writes the token's vector writes its element again.
template <bool FAR, typename T>
__device__ __forceinline__ void put_grad(const Vec<T>& v, int j, T* out, const RowCut& c, const GradRow& r, bool same,
                                         float c_hi, float c_lo) {
  constexpr int N = Vec<T>::N;
  const Vec<T> o = vec_grad<FAR>(v, r, c_hi, c_lo);
  const int i0 = c.head + j * N;
  if (same) {
    *reinterpret_cast<Vec<T>*>(out + i0) = o;
  } else {
    float x[N];  // rounded to T already
    unpack(o, x);
#pragma unroll
    for (int k = 0; k < N; ++k) out[i0 + k] = from_f32<T>(x[k]);
  }
  if ((unsigned)(r.tok - i0) < (unsigned)N) out[r.tok] = one_grad<T>(r.at, r, 1.f, c_hi, c_lo);
}
// The single elements before and behind a row's vectors.
template <typename T>
__device__ __forceinline__ void put_ends(const T* row, T* out, int V, const RowCut& c, const GradRow& r, int tid, int nt,
                                         float c_hi, float c_lo) {
  for (int i = tid; i < c.head; i += nt) out[i] = one_grad<T>(to_f32(row[i]), r, i == r.tok ? 1.f : 0.f, c_hi, c_lo);
  for (int i = c.tail0 + tid; i < V; i += nt)
    out[i] = one_grad<T>(to_f32(row[i]), r, i == r.tok ? 1.f : 0.f, c_hi, c_lo);
}
template <typename T>
__device__ __forceinline__ bool same_boundary(const T* out, const RowCut& c) {
  return (reinterpret_cast<uintptr_t>(out + c.head) & 15) == 0;
}

// `value` into elements [i0, i1) of a row
template <typename T>
__device__ __forceinline__ void fill(T* out, int i0, int i1, int tid, int nt, T value) {
  constexpr int N = Vec<T>::N;
  const int h = min(i1, i0 + (int)(((16 - (reinterpret_cast<uintptr_t>(out + i0) & 15)) & 15) / sizeof(T)));
  const int nv = (i1 - h) / N;
  float f[N];
#pragma unroll
  for (int k = 0; k < N; ++k) f[k] = to_f32(value);
  const Vec<T> z = pack<T>(f);
  for (int j = tid; j < nv; j += nt) *reinterpret_cast<Vec<T>*>(out + h + j * N) = z;
  for (int i = i0 + tid; i < h; i += nt) out[i] = value;
  for (int i = h + nv * N + tid; i < i1; i += nt) out[i] = value;
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Results of a position that does not count.
template <bool POLICY>
__device__ __forceinline__ void skip_row(const RowOut& o, const PolicyWs& w, int64_t r) {
  o.logp[r] = 0.f;
  if (o.logp64) o.logp64[r] = 0.0;
  if (o.stats) o.stats[r] = make_float2(0.f, 1.f);
  if constexpr (POLICY) {
    w.rows[r] = RowResult{0.f, 0.f, 0.f};
    if (o.coef) o.coef[r] = 0.f;
  }
}
// From a row's sum to its results; `lead` writes them. Returns g, the gradient's factor.
template <bool POLICY>
__device__ __forceinline__ float finish_row(const TokenRows& p, const PolicyArgs& a, const PolicyWs& w, const RowOut& o,
                                            const TokenOps& x, int64_t r, float at_token, const Base& base, float S,
                                            bool lead) {
  // the token's exponent exactly as the sum's elements have theirs: relative to base.k
  const double c = p.scale * 1.44269504088896340736;
  const double at = base.far ? ((double)at_token - (double)base.m) * c : fma((double)at_token, c, (double)base.k);
  const double logp = at * kLn2 - log_sum(S);
  float coef = 0.f;
  if constexpr (POLICY) {
    const TokenLoss tl = policy_token(a, x, logp);
    coef = (float)(x.weight * (double)tl.dlogp);
    if (lead) {
      w.rows[r] = RowResult{(float)(x.weight * (double)tl.loss), tl.kl, tl.clipped ? 1.f : 0.f};
      if (o.coef) o.coef[r] = coef;
    }
  }
  if (lead) {
    o.logp[r] = (float)logp;
    if (o.logp64) o.logp64[r] = logp;
    if (o.stats) o.stats[r] = make_float2(base.m, S);
  }
  return (float)((double)coef * p.scale);
}

// Whether a sum over an assumed base can be trusted (false for NaN too).
__device__ __forceinline__ bool in_range(float S) { return S > 8.673617e-19f && S < 1.2676506e30f; }  // 2^-60, 2^100

// One cluster of CTAs (of one CTA where there are rows enough) per row. With KEEP a CTA's part
// stays in shared memory between the sum and the gradient; each thread reads there what it
// copied itself, so the copies need no barrier. Without, the gradient reads the row again
// (from the L2 cache, as a rule).
template <typename T, bool POLICY, bool KEEP>
__global__ void __launch_bounds__(kRowThreads) token_rows_kernel(TokenRows p, PolicyArgs a, PolicyWs w, RowOut o) {
  constexpr int U = 4;  // loads in flight per thread
  extern __shared__ uint4 kept_raw[];
  Vec<T>* kept = reinterpret_cast<Vec<T>*>(kept_raw);
  __shared__ float part[kRowWarps];
  __shared__ GradRow sh;
  __shared__ bool again;
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int64_t r = blockIdx.x / C;
  const int64_t b = r / p.T, t = r - b * p.T;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, W = nt >> 5;
  const T* row = static_cast<const T*>(p.logits) + b * p.sb + t * p.st;
  T* drow = nullptr;
  if constexpr (POLICY)
    if (o.dlogits) drow = static_cast<T*>(o.dlogits) + b * o.dsb + t * o.dst;
  const int e0 = (int)((int64_t)p.V * rank / C), e1 = (int)((int64_t)p.V * (rank + 1) / C);  // this CTA's part of a fill
  const Position pos = position(p, b, t);
  if (!pos.keep) {  // the same for the whole cluster
    if (rank == 0 && tid == 0) skip_row<POLICY>(o, w, r);
    if (drow) fill<T>(drow, e0, e1, tid, nt, from_f32<T>(0.f));
    return;
  }
  const RowCut c = cut_row(row, p.V);
  const int v0 = (int)((int64_t)c.nv * rank / C), v1 = (int)((int64_t)c.nv * (rank + 1) / C), n = v1 - v0;
  const Vec<T>* rv = reinterpret_cast<const Vec<T>*>(row + c.head);
  const Vec<T>* mine = rv + v0;
  const int quarter = (n + 4 * nt - 1) / (4 * nt) * nt;  // of the part, in whole rounds of the CTA
  if constexpr (KEEP) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      for (int j = q * quarter + tid; j < min(n, (q + 1) * quarter); j += nt) cp_async16(kept + j, mine + j);
      cp_async_commit();
    }
  }
  // the base: the largest of the row's first 32 vectors (of all, where there is no vector)
  float m = -INFINITY;
  if (c.nv > 0) {
    if (lane < c.nv) m = vec_max(rv[lane]);
  } else if (lane < p.V) {
    m = to_f32(row[lane]);
  }
  TokenOps x{};
  float at_token = 0.f;
  if (tid == 0) {
    at_token = pos.known ? to_f32(row[pos.tok]) : NAN;
    if constexpr (POLICY) x = token_ops(a, w, b, t);
  }
  Base base = base_at(warp_max(m), p.c_hi);
  float s = 0.f;
  if constexpr (KEEP) {
    auto sum_quarter = [&](int q) {
      for (int j = q * quarter + tid; j < min(n, (q + 1) * quarter); j += nt)
        s += vec_sum<false>(kept[j], base, p.c_hi, p.c_lo);
    };
    cp_async_wait<3>();
    sum_quarter(0);
    cp_async_wait<2>();
    sum_quarter(1);
    cp_async_wait<1>();
    sum_quarter(2);
    cp_async_wait<0>();
    sum_quarter(3);
  } else {
    int j = tid;
    for (; j + (U - 1) * nt < n; j += U * nt) {
      Vec<T> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = mine[j + u * nt];
#pragma unroll
      for (int u = 0; u < U; ++u) s += vec_sum<false>(v[u], base, p.c_hi, p.c_lo);
    }
    for (; j < n; j += nt) s += vec_sum<false>(mine[j], base, p.c_hi, p.c_lo);
  }
  auto ends = [&](auto f) {
    if (rank == 0) {
      for (int i = tid; i < c.head; i += nt) f(to_f32(row[i]));
      for (int i = c.tail0 + tid; i < p.V; i += nt) f(to_f32(row[i]));
    }
  };
  ends([&](float l) { s += exp2_approx(exponent<false>(l, base, p.c_hi, p.c_lo)); });
  s = warp_sum(s);
  if (lane == 0) part[warp] = s;
  auto meet = [&]() {
    if (C > 1) cl.sync();
    else __syncthreads();
  };
  meet();
  if (warp == 0) {
    float S = 0.f;
    for (int i = lane; i < W * C; i += 32) S += C > 1 ? cl.map_shared_rank(part, i / W)[i % W] : part[i];
    S = warp_sum(S);
    if (lane == 0) {
      again = base.far || !in_range(S);
      if (!again) {
        const float g = finish_row<POLICY>(p, a, w, o, x, r, at_token, base, S, rank == 0);
        sh = GradRow{base, g, 1.f / S, pos.known ? (int)pos.tok : -1, at_token};
      }
    }
  }
  __syncthreads();
  if (again) {
    // rare: the row's true maximum, then its sum
    auto all = [&](float v, bool largest) {
      meet();  // the parts of the last sum have been read
      if (lane == 0) part[warp] = v;
      meet();
      float y = largest ? -INFINITY : 0.f;
      for (int i = 0; i < W * C; ++i) {
        const float z = C > 1 ? cl.map_shared_rank(part, i / W)[i % W] : part[i];
        y = largest ? fmaxf(y, z) : y + z;
      }
      return y;
    };
    float mx = -INFINITY;
    for (int j = tid; j < n; j += nt) mx = fmaxf(mx, vec_max(mine[j]));
    ends([&](float l) { mx = fmaxf(mx, l); });
    base = base_at(all(warp_max(mx), true), p.c_hi);
    s = 0.f;
    for (int j = tid; j < n; j += nt)
      s += base.far ? vec_sum<true>(mine[j], base, p.c_hi, p.c_lo) : vec_sum<false>(mine[j], base, p.c_hi, p.c_lo);
    ends([&](float l) {
      s += exp2_approx(base.far ? exponent<true>(l, base, p.c_hi, p.c_lo) : exponent<false>(l, base, p.c_hi, p.c_lo));
    });
    const float S = all(warp_sum(s), false);
    if (tid == 0) {
      const float g = finish_row<POLICY>(p, a, w, o, x, r, at_token, base, S, rank == 0);
      sh = GradRow{base, g, 1.f / S, pos.known ? (int)pos.tok : -1, at_token};
    }
    __syncthreads();
  }
  if (C > 1) cl.barrier_arrive();  // this CTA reads no other's part from here on
  if constexpr (POLICY) {
    if (drow) {
      const GradRow gr = sh;
      if (gr.g == 0.f) {
        fill<T>(drow, e0, e1, tid, nt, from_f32<T>(0.f));
      } else {
        const bool same = same_boundary(drow, c);
        auto put = [&](auto far) {
          for (int j = tid; j < n; j += nt)
            put_grad<decltype(far)::value>(KEEP ? kept[j] : mine[j], v0 + j, drow, c, gr, same, p.c_hi, p.c_lo);
        };
        if (gr.base.far) put(std::true_type{});
        else put(std::false_type{});
        if (rank == 0) put_ends(row, drow, p.V, c, gr, tid, nt, p.c_hi, p.c_lo);
      }
    }
  }
  if (C > 1) cl.barrier_wait();  // no CTA leaves while another reads its part
}

// Short rows (up to 4 KB): a warp per row, the row in its registers.
constexpr int kShortBytes = 4096, kShortVecs = kShortBytes / (16 * 32), kShortThreads = 128;
template <typename T, bool POLICY>
__global__ void __launch_bounds__(kShortThreads) token_short_rows_kernel(TokenRows p, PolicyArgs a, PolicyWs w, RowOut o) {
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * (kShortThreads / 32) + (threadIdx.x >> 5);
  if (r >= p.R) return;
  const int64_t b = r / p.T, t = r - b * p.T;
  const T* row = static_cast<const T*>(p.logits) + b * p.sb + t * p.st;
  T* drow = nullptr;
  if constexpr (POLICY)
    if (o.dlogits) drow = static_cast<T*>(o.dlogits) + b * o.dsb + t * o.dst;
  const Position pos = position(p, b, t);
  if (!pos.keep) {
    if (lane == 0) skip_row<POLICY>(o, w, r);
    if (drow) fill<T>(drow, 0, p.V, lane, 32, from_f32<T>(0.f));
    return;
  }
  const RowCut c = cut_row(row, p.V);
  const Vec<T>* rv = reinterpret_cast<const Vec<T>*>(row + c.head);
  Vec<T> v[kShortVecs];
#pragma unroll
  for (int u = 0; u < kShortVecs; ++u)
    if (lane + 32 * u < c.nv) v[u] = rv[lane + 32 * u];
  // at most seven single elements on each side
  const float first = lane < c.head ? to_f32(row[lane]) : -INFINITY;
  const float last = c.tail0 + lane < p.V ? to_f32(row[c.tail0 + lane]) : -INFINITY;
  const float at_token = pos.known ? to_f32(row[pos.tok]) : NAN;
  TokenOps x{};
  if constexpr (POLICY) x = token_ops(a, w, b, t);
  float m = fmaxf(first, last);
#pragma unroll
  for (int u = 0; u < kShortVecs; ++u)
    if (lane + 32 * u < c.nv) m = fmaxf(m, vec_max(v[u]));
  const Base base = base_at(warp_max(m), p.c_hi);
  auto sum = [&](auto far) {
    constexpr bool FAR = decltype(far)::value;
    // a lane without a single element holds -inf there, which adds nothing
    float s = (lane < c.head ? exp2_approx(exponent<FAR>(first, base, p.c_hi, p.c_lo)) : 0.f) +
              (c.tail0 + lane < p.V ? exp2_approx(exponent<FAR>(last, base, p.c_hi, p.c_lo)) : 0.f);
#pragma unroll
    for (int u = 0; u < kShortVecs; ++u)
      if (lane + 32 * u < c.nv) s += vec_sum<FAR>(v[u], base, p.c_hi, p.c_lo);
    return s;
  };
  const float S = warp_sum(base.far ? sum(std::true_type{}) : sum(std::false_type{}));
  const float g = finish_row<POLICY>(p, a, w, o, x, r, at_token, base, S, lane == 0);
  if constexpr (POLICY) {
    if (drow) {
      const GradRow gr{base, g, 1.f / S, pos.known ? (int)pos.tok : -1, at_token};
      if (g == 0.f) {
        fill<T>(drow, 0, p.V, lane, 32, from_f32<T>(0.f));
      } else {
        const bool same = same_boundary(drow, c);
        auto put = [&](auto far) {
#pragma unroll
          for (int u = 0; u < kShortVecs; ++u)
            if (lane + 32 * u < c.nv)
              put_grad<decltype(far)::value>(v[u], lane + 32 * u, drow, c, gr, same, p.c_hi, p.c_lo);
        };
        if (base.far) put(std::true_type{});
        else put(std::false_type{});
        put_ends(row, drow, p.V, c, gr, lane, 32, p.c_hi, p.c_lo);
      }
    }
  }
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

// The gradient of the logits from the rows' (m, S). A warp takes a part of a row at a time,
// parts from the end (the forward read the end last, so some of it is still in the L2 cache).
constexpr int kGradThreads = 256, kGradWarps = kGradThreads / 32;
constexpr int kGradU = 4;                    // loads in flight per lane
constexpr int kGradPart = 32 * kGradU * 4;   // vectors of one part
template <typename T>
__global__ void __launch_bounds__(kGradThreads, 3)
    token_grad_kernel(TokenRows p, const float2* stats, Map2<const float> coef, const float* up, bool keep_if_one,
                      T* dlogits, int64_t dsb, int64_t dst, int parts, int64_t units) {
  const float u = up ? *up : 1.f;
  if (keep_if_one && u == 1.f) return;
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * kGradWarps;
  for (int64_t i = (int64_t)blockIdx.x * kGradWarps + (threadIdx.x >> 5); i < units; i += step) {
    const int64_t at = units - 1 - i, r = at / parts, b = r / p.T, t = r - b * p.T;
    const int part = (int)(at - r * parts);
    const T* row = static_cast<const T*>(p.logits) + b * p.sb + t * p.st;
    T* out = dlogits + b * dsb + t * dst;
    const Position pos = position(p, b, t);
    const float co = map_at(coef, b, t);
    const float2 st = stats[r];
    const RowCut c = cut_row(row, p.V);
    const int v0 = min(c.nv, part * kGradPart), v1 = min(c.nv, v0 + kGradPart);
    GradRow gr;
    gr.g = 0.f;
    if (pos.keep) gr.g = pos.known ? (float)((double)u * (double)co * p.scale) : NAN;
    if (gr.g == 0.f) {
      constexpr int N = Vec<T>::N;
      fill<T>(out, part == 0 ? 0 : c.head + v0 * N, part == parts - 1 ? p.V : c.head + v1 * N, lane, 32,
              from_f32<T>(0.f));
      continue;
    }
    gr.base = base_at(st.x, p.c_hi);
    gr.inv = 1.f / st.y;
    gr.tok = pos.known ? (int)pos.tok : -1;
    gr.at = pos.known ? to_f32(row[pos.tok]) : 0.f;
    const Vec<T>* rv = reinterpret_cast<const Vec<T>*>(row + c.head);
    const bool same = same_boundary(out, c);
    auto put = [&](auto far) {
      for (int j0 = v0; j0 < v1; j0 += 32 * kGradU) {
        Vec<T> v[kGradU];
#pragma unroll
        for (int k = 0; k < kGradU; ++k)
          if (j0 + lane + 32 * k < v1) v[k] = rv[j0 + lane + 32 * k];
#pragma unroll
        for (int k = 0; k < kGradU; ++k)
          if (j0 + lane + 32 * k < v1)
            put_grad<decltype(far)::value>(v[k], j0 + lane + 32 * k, out, c, gr, same, p.c_hi, p.c_lo);
      }
    };
    if (gr.base.far) put(std::true_type{});
    else put(std::false_type{});
    if (part == 0) put_ends(row, out, p.V, c, gr, lane, 32, p.c_hi, p.c_lo);
  }
}

// How the rows are laid over the device.
struct RowPlan {
  int C, threads;
  size_t smem;
};
constexpr int64_t kKeepBytes = 110 * 1024;  // of a CTA's part: two CTAs of an SM then hold one each
constexpr int64_t kKeepMost = 220 * 1024;
int plan_rows(const TokenRows& p, int64_t elem, bool policy, bool keep, RowPlan* out) {
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  const int64_t bytes = (int64_t)p.V * elem;
  int C = 1;
  // few rows: split each so that the device is filled, down to parts of 16 KB
  while (C < 8 && p.R * C * 2 <= 2 * (int64_t)sms && bytes / (2 * C) >= 16384) C *= 2;
  // the same with and without a gradient, so that both give the same bits
  if (policy)
    while (C < 8 && bytes / C > kKeepBytes) C *= 2;
  // about eight vectors a thread
  const int64_t want = bytes / C / 16 / 8;
  int threads = 64;
  while (threads < kRowThreads && threads < want) threads *= 2;
  out->C = C;
  out->threads = threads;
  out->smem = keep ? (size_t)(bytes / C / 16 + 2) * 16 : 0;
  if (out->smem > (size_t)kKeepMost) out->smem = 0;
  return M3_OK;
}

template <typename T, bool POLICY, bool KEEP>
int launch_cluster_rows(const TokenRows& p, const PolicyArgs& a, const PolicyWs& w, const RowOut& o, const RowPlan& plan,
                        cudaStream_t s) {
  if (p.R > INT32_MAX / plan.C) return fail(M3_ERR_UNSUPPORTED, "token rows: too many positions");
  auto kernel = token_rows_kernel<T, POLICY, KEEP>;
  if constexpr (KEEP) {
    static std::atomic<bool> done[kMaxDevices];
    M3_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), (size_t)kKeepMost, done));
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.R * plan.C));
  cfg.blockDim = dim3((unsigned)plan.threads);
  cfg.dynamicSmemBytes = KEEP ? plan.smem : 0;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)plan.C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, a, w, o);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(M3_ERR_CUDA, std::string("token_rows_kernel: ") + cudaGetErrorString(e));
  }
  return M3_OK;
}

template <typename T, bool POLICY>
int launch_rows(const TokenRows& p, const PolicyArgs& a, const PolicyWs& w, const RowOut& o, cudaStream_t s) {
  if (p.R == 0) return M3_OK;
  if ((int64_t)p.V * (int64_t)sizeof(T) <= kShortBytes) {
    const int64_t per = kShortThreads / 32;
    token_short_rows_kernel<T, POLICY><<<(unsigned)((p.R + per - 1) / per), kShortThreads, 0, s>>>(p, a, w, o);
    return check_launch("token_short_rows_kernel");
  }
  RowPlan plan;
  M3_TRY(plan_rows(p, (int64_t)sizeof(T), POLICY, o.dlogits != nullptr, &plan));
  if constexpr (POLICY)
    if (plan.smem > 0) return launch_cluster_rows<T, POLICY, true>(p, a, w, o, plan, s);
  return launch_cluster_rows<T, POLICY, false>(p, a, w, o, plan, s);
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
  const unsigned grid = (unsigned)std::min<int64_t>((units + kGradWarps - 1) / kGradWarps, (int64_t)sms * 8);
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
