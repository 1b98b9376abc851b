// Losses over the tokens of a language model's logits, forward and backward.
//
// A row is the V logits l of one position, s = 1 / temperature, c = s log2(e):
//   logp = s l[tok] - log sum_v exp(s l[v]) = ln 2 (c (l[tok] - m) - log2 S),
//   S = sum_v 2^(c (l[v] - m)),  m any value near max(l)
//   d logp / d l[v] = s (1[v = tok] - 2^(c (l[v] - m)) / S)
// m is the largest of the row's first elements and the token's own (a likely one, in earnest):
// every warp finds the same m by itself, sums of all warps (and CTAs) join by addition, and no
// element passes through a second rounding exponential. Where S then leaves 2^-60 .. 2^20 the
// row is done again with its true maximum (in_range says why).
// c is held in two floats: one float's rounding (up to 6e-8 of c) would move every
// log-probability of a sequence the same way, and the preference loss sums them. The policy loss
// takes c rounded to the nearest float.
// The element work runs in 32 bits; log-probabilities and their differences, once a row, in 64.
//
// What bounds it: every logit is read once (twice where the gradient has to wait for other rows,
// as in the preference loss) and every gradient written once, 2 or 4 bytes each, against one or
// two exponentials: at the copy rate of the memory an SM has to form 12 (forward) or 6 (policy,
// twice) exponentials a cycle in bf16, of the 16 that its unit can, so the rest of an element's
// work is kept to four or five instructions.
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

#include "copy_rounds.cuh"
#include "m3_common.cuh"
#include "sm100.cuh"
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

// What comes off a row's logits before the exponential. `far`: so large (a mask's constant in a
// row that has nothing else, or an infinity) that the rounding of c * base, which every exponent
// of the row has in common, could leave an exponent's range; the difference is then formed first.
// Below 2^20 that rounding is 2^-5 at most, and base * c_lo 2^-3.
struct Base {
  float m, k;  // the base and -c_hi * base
  bool far;
};
__device__ __forceinline__ Base base_at(float m, float c_hi) {
  if (m == -INFINITY) m = 0.f;
  const bool far = !(fabsf(m) * c_hi < 1048576.f);
  return Base{m, far ? 0.f : -(m * c_hi), far};
}

// The exponent of a logit. FINE: with c's lower half too (c_lo is positive, so that l = -inf
// stays -inf); it then carries m c_lo, which norm_sum takes off the sum. The policy loss does
// without, c_hi being the float nearest to c: scale is then off by 2^-24 of itself at most, for
// S and for the token alike, which moves a log-probability by 2^-24 s (l[tok] - mean of l under
// p). By -logp = entropy of p - s (l[tok] - mean) that is at most 2^-24 of an unlikely token's own
// value, and 2^-24 ln V of a likely one's.
template <bool FAR, bool FINE>
__device__ __forceinline__ float exponent(float l, const Base& b, float c_hi, float c_lo) {
  if constexpr (FAR) {
    const float d = l - b.m;
    return fmaf(d, c_hi, d * c_lo);
  } else if constexpr (FINE) {
    return fmaf(l, c_lo, fmaf(l, c_hi, b.k));
  } else {
    return fmaf(l, c_hi, b.k);
  }
}
// 2^(exponent) of one logit, whichever kind its base is
template <bool FINE>
__device__ __forceinline__ float exp_one(float l, const Base& b, float c_hi, float c_lo) {
  return exp2_approx(b.far ? exponent<true, FINE>(l, b, c_hi, c_lo) : exponent<false, FINE>(l, b, c_hi, c_lo));
}
// A sum of fine exponentials in terms of plain ones, as the gradient forms them.
template <bool FINE>
__device__ __forceinline__ float norm_sum(float S, const Base& b, float c_lo) {
  return FINE && !b.far ? S * exp2_approx(-b.m * c_lo) : S;
}

// Two running sums, for their latency.
struct Sum {
  float a, b;
  __device__ __forceinline__ float total() const { return a + b; }
};
template <bool FAR, bool FINE, typename T>
__device__ __forceinline__ void add_vec(Sum& s, const Vec<T>& v, const Base& b, float c_hi, float c_lo) {
  constexpr int N = Vec<T>::N;
  float l[N];
  unpack(v, l);
  if constexpr (N == 8) {
    // a vector's terms first: as many additions, a quarter of them to a large sum
#pragma unroll
    for (int k = 0; k < N; ++k) l[k] = exp2_approx(exponent<FAR, FINE>(l[k], b, c_hi, c_lo));
    s.a += (l[0] + l[2]) + (l[4] + l[6]);
    s.b += (l[1] + l[3]) + (l[5] + l[7]);
  } else {
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      s.a += exp2_approx(exponent<FAR, FINE>(l[k], b, c_hi, c_lo));
      s.b += exp2_approx(exponent<FAR, FINE>(l[k + 1], b, c_hi, c_lo));
    }
  }
}
template <bool FINE, typename T>
__device__ __forceinline__ void add_any(Sum& s, const Vec<T>& v, const Base& b, float c_hi, float c_lo) {
  if (b.far) add_vec<true, FINE>(s, v, b, c_hi, c_lo);
  else add_vec<false, FINE>(s, v, b, c_hi, c_lo);
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
// The type in which a row's partial sums are joined: a thread's own sum is of 32 bits, but what
// is rounded here is a whole row's, and sums of log-probabilities (the rewards) add it up.
template <bool POLICY>
using Joined = std::conditional_t<POLICY, float, double>;
template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, s));
  return v;
}

// log S. ex2.approx falls short by kExpShort of its value on average (measured for negative
// exponents over the whole range of fractions; about 3e-8 too much for positive ones, which are
// few); all terms but the base's own, which is exact, carry that. From a 32-bit S the integer
// part of the logarithm is scaled in 64 bits, so that the result is off by 3e-8 (a step of its
// fraction's logarithm) instead of half a step of a value near 10 (5e-7).
constexpr double kExpShort = 5.05e-8;
__device__ __forceinline__ double log_sum(double S) {
  if (!(S > 0.0 && S < INFINITY)) return (double)NAN;
  return log(S) + (S > 1.0 ? kExpShort * ((S - 1.0) / S) : 0.0);
}
__device__ __forceinline__ double log_sum(float S) {
  if (!(S > 0.f && S < INFINITY)) return (double)NAN;
  int e;
  float m = frexpf(S, &e);  // 0.5 .. 1
  if (m < 0.75f) { m *= 2.f; --e; }
  return (double)e * kLn2 + (double)log1pf(m - 1.f) + (S > 1.f ? kExpShort * (double)((S - 1.f) / S) : 0.0);
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
struct PolicyHead {
  int kept, skipped;  // positions that count and that do not
  int sequences;      // with any that counts
  unsigned done;      // CTAs of the final sum that have finished
};
struct RowResult {
  float loss, kl, clipped;  // weighted loss; KL and 0 / 1, zero where the position does not count
};
constexpr int kSumRows = 512;  // rows of one CTA of the final sum
struct SumPart {
  double loss, kl, clipped;
};
struct PolicyWs {
  float2* stats;
  float* coef;
  PolicyHead* head;
  int* counts;
  int* order;  // the positions that count, then the others
  RowResult* rows;
  SumPart* parts;
  size_t zeroed;
};
__host__ __device__ inline size_t up16(size_t n) { return (n + 15) & ~size_t(15); }
inline PolicyWs policy_ws(void* ws, int64_t batch, int64_t rows, size_t* bytes) {
  char* q = static_cast<char*>(ws);
  size_t at = 0;
  PolicyWs w;
  w.stats = reinterpret_cast<float2*>(q + at);
  at += up16(sizeof(float2) * (size_t)rows);
  w.coef = reinterpret_cast<float*>(q + at);
  at += up16(sizeof(float) * (size_t)rows);
  w.head = reinterpret_cast<PolicyHead*>(q + at);
  at += up16(sizeof(PolicyHead));
  w.counts = reinterpret_cast<int*>(q + at);  // with the head, what is zero at the start
  at += up16(sizeof(int) * (size_t)batch);
  w.zeroed = (size_t)(q + at - reinterpret_cast<char*>(w.head));
  w.parts = reinterpret_cast<SumPart*>(q + at);
  at += up16(sizeof(SumPart) * (size_t)((rows + kSumRows - 1) / kSumRows));
  w.order = reinterpret_cast<int*>(q + at);
  at += up16(sizeof(int) * (size_t)rows);
  w.rows = reinterpret_cast<RowResult*>(q + at);
  at += up16(sizeof(RowResult) * (size_t)rows);
  *bytes = at;
  return w;
}

// Positions that count, by sequence and in all, and the rows' order: those first, so that
// they spread evenly whatever the mask. A warp takes 256 positions and adds its (whole) numbers
// to counters that are zero at the start, so the counts do not depend on the schedule. The
// order within the two groups does, but no result depends on it. A single CTA, which few
// positions need, zeroes the counters itself.
constexpr int kCountThreads = 256, kCountRows = 256;
__global__ void __launch_bounds__(kCountThreads) policy_count_kernel(TokenRows p, bool by_sequence, PolicyWs w) {
  const int lane = threadIdx.x & 31, R = (int)p.R;
  const int r0 = ((blockIdx.x * kCountThreads + threadIdx.x) >> 5) * kCountRows;
  if (gridDim.x == 1) {
    for (int i = threadIdx.x; i < (int)(w.zeroed / 4); i += kCountThreads) reinterpret_cast<int*>(w.head)[i] = 0;
    __syncthreads();
  }
  if (r0 >= R) return;
  unsigned flags = 0;  // bit k: position r0 + 32 k + lane
#pragma unroll
  for (int k = 0; k < kCountRows / 32; ++k) {
    const int r = r0 + 32 * k + lane, b = r / p.T;
    if (r < R && position(p, b, r - b * p.T).keep) flags |= 1u << k;
  }
  const int n = __reduce_add_sync(0xffffffffu, __popc(flags));
  int at = 0, skip = 0;
  if (lane == 0) {
    if (n > 0) at = atomicAdd(&w.head->kept, n);
    skip = atomicAdd(&w.head->skipped, min(kCountRows, R - r0) - n);
  }
  at = __shfl_sync(0xffffffffu, at, 0);
  skip = R - 1 - __shfl_sync(0xffffffffu, skip, 0);
  const unsigned below = (1u << lane) - 1;
#pragma unroll
  for (int k = 0; k < kCountRows / 32; ++k) {
    const int r = r0 + 32 * k + lane;
    const bool in = r < R, keep = flags >> k & 1;
    const unsigned yes = __ballot_sync(0xffffffffu, keep), no = __ballot_sync(0xffffffffu, in && !keep);
    if (keep) w.order[at + __popc(yes & below)] = r;
    else if (in) w.order[skip - __popc(no & below)] = r;
    at += __popc(yes);
    skip -= __popc(no);
    if (by_sequence && yes != 0) {
      // one addition where the 32 positions are of one sequence
      const int b = r / p.T, first = __shfl_sync(0xffffffffu, b, 0);
      const bool one = __all_sync(0xffffffffu, b == first || !in);
      const int add = one ? (lane == 0 ? __popc(yes) : 0) : keep ? 1 : 0;
      // whoever finds a sequence's counter at zero is its first
      if (add > 0 && atomicAdd(&w.counts[b], add) == 0) atomicAdd(&w.head->sequences, 1);
    }
  }
}

// A position's operands of the policy loss, loaded ahead of the row's sum.
struct TokenOps {
  float old_logp, adv, ref;
  double weight;
};
// The weight of a position, where it is the same for all.
__device__ __forceinline__ double even_weight(const PolicyArgs& a, const PolicyWs& w) {
  return a.by_sequence ? 0.0 : 1.0 / (double)w.head->kept;
}
__device__ __forceinline__ TokenOps token_ops(const PolicyArgs& a, const PolicyWs& w, int64_t b, int64_t t, double even) {
  TokenOps o;
  o.old_logp = map_at(a.old_logp, b, t);
  o.adv = map_at(a.adv, b, t);
  o.ref = a.ref.p ? map_at(a.ref, b, t) : 0.f;
  o.weight = a.by_sequence ? 1.0 / ((double)w.counts[b] * (double)w.head->sequences) : even;
  return o;
}

// exp(d) - 1 - d without the cancellation of a small d: the series to d^9 below 1/2 (its
// remainder is 2^-30 of the result), the difference above (infinite for an infinite d).
__device__ __forceinline__ float kl_term(float d) {
  if (d == INFINITY) return d;
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
    if (k != 0.f) {  // else it is only reported, also where it overflows
      o.loss = fmaf(k, o.kl, o.loss);
      o.dlogp = fmaf(-k, expm1f(d), o.dlogp);
    }
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
  unsigned* clear;  // zero for the kernel that follows; may be null
};

// The gradient of one row: g (one-hot - softmax). tok < 0: no element is the token's.
struct GradRow {
  Base base;
  float g, inv;  // inv = 1 / S
  int tok;
  float at;      // the token's logit
  // For 16-bit results |g| / S goes into the exponent, so that a multiplication is spared:
  // its rounding there, at most 2^-19 for |kg| < 64, is far below the result's own (2^-12).
  float kg;
  bool negative;  // -g < 0
  bool folded;
};
__device__ __forceinline__ GradRow grad_row(const Base& base, float g, float S, int tok, float at) {
  GradRow r{base, g, 1.f / S, tok, at, 0.f, g > 0.f, false};
  r.kg = base.k + log2f(fabsf(g) * r.inv);
  r.folded = !base.far && fabsf(r.kg) < 64.f && fabsf(base.k) < 64.f;  // false for NaN
  return r;
}
// Two floats of at least 0 to two 16-bit values in a word, their signs set. For bf16 by an
// addition (which rounds, ties up instead of to even, and sets the sign) and a byte selection:
// the conversion instruction shares the exponential's unit, which bounds these kernels.
__device__ __forceinline__ uint32_t signed_word(float a, float b, bool negative, __nv_bfloat16) {
  const uint32_t add = negative ? 0x80008000u : 0x8000u;
  return __byte_perm(__float_as_uint(a) + add, __float_as_uint(b) + add, 0x7632);
}
__device__ __forceinline__ uint32_t signed_word(float a, float b, bool negative, __half t) {
  return word(a, b, t) ^ (negative ? 0x80008000u : 0u);
}
template <typename T>
__device__ __forceinline__ Vec<T> vec_grad_folded(const Vec<T>& v, float kg, bool negative, float c_hi) {
  constexpr int N = Vec<T>::N;
  float l[N];
  unpack(v, l);
#pragma unroll
  for (int k = 0; k < N; ++k) l[k] = exp2_approx(fmaf(l[k], c_hi, kg));
  uint32_t o[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) o[k] = signed_word(l[2 * k], l[2 * k + 1], negative, T{});
  return Vec<T>{make_uint4(o[0], o[1], o[2], o[3])};
}
template <bool FAR, typename T>
__device__ __forceinline__ Vec<T> vec_grad(const Vec<T>& v, const GradRow& r, float c_hi, float c_lo) {
  float l[Vec<T>::N];
  unpack(v, l);
  const float q = -r.g * r.inv;
#pragma unroll
  for (int k = 0; k < Vec<T>::N; ++k) l[k] = q * exp2_approx(exponent<FAR, false>(l[k], r.base, c_hi, c_lo));
  return pack<T>(l);
}
template <typename T>
__device__ __forceinline__ T one_grad(float l, const GradRow& r, float hot, float c_hi, float c_lo) {
  return from_f32<T>(r.g * (hot - exp_one<false>(l, r.base, c_hi, c_lo) * r.inv));
}
// Vector j of a row to its place (the token's element is written again afterwards).
template <typename T>
__device__ __forceinline__ void put_grad(const Vec<T>& v, int j, T* out, const RowCut& c, const GradRow& r, bool same,
                                         float c_hi, float c_lo) {
  constexpr int N = Vec<T>::N;
  const Vec<T> o = r.base.far ? vec_grad<true>(v, r, c_hi, c_lo) : vec_grad<false>(v, r, c_hi, c_lo);
  const int i0 = c.head + j * N;
  if (same) {
    *reinterpret_cast<Vec<T>*>(out + i0) = o;
  } else {
    float x[N];  // rounded to T already
    unpack(o, x);
#pragma unroll
    for (int k = 0; k < N; ++k) out[i0 + k] = from_f32<T>(x[k]);
  }
}
// Vectors first, first + nt, ... below n, which go to places v0 + j of the row.
template <typename T, typename Get>
__device__ __forceinline__ void put_vecs(int first, int n, int nt, int v0, T* out, const RowCut& c, const GradRow& r,
                                         bool same, float c_hi, float c_lo, Get get) {
  Vec<T>* const dst = reinterpret_cast<Vec<T>*>(out + c.head) + v0;
  if (same && sizeof(T) == 2 && r.folded) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll 4
      for (int j = first; j < n; j += nt) dst[j] = vec_grad_folded(get(j), r.kg, r.negative, c_hi);
    }
  } else if (same && !r.base.far) {
#pragma unroll 4
    for (int j = first; j < n; j += nt) dst[j] = vec_grad<false>(get(j), r, c_hi, c_lo);
  } else {
    for (int j = first; j < n; j += nt) put_grad(get(j), v0 + j, out, c, r, same, c_hi, c_lo);
  }
}
// The token's element, by the thread that has written its vector: vectors v0 + tid, v0 + tid +
// nt, ... of [v0, v1). One before or behind the vectors is put_ends' work.
template <typename T>
__device__ __forceinline__ void put_token(T* out, const RowCut& c, const GradRow& r, int v0, int v1, int tid, int nt,
                                          float c_hi, float c_lo) {
  constexpr int N = Vec<T>::N;
  if (r.tok < c.head || r.tok >= c.tail0) return;
  const int j = (r.tok - c.head) / N;
  if (j >= v0 && j < v1 && (j - v0) % nt == tid) out[r.tok] = one_grad<T>(r.at, r, 1.f, c_hi, c_lo);
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
// From a row's sum to its results (`lead` writes them) and to what its gradient needs.
template <bool POLICY>
__device__ __forceinline__ GradRow finish_row(const TokenRows& p, const PolicyArgs& a, const PolicyWs& w, const RowOut& o,
                                              const TokenOps& x, int64_t r, float at_token, int tok, const Base& base,
                                              Joined<POLICY> S, bool lead) {
  // the token's exponent exactly as the sum's elements have theirs
  const double c = POLICY ? (double)p.c_hi : (double)p.c_hi + (double)p.c_lo;
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
  const float Sn = norm_sum<!POLICY>((float)S, base, p.c_lo);
  if (lead) {
    o.logp[r] = (float)logp;
    if (o.logp64) o.logp64[r] = logp;
    if (o.stats) o.stats[r] = make_float2(base.m, Sn);
  }
  return grad_row(base, (float)((double)coef * p.scale), Sn, tok, at_token);
}

// Whether a sum over an assumed base can be trusted (false for NaN too). Logits up to log2 S above
// the base have exponents that large, whose roundings (three of half a step) and lacking lower half
// of c (2^-23 of the exponent) move p by ln 2 (3 * 2^-20 + 20 * 2^-23) = 2^-18 at S = 2^20. Far above
// that p loses more, and the gradient's factor g / S leaves the normal numbers where g is small.
// Logits that are all alike have S = V, so that the bound has to be above a vocabulary's size.
__device__ __forceinline__ bool in_range(float S) { return S > 8.673617e-19f && S < 1048576.f; }  // 2^-60, 2^20

template <bool POLICY>
struct RowShared {
  Joined<POLICY> part[kRowWarps];  // the warps' sums
  GradRow row;
  bool again;
};

// The largest of a row's first vectors (of all elements, where there is no vector).
template <typename T>
__device__ __forceinline__ float first_max(const T* row, int V, const RowCut& c, int lane) {
  if (c.nv > 0) return lane < c.nv ? vec_max(reinterpret_cast<const Vec<T>*>(row + c.head)[lane]) : -INFINITY;
  return lane < V ? to_f32(row[lane]) : -INFINITY;
}

// Joins the threads' sums over the cluster and finishes the row. `s`: this thread's sum over
// `base`; `get(j)`: vector j of this CTA's part. On return sh.row holds the row.
template <typename T, bool POLICY, typename Get>
__device__ __forceinline__ void join_row(const TokenRows& p, const PolicyArgs& a, const PolicyWs& w, const RowOut& o,
                                         RowShared<POLICY>& sh, const TokenOps& x, int64_t r, const T* row,
                                         const RowCut& c, int n, Base base, float s, float at_token, int tok, Get get) {
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, W = nt >> 5;
  auto meet = [&]() {
    if (C > 1) cl.sync();
    else __syncthreads();
  };
  using F = Joined<POLICY>;
  F* part = sh.part;
  const F mine = warp_sum((F)s);
  if (lane == 0) part[warp] = mine;
  meet();
  if (warp == 0) {
    // by CTA first: the order of token_grad_rows_kernel, for the same bits
    F S = 0;
    for (int k = 0; k < C; ++k) S += warp_sum(lane < W ? (C > 1 ? cl.map_shared_rank(part, k)[lane] : part[lane]) : F(0));
    if (lane == 0) {
      sh.again = base.far || !in_range((float)S);
      if (!sh.again) sh.row = finish_row<POLICY>(p, a, w, o, x, r, at_token, tok, base, S, rank == 0);
    }
  }
  __syncthreads();
  if (!sh.again) return;
  // rare: the row's true maximum, then its sum
  auto ends = [&](auto f) {
    if (rank == 0) {
      for (int i = tid; i < c.head; i += nt) f(to_f32(row[i]));
      for (int i = c.tail0 + tid; i < p.V; i += nt) f(to_f32(row[i]));
    }
  };
  auto all = [&](F v, bool largest) {
    meet();  // the parts of the last sum have been read
    if (lane == 0) part[warp] = v;
    meet();
    F y = largest ? -INFINITY : F(0);
    for (int k = 0; k < C; ++k) {  // in the same order as the first sum
      const F z = lane >= W ? (largest ? -INFINITY : F(0)) : C > 1 ? cl.map_shared_rank(part, k)[lane] : part[lane];
      if (largest) y = fmaxf((float)y, warp_max((float)z));
      else y += warp_sum(z);
    }
    return y;
  };
  float mx = -INFINITY;
  for (int j = tid; j < n; j += nt) mx = fmaxf(mx, vec_max(get(j)));
  ends([&](float l) { mx = fmaxf(mx, l); });
  base = base_at((float)all(warp_max(mx), true), p.c_hi);
  Sum s2{0.f, 0.f};
  for (int j = tid; j < n; j += nt) add_any<!POLICY>(s2, get(j), base, p.c_hi, p.c_lo);
  s = s2.total();
  ends([&](float l) { s += exp_one<!POLICY>(l, base, p.c_hi, p.c_lo); });
  const F S = all(warp_sum((F)s), false);
  if (tid == 0) sh.row = finish_row<POLICY>(p, a, w, o, x, r, at_token, tok, base, S, rank == 0);
  __syncthreads();
}

// One cluster of CTAs (of one CTA where there are rows enough) per row. A policy gradient of
// rows too long for token_grad_rows_kernel is written from a second reading.
// Bound by the memory: 7952 rows of 50277 bf16 logits in 126 us, 6.3 TB/s, 97% of a copy's rate;
// 1200 such rows of 2000 in 25 us (4.9 TB/s: the last rows run beside few others). Eight loads in
// flight per thread, the first while the base is found and the last, which do not fill a turn,
// all at once as well: with those one by one rows of 24000 logits had 4.8 TB/s instead of 6.1.
template <typename T, bool POLICY, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) token_rows_kernel(TokenRows p, PolicyArgs a, PolicyWs w, RowOut o) {
  constexpr int U = 8;  // loads in flight per thread
  __shared__ RowShared<POLICY> sh;
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int64_t r = blockIdx.x / C;
  const int64_t b = r / p.T, t = r - b * p.T;
  constexpr int nt = NT;
  const int tid = threadIdx.x, lane = tid & 31;
  if constexpr (!POLICY)
    if (o.clear && blockIdx.x == 0 && threadIdx.x == 0) *o.clear = 0;
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
  const Vec<T>* mine = reinterpret_cast<const Vec<T>*>(row + c.head) + v0;
  const float at_token = pos.known ? to_f32(row[pos.tok]) : NAN;
  TokenOps x{};
  if constexpr (POLICY)
    if (tid == 0) x = token_ops(a, w, b, t, even_weight(a, w));
  Vec<T> v[U];
  auto load = [&](int j0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j0 + tid + u * nt < n) v[u] = mine[j0 + tid + u * nt];
  };
  load(0);  // while the base is found
  const Base base = base_at(fmaxf(warp_max(first_max(row, p.V, c, lane)), at_token), p.c_hi);
  Sum s2{0.f, 0.f};
  for (int j0 = 0; j0 < n; j0 += U * nt) {
    if (j0 > 0) load(j0);
    if (j0 + U * nt <= n) {
#pragma unroll
      for (int u = 0; u < U; ++u) add_vec<false, !POLICY>(s2, v[u], base, p.c_hi, p.c_lo);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (j0 + tid + u * nt < n) add_vec<false, !POLICY>(s2, v[u], base, p.c_hi, p.c_lo);
    }
  }
  float s = s2.total();
  if (rank == 0) {
    for (int i = tid; i < c.head; i += nt) s += exp_one<!POLICY>(to_f32(row[i]), base, p.c_hi, p.c_lo);
    for (int i = c.tail0 + tid; i < p.V; i += nt) s += exp_one<!POLICY>(to_f32(row[i]), base, p.c_hi, p.c_lo);
  }
  join_row<T, POLICY>(p, a, w, o, sh, x, r, row, c, n, base, s, at_token, pos.known ? (int)pos.tok : -1,
                      [&](int k) { return mine[k]; });
  if (C > 1) cl.barrier_arrive();  // this CTA reads no other's part from here on
  if constexpr (POLICY) {
    if (drow) {
      const GradRow gr = sh.row;
      if (gr.g == 0.f) {
        fill<T>(drow, e0, e1, tid, nt, from_f32<T>(0.f));
      } else {
        const bool same = same_boundary(drow, c);
        put_vecs<T>(tid, n, nt, v0, drow, c, gr, same, p.c_hi, p.c_lo, [&](int k) { return mine[k]; });
        put_token(drow, c, gr, v0, v1, tid, nt, p.c_hi, p.c_lo);
        if (rank == 0) put_ends(row, drow, p.V, c, gr, tid, nt, p.c_hi, p.c_lo);
      }
    }
  }
  if (C > 1) cl.barrier_wait();  // no CTA leaves while another reads its part
}

// The policy loss and its gradient, the logits read once. CTAs (clusters of them, where a row
// is split) stay on the device and take the rows that count in turn; a CTA keeps its part of
// a row in shared memory between the sum and the gradient. One warp copies: it fetches what
// the row needs beside its logits a row ahead, refills each piece of the part with the next
// row's as soon as the other warps have read it for the gradient, and writes the zeros of the
// positions that do not count, so that the memory stays busy while the others compute.
// 32 x 1024 x 50280 bf16, 0.6 of the positions counting: 0.91 ms in all, 5.27 GB at 5.8 TB/s,
// 88% of a copy's rate. Before: every row read again from the L2 cache 1.14 ms; copies through
// the threads' own cp.async, two rows' places 1.77 ms (a thread's copies in flight are few, and
// were only issued while gradients were written); without the pieces' fixed number of vectors
// (a bound check and a wait for two vectors) 1.19 ms, bound by instructions. Where a part leaves
// room for one CTA of an SM only (above kPlaceBytes) the row goes to a cluster of two or more.
constexpr int kPieces = 8;           // at most
constexpr int kPieceVecs = 4;        // vectors of a piece per thread: few enough waits and bounds beside the work
constexpr int kZeroBytes = 2048;
constexpr uint32_t kWaitLimit = 1u << 24;

template <typename T>
struct RowInfo {
  const T* row;
  T* drow;
  int64_t r;
  RowCut c;
  int v0, n;
  Base base;
  TokenOps x;
  float at_token;
  int tok;
};
template <typename T>
struct GradRowsShared {
  alignas(16) unsigned char zeros[kZeroBytes];
  uint64_t full[kPieces], empty[kPieces], info_full[2], info_empty[2], met[2];
  float part[2][kRowWarps];
  float other[2][8];  // sums of the cluster's CTAs
  float sum;
  bool again[2], stop[2];
  int dead;           // a wait gave up: everyone leaves
  GradRow row[2];
  RowInfo<T> info[2];
};

__device__ unsigned g_token_error;

// A bounded wait of one thread. Where it gives up, so does everyone who waits in this CTA.
__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity, int* dead) {
  if (sm100::mbar_try_wait(bar, parity)) return true;
  for (uint32_t i = 0; i < kWaitLimit; ++i) {
    if (sm100::mbar_try_wait(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(dead)) return false;
  }
  *reinterpret_cast<volatile int*>(dead) = 1;
  atomicOr(&g_token_error, 1u);
  return false;
}
// The same for a whole warp, which agrees on the answer.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, int* dead) {
  return __all_sync(0xffffffffu, wait_one(bar, parity, dead));
}
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(sm100::smem_u32(src)),
               "r"(bytes)
               : "memory");
}
// v into other[slot] of CTA `to` of the cluster, counted on its barrier `met`
__device__ __forceinline__ void send(float* slot, uint64_t* met, int to, float v) {
  uint32_t at, bar;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(sm100::smem_u32(slot)), "r"(to));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(sm100::smem_u32(met)), "r"(to));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(at),
               "r"(__float_as_uint(v)), "r"(bar)
               : "memory");
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT + 32, NT == 128 ? 6 : 1024 / NT)
    token_grad_rows_kernel(TokenRows p, PolicyArgs a, PolicyWs w, RowOut o, int pieces) {
  constexpr int W = NT / 32, kPiece = kPieceVecs * NT;
  extern __shared__ __align__(16) uint4 kept_raw[];
  __shared__ GradRowsShared<T> sh;
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int cid = blockIdx.x / C, ncl = gridDim.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Vec<T>* const kept = reinterpret_cast<Vec<T>*>(kept_raw);
  for (int i = tid; i < kZeroBytes / 16; i += NT + 32) reinterpret_cast<uint4*>(sh.zeros)[i] = make_uint4(0, 0, 0, 0);
  sm100::fence_proxy_async_smem();  // the zeros, for the copies that read them
  if (tid == 0) {
    for (int k = 0; k < kPieces; ++k) {
      sm100::mbar_init(&sh.full[k], 1);
      sm100::mbar_init(&sh.empty[k], W);
    }
    for (int k = 0; k < 2; ++k) {
      sm100::mbar_init(&sh.info_full[k], 1);
      sm100::mbar_init(&sh.info_empty[k], W);
      sm100::mbar_init(&sh.met[k], 1);
    }
    sh.dead = 0;
    sm100::fence_barrier_init();
  }
  if (C > 1) cl.sync();
  else __syncthreads();
  const int kept_rows = w.head->kept;

  if (warp == W) {
    // ------------------------------------------------------------------ the copying warp
    const double even = even_weight(a, w);
    CopyRounds rounds;  // lane 0 issues
    bool ok = true;
    // zeros to a position that does not count, this CTA's part of the row
    auto skip = [&](int i) {
      const int r = w.order[i];
      const int64_t b = r / p.T, t = r - b * p.T;
      T* const drow = static_cast<T*>(o.dlogits) + b * o.dsb + t * o.dst;
      if (rank == 0 && lane == 0) skip_row<true>(o, w, r);
      const RowCut c = cut_row(drow, p.V);
      const int v0 = (int)((int64_t)c.nv * rank / C), v1 = (int)((int64_t)c.nv * (rank + 1) / C);
      Vec<T>* const dst = reinterpret_cast<Vec<T>*>(drow + c.head);
      constexpr int per = kZeroBytes / 16;
      for (int v = v0 + lane * per; v < v1; v += 32 * per) bulk_store(dst + v, sh.zeros, (uint32_t)min(per, v1 - v) * 16u);
      if (rank == 0) {
        if (lane < c.head) drow[lane] = from_f32<T>(0.f);
        if (c.tail0 + lane < p.V) drow[c.tail0 + lane] = from_f32<T>(0.f);
      }
      sm100::bulk_commit();
    };
    const int mine = cid < kept_rows ? (kept_rows - cid + ncl - 1) / ncl : 0;  // rows that count
    const int rest = p.R - kept_rows, skips = cid < rest ? (int)(rest - cid + ncl - 1) / ncl : 0;
    int skipped = 0;
    for (int i = cid; i < kept_rows; i += ncl, rounds.next()) {
      const uint32_t round = rounds.round;
      const int slot = round & 1;
      if (round >= 2 && !(ok = wait_warp(&sh.info_empty[slot], ((round >> 1) - 1) & 1, &sh.dead))) break;
      RowInfo<T> q;
      q.r = w.order[i];
      const int b = (int)q.r / p.T, t = (int)q.r - b * p.T;
      q.row = static_cast<const T*>(p.logits) + b * p.sb + t * p.st;
      q.drow = static_cast<T*>(o.dlogits) + b * o.dsb + t * o.dst;
      q.c = cut_row(q.row, p.V);
      q.v0 = (int)((int64_t)q.c.nv * rank / C);
      q.n = (int)((int64_t)q.c.nv * (rank + 1) / C) - q.v0;
      const int64_t tok = map_at(p.tok, b, t);
      const bool known = tok >= 0 && tok < p.V;
      q.tok = known ? (int)tok : -1;
      q.x = token_ops(a, w, b, t, even);
      q.at_token = known ? to_f32(q.row[tok]) : NAN;
      q.base = base_at(fmaxf(warp_max(first_max(q.row, p.V, q.c, lane)), q.at_token), p.c_hi);
      if (lane == 0) {
        sh.info[slot] = q;
        sm100::mbar_arrive(&sh.info_full[slot]);
        const Vec<T>* src = reinterpret_cast<const Vec<T>*>(q.row + q.c.head) + q.v0;
        for (int k = 0; k < pieces; ++k) {
          if (round >= 1 && !(ok = wait_one(&sh.empty[k], (round - 1) & 1, &sh.dead))) break;
          const int n = min(kPiece, q.n - k * kPiece);
          sm100::mbar_expect_tx(&sh.full[k], n > 0 ? (uint32_t)n * 16u : 0u);
          if (n > 0) sm100::bulk_load(kept + k * kPiece, src + k * kPiece, (uint32_t)n * 16u, &sh.full[k]);
          rounds.issue(k);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      // in step with the rows that count
      for (const int until = (int)((int64_t)skips * (round + 1) / mine); skipped < until; ++skipped)
        skip(kept_rows + cid + skipped * ncl);
    }
    for (; ok && skipped < skips; ++skipped) skip(kept_rows + cid + skipped * ncl);
    if (lane == 0) {
      // copies in flight end before the CTA does, also where the others have given up on them
      for (int k = 0; k < pieces; ++k)
        if (rounds.copied(k)) sm100::mbar_wait(&sh.full[k], rounds.last_phase(k), kWaitLimit);
    }
    sm100::bulk_wait0();
  } else {
    // ---------------------------------------------------- the warps that sum and write
    uint32_t meets = 0;
    // The sum (or maximum) over the cluster, by warp 0. Two barriers in turn: a CTA may be one
    // exchange ahead of this one, whose values must not count for the present one.
    auto over_cluster = [&](float v, bool largest) {
      if (C == 1) return v;
      const int s = meets & 1;
      if (lane == 0) sm100::mbar_expect_tx(&sh.met[s], 4u * C);
      __syncwarp();
      if (lane < C) send(&sh.other[s][rank], &sh.met[s], lane, v);
      wait_warp(&sh.met[s], (meets >> 1) & 1, &sh.dead);
      ++meets;
      float y = sh.other[s][0];
      for (int k = 1; k < C; ++k) y = largest ? fmaxf(y, sh.other[s][k]) : y + sh.other[s][k];
      return y;
    };
    uint32_t round = 0;
    for (int i = cid; i < kept_rows; i += ncl, ++round) {
      const int slot = round & 1;
      // where a wait gives up the warp does no more work, but still meets the others below,
      // where all learn of it
      bool ok = wait_warp(&sh.info_full[slot], (round >> 1) & 1, &sh.dead);
      const RowInfo<T>& q = sh.info[slot];
      const RowCut c = ok ? q.c : RowCut{0, 0, p.V};
      const int n = ok ? q.n : 0, v0 = q.v0;
      const T* const row = q.row;
      T* const drow = q.drow;
      Base base = q.base;
      Sum s2{0.f, 0.f};
      for (int k = 0; k < pieces; ++k) {
        const int left = n - k * kPiece;
        if (left <= 0) break;
        if (!(ok = wait_warp(&sh.full[k], round & 1, &sh.dead))) break;
        const Vec<T>* const at = kept + k * kPiece + tid;
        if (left >= kPiece) {
          Vec<T> v[kPieceVecs];
#pragma unroll
          for (int u = 0; u < kPieceVecs; ++u) v[u] = at[u * NT];
#pragma unroll
          for (int u = 0; u < kPieceVecs; ++u) add_vec<false, false>(s2, v[u], base, p.c_hi, p.c_lo);
        } else {
          for (int j = tid; j < left; j += NT) add_vec<false, false>(s2, at[j - tid], base, p.c_hi, p.c_lo);
        }
      }
      float s = s2.total();
      auto ends = [&](auto f) {
        if (rank == 0) {
          if (tid < c.head) f(to_f32(row[tid]));
          if (c.tail0 + tid < p.V) f(to_f32(row[c.tail0 + tid]));
        }
      };
      ends([&](float l) { s += exp_one<false>(l, base, p.c_hi, p.c_lo); });
      s = warp_sum(s);
      if (lane == 0) sh.part[slot][warp] = s;
      bar_sync(1, NT);
      if (warp == 0) {
        const float S = over_cluster(warp_sum(lane < W ? sh.part[slot][lane] : 0.f), false);
        if (lane == 0) {
          const bool stop = *reinterpret_cast<volatile int*>(&sh.dead) != 0;
          sh.stop[slot] = stop;
          sh.again[slot] = base.far || !in_range(S);
          if (!stop && !sh.again[slot])
            sh.row[slot] = finish_row<true>(p, a, w, o, q.x, q.r, q.at_token, q.tok, base, S, rank == 0);
        }
      }
      bar_sync(1, NT);
      if (sh.stop[slot]) break;
      if (sh.again[slot]) {
        // rare: the row's true maximum, then its sum
        auto all = [&](float v, bool largest) {
          if (lane == 0) sh.part[slot][warp] = v;
          bar_sync(1, NT);
          if (warp == 0) {
            float y = lane < W ? sh.part[slot][lane] : (largest ? -INFINITY : 0.f);
            y = over_cluster(largest ? warp_max(y) : warp_sum(y), largest);
            if (lane == 0) sh.sum = y;
          }
          bar_sync(1, NT);
          return sh.sum;
        };
        float mx = -INFINITY;
        for (int j = tid; j < n; j += NT) mx = fmaxf(mx, vec_max(kept[j]));
        ends([&](float l) { mx = fmaxf(mx, l); });
        base = base_at(all(warp_max(mx), true), p.c_hi);
        s2 = Sum{0.f, 0.f};
        for (int j = tid; j < n; j += NT) add_any<false>(s2, kept[j], base, p.c_hi, p.c_lo);
        s = s2.total();
        ends([&](float l) { s += exp_one<false>(l, base, p.c_hi, p.c_lo); });
        const float S = all(warp_sum(s), false);
        if (tid == 0) sh.row[slot] = finish_row<true>(p, a, w, o, q.x, q.r, q.at_token, q.tok, base, S, rank == 0);
        bar_sync(1, NT);
      }
      const GradRow gr = sh.row[slot];
      const bool same = same_boundary(drow, c), zero = gr.g == 0.f;
      const int kind = zero ? 0 : !same || gr.base.far ? 3 : sizeof(T) == 2 && gr.folded ? 1 : 2;
      if (zero)
        fill<T>(drow, (int)((int64_t)p.V * rank / C), (int)((int64_t)p.V * (rank + 1) / C), tid, NT, from_f32<T>(0.f));
      Vec<T>* const dst = reinterpret_cast<Vec<T>*>(drow + c.head) + v0 + tid;
      for (int k = 0; k < pieces; ++k) {
        const int left = n - k * kPiece;
        const Vec<T>* const at = kept + k * kPiece + tid;
        Vec<T>* const to = dst + k * kPiece;
        if (left >= kPiece && (kind == 1 || kind == 2)) {
          Vec<T> v[kPieceVecs];
#pragma unroll
          for (int u = 0; u < kPieceVecs; ++u) v[u] = at[u * NT];
          __syncwarp();
          if (lane == 0) sm100::mbar_arrive(&sh.empty[k]);  // read: its place can be filled again
          if (kind == 1) {
            if constexpr (sizeof(T) == 2) {
#pragma unroll
              for (int u = 0; u < kPieceVecs; ++u) to[u * NT] = vec_grad_folded(v[u], gr.kg, gr.negative, p.c_hi);
            }
          } else {
#pragma unroll
            for (int u = 0; u < kPieceVecs; ++u) to[u * NT] = vec_grad<false>(v[u], gr, p.c_hi, p.c_lo);
          }
        } else {
          if (!zero)
            for (int j = tid; j < left; j += NT)
              put_grad(at[j - tid], v0 + k * kPiece + j, drow, c, gr, same, p.c_hi, p.c_lo);
          __syncwarp();
          if (lane == 0) sm100::mbar_arrive(&sh.empty[k]);
        }
      }
      if (!zero) {
        // the token's element again, by the thread that wrote its vector
        const int jt = gr.tok >= c.head && gr.tok < c.tail0 ? (gr.tok - c.head) / Vec<T>::N - v0 : -1;
        if (jt >= 0 && jt < n && jt % NT == tid) drow[gr.tok] = one_grad<T>(gr.at, gr, 1.f, p.c_hi, p.c_lo);
        if (rank == 0) put_ends(row, drow, p.V, c, gr, tid, NT, p.c_hi, p.c_lo);
      }
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&sh.info_empty[slot]);
    }
  }
  if (C > 1) cl.sync();  // no CTA leaves while another sends to it
}

// Rows of up to 24 KB. A warp takes 32 / G consecutive rows at a time, which bulk copies bring to
// its place in shared memory, sums each with G lanes and writes their gradients from there. A lane
// is a row where a row's few numbers are concerned: its token, logarithm, loss and gradient's
// factor cost a warp as much for one row as for eight. No warp waits for another, and none copies
// ahead: twice the warps hide a copy better than a second place each (4096 bf16 logits a row, loss
// and gradient: 5.1 TB/s read and written against 4.3). What bounds it: in short 16-bit rows the
// latency of loads that depend on one another (position, token's logit, ends; at 300 logits 57% of
// the issue slots are busy, at 1000 50-66% of the exponential's unit, with 30-42% of the warps
// active), the memory else.
// 400 million logits, at most 262144 rows, TB/s, without a gradient | with the policy's:
//   bf16, rows of 300, 1000, 2500, 4096, 8192: 2.9 4.3 4.7 5.5 5.7 | 2.8 4.2 4.7 5.4 5.4
//   fp32, rows of 300, 1000, 2500, 4096, 6000: 5.8 6.5 6.6 6.9 6.6 | 4.5 5.4 5.6 5.6 6.1
// A warp per row in registers (up to 4 KB) and a CTA per row (above) had 0.9 2.7 1.2 2.3 3.9 for
// bf16 rows without a gradient and 0.9 2.7 2.1 2.9 4.0 with it.
constexpr int kWarpThreads = 64;
template <bool POLICY>
constexpr int kWarpCtas = POLICY ? 14 : 16;  // of an SM at most: 72 and 64 registers
constexpr int64_t kWarpRow = 24 * 1024;      // rows of fp32 logits of 32 KB: a CTA per row 6.8 TB/s, this 6.2
constexpr int64_t kSmSmem = 227 * 1024;
template <typename T, int G>
struct WarpRowsShared {
  static constexpr int E = 32 / sizeof(T);  // single elements before and behind a row's vectors: fewer than this
  uint64_t full[kWarpThreads / 32];
  int dead;
  T ends[kWarpThreads / 32][32 / G * E];
};
struct LaneRow {
  int r, b, t, tok, head, nv;
  bool mine, keep;
  float at_token;
  TokenOps x;
};
template <typename T, bool POLICY, int G>
__global__ void __launch_bounds__(kWarpThreads, kWarpCtas<POLICY>)
    token_warp_rows_kernel(TokenRows p, PolicyArgs a, PolicyWs w, RowOut o, int row_vecs) {
  constexpr int N = Vec<T>::N, E = WarpRowsShared<T, G>::E, W = kWarpThreads / 32;
  constexpr int each = 32 / G;  // rows of a batch
  using F = Joined<POLICY>;
  extern __shared__ __align__(16) uint4 places_raw[];
  __shared__ WarpRowsShared<T, G> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Vec<T>* const place = reinterpret_cast<Vec<T>*>(places_raw) + (size_t)warp * each * row_vecs;
  if constexpr (!POLICY)
    if (o.clear && blockIdx.x == 0 && threadIdx.x == 0) *o.clear = 0;
  if (threadIdx.x == 0) {
    for (int k = 0; k < W; ++k) sm100::mbar_init(&sh.full[k], 1);
    sh.dead = 0;
    sm100::fence_barrier_init();
  }
  __syncthreads();
  const T* const logits = static_cast<const T*>(p.logits);
  auto row_at = [&](int b, int t) { return logits + b * p.sb + t * p.st; };
  auto of = [](auto v, int i) { return __shfl_sync(0xffffffffu, v, i); };

  double even = 0.0;
  if constexpr (POLICY) even = even_weight(a, w);

  // the rows of a batch: their vectors on the way to its place, the rest here
  auto fetch = [&](int batch) {
    const int r0 = batch * each, rows = min(each, (int)p.R - r0);
    LaneRow q;
    q.mine = lane < rows;
    q.r = r0 + min(lane, rows - 1);
    q.b = q.r / p.T;
    q.t = q.r - q.b * p.T;
    const Position pos = position(p, q.b, q.t);
    q.keep = q.mine && pos.keep;
    q.tok = pos.known ? (int)pos.tok : -1;
    const T* const row = row_at(q.b, q.t);
    const RowCut c = cut_row(row, p.V);
    q.head = c.head;
    q.nv = c.nv;
    const uint32_t bytes = q.keep ? 16u * c.nv : 0u, all = __reduce_add_sync(0xffffffffu, bytes);
    if (lane == 0) sm100::mbar_expect_tx(&sh.full[warp], all);
    __syncwarp();
    if (bytes) sm100::bulk_load(place + lane * row_vecs, row + c.head, bytes, &sh.full[warp]);
    q.at_token = NAN;
    q.x = TokenOps{};
    if (q.keep) {
      if (pos.known) q.at_token = to_f32(row[pos.tok]);
      if constexpr (POLICY) q.x = token_ops(a, w, q.b, q.t, even);
    }
    if (const unsigned need = __ballot_sync(0xffffffffu, q.keep && p.V != c.nv * N)) {
      T* const ends = sh.ends[warp];
#pragma unroll
      for (int k0 = 0; k0 < each; k0 += 32 / E) {
        const int k = k0 + lane / E, e = lane % E;
        const int head = of(q.head, k), nv = of(q.nv, k), b = of(q.b, k), t = of(q.t, k);
        if ((need >> k & 1) && e < p.V - nv * N) ends[k * E + e] = row_at(b, t)[e < head ? e : nv * N + e];
      }
    }
    __syncwarp();  // the ends
    return q;
  };

  // a row is summed and written by G lanes, of which this is number l
  const int i = lane / G, l = lane % G;
  auto work = [&](const LaneRow& q) {
    const int rows = __popc(__ballot_sync(0xffffffffu, q.mine));
    const unsigned keeps = __ballot_sync(0xffffffffu, q.keep);
    Base my_base{};
    F my_S = 0;
    if (keeps) {
      const int nv = of(q.nv, i), singles = p.V - nv * N;
      const bool keep = keeps >> i & 1;
      const Vec<T>* const v = place + i * row_vecs;
      const T* const ends = sh.ends[warp] + i * E;
      // over the row's lanes
      auto all_max = [](float x) {
#pragma unroll
        for (int k = G / 2; k > 0; k >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, k));
        return x;
      };
      auto all_sum = [](F x) {
#pragma unroll
        for (int k = G / 2; k > 0; k >>= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
        return x;
      };
      auto ends_max = [&] {
        float m = -INFINITY;
        if (keep)
          for (int e = l; e < singles; e += G) m = fmaxf(m, to_f32(ends[e]));
        return m;
      };
      float m = ends_max();
      if (keep && l < nv) m = fmaxf(m, vec_max(v[l]));
      Base base = base_at(fmaxf(all_max(m), of(q.at_token, i)), p.c_hi);
      auto sum = [&](auto known, bool sums) {
        Sum s2{0.f, 0.f};
        if (sums) {
#pragma unroll 4
          for (int j = l; j < nv; j += G) {
            if constexpr (decltype(known)::value) add_any<!POLICY>(s2, v[j], base, p.c_hi, p.c_lo);
            else add_vec<false, !POLICY>(s2, v[j], base, p.c_hi, p.c_lo);
          }
          for (int e = l; e < singles; e += G) s2.a += exp_one<!POLICY>(to_f32(ends[e]), base, p.c_hi, p.c_lo);
        }
        return all_sum((F)s2.total());
      };
      F S = sum(std::false_type{}, keep);
      const bool again = keep && (base.far || !in_range((float)S));
      if (__any_sync(0xffffffffu, again)) {
        // rare: the row's true maximum, then its sum
        m = ends_max();
        if (again)
          for (int j = l; j < nv; j += G) m = fmaxf(m, vec_max(v[j]));
        m = all_max(m);
        if (again) base = base_at(m, p.c_hi);
        const F y = sum(std::true_type{}, again);
        if (again) S = y;
      }
      // to the row's lane
      const int from = lane * G & 31;
      my_base = Base{of(base.m, from), of(base.k, from), of((int)base.far, from) != 0};
      my_S = of(S, from);
    }
    GradRow gr{};
    if (q.keep) {
      gr = finish_row<POLICY>(p, a, w, o, q.x, q.r, q.at_token, q.tok, my_base, my_S, true);
    } else if (q.mine) {
      skip_row<POLICY>(o, w, q.r);
    }
    if constexpr (POLICY) {
      if (!o.dlogits) return;
      const int b = of(q.b, i), t = of(q.t, i);
      T* const drow = static_cast<T*>(o.dlogits) + b * o.dsb + t * o.dst;
      const GradRow y{Base{of(gr.base.m, i), of(gr.base.k, i), of((int)gr.base.far, i) != 0}, of(gr.g, i), of(gr.inv, i),
                      of(gr.tok, i), of(gr.at, i), of(gr.kg, i), of((int)gr.negative, i) != 0,
                      of((int)gr.folded, i) != 0};
      RowCut c;
      c.head = of(q.head, i);
      c.nv = of(q.nv, i);
      c.tail0 = c.head + c.nv * N;
      if (i >= rows) return;
      if (y.g == 0.f) {  // a position that does not count among them
        fill<T>(drow, 0, p.V, l, G, from_f32<T>(0.f));
        return;
      }
      const Vec<T>* const v = place + i * row_vecs;
      put_vecs<T>(l, c.nv, G, 0, drow, c, y, same_boundary(drow, c), p.c_hi, p.c_lo, [&](int j) { return v[j]; });
      put_token(drow, c, y, 0, c.nv, l, G, p.c_hi, p.c_lo);
      for (int e = l; e < p.V - c.nv * N; e += G) {
        const int j = e < c.head ? e : c.nv * N + e;
        drow[j] = one_grad<T>(to_f32(sh.ends[warp][i * E + e]), y, j == y.tok ? 1.f : 0.f, p.c_hi, p.c_lo);
      }
    }
  };

  const int batches = (int)((p.R + each - 1) / each), warps = gridDim.x * W;
  int batch = blockIdx.x * W + warp;
  if (batch >= batches) return;
  for (uint32_t n = 0;; ++n) {
    const LaneRow q = fetch(batch);
    if (!wait_warp(&sh.full[warp], n & 1, &sh.dead)) {
      sm100::mbar_wait(&sh.full[warp], n & 1, kWaitLimit);  // copies in flight end before the CTA does
      return;
    }
    work(q);
    __syncwarp();  // all have read the place
    if (batch >= batches - warps) return;
    batch += warps;
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
    const double n = w.head->kept > 0 ? (double)w.head->kept : 1.0;
    *loss = (float)s.loss;
    *kl = (float)(s.kl / n);
    *clipped = (float)(s.clipped / n);
  }
}

// Rewards of the answers, then (by the CTA that finishes last) the loss of the pairs and the
// derivative by each answer's log-probabilities. One CTA per answer.
struct PrefWs {
  float2* stats;
  float* coef;      // (2 N)
  unsigned* done;
  double* rewards;  // (2 N)
  double* logp;     // (2 N, T)
};
inline PrefWs pref_ws(void* ws, int64_t batch, int64_t rows, size_t* bytes) {
  char* q = static_cast<char*>(ws);
  size_t at = 0;
  PrefWs w;
  w.stats = reinterpret_cast<float2*>(q + at);
  at += up16(sizeof(float2) * (size_t)rows);
  w.coef = reinterpret_cast<float*>(q + at);
  at += up16(sizeof(float) * (size_t)batch);
  w.done = reinterpret_cast<unsigned*>(q + at);
  at += 16;
  w.rewards = reinterpret_cast<double*>(q + at);
  at += up16(sizeof(double) * (size_t)batch);
  w.logp = reinterpret_cast<double*>(q + at);
  at += up16(sizeof(double) * (size_t)rows);
  *bytes = at;
  return w;
}

__global__ void __launch_bounds__(kSumThreads)
    preference_pairs_kernel(TokenRows p, Map2<const float> ref, double beta, double smoothing, int pairs,
                            PrefWs w, float* loss, float* rewards) {
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
    const double q = exp(-fabs(z)), l = log1p(q);  // softplus(-|z|)
    // a side without weight counts nothing, also where it is infinite
    if (smoothing < 1.0) s += (1.0 - smoothing) * (l + fmax(-z, 0.0));
    if (smoothing > 0.0) s += smoothing * (l + fmax(z, 0.0));
    // e sigma(z) - (1 - e) sigma(-z): sigma(z) - (1 - e) would lose sigma(-z) in the 1
    const double less = q / (1.0 + q), more = 1.0 / (1.0 + q);  // sigma(-|z|), sigma(|z|)
    const double dz = (smoothing * (z < 0.0 ? less : more) - (1.0 - smoothing) * (z < 0.0 ? more : less)) * beta / pairs;
    w.coef[i] = (float)dz;
    w.coef[pairs + i] = (float)-dz;
  }
  s = block_sum(s, sh);
  if (threadIdx.x == 0) *loss = (float)(s / pairs);
}

// The gradient of the logits from the rows' (m, S). A group of G threads takes a part of a row
// at a time, parts from the end (the forward read the end last, so some of it is still in the
// L2 cache; the stores are marked to leave it there). Bound by the memory: 11200 rows of 50280
// bf16 logits, 0.6 of them counting, 1.80 GB in 0.28 ms, 6.4 TB/s. The last loads of a thread,
// fewer than kGradU, are in flight together too (rows of 6000 logits 6.55 TB/s, 6.0 one by one).
constexpr int kGradThreads = 256;
constexpr int kGradU = 4;  // loads in flight per thread
template <typename T, int G>
__global__ void __launch_bounds__(kGradThreads, 4)
    token_grad_kernel(TokenRows p, const float2* stats, Map2<const float> coef, const float* up, bool keep_if_one,
                      T* dlogits, int64_t dsb, int64_t dst, int parts, int units) {
  const float u = up ? *up : 1.f;
  if (keep_if_one && u == 1.f) return;
  constexpr int groups = kGradThreads / G;
  const int tid = threadIdx.x % G;
  const int step = gridDim.x * groups;
  for (int i = blockIdx.x * groups + threadIdx.x / G; i < units; i += step) {
    const int at = units - 1 - i, r = at / parts, part = at - r * parts, b = r / p.T, t = r - b * p.T;
    const T* row = static_cast<const T*>(p.logits) + b * p.sb + t * p.st;
    T* out = dlogits + b * dsb + t * dst;
    const Position pos = position(p, b, t);
    const float co = map_at(coef, b, t);
    const float2 st = stats[r];
    const RowCut c = cut_row(row, p.V);
    const int v0 = (int)((int64_t)c.nv * part / parts), v1 = (int)((int64_t)c.nv * (part + 1) / parts);
    float g = 0.f;
    if (pos.keep) g = pos.known ? (float)((double)u * (double)co * p.scale) : NAN;
    if (g == 0.f) {
      constexpr int N = Vec<T>::N;
      fill<T>(out, part == 0 ? 0 : c.head + v0 * N, part == parts - 1 ? p.V : c.head + v1 * N, tid, G, from_f32<T>(0.f));
      continue;
    }
    GradRow gr = grad_row(base_at(st.x, p.c_hi), g, st.y, pos.known ? (int)pos.tok : -1, 0.f);
    const Vec<T>* rv = reinterpret_cast<const Vec<T>*>(row + c.head);
    uint4* const to = reinterpret_cast<uint4*>(out + c.head);
    const bool same = same_boundary(out, c);
    const int kind = !same || gr.base.far ? 3 : sizeof(T) == 2 && gr.folded ? 1 : 2;
    for (int j = v0 + tid; j < v1; j += kGradU * G) {
      Vec<T> v[kGradU];
      const bool full = j + (kGradU - 1) * G < v1;
#pragma unroll
      for (int k = 0; k < kGradU; ++k)
        if (full || j + k * G < v1) v[k] = rv[j + k * G];
      if (kind == 1) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int k = 0; k < kGradU; ++k)
            if (full || j + k * G < v1) __stcs(to + j + k * G, vec_grad_folded(v[k], gr.kg, gr.negative, p.c_hi).u);
        }
      } else if (kind == 2) {
#pragma unroll
        for (int k = 0; k < kGradU; ++k)
          if (full || j + k * G < v1) __stcs(to + j + k * G, vec_grad<false>(v[k], gr, p.c_hi, p.c_lo).u);
      } else {
#pragma unroll
        for (int k = 0; k < kGradU; ++k)
          if (full || j + k * G < v1) put_grad(v[k], j + k * G, out, c, gr, same, p.c_hi, p.c_lo);
      }
    }
    if (gr.tok >= 0) gr.at = to_f32(row[gr.tok]);  // a row's loads need not wait for it
    put_token(out, c, gr, v0, v1, tid, G, p.c_hi, p.c_lo);
    if (part == 0) put_ends(row, out, p.V, c, gr, tid, G, p.c_hi, p.c_lo);
  }
}

// Positions are counted in 32 bits, and a kernel's stride is added to them.
int check_rows(const TokenRows& p) {
  return p.R > INT32_MAX / 2 - 4096 ? fail(M3_ERR_UNSUPPORTED, "token rows: too many positions") : M3_OK;
}

// How the rows are laid over the device.
struct RowPlan {
  int C, threads;
  int slot_vecs;  // of one row's place in shared memory; 0: none
};
constexpr int64_t kPlaceBytes = 104 * 1024;  // of a CTA's part of a row: two CTAs share an SM
int plan_rows(const TokenRows& p, int64_t elem, bool policy, RowPlan* out) {
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  const int64_t bytes = (int64_t)p.V * elem;
  int C = 1;
  // few rows: split each so that the device is filled, down to parts of 16 KB
  while (C < 8 && p.R * C * 2 <= 2 * (int64_t)sms && bytes / (2 * C) >= 16384) C *= 2;
  // a place for each part, with and without a gradient, so that both give the same bits
  if (policy)
    while (C < 8 && bytes / C > kPlaceBytes) C *= 2;
  out->C = C;
  // small CTAs stream best (1200 rows of 100 KB: 24.9 us with 128 threads, 25.4 with 256, 31.7
  // with 512); a CTA that keeps its part needs warps enough for the whole of it. 16-bit rows want
  // as many bytes of an SM's shared memory in use as there are (six, four to three, or two CTAs;
  // bf16 loss and gradient read and written, with the limits of wide rows and with these: rows of
  // 16384 logits 5.0, 5.3 TB/s, of 32000 4.7, 5.25, of 131072 4.4, 5.0); 32-bit rows, whose
  // arithmetic is half as much a byte, do better with less of it (17000 logits with 512 threads
  // twice 6.2 TB/s, with 256 three times 5.6) unless larger clusters wait for one another (57000
  // logits: 4.9, 6.2). Few rows: more threads to each.
  const int64_t part = bytes / C;
  const bool wide = (elem == 4 && C < 4) || p.R * C < 4 * (int64_t)sms;
  out->threads = !policy || part <= (wide ? 16 : 34) * 1024 ? 128 : part <= (wide ? 52 : 72) * 1024 ? 256 : 512;
  out->slot_vecs = bytes / C <= kPlaceBytes ? (int)(bytes / C / 16 + 2) : 0;
  return M3_OK;
}

// Clusters of one kernel that the device holds at once, remembered for the last launch shape of
// each device: (shared memory << 32) | (cluster size << 16) | clusters.
struct ClusterCache {
  std::atomic<long long> word[kMaxDevices];
};

// A launch of clusters. With a cache: as many as the device holds at once, at most `most`;
// without: `most` of them.
template <typename K, typename... A>
int launch_clusters(K kernel, const RowPlan& plan, int64_t most, ClusterCache* cache, size_t smem, cudaStream_t s,
                    A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3((unsigned)plan.threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)plan.C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cache) {
    int dev = 0;
    M3_TRY(current_device(&dev));
    const long long shape = ((long long)smem << 16) | plan.C, word = cache->word[dev].load(std::memory_order_acquire);
    int n = (int)(word & 0xffff);
    if (n == 0 || (word >> 16) != shape) {
      cfg.gridDim = dim3((unsigned)plan.C);
      cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
      if (e != cudaSuccess || n <= 0) {
        cudaGetLastError();
        return fail(M3_ERR_CUDA, std::string("token rows: occupancy query: ") + cudaGetErrorString(e));
      }
      n = std::min(n, 0xffff);
      cache->word[dev].store((shape << 16) | n, std::memory_order_release);
    }
    most = std::min<int64_t>(n, most);
  }
  cfg.gridDim = dim3((unsigned)(most * plan.C));
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(M3_ERR_CUDA, std::string("token rows: ") + cudaGetErrorString(e));
  }
  return M3_OK;
}

template <typename T, int NT>
int launch_grad_rows(const TokenRows& p, const PolicyArgs& a, const PolicyWs& w, const RowOut& o, RowPlan plan,
                     cudaStream_t s) {
  auto kernel = token_grad_rows_kernel<T, NT>;
  static std::atomic<bool> done[kMaxDevices];
  M3_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), (size_t)kPlaceBytes + 64, done));
  const int pieces = (plan.slot_vecs + kPieceVecs * NT - 1) / (kPieceVecs * NT);
  if (pieces > kPieces) return fail(M3_ERR_UNSUPPORTED, "token rows: row too long");
  plan.threads = NT + 32;
  static ClusterCache cache;
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  const size_t smem = (size_t)plan.slot_vecs * 16;
  // 32-bit rows: up to 144 KB of an SM in use (rows of 10000 logits: three CTAs 6.17 TB/s, four
  // 5.6; of 11000: three 6.17, two 5.3)
  const int64_t some = sizeof(T) == 4 && plan.C == 1 ? sms * std::max<int64_t>(2, 144 * 1024 / (int64_t)smem) : p.R;
  return launch_clusters(kernel, plan, std::min(some, p.R), &cache, smem, s, p, a, w, o, pieces);
}

template <typename T, bool POLICY, int G>
int launch_warp_rows(const TokenRows& p, const PolicyArgs& a, const PolicyWs& w, const RowOut& o, cudaStream_t s) {
  constexpr int W = kWarpThreads / 32, each = 32 / G;
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  const int row_vecs = (int)(((int64_t)p.V * (int64_t)sizeof(T) + 15) / 16);
  const size_t smem = (size_t)W * each * row_vecs * 16;
  // 1 KB of each CTA is the system's
  const int64_t fit = kSmSmem / (int64_t)(smem + sizeof(WarpRowsShared<T, G>) + 1024);
  const int64_t most = sms * std::min<int64_t>(kWarpCtas<POLICY>, fit);
  if constexpr (G < 32)  // few rows: more lanes for each
    if (p.R < most * W * each) return launch_warp_rows<T, POLICY, 2 * G>(p, a, w, o, s);
  auto kernel = token_warp_rows_kernel<T, POLICY, G>;
  static std::atomic<bool> done[kMaxDevices];
  M3_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), (size_t)W * kWarpRow, done));
  const int64_t batches = (p.R + each - 1) / each;
  kernel<<<(unsigned)std::min(most, (batches + W - 1) / W), kWarpThreads, smem, s>>>(p, a, w, o, row_vecs);
  return check_launch("token_warp_rows_kernel");
}

template <typename T, bool POLICY>
int launch_rows(const TokenRows& p, const PolicyArgs& a, const PolicyWs& w, const RowOut& o, cudaStream_t s) {
  if (p.R == 0) return M3_OK;
  M3_TRY(check_rows(p));
  const int64_t bytes = (int64_t)p.V * (int64_t)sizeof(T);
  // Lanes of a row, so that a warp's rows are 5 to 24 KB (without a gradient, TB/s, of 4, 8, 16
  // and 32 lanes: 300 bf16 logits 2.7, 2.0, 1.8, 1.3; 1000 4.6, 4.4, 3.2, 2.9; 2047 -, 4.4, 4.0,
  // 3.0; 4096 -, -, 5.4, 4.8; 600 fp32 logits 5.9, 6.4, 5.3, 5.2; 2500 -, -, 6.5, 6.9).
  if (bytes <= 1280) return launch_warp_rows<T, POLICY, 4>(p, a, w, o, s);
  if (bytes <= 4096) return launch_warp_rows<T, POLICY, 8>(p, a, w, o, s);
  if (bytes <= kWarpRow / 2) return launch_warp_rows<T, POLICY, 16>(p, a, w, o, s);
  if (bytes <= kWarpRow) return launch_warp_rows<T, POLICY, 32>(p, a, w, o, s);
  RowPlan plan;
  M3_TRY(plan_rows(p, (int64_t)sizeof(T), POLICY, &plan));
  if constexpr (POLICY) {
    if (o.dlogits && plan.slot_vecs > 0) {
      if (plan.threads == 128) return launch_grad_rows<T, 128>(p, a, w, o, plan, s);
      if (plan.threads == 256) return launch_grad_rows<T, 256>(p, a, w, o, plan, s);
      return launch_grad_rows<T, 512>(p, a, w, o, plan, s);
    }
  }
  if constexpr (POLICY) {
    if (plan.threads == 512) return launch_clusters(token_rows_kernel<T, POLICY, 512>, plan, p.R, nullptr, 0, s, p, a, w, o);
    if (plan.threads == 256) return launch_clusters(token_rows_kernel<T, POLICY, 256>, plan, p.R, nullptr, 0, s, p, a, w, o);
  }
  return launch_clusters(token_rows_kernel<T, POLICY, 128>, plan, p.R, nullptr, 0, s, p, a, w, o);
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

int token_error_word(bool reset, int* out) {
  unsigned v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_token_error, sizeof(v));
  if (e == cudaSuccess && reset) {
    const unsigned z = 0;
    e = cudaMemcpyToSymbol(g_token_error, &z, sizeof(z));
  }
  if (e != cudaSuccess) return fail(M3_ERR_CUDA, std::string("device timeouts: ") + cudaGetErrorString(e));
  *out = (int)v;
  return M3_OK;
}

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
  return launch_rows_of<false>(p, dtype, PolicyArgs{}, PolicyWs{}, RowOut{logp, nullptr, stats, nullptr, nullptr, 0, 0, nullptr}, s);
}

int launch_policy_loss(const TokenRows& p, int dtype, const PolicyArgs& a, int64_t batch, float* loss, float* kl,
                       float* clipped, float* logp, void* dlogits, int64_t dsb, int64_t dst, void* ws, cudaStream_t s) {
  M3_TRY(check_rows(p));
  size_t bytes = 0;
  const PolicyWs w = policy_ws(ws, batch, p.R, &bytes);
  const int64_t warps = (p.R + kCountRows - 1) / kCountRows, per = kCountThreads / 32;
  const int64_t ctas = std::max<int64_t>(1, (warps + per - 1) / per);
  if (ctas > 1) {
    cudaError_t e = cudaMemsetAsync(w.head, 0, w.zeroed, s);
    if (e != cudaSuccess) return fail(M3_ERR_CUDA, std::string("policy loss: ") + cudaGetErrorString(e));
  }
  policy_count_kernel<<<(unsigned)ctas, kCountThreads, 0, s>>>(p, a.by_sequence != 0, w);
  M3_TRY(check_launch("policy_count_kernel"));
  M3_TRY(launch_rows_of<true>(p, dtype, a, w, RowOut{logp, nullptr, w.stats, w.coef, dlogits, dsb, dst, nullptr}, s));
  policy_sum_kernel<<<(unsigned)((p.R + kSumRows - 1) / kSumRows), kSumThreads, 0, s>>>(p.R, w, loss, kl, clipped);
  return check_launch("policy_sum_kernel");
}

int launch_preference_loss(const TokenRows& p, int dtype, Map2<const float> ref, double beta, double smoothing,
                           int64_t pairs, float* loss, float* rewards, float* logp, void* ws, cudaStream_t s) {
  M3_TRY(check_rows(p));
  size_t bytes = 0;
  const PrefWs w = pref_ws(ws, 2 * pairs, p.R, &bytes);
  if (p.R == 0) {  // else the rows' kernel does it
    cudaError_t e = cudaMemsetAsync(w.done, 0, sizeof(unsigned), s);
    if (e != cudaSuccess) return fail(M3_ERR_CUDA, std::string("preference loss: ") + cudaGetErrorString(e));
  }
  M3_TRY(launch_rows_of<false>(p, dtype, PolicyArgs{}, PolicyWs{},
                               RowOut{logp, w.logp, w.stats, nullptr, nullptr, 0, 0, w.done}, s));
  preference_pairs_kernel<<<(unsigned)(2 * pairs), kSumThreads, 0, s>>>(p, ref, beta, smoothing, (int)pairs, w, loss,
                                                                       rewards);
  return check_launch("preference_pairs_kernel");
}

const float2* workspace_stats(const void* ws) { return static_cast<const float2*>(ws); }
Map2<const float> policy_coef(const void* ws, const TokenRows& p) {
  size_t bytes = 0;
  return Map2<const float>{policy_ws(const_cast<void*>(ws), p.R / p.T, p.R, &bytes).coef, p.T, 1};
}
Map2<const float> preference_coef(const void* ws, const TokenRows& p) {
  size_t bytes = 0;
  return Map2<const float>{pref_ws(const_cast<void*>(ws), p.R / p.T, p.R, &bytes).coef, 1, 0};
}

template <typename T>
static int launch_grad(const TokenRows& p, const float2* stats, Map2<const float> coef, const float* up,
                       bool keep_if_one, void* dlogits, int64_t dsb, int64_t dst, cudaStream_t s) {
  int sms = 0;
  M3_TRY(check_rows(p));
  M3_TRY(device_sm_count(&sms));
  const int64_t bytes = (int64_t)p.V * (int64_t)sizeof(T), ctas = (int64_t)sms * 4;
  T* const d = static_cast<T*>(dlogits);
  // where the kernel may find nothing to do its grid is small, else as large as the work
  auto by_rows = [&](auto lanes) {
    constexpr int G = decltype(lanes)::value;
    const int64_t need = (p.R + kGradThreads / G - 1) / (kGradThreads / G);
    token_grad_kernel<T, G><<<(unsigned)(keep_if_one ? std::min(need, ctas) : need), kGradThreads, 0, s>>>(
        p, stats, coef, up, keep_if_one, d, dsb, dst, 1, (int)p.R);
  };
  // a warp or less per row: up to 40 KB where there are rows for all warps (13000 bf16 logits 6.3
  // TB/s, 5.4 with a CTA per row; 20000 6.2, 6.0; 24000 6.2, 6.4)
  if (bytes <= 8192 || (bytes <= 40960 && p.R >= 8 * ctas)) {
    // Lanes of a row: short rows leave a warp's idle, and each has its position to find (bf16, of
    // 4, 8, 16 and 32 lanes: 300 logits 5.0, 4.5, 2.5, 1.6 TB/s; 1000 5.1, 5.9, 5.2, 3.7; 2047 5.2,
    // 6.1, 6.4, 5.7; 4096 6.7 with 32). Few rows: as many lanes as keep the device's busy.
    int g = bytes <= 1024 ? 4 : bytes <= 2560 ? 8 : bytes <= 6144 ? 16 : 32;
    while (g < 32 && p.R * g < ctas * kGradThreads) g *= 2;
    if (g == 4) by_rows(std::integral_constant<int, 4>{});
    else if (g == 8) by_rows(std::integral_constant<int, 8>{});
    else if (g == 16) by_rows(std::integral_constant<int, 16>{});
    else by_rows(std::integral_constant<int, 32>{});
  } else {
    // a CTA per row, or per part of a row (16 KB or more) where there are few rows
    int64_t parts = 1;
    while (p.R * parts < 4 * ctas && bytes / (2 * parts) >= 16384) parts *= 2;
    const int64_t units = p.R * parts;
    token_grad_kernel<T, kGradThreads><<<(unsigned)(keep_if_one ? std::min(units, ctas) : units), kGradThreads, 0, s>>>(
        p, stats, coef, up, keep_if_one, d, dsb, dst, (int)parts, (int)units);
  }
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
