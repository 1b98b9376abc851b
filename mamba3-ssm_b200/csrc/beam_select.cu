// Selection of a step of beam search: with lse_j = log sum_v exp(l[j, v]) of beam j's logits,
//   the `num` largest of score_j + l[j, v] - lse_j over all beams j and tokens v. Of equal ones the lower beam's come first, and
//   within a beam the larger logit's, then the lower token's (the order of the sums before they are rounded).
// A beam that has ended offers its end token at no cost; one whose score is -inf, or all of whose logits
// are, offers -inf; one with a NaN or an infinite logit or score offers NaN, which ranks first.
// beam_rows_kernel reads the logits once: a CTA a part of a row keeps its largest element and the sum of
// exponentials (one float a thread, two where they join) and the part's `num` largest elements. Those pass a
// threshold, at first the num-th largest of the threads' maxima, which rises whenever the list of those that
// passed has grown, so that later tiles are mostly dismissed by one comparison a vector. Where more pass than the list
// holds (rising or equal logits), the rest of the tile waits for the risen threshold; keys are unique (value, then the
// lower index), so that each look lists a full list's worth of them. beam_join_kernel, a CTA a prompt,
// joins the sums and ranks the parts' elements by their score, both in two floats (about 48 bits).
// beam_cluster_kernel does both for few and short rows.
// Bound by latency where there are few rows: 1 x 4 x 50000 of bf16 take 12 us in one launch (0.4 MB), of which the rows are 5,
// the join 3. Where there are many, by the rows' threads between two barriers: 64 x 8 x 131072 of bf16, a quarter ended, take
// 42 us (101 MB, 15 us of memory; with groups' maxima and a list cut at every tile 158) and 8 to join.
#include <algorithm>
#include <type_traits>

#include "beam.cuh"
#include "m3_common.cuh"
#include "pairs.cuh"

namespace m3 {
namespace {

constexpr int NT = 256;

struct Part { Two sum; float max; int n; };  // of a row's part: sum of exp(l - max), and listed elements

// floats in the order of unsigned integers; -0 counts as +0
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(float v, int i) { return ((uint64_t)ordered(v) << 32) | (uint32_t)~i; }

// Scores are held in two floats, hi + lo with |lo| at most half a step of hi: an infinite or NaN hi has lo = 0.
__device__ __forceinline__ Two two_sum(float a, float b) {
  Two r{a, 0.f};
  r.add(b);
  if (!(fabsf(r.hi) < INFINITY)) r.lo = 0.f;
  return r;
}
__device__ __forceinline__ Two plus(const Two& a, const Two& b) {
  Two r = two_sum(a.hi, b.hi);
  if (fabsf(r.hi) < INFINITY) {
    const float l = __fadd_rn(r.lo, __fadd_rn(a.lo, b.lo)), h = __fadd_rn(r.hi, l);
    r.lo = __fsub_rn(l, __fsub_rn(h, r.hi));
    r.hi = h;
  }
  return r;
}
// in the order of unsigned integers, a NaN above all
__device__ __forceinline__ uint64_t ordered64(const Two& v) {
  return v.hi != v.hi ? ~0ull : ((uint64_t)ordered(v.hi) << 32) | ordered(v.lo);
}
__device__ __forceinline__ float score_of(uint64_t k) {
  return k == ~0ull ? __int_as_float(0x7fc00000) : __fadd_rn(unordered((uint32_t)(k >> 32)), unordered((uint32_t)k));
}

// log of a sum s > 0, to a few 1e-9: s = 2^n m with m in [3/4, 3/2), log m = 2 atanh(t), t = (m - 1) / (m + 1), |t| <= 1/5, of which
// t itself is formed in two floats and the rest of the series, 125 times smaller, in one.
__device__ __forceinline__ Two log_two(const Two& s) {
  const float top = __fadd_rn(s.hi, s.lo);
  if (!(top > 0.f && top < INFINITY)) return Two{logf(top), 0.f};
  int n = (__float_as_int(top) - 0x3f400000) >> 23;  // of 3/4
  const float scale = __int_as_float((127 - n) << 23);  // (sums of at most 2^24 terms of at most 1)
  const float m = s.hi * scale, ml = s.lo * scale;
  const Two a = two_sum(m, -1.f), b = two_sum(m, 1.f);
  const float al = a.lo + ml, bl = b.lo + ml;
  const float th = __fdiv_rn(a.hi, b.hi);
  // what the quotient leaves: (a - th b) / b
  const float tl = __fdiv_rn(__fadd_rn(fmaf(-th, b.hi, a.hi), al - th * bl), b.hi);
  const float q = th * th;
  float r = fmaf(q, 1.f / 13, 1.f / 11);
  r = fmaf(q, r, 1.f / 9);
  r = fmaf(q, r, 1.f / 7);
  r = fmaf(q, r, 1.f / 5);
  r = fmaf(q, r, 1.f / 3);
  const Two logm = two_sum(2.f * th, 2.f * fmaf(q * th, r, tl));
  // n log 2, log 2 in two parts of which the first has few enough bits for an exact product
  return plus(plus(Two{n * 0.693145751953125f, 0.f}, Two{n * 1.42860682030941723212e-6f, 0.f}), logm);
}

// put(i, r) for each of n <= NT elements, r of which are above element i. As many threads an element as there are for it
// (one thread an element, or a warp, took 14000 cycles for 128 elements where this takes 1000).
template <typename X, typename Above, typename Put>
__device__ __forceinline__ void ranks(const X* x, int n, Above&& above, Put&& put) {
  int per = 1;
  while (per < 32 && 2 * per * n <= NT) per *= 2;
  const int part = threadIdx.x & (per - 1), i = threadIdx.x / per;
  int r = 0;
  if (i < n) {
    const X mine = x[i];
#pragma unroll 4
    for (int k = part; k < n; k += per) r += above(x[k], mine);
  }
  for (int o = per / 2; o > 0; o /= 2) r += __shfl_xor_sync(0xffffffffu, r, o);
  if (i < n && part == 0) put(i, r);
}

// A t with count(t) >= num, bit by bit from the highest of `bits` down to `lowest`: the largest one, or the first whose
// count, which falls as t rises, is `enough` at most. had: the count, left alone where no bit could be set.
template <typename Count>
__device__ __forceinline__ uint64_t bisect(int bits, int lowest, int num, int enough, int* had, Count&& count) {
  uint64_t t = 0;
  for (int bit = bits - 1; bit >= lowest; --bit) {
    const uint64_t with = t | 1ull << bit;
    const int c = count(with);
    if (c >= num) {
      t = with;
      *had = c;
      if (c <= enough) break;
    }
  }
  return t;
}
constexpr int kRanked = NT / 2;  // more elements than these are cut before they are ranked
static_assert(kRanked >= kMaxCandidates, "the candidates themselves have to be ranked");

template <typename T, int U>
struct Rows {
  static constexpr int VN = 16 / sizeof(T), TILE = NT * U * VN;
  static constexpr int CAP = 1024;  // listed elements; more of a tile wait until the threshold has risen
  uint64_t list[CAP], best[kRanked];
  Two sum[NT / 32];
  float max[NT / 32];
  int n;
  uint64_t tau;  // keys above it pass
};

// Keeps the `num` largest keys of the list, in order, and the last of them as the threshold; returns how many there are.
template <typename R>
__device__ __forceinline__ int compact(R& sh, int num) {
  __syncthreads();
  const int n = min(sh.n, R::CAP), m = min(n, num);
  auto larger = [](uint64_t a, uint64_t b) { return a > b; };
  if (n > kRanked) {  // (pairs of a full list's elements are too many to compare)
    int had = n;
    const uint64_t low = bisect(64, 0, num, kRanked, &had, [&](uint64_t t) {
      int c = 0;
      for (int i0 = 0; i0 < n; i0 += NT) c += __syncthreads_count(i0 + (int)threadIdx.x < n && sh.list[i0 + threadIdx.x] >= t);
      return c;
    });
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT)
      if (sh.list[i] >= low) sh.best[atomicAdd(&sh.n, 1)] = sh.list[i];
    __syncthreads();
    ranks(sh.best, had, larger, [&](int i, int r) {
      if (r < num) sh.list[r] = sh.best[i];
    });
  } else {
    ranks(sh.list, n, larger, [&](int i, int r) {
      if (r < num) sh.best[r] = sh.list[i];
    });
    __syncthreads();
    if (threadIdx.x < m) sh.list[threadIdx.x] = sh.best[threadIdx.x];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    sh.n = m;
    if (m == num) sh.tau = max(sh.tau, sh.list[num - 1]);
  }
  __syncthreads();
  return m;
}

// Whether a beam's logits are needed at all.
__device__ __forceinline__ bool beam_counts(const BeamParams& p, int64_t b, int j) {
  return !(p.finished != nullptr && p.finished[b * p.fb + j * p.fk] != 0) && p.scores[b * p.sb + j * p.sk] != -INFINITY;
}

// 16 bytes of the 32 in a and b, from byte 4 W + bits / 8 on.
template <int W>
__device__ __forceinline__ uint4 funnel(const uint4& a, const uint4& b, int bits) {
  const uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __funnelshift_r(v[W + i], v[W + i + 1], bits);
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// Elements s0 .. s1 - 1 of a row, by one CTA. Which thread takes which elements, and so the sum's last bits, goes by their indices
// alone: beams with the same logits have the same scores wherever their rows lie. Where these are not all on 16-byte boundaries
// (ALIGNED false), floats are loaded one by one (64 x 8 x 50257: 44 us, as many as with aligned rows), and of 16-bit elements the
// 16 bytes from the boundary in front of the thread's own and those behind it, which are shifted (36 us, 32 with aligned rows). Both
// kernels in a graph: floats 55 us, shifted 63; 16-bit elements 47, by shuffles from the neighbour's registers 51.
template <typename T, int U, bool ALIGNED>
__device__ __forceinline__ void row_part(const BeamParams& p, Rows<T, U>& sh, const T* x, int s0, int s1, Part* part, uint64_t* keys) {
  using R = Rows<T, U>;
  constexpr int VN = R::VN, TILE = R::TILE;
  const int tid = threadIdx.x;
  constexpr bool SHIFT = !ALIGNED && sizeof(T) == 2;
  const int off = !SHIFT ? 0 : (int)((reinterpret_cast<uintptr_t>(x + s0) & 15) / sizeof(T));
  if (tid == 0) { sh.n = 0; sh.tau = 0; }
  // 16 bytes, element i0 the first; -inf outside the part
  auto load = [&](int i0) {
    if ((!SHIFT || i0 >= s0) && i0 + VN <= s1) {
      if constexpr (!ALIGNED && !SHIFT) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(x + i0);
        return make_uint4(w[0], w[1], w[2], w[3]);
      }
      return *reinterpret_cast<const uint4*>(x + i0);
    }
    alignas(16) T e[VN];
#pragma unroll
    for (int k = 0; k < VN; ++k) e[k] = i0 + k >= s0 && i0 + k < s1 ? x[i0 + k] : from_f32<T>(-INFINITY);
    return *reinterpret_cast<const uint4*>(e);
  };
  uint4 next[U];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = load(t0 + (u * NT + tid) * VN - off);
  };
  // this thread's elements of the tile at t0, which has been fetched; its neighbours' bytes are in L1
  auto take = [&](int t0, uint4 (&raw)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = next[u];
    if (!SHIFT || off == 0) return;
    uint4 b[U];
    const int i0 = t0 + (tid + 1) * VN - off;
    if (t0 + TILE + VN <= s1) {
#pragma unroll
      for (int u = 0; u < U; ++u) b[u] = *reinterpret_cast<const uint4*>(x + i0 + u * NT * VN);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) b[u] = load(i0 + u * NT * VN);
    }
    const int bits = off % 2 * 16;
    auto shift = [&](auto words) {
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = funnel<decltype(words)::value>(raw[u], b[u], bits);
    };
    switch (off / 2) {
      case 0: return shift(std::integral_constant<int, 0>{});
      case 1: return shift(std::integral_constant<int, 1>{});
      case 2: return shift(std::integral_constant<int, 2>{});
      default: return shift(std::integral_constant<int, 3>{});
    }
  };
  // Lists the tile's elements above the threshold, of those left; false where some found no place.
  auto look = [&](const uint4 (&raw)[U], const float (&vm)[U], float tm, int t0, uint32_t& left) {
    const uint64_t tau = sh.tau;
    const float tau_v = unordered((uint32_t)((tau + 1) >> 32));  // the lowest value that may pass,
    const bool ties = key_of(tau_v, t0) > tau;                    // and whether it may from this tile on
    auto may = [&](float v) { return ties ? v >= tau_v : v > tau_v; };
    const uint32_t all = 0xffffffffu;
    bool placed = true;
    if (__any_sync(all, may(tm))) {
      uint32_t pass = 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (__any_sync(all, may(vm[u]))) {
          const T* e = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
          for (int k = 0; k < VN; ++k)
            if (may(to_f32(e[k]))) pass |= 1u << (u * VN + k);
        }
      pass &= left;
      while (pass) {
        const int bit = __ffs(pass) - 1, i = t0 + (bit / VN * NT + tid) * VN + bit % VN;
        pass &= pass - 1;
        const uint64_t key = i < s1 ? key_of(to_f32(x[i]), i) : 0;
        if (key > tau) {
          const int at = *const_cast<volatile int*>(&sh.n) < R::CAP ? atomicAdd(&sh.n, 1) : R::CAP;
          if (at >= R::CAP) {
            placed = false;
            break;
          }
          sh.list[at] = key;
        }
        left &= ~(1u << bit);
      }
    }
    return placed;
  };
  // the largest elements of the vectors, and of all of them
  auto largest = [&](const uint4 (&raw)[U], float (&vm)[U]) {
    float tm = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const T* e = reinterpret_cast<const T*>(&raw[u]);
      vm[u] = to_f32(e[0]);
#pragma unroll
      for (int k = 1; k < VN; ++k) vm[u] = fmaxf(vm[u], to_f32(e[k]));
      tm = fmaxf(tm, vm[u]);
    }
    return tm;
  };
  fetch(s0);
  float run = -INFINITY, sum = 0.f;
  int held = 0;  // listed elements at the last barrier
  __syncthreads();
  // a few tiles between two barriers, at which the list is cut to its best and the threshold rises (64 x 8 x 131072: 43 us with
  // four, 46 with two, 45 with eight; half as many vectors a thread at four CTAs an SM 61)
  constexpr int kTiles = 4;
#pragma unroll 1
  for (int g0 = s0; g0 < s1; g0 += kTiles * TILE) {
    const int g1 = min(g0 + kTiles * TILE, s1);
    bool placed = true;
#pragma unroll 1
    for (int t0 = g0; t0 < g1; t0 += TILE) {
      uint4 raw[U];
      take(t0, raw);
      if (t0 + TILE < s1) fetch(t0 + TILE);
      float vm[U];
      const float tm = largest(raw, vm);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (vm[u] > run) {
          sum *= ex2((run - vm[u]) * kLog2e);
          run = vm[u];
        }
        // elements of -inf in front of the first finite one: the difference to -inf would be NaN
        const float base = run == -INFINITY ? 0.f : -run;
        const f2 less = pack2(base, base), scale = pack2(kLog2e, kLog2e);
        const T* e = reinterpret_cast<const T*>(&raw[u]);
        f2 s = 0;
#pragma unroll
        for (int k = 0; k < VN; k += 2) {
          float d0, d1;
          unpack2(mul2(add2(pack2(to_f32(e[k]), to_f32(e[k + 1])), less), scale), d0, d1);
          s = add2(s, pack2(ex2(d0), ex2(d1)));
        }
        float a0, a1;
        unpack2(s, a0, a1);
        sum += a0 + a1;
      }
      if (t0 == s0) {
        // the first threshold: just below what the maxima of `num` threads reach, to the upper 16 bits
        const uint32_t o = ordered(tm);
        int had = 0;
        const uint32_t low = (uint32_t)bisect(32, 16, p.num, p.num, &had, [&](uint64_t t) { return __syncthreads_count(o >= (uint32_t)t); });
        if (tid == 0) sh.tau = ((uint64_t)max(low, ordered(-INFINITY)) << 32) - 1;  // (what lies below -inf are NaNs)
        __syncthreads();
      }
      uint32_t left = ~0u;
      placed &= look(raw, vm, tm, t0, left);
    }
    if (__syncthreads_or(!placed)) {
      // more passed than the list holds: these tiles again, each as often as it takes, the threshold rising in between
      if (tid == 0) sh.n = held;
      __syncthreads();
#pragma unroll 1
      for (int t0 = g0; t0 < g1; t0 += TILE) {
        uint4 keep[U], raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) keep[u] = next[u];
        fetch(t0);
        take(t0, raw);
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = keep[u];
        float vm[U];
        const float tm = largest(raw, vm);
        uint32_t left = ~0u;  // of this thread's U VN elements
        bool again;
        do {
          again = __syncthreads_or(!look(raw, vm, tm, t0, left));
          compact(sh, p.num);
        } while (again);
      }
    }
    held = compact(sh, p.num);
  }
  const int n = held;
  if (tid < n) keys[tid] = sh.list[tid];
  // the sum over the CTA, to one base
  float m = run;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((tid & 31) == 0) sh.max[tid >> 5] = m;
  __syncthreads();
  m = sh.max[0];
#pragma unroll
  for (int w = 1; w < NT / 32; ++w) m = fmaxf(m, sh.max[w]);
  Two d{run == -INFINITY ? sum : sum * ex2((run - m) * kLog2e), 0.f};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d.add(d.shuffled(o));
  if ((tid & 31) == 0) sh.sum[tid >> 5] = d;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < NT / 32; ++w) d.add(sh.sum[w]);
    *part = Part{d, m, n};
  }
}

// (three CTAs an SM, at 80 registers a thread: 43 us at 64 x 8 x 131072; two 50, four, which spill, 72)
template <typename T, int U, bool ALIGNED>
__global__ void __launch_bounds__(NT, 3) beam_rows_kernel(const BeamParams p, Part* parts, uint64_t* keys, int seg) {
  __shared__ Rows<T, U> sh;
  const int64_t row = blockIdx.y, b = row / p.beams;
  const int j = (int)(row % p.beams), s0 = blockIdx.x * seg;
  if (!beam_counts(p, b, j)) return;
  const int64_t part = row * gridDim.x + blockIdx.x;
  row_part<T, U, ALIGNED>(p, sh, static_cast<const T*>(p.logits) + b * p.lb + j * p.lk, s0, min(p.V, s0 + seg), parts + part, keys + part * p.num);
}

struct Cand { uint64_t value, tie; };  // score in order of integers; then beam, logit, token
__device__ __forceinline__ bool above(const Cand& a, const Cand& b) {
  return a.value > b.value || (a.value == b.value && a.tie > b.tie);
}
constexpr int kTokenBits = 24;
static_assert(kMaxVocab <= 1 << kTokenBits && kMaxBeams <= 64, "a tie's key holds 6 + 32 + 24 bits");
__device__ __forceinline__ uint64_t tie_of(int beam, uint32_t logit, int token) {
  return ((uint64_t)(63 - beam) << (32 + kTokenBits)) | ((uint64_t)logit << kTokenBits) | (uint32_t)((1 << kTokenBits) - 1 - token);
}

// Lists that reach into the num best are num at most, with num elements each; twice as many are let through where they are
// not told apart at once.
constexpr int kHeads = 2;
__host__ __device__ inline int most_candidates(int lists, int num) { return (lists < kHeads * num ? lists : kHeads * num) * num; }

__host__ __device__ inline size_t join_bytes(int lists, int num) { return (size_t)(lists + most_candidates(lists, num)) * sizeof(Cand); }

// A prompt's continuations from the parts of its beams' rows, by one CTA. room: join_bytes.
__device__ __forceinline__ void join_parts(const BeamParams& p, int64_t b, const Part* parts, const uint64_t* keys, int splits,
                                           unsigned char* room) {
  Cand* head = reinterpret_cast<Cand*>(room);  // beams * splits
  Cand* cand = head + p.beams * splits;        // most_candidates
  // a logarithm of probability is (l - max) - log(sum): l - (max + log(sum)) would lose the digits of large logits
  __shared__ float s_max[kMaxBeams], s_score[kMaxBeams];
  __shared__ Two s_log[kMaxBeams];
  __shared__ int s_kind[kMaxBeams];  // 0 listed, 1 ended, 2 nothing, 3 NaN
  __shared__ int s_n, s_lists, s_list[kHeads * kMaxCandidates];  // candidates; lists that may hold some of the best
  __shared__ uint64_t s_tau;
  __shared__ Cand s_best[kRanked];
  const int tid = threadIdx.x, lane = tid & 31, K = p.beams, lists = K * splits;
  if (tid == 0) { s_n = 0; s_lists = 0; s_tau = 0; }
  // what the first element of this thread's list will need, on its way while the sums are joined (not used where it was not written)
  const int first_n = tid < lists ? parts[tid].n : 0;
  const uint64_t first_key = tid < lists ? keys[tid * p.num] : 0;
  // a warp a beam joins its parts' sums
  for (int j = tid >> 5; j < K; j += NT / 32) {
    const float score = p.scores[b * p.sb + j * p.sk];
    int kind = 0;
    float peak = 0.f;
    Two logs{0.f, 0.f};
    if (score == -INFINITY) kind = 2;
    else if (!(score < INFINITY)) kind = 3;
    else if (p.finished != nullptr && p.finished[b * p.fb + j * p.fk] != 0) kind = 1;
    else {
      const Part* q = parts + j * splits;
      const Part mine = lane < splits ? q[lane] : Part{Two{0.f, 0.f}, -INFINITY, 0};
      float m = mine.max;
      for (int i = lane + 32; i < splits; i += 32) m = fmaxf(m, q[i].max);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      auto part = [&](const Part& x) {
        const float f = x.max == m || x.max == -INFINITY ? 1.f : ex2((x.max - m) * kLog2e);
        return Two{x.sum.hi * f, x.sum.lo * f};
      };
      Two s = part(mine);
      for (int i = lane + 32; i < splits; i += 32) s.add(part(q[i]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s.add(s.shuffled(o));
      peak = m;
      const float total = s.value();
      if (!(total == total) || m == INFINITY) kind = 3;
      else if (m == -INFINITY) kind = 2;
      else logs = log_two(s);
    }
    if (lane == 0) {
      s_kind[j] = kind;
      s_max[j] = peak;
      s_log[j] = Two{-logs.hi, -logs.lo};
      s_score[j] = score;
    }
  }
  __syncthreads();
  // element i of list l, of n listed ones the one with this key: false behind its end
  auto make = [&](int l, int i, int n, uint64_t key, Cand* c) {
    const int j = l / splits, kind = s_kind[j];
    if (kind == 0) {
      if (i >= n) return false;
      const uint32_t o = (uint32_t)(key >> 32);
      const Two logp = plus(two_sum(unordered(o), -s_max[j]), s_log[j]);
      *c = Cand{ordered64(plus(Two{s_score[j], 0.f}, logp)), tie_of(j, o, (int)~(uint32_t)key)};
      return true;
    }
    if (l % splits != 0 || i >= p.V) return false;
    if (kind == 1 && i == 0) {
      *c = Cand{ordered64(Two{s_score[j], 0.f}), tie_of(j, ~0u, p.end_token)};
      return true;
    }
    const int token = kind == 1 && i <= p.end_token ? i - 1 : i;
    *c = Cand{kind == 3 ? ~0ull : ordered64(Two{-INFINITY, 0.f}), tie_of(j, 0, token)};
    return true;
  };
  auto get = [&](int l, int i, Cand* c) { return make(l, i, parts[l].n, keys[l * p.num + i], c); };
  if (tid < lists && !make(tid, 0, first_n, first_key, &head[tid])) head[tid] = Cand{0, 0};
  for (int l = tid + NT; l < lists; l += NT)
    if (!get(l, 0, &head[l])) head[l] = Cand{0, 0};
  __syncthreads();
  // nothing below the num-th best head can be among the num best
  uint64_t tau = 0;
  if (lists <= kRanked) {
    ranks(head, lists, [](const Cand& a, const Cand& b) { return above(a, b); }, [&](int l, int r) {
      if (r == p.num - 1) s_tau = head[l].value;
      if (r < p.num && head[l].tie != 0) s_list[atomicAdd(&s_lists, 1)] = l;
    });
    __syncthreads();
    tau = s_tau;
  } else {
    int had = 0;
    tau = bisect(64, 0, p.num, kHeads * p.num, &had, [&](uint64_t t) {
      int c = 0;
      for (int l0 = 0; l0 < lists; l0 += NT) c += __syncthreads_count(l0 + tid < lists && head[l0 + tid].value >= t);
      return c;
    });
    const bool equal = had > kHeads * p.num;  // heads, which their ties' keys tell apart
    for (int l = tid; l < lists; l += NT) {
      const Cand mine = head[l];
      if (mine.tie == 0 || mine.value < tau) continue;
      int r = 0;
      if (equal) {
        for (int i = 0; i < lists; ++i) r += above(head[i], mine);
      }
      if (r < p.num) s_list[atomicAdd(&s_lists, 1)] = l;
    }
    __syncthreads();
  }
  const int left = s_lists * p.num;
  for (int i = tid; i < left; i += NT) {
    Cand c;
    if (get(s_list[i / p.num], i % p.num, &c) && c.value >= tau) cand[atomicAdd(&s_n, 1)] = c;
  }
  __syncthreads();
  int n = s_n;
  const Cand* from = cand;
  if (n > kRanked) {  // the best of them, the last of which is found bit by bit: its value, and among many equal ones its tie
    int had = n;
    auto at_least = [&](uint64_t value, uint64_t tie) {
      int c = 0;
      for (int i0 = 0; i0 < n; i0 += NT) {
        const int i = i0 + tid;
        c += __syncthreads_count(i < n && (cand[i].value > value || (cand[i].value == value && cand[i].tie >= tie)));
      }
      return c;
    };
    Cand low{0, 0};
    low.value = bisect(64, 0, p.num, kRanked, &had, [&](uint64_t t) { return at_least(t, 0); });
    if (had > kRanked) low.tie = bisect(64, 0, p.num, kRanked, &had, [&](uint64_t t) { return at_least(low.value, t); });
    if (tid == 0) s_n = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NT)
      if (!above(low, cand[i])) s_best[atomicAdd(&s_n, 1)] = cand[i];
    __syncthreads();
    from = s_best;
    n = had;
  }
  ranks(from, n, [](const Cand& a, const Cand& b) { return above(a, b); }, [&](int i, int r) {
    if (r >= p.num) return;
    const Cand c = from[i];
    const int64_t at = b * p.num + r;
    p.out_scores[at] = score_of(c.value);
    p.parents[at] = 63 - (int)(c.tie >> (32 + kTokenBits));
    p.tokens[at] = (1 << kTokenBits) - 1 - (int)(c.tie & ((1 << kTokenBits) - 1));
  });
}

__global__ void __launch_bounds__(NT) beam_join_kernel(const BeamParams p, const Part* parts, const uint64_t* keys, int splits) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const int64_t b = blockIdx.x, lists = (int64_t)p.beams * splits;
  join_parts(p, b, parts + b * lists, keys + b * lists * p.num, splits, smem_raw);
}

// Both in one launch for few and small prompts, where the second launch and the workspace would cost more than they
// spread: a cluster of eight CTAs a prompt, with a part each, which go into the first one's shared memory, which joins them.
constexpr int kCluster = 8;
constexpr int kClusterPart = 32768;  // elements a CTA

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
template <typename X>
__device__ __forceinline__ X* of_first(X* p) {  // the same place in the shared memory of the cluster's first CTA
  uint64_t r;
  asm("mapa.u64 %0, %1, 0;" : "=l"(r) : "l"((uint64_t)p));
  return reinterpret_cast<X*>(r);
}

template <typename T, int U, bool ALIGNED>
__global__ void __launch_bounds__(NT) beam_cluster_kernel(const BeamParams p, int splits, int seg) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ Rows<T, U> sh;
  const int lists = p.beams * splits, rank = blockIdx.x % kCluster;
  const int64_t b = blockIdx.x / kCluster;
  Part* parts = reinterpret_cast<Part*>(smem_raw);
  uint64_t* keys = reinterpret_cast<uint64_t*>(parts + lists);
  cluster_arrive();  // every CTA runs before any writes into the first one's memory
  cluster_wait();
  if (rank < lists) {
    const int j = rank / splits, s0 = rank % splits * seg;
    if (beam_counts(p, b, j) && s0 < p.V)
      row_part<T, U, ALIGNED>(p, sh, static_cast<const T*>(p.logits) + b * p.lb + j * p.lk, s0, min(p.V, s0 + seg), of_first(parts + rank),
                              of_first(keys + rank * p.num));
    else if (threadIdx.x == 0)
      *of_first(parts + rank) = Part{Two{0.f, 0.f}, -INFINITY, 0};
  }
  cluster_arrive();
  cluster_wait();
  if (rank == 0) join_parts(p, b, parts, keys, splits, reinterpret_cast<unsigned char*>(keys + lists * p.num));
}

struct BeamPlan {
  bool cluster;
  int u, seg, splits;
};

// In one launch, as many parts a row as there are CTAs of the cluster for it. In two, tiles of four vectors a
// thread where the rows alone fill the GPU, of one where they do not, and as many parts as bring the rows to about four CTAs
// an SM (finer parts cost more in thresholds than their balance gives: 48 us at eight an SM, 42 at four, 64 x 8 rows of 131072).
BeamPlan plan(int64_t batch, int beams, int V, int num, int es, int sms) {
  const int vn = 16 / es;
  BeamPlan w;
  const int64_t rows = batch * beams;
  w.splits = beams <= kCluster ? kCluster / beams : 0;
  const int one = w.splits > 0 ? (V + w.splits - 1) / w.splits : 0;
  // One launch, two launches, us a call by itself (and in a CUDA graph, without the host): 1 x 4 x 16384 of 8: 19.0, 24.8
  // (9.3, 8.8); 32 x 4 x 16384 of 8: 19.0, 24.6 (10.5, 12.6); 1 x 4 x 50000 of 4: 19.0, 25.0 (12.1, 11.3), of 16: 20.7, 24.8
  // (18.6, 11.7). Of more prompts than the GPU holds at once the clusters would take turns.
  w.cluster = w.splits > 0 && one <= kClusterPart && batch * kCluster <= 2 * sms;
  if (w.cluster) {
    w.seg = (one + vn - 1) / vn * vn;
    w.u = w.seg > 2 * NT * vn ? 4 : 1;
    return w;
  }
  const int64_t big = (V + 4 * NT * vn - 1) / (4 * NT * vn);
  w.u = rows * big >= 2 * sms ? 4 : 1;
  const int tile = NT * w.u * vn;
  const int64_t tiles = (V + tile - 1) / tile;
  const int64_t want = std::max<int64_t>(1, (int64_t)4 * sms / std::max<int64_t>(1, rows));
  const int64_t per = (tiles + std::min(want, tiles) - 1) / std::min(want, tiles);
  w.seg = (int)(per * tile);
  w.splits = (int)((V + w.seg - 1) / w.seg);
  return w;
}

constexpr int kMaxLists = 4096;

}  // namespace

size_t beam_workspace_bytes(int64_t batch, int beams, int V, int num, int dtype, int sms) {
  const BeamPlan w = plan(batch, beams, V, num, (int)dtype_size(dtype), sms);
  return w.cluster ? 0 : (size_t)batch * beams * w.splits * (sizeof(Part) + (size_t)num * sizeof(uint64_t));
}

template <typename T, int U, bool ALIGNED>
static int launch_cluster(const BeamParams& p, const BeamPlan& w, cudaStream_t s) {
  const int lists = p.beams * w.splits;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kCluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.batch * kCluster));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = (size_t)lists * (sizeof(Part) + p.num * sizeof(uint64_t)) + join_bytes(lists, p.num);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, beam_cluster_kernel<T, U, ALIGNED>, p, w.splits, w.seg);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(M3_ERR_CUDA, std::string("beam_cluster_kernel: ") + cudaGetErrorString(e));
  }
  return M3_OK;
}

int launch_beam_select(const BeamParams& p, int dtype, void* ws, cudaStream_t s) {
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  const int64_t rows = p.batch * p.beams;
  const BeamPlan w = plan(p.batch, p.beams, p.V, p.num, (int)dtype_size(dtype), sms);
  if (p.beams * w.splits > kMaxLists) return fail(M3_ERR_UNSUPPORTED, "beam_select: too many parts");
  Part* parts = static_cast<Part*>(ws);
  uint64_t* keys = reinterpret_cast<uint64_t*>(parts + rows * w.splits);
  const dim3 grid((unsigned)w.splits, (unsigned)rows);
  // parts of a row begin at multiples of a vector
  const uint64_t any = reinterpret_cast<uintptr_t>(p.logits) | (uint64_t)(p.batch > 1 ? p.lb : 0) * dtype_size(dtype) |
                       (uint64_t)(p.beams > 1 ? p.lk : 0) * dtype_size(dtype);
  auto launch = [&](auto t, auto u, auto aligned) {
    using T = decltype(t);
    constexpr int U = decltype(u)::value;
    constexpr bool ALIGNED = decltype(aligned)::value;
    if (w.cluster) return launch_cluster<T, U, ALIGNED>(p, w, s);
    beam_rows_kernel<T, U, ALIGNED><<<grid, NT, 0, s>>>(p, parts, keys, w.seg);
    return check_launch("beam_rows_kernel");
  };
  auto by_place = [&](auto t, auto u) {
    return any % 16 == 0 ? launch(t, u, std::true_type{}) : launch(t, u, std::false_type{});
  };
  auto go = [&](auto t) {
    return w.u == 4 ? by_place(t, std::integral_constant<int, 4>{}) : by_place(t, std::integral_constant<int, 1>{});
  };
  if (dtype == M3_FLOAT32) M3_TRY(go(float{}));
  else if (dtype == M3_BFLOAT16) M3_TRY(go(__nv_bfloat16{}));
  else M3_TRY(go(__half{}));
  if (w.cluster) return M3_OK;
  static std::atomic<bool> done[kMaxDevices];
  const size_t most = join_bytes(kMaxLists, kMaxCandidates);
  M3_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(&beam_join_kernel), most, done));
  beam_join_kernel<<<(unsigned)p.batch, NT, join_bytes(p.beams * w.splits, p.num), s>>>(p, parts, keys, w.splits);
  return check_launch("beam_join_kernel");
}

}  // namespace m3
