// Selection of a step of beam search: with lse_j = log sum_v exp(l[j, v]) of beam j's logits,
//   the `num` largest of score_j + l[j, v] - lse_j over all beams j and tokens v, ties to the lowest (j, v).
// A beam that has ended offers its end token at no cost; one whose score is -inf, or all of whose logits
// are, offers -inf; one with a NaN or an infinite logit or score offers NaN, which ranks first.
// beam_rows_kernel reads the logits once: a CTA a part of a row keeps its largest element and the sum of
// exponentials (32 bits a thread, joined in 64) and the part's `num` largest elements. Those pass a
// threshold: the num-th largest of the threads' own maxima of the first tile, so that later tiles are mostly
// dismissed by one comparison a vector. Keys are unique (value, then the lower index), so a
// tile passes at most num threads' elements whatever the logits are. beam_join_kernel, a CTA a prompt,
// joins the sums in 64 bits and ranks the parts' elements by their score in 64 bits.
// Bound by the memory where there are many rows, by latency where there are few.
#include <algorithm>

#include "beam.cuh"
#include "m3_common.cuh"

namespace m3 {
namespace {

constexpr int NT = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct Part { double sum; float max; int n; };  // of a row's part: sum of exp(l - max), and listed elements

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// floats in the order of unsigned integers; -0 counts as +0
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(float v, int i) { return ((uint64_t)ordered(v) << 32) | (uint32_t)~i; }

__device__ __forceinline__ uint64_t ordered64(double v) {
  if (v != v) return ~0ull;
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ double unordered64(uint64_t k) {
  if (k == ~0ull) return __longlong_as_double(0x7ff8000000000000ll);
  return __longlong_as_double((long long)(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
}

template <typename T, int U>
struct Rows {
  static constexpr int VN = 16 / sizeof(T), TILE = NT * U * VN;
  static constexpr int CAP = kMaxCandidates * U * VN + kMaxCandidates;
  uint64_t list[CAP], best[kMaxCandidates], thread_max[NT];
  double sum[NT / 32];
  float max[NT / 32];
  int total, n;
  uint64_t tau;
};

// Keeps the `num` largest keys of the list, in order, and the last of them as the threshold.
template <typename R>
__device__ __forceinline__ void compact(R& sh, int num) {
  __syncthreads();
  const int n = sh.n;
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint64_t k = sh.list[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += sh.list[j] > k;
    if (r < num) sh.best[r] = k;
  }
  __syncthreads();
  const int m = min(n, num);
  if (threadIdx.x < m) sh.list[threadIdx.x] = sh.best[threadIdx.x];
  if (threadIdx.x == 0) {
    sh.n = m;
    if (m == num) sh.tau = max(sh.tau, sh.best[num - 1]);
  }
  __syncthreads();
}

template <typename T, int U>
__global__ void __launch_bounds__(NT) beam_rows_kernel(const BeamParams p, Part* parts, uint64_t* keys, int seg) {
  using R = Rows<T, U>;
  constexpr int VN = R::VN;
  __shared__ R sh;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y;
  const int64_t b = row / p.beams;
  const int j = (int)(row % p.beams);
  if (p.finished != nullptr && p.finished[b * p.fb + j * p.fk] != 0) return;
  if (p.scores[b * p.sb + j * p.sk] == -INFINITY) return;
  const T* x = static_cast<const T*>(p.logits) + b * p.lb + j * p.lk;
  const int s0 = blockIdx.x * seg, s1 = min(p.V, s0 + seg);
  // vectors lie on 16-byte boundaries: the first begins up to VN - 1 elements in front of the part
  const int off = (int)((reinterpret_cast<uintptr_t>(x + s0) & 15) / sizeof(T));
  if (tid == 0) { sh.n = 0; sh.tau = 0; sh.total = 0; }
  float run = -INFINITY, sum = 0.f;
  __syncthreads();
  for (int t0 = s0 - off; t0 < s1; t0 += R::TILE) {
    float v[U][VN];
    float tm = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i0 = t0 + (u * NT + tid) * VN;
      if (i0 >= s0 && i0 + VN <= s1) {
        const uint4 raw = *reinterpret_cast<const uint4*>(x + i0);
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int k = 0; k < VN; ++k) v[u][k] = to_f32(e[k]);
      } else {
#pragma unroll
        for (int k = 0; k < VN; ++k) v[u][k] = i0 + k >= s0 && i0 + k < s1 ? to_f32(x[i0 + k]) : -INFINITY;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float m = v[u][0];
#pragma unroll
      for (int k = 1; k < VN; ++k) m = fmaxf(m, v[u][k]);
      if (m > run) {
        sum *= ex2f((run - m) * kLog2e);
        run = m;
      }
      tm = fmaxf(tm, m);
      // elements of -inf in front of the first finite one: the difference to -inf would be NaN
      const float base = run == -INFINITY ? 0.f : run;
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < VN; ++k) s += ex2f((v[u][k] - base) * kLog2e);
      sum += s;
    }
    // elements above the threshold
    const float tau_v = sh.tau == 0 ? -INFINITY : unordered((uint32_t)(sh.tau >> 32));
    const bool some = tm >= tau_v;
    if (!__syncthreads_or(some)) continue;
    auto count = [&]() {
      const uint64_t tau = sh.tau;
      int c = 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < VN; ++k) {
          const int i = t0 + (u * NT + tid) * VN + k;
          c += i >= s0 && i < s1 && key_of(v[u][k], i) > tau;
        }
      return c;
    };
    int c = some ? count() : 0;
    if (c) atomicAdd(&sh.total, c);
    __syncthreads();
    const int would = sh.n + sh.total;
    __syncthreads();  // the list grows only once every thread has read its length
    if (would > R::CAP) {
      // the num-th largest of the threads' maxima: at most num threads hold elements from there on
      uint64_t mine = 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < VN; ++k) {
          const int i = t0 + (u * NT + tid) * VN + k;
          if (i >= s0 && i < s1) mine = max(mine, key_of(v[u][k], i));
        }
      sh.thread_max[tid] = mine;
      compact(sh, p.num);
      int r = 0;
#pragma unroll 8
      for (int i = 0; i < NT; ++i) r += sh.thread_max[i] > mine;
      if (tid == 0) sh.total = 0;
      __syncthreads();
      // keys from the threshold on pass: the threshold itself is that of an element
      if (r == p.num - 1 && mine != 0 && mine - 1 > sh.tau) sh.tau = mine - 1;
      __syncthreads();
      c = count();
    }
    if (c) {
      const uint64_t tau = sh.tau;
      int at = atomicAdd(&sh.n, c);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < VN; ++k) {
          const int i = t0 + (u * NT + tid) * VN + k;
          const uint64_t key = key_of(v[u][k], i);
          if (i >= s0 && i < s1 && key > tau) sh.list[at++] = key;
        }
    }
    __syncthreads();
    if (tid == 0) sh.total = 0;
  }
  compact(sh, p.num);
  const int n = sh.n;
  const int64_t part = row * gridDim.x + blockIdx.x;
  if (tid < n) keys[part * p.num + tid] = sh.list[tid];
  // the sum over the CTA, to one base
  float m = run;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((tid & 31) == 0) sh.max[tid >> 5] = m;
  __syncthreads();
  m = sh.max[0];
#pragma unroll
  for (int w = 1; w < NT / 32; ++w) m = fmaxf(m, sh.max[w]);
  double d = run == -INFINITY ? (double)sum : (double)sum * exp((double)run - (double)m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  if ((tid & 31) == 0) sh.sum[tid >> 5] = d;
  __syncthreads();
  if (tid == 0) {
    d = sh.sum[0];
#pragma unroll
    for (int w = 1; w < NT / 32; ++w) d += sh.sum[w];
    parts[part] = Part{d, m, n};
  }
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

constexpr int kCands = kMaxCandidates * kMaxCandidates;

__global__ void __launch_bounds__(NT) beam_join_kernel(const BeamParams p, const Part* parts, const uint64_t* keys, int splits) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Cand* cand = reinterpret_cast<Cand*>(smem_raw);        // kCands
  Cand* head = cand + kCands;                            // beams * splits
  // a logarithm of probability is (l - max) - log(sum): l - (max + log(sum)) would lose the digits of large logits
  __shared__ double s_max[kMaxBeams], s_log[kMaxBeams], s_score[kMaxBeams];
  __shared__ int s_kind[kMaxBeams], s_n;                 // 0 listed, 1 ended, 2 nothing, 3 NaN
  __shared__ Cand s_tau;
  const int tid = threadIdx.x, K = p.beams, lists = K * splits;
  const int64_t b = blockIdx.x;
  if (tid == 0) { s_n = 0; s_tau = Cand{0, 0}; }
  if (tid < K) {
    const float score = p.scores[b * p.sb + tid * p.sk];
    int kind = 0;
    double peak = 0.0, logs = 0.0;
    if (score == -INFINITY) kind = 2;
    else if (!(score < INFINITY)) kind = 3;
    else if (p.finished != nullptr && p.finished[b * p.fb + tid * p.fk] != 0) kind = 1;
    else {
      const Part* q = parts + (b * K + tid) * splits;
      float m = -INFINITY;
      for (int i = 0; i < splits; ++i) m = fmaxf(m, q[i].max);
      double s = 0.0;
      for (int i = 0; i < splits; ++i) s += q[i].max == -INFINITY ? q[i].sum : q[i].sum * exp((double)q[i].max - (double)m);
      peak = (double)m;
      logs = log(s);
      if (!(s == s) || m == INFINITY) kind = 3;
      else if (m == -INFINITY) kind = 2;
    }
    s_kind[tid] = kind;
    s_max[tid] = peak;
    s_log[tid] = logs;
    s_score[tid] = (double)score;
  }
  __syncthreads();
  // element i of list l: false behind its end
  auto get = [&](int l, int i, Cand* c) {
    const int j = l / splits, kind = s_kind[j];
    if (i >= p.num) return false;
    if (kind == 0) {
      const int64_t part = (b * K + j) * splits + l % splits;
      if (i >= parts[part].n) return false;
      const uint64_t key = keys[part * p.num + i];
      const uint32_t o = (uint32_t)(key >> 32);
      *c = Cand{ordered64(s_score[j] + (((double)unordered(o) - s_max[j]) - s_log[j])), tie_of(j, o, (int)~(uint32_t)key)};
      return true;
    }
    if (l % splits != 0 || i >= p.V) return false;
    if (kind == 1 && i == 0) {
      *c = Cand{ordered64(s_score[j]), tie_of(j, ~0u, p.end_token)};
      return true;
    }
    const int token = kind == 1 && i <= p.end_token ? i - 1 : i;
    *c = Cand{kind == 3 ? ~0ull : ordered64(-(double)INFINITY), tie_of(j, 0, token)};
    return true;
  };
  for (int l = tid; l < lists; l += NT)
    if (!get(l, 0, &head[l])) head[l] = Cand{0, 0};
  __syncthreads();
  // nothing below the num-th best head can be among the num best
  if (lists > p.num) {
    for (int l = tid; l < lists; l += NT) {
      const Cand mine = head[l];
      int r = 0;
      for (int i = 0; i < lists; ++i) r += above(head[i], mine);
      if (r == p.num - 1 && mine.tie != 0) s_tau = mine;
    }
    __syncthreads();
  }
  const Cand tau = s_tau;
  for (int l = tid; l < lists; l += NT) {
    Cand c;
    for (int i = 0; get(l, i, &c) && !above(tau, c); ++i) cand[atomicAdd(&s_n, 1)] = c;
  }
  __syncthreads();
  const int n = s_n;
  for (int i = tid; i < n; i += NT) {
    const Cand mine = cand[i];
    int r = 0;
    for (int k = 0; k < n; ++k) r += above(cand[k], mine);
    if (r < p.num) {
      const int64_t at = b * p.num + r;
      p.out_scores[at] = (float)unordered64(mine.value);
      p.parents[at] = 63 - (int)(mine.tie >> (32 + kTokenBits));
      p.tokens[at] = (1 << kTokenBits) - 1 - (int)(mine.tie & ((1 << kTokenBits) - 1));
    }
  }
}

struct BeamPlan { int u, seg, splits; };

// Parts of a row: tiles of four vectors a thread where the rows alone fill the GPU, of one where they do not;
// then as many parts as bring the rows to about four CTAs an SM.
BeamPlan plan(int64_t rows, int V, int es, int sms) {
  const int vn = 16 / es;
  BeamPlan w;
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
  const int64_t rows = batch * beams;
  const BeamPlan w = plan(rows, V, (int)dtype_size(dtype), sms);
  return (size_t)rows * w.splits * (sizeof(Part) + (size_t)num * sizeof(uint64_t));
}

int launch_beam_select(const BeamParams& p, int dtype, void* ws, cudaStream_t s) {
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  const int64_t rows = p.batch * p.beams;
  const BeamPlan w = plan(rows, p.V, (int)dtype_size(dtype), sms);
  if (p.beams * w.splits > kMaxLists) return fail(M3_ERR_UNSUPPORTED, "beam_select: too many parts");
  Part* parts = static_cast<Part*>(ws);
  uint64_t* keys = reinterpret_cast<uint64_t*>(parts + rows * w.splits);
  const dim3 grid((unsigned)w.splits, (unsigned)rows);
  auto go = [&](auto t) {
    using T = decltype(t);
    if (w.u == 4) beam_rows_kernel<T, 4><<<grid, NT, 0, s>>>(p, parts, keys, w.seg);
    else beam_rows_kernel<T, 1><<<grid, NT, 0, s>>>(p, parts, keys, w.seg);
    return check_launch("beam_rows_kernel");
  };
  if (dtype == M3_FLOAT32) M3_TRY(go(float{}));
  else if (dtype == M3_BFLOAT16) M3_TRY(go(__nv_bfloat16{}));
  else M3_TRY(go(__half{}));
  static std::atomic<bool> done[kMaxDevices];
  const size_t most = (size_t)(kCands + kMaxLists) * sizeof(Cand);
  M3_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(&beam_join_kernel), most, done));
  const size_t smem = (size_t)(kCands + p.beams * w.splits) * sizeof(Cand);
  beam_join_kernel<<<(unsigned)p.batch, NT, smem, s>>>(p, parts, keys, w.splits);
  return check_launch("beam_join_kernel");
}

}  // namespace m3
