// Global gradient norm over many tensors, with scaling and clipping:
//   n = scale * sqrt(sum_i sum_j g_ij^2)   (or scale * max |g_ij|)
//   f = scale * min(1, max_norm / (n + 1e-6)),   g <- f g  (or out <- f g)
// A NaN among the gradients makes n and everything that is written NaN; an infinite n makes f 0, or
// NaN where max_norm is infinite too. In place with scale 1 and max_norm infinite only n is formed.
// Two launches: partial norms of fixed parts, then every CTA adds the partial norms in the
// same order (so all agree on f, and the result does not depend on the schedule) and scales
// its parts. The tensors' table travels in the kernel's parameters, so a captured graph holds
// it and nothing is copied to the device.
// Bound by the memory: 2.73 G bf16 gradients, norm 0.79 ms (5.5 GB read at 6.9 TB/s), scaled into
// fp32 2.75 ms (16.4 GB at 6.0 TB/s). They are read twice because the factor depends on all of
// them; what the L2 cache still holds (126 MB) is read back from it. A model's 156 M fp32
// gradients whose norm is in bounds: 0.10 ms, one reading at 6.2 TB/s.
#include <algorithm>

#include "grad_clip.cuh"
#include "m3_common.cuh"

namespace m3 {
namespace {

constexpr int kThreads = 256;
constexpr int kCtasPerSm = 8;
constexpr int kMaxCtas = 2048;       // of one launch
constexpr int kFew = 64, kMany = 1000;  // tensors of one launch: parameters of 2 KB / 31 KB

constexpr int64_t kMaxElements = int64_t(1) << 44;  // 2^30 parts of 16384

template <int K>
struct Table {
  const void* g[K];
  void* o[K];
  int64_t n[K];
  uint32_t first[K];   // the tensor's first part
  uint8_t type[K];     // gradient's dtype | out's dtype << 4
  int count;
  uint32_t parts;
  int part;            // elements of one part, a multiple of 16
};
static_assert(sizeof(Table<kMany>) + 64 <= 32764, "kernel parameters are limited to 32764 bytes");

template <typename T>
struct alignas(16) Vec {
  static constexpr int N = 16 / sizeof(T);
  T e[N];
};

// The part's tensor: the last one that begins at or before it.
template <int K>
__device__ __forceinline__ int tensor_of(const Table<K>& t, uint32_t part) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= part) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// larger magnitude, a NaN above all
__device__ __forceinline__ float larger(float a, float b) { return (a > b || a != a) ? a : b; }

// rows of an embedding that no token used are zeros: they need no second look
template <typename T, int N>
__device__ __forceinline__ bool nonzero(const T (&e)[N]) {
  bool any = false;
#pragma unroll
  for (int k = 0; k < N; ++k) any |= to_f32(e[k]) != 0.f;
  return any;
}

template <typename T, bool LARGEST>
struct Acc {
  double sum = 0.0;
  float mx = 0.f;
  // Squares of one vector are added in 32 bits, vectors in 64. Where the 32-bit sum could
  // have overflowed or lost what underflows, the vector's squares are formed in 64 bits.
  template <int N>
  __device__ __forceinline__ void take(const T (&e)[N]) {
    if constexpr (LARGEST) {
#pragma unroll
      for (int k = 0; k < N; ++k) mx = larger(fabsf(to_f32(e[k])), mx);
    } else {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < N; ++k) s = fmaf(to_f32(e[k]), to_f32(e[k]), s);
      if (s > 1e-28f && s < 1e37f) {
        sum += (double)s;
      } else if (nonzero(e)) {
#pragma unroll
        for (int k = 0; k < N; ++k) sum = fma((double)to_f32(e[k]), (double)to_f32(e[k]), sum);
      }
    }
  }
};

template <typename T, bool LARGEST>
__device__ __forceinline__ void take_part(Acc<T, LARGEST>& acc, const T* g, int n) {
  constexpr int N = Vec<T>::N;
  const int head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) / sizeof(T)));
  const int nv = (n - head) / N;
  const Vec<T>* v = reinterpret_cast<const Vec<T>*>(g + head);
  constexpr int U = 4;
  int j = threadIdx.x;
  for (; j + (U - 1) * kThreads < nv; j += U * kThreads) {
    Vec<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = v[j + u * kThreads];
#pragma unroll
    for (int u = 0; u < U; ++u) acc.take(x[u].e);
  }
  for (; j < nv; j += kThreads) acc.take(v[j].e);
  for (int i = threadIdx.x; i < head; i += kThreads) { const T e[1] = {g[i]}; acc.take(e); }
  for (int i = head + nv * N + threadIdx.x; i < n; i += kThreads) { const T e[1] = {g[i]}; acc.take(e); }
}

template <bool LARGEST>
__device__ __forceinline__ double block_join(double sum, float mx, double* sh) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    if constexpr (LARGEST) mx = larger(__shfl_xor_sync(0xffffffffu, mx, s), mx);
    else sum += __shfl_xor_sync(0xffffffffu, sum, s);
  }
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = LARGEST ? (double)mx : sum;
  __syncthreads();
  double t = sh[0];
  for (int i = 1; i < kThreads / 32; ++i) t = LARGEST ? (double)larger((float)sh[i], (float)t) : t + sh[i];
  return t;
}

template <int K, bool LARGEST>
__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const __grid_constant__ Table<K> t, double* partial) {
  __shared__ double sh[kThreads / 32];
  double sum = 0.0;
  float mx = 0.f;
  for (uint32_t part = blockIdx.x; part < t.parts; part += gridDim.x) {
    const int i = tensor_of(t, part);
    const int64_t at = (int64_t)(part - t.first[i]) * t.part;
    const int n = (int)min((int64_t)t.part, t.n[i] - at);
    auto go = [&](auto* g) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(g)>>;
      Acc<T, LARGEST> acc;
      take_part(acc, g + at, n);
      if constexpr (LARGEST) mx = larger(acc.mx, mx);
      else sum += acc.sum;
    };
    const int type = t.type[i] & 15;
    if (type == M3_FLOAT32) go(static_cast<const float*>(t.g[i]));
    else if (type == M3_BFLOAT16) go(static_cast<const __nv_bfloat16*>(t.g[i]));
    else go(static_cast<const __half*>(t.g[i]));
  }
  const double v = block_join<LARGEST>(sum, mx, sh);
  if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

// `n` gradients, scaled. A thread moves as many elements at once as make one 16-byte store, so
// that the stores of a warp are one run of memory also where a 16-bit gradient becomes an fp32
// one (its loads are then 8 bytes wide).
template <typename T, typename O>
__device__ __forceinline__ void scale_part(const T* g, O* o, int n, float f) {
  constexpr int M = 16 / sizeof(O), kBytes = M * sizeof(T);
  struct alignas(kBytes) In { T e[M]; };
  struct alignas(16) Out { O e[M]; };
  const int head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(o) & 15)) & 15) / sizeof(O)));
  const bool same = (reinterpret_cast<uintptr_t>(g + head) & (kBytes - 1)) == 0;
  const int nv = same ? (n - head) / M : 0;
  const In* v = reinterpret_cast<const In*>(g + head);
  Out* w = reinterpret_cast<Out*>(o + head);
  auto put = [&](int j, const In& x) {
    Out y;
#pragma unroll
    for (int k = 0; k < M; ++k) y.e[k] = from_f32<O>(to_f32(x.e[k]) * f);
    __stcs(reinterpret_cast<float4*>(w + j), *reinterpret_cast<const float4*>(&y));  // not needed again here
  };
  constexpr int U = kBytes == 16 ? 4 : 8;
  int j = threadIdx.x;
  for (; j + (U - 1) * kThreads < nv; j += U * kThreads) {
    In x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = v[j + u * kThreads];
#pragma unroll
    for (int u = 0; u < U; ++u) put(j + u * kThreads, x[u]);
  }
  for (; j < nv; j += kThreads) put(j, v[j]);
  // before the vectors and behind them (everything, where the two sides' boundaries differ)
  for (int i = threadIdx.x; i < head; i += kThreads) o[i] = from_f32<O>(to_f32(g[i]) * f);
  for (int i = head + nv * M + threadIdx.x; i < n; i += kThreads) o[i] = from_f32<O>(to_f32(g[i]) * f);
}

template <int K, bool LARGEST>
__global__ void __launch_bounds__(kThreads)
    grad_scale_kernel(const __grid_constant__ Table<K> t, const double* partial, int partials, double max_norm,
                      double scale, bool in_place, bool norm_alone, float* norm) {
  __shared__ double sh[kThreads / 32];
  double sum = 0.0;
  float mx = 0.f;
  for (int i = threadIdx.x; i < partials; i += kThreads) {
    if constexpr (LARGEST) mx = larger((float)partial[i], mx);
    else sum += partial[i];
  }
  const double all = block_join<LARGEST>(sum, mx, sh);
  const double n = scale * (LARGEST ? all : sqrt(all));
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  if (norm_alone) return;
  double c = max_norm / (n + 1e-6);
  if (c > 1.0) c = 1.0;  // a NaN stays
  if (in_place && c == 1.0 && scale == 1.0) return;
  const float f = (float)(c * scale);
  // from the last part back: what the norm read last may still be in the L2 cache
  for (uint32_t q = blockIdx.x; q < t.parts; q += gridDim.x) {
    const uint32_t part = t.parts - 1 - q;
    const int i = tensor_of(t, part);
    const int64_t at = (int64_t)(part - t.first[i]) * t.part;
    const int m = (int)min((int64_t)t.part, t.n[i] - at);
    auto go = [&](auto* g, auto* o) { scale_part(g + at, o + at, m, f); };
    const int type = t.type[i] & 15, to = t.type[i] >> 4;
    if (type == M3_FLOAT32) {
      go(static_cast<const float*>(t.g[i]), static_cast<float*>(t.o[i]));
    } else if (type == M3_BFLOAT16) {
      if (to == M3_FLOAT32) go(static_cast<const __nv_bfloat16*>(t.g[i]), static_cast<float*>(t.o[i]));
      else go(static_cast<const __nv_bfloat16*>(t.g[i]), static_cast<__nv_bfloat16*>(t.o[i]));
    } else {
      if (to == M3_FLOAT32) go(static_cast<const __half*>(t.g[i]), static_cast<float*>(t.o[i]));
      else go(static_cast<const __half*>(t.g[i]), static_cast<__half*>(t.o[i]));
    }
  }
}

// Elements of one part: the work in about four parts a CTA, between 2048 (a part's search
// and reduction are then still small beside it) and 16384 elements.
int part_elements(int64_t total, int64_t ctas) {
  int64_t want = total / (ctas * 4);
  int part = 2048;
  while (part < 16384 && part < want) part *= 2;
  return part;
}

template <int K>
int run(const ClipArgs& a, double* partial, cudaStream_t s) {
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  const int ctas = std::min(kMaxCtas, sms * kCtasPerSm);
  int64_t total = 0;
  for (int64_t i = 0; i < a.count; ++i) {
    total += a.numel[i];
    if (a.numel[i] > kMaxElements || total > kMaxElements)
      return fail(M3_ERR_UNSUPPORTED, "clip_grads: too many elements");
  }
  Table<K> t;
  t.part = part_elements(total, ctas);
  // one launch's tensors from i on; returns the next one
  auto fill = [&](int64_t i) {
    uint64_t parts = 0;
    t.count = 0;
    for (; i < a.count && t.count < K; ++i) {
      const uint64_t mine = (uint64_t)((a.numel[i] + t.part - 1) / t.part);
      if (mine == 0) continue;
      const int k = t.count++;
      t.g[k] = a.grads[i];
      t.o[k] = a.outs ? a.outs[i] : const_cast<void*>(a.grads[i]);
      t.n[k] = a.numel[i];
      t.first[k] = (uint32_t)parts;
      const int32_t to = a.outs ? a.out_dtypes[i] : a.dtypes[i];
      t.type[k] = (uint8_t)(a.dtypes[i] | (to << 4));
      parts += mine;
    }
    t.parts = (uint32_t)parts;
    return i;
  };
  int partials = 0;
  for (int64_t i = 0; i < a.count;) {
    i = fill(i);
    if (t.parts == 0) continue;
    const int grid = (int)std::min<int64_t>(t.parts, ctas);
    if (a.largest) grad_norm_kernel<K, true><<<grid, kThreads, 0, s>>>(t, partial + partials);
    else grad_norm_kernel<K, false><<<grid, kThreads, 0, s>>>(t, partial + partials);
    M3_TRY(check_launch("grad_norm_kernel"));
    partials += grid;
  }
  float* norm = a.norm;
  for (int64_t i = 0; i < a.count;) {
    i = fill(i);
    if (t.parts == 0 && norm == nullptr) continue;
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(t.parts, ctas));
    if (a.largest)
      grad_scale_kernel<K, true><<<grid, kThreads, 0, s>>>(t, partial, partials, a.max_norm, a.scale, a.in_place,
                                                           a.norm_alone, norm);
    else
      grad_scale_kernel<K, false><<<grid, kThreads, 0, s>>>(t, partial, partials, a.max_norm, a.scale, a.in_place,
                                                            a.norm_alone, norm);
    M3_TRY(check_launch("grad_scale_kernel"));
    norm = nullptr;  // the first launch writes it
  }
  return M3_OK;
}

}  // namespace

size_t clip_grads_workspace_bytes(int64_t count) {
  return sizeof(double) * kMaxCtas * (size_t)(count / kMany + 1);  // one partial norm a CTA and launch
}

int launch_clip_grads(const ClipArgs& a, void* ws, cudaStream_t s) {
  if (a.count == 0) {
    cudaError_t e = cudaMemsetAsync(a.norm, 0, sizeof(float), s);
    if (e != cudaSuccess) return fail(M3_ERR_CUDA, std::string("clip_grads: ") + cudaGetErrorString(e));
    return M3_OK;
  }
  double* partial = static_cast<double*>(ws);
  return a.count <= kFew ? run<kFew>(a, partial, s) : run<kMany>(a, partial, s);
}

}  // namespace m3
