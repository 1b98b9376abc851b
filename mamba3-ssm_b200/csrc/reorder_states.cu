// Rows of many state tensors moved to the beams that continue them, in one launch:
//   dst row b T + j  <-  src row b S + parents[b, j]; zeros where the parent is outside [0, S).
// In place (S = T) a thread takes one column of a whole group: it reads what the moved rows need before it
// writes any, so no other thread's column matters, rows that stay are neither read nor written, and
// nothing is staged. The tensors' table travels in the kernel's parameters.
// Bound by the memory: distinct moved parents read once, moved rows written (1.5 GB in 253 us, 5.9 TB/s).
#include <algorithm>

#include "beam.cuh"
#include "m3_common.cuh"

namespace m3 {
namespace {

constexpr int kThreads = 128;
constexpr int kFew = 64, kMany = 512;  // tensors of one launch

template <int K>
struct Table {
  const char* src[K];
  char* dst[K];
  int64_t src_pitch[K], dst_pitch[K];
  int64_t units[K];     // of a row
  uint32_t first[K];    // the tensor's first part
  uint8_t log_unit[K];  // bytes moved at a time: 2^log_unit
  int count;
  uint32_t parts;
  const int64_t* parents;
  int64_t pb, pk;
  int batch, source, rows;
  bool in_place;
};
static_assert(sizeof(Table<kMany>) + 64 <= 32764, "kernel parameters are limited to 32764 bytes");

template <int R, typename U, int K>
__device__ __forceinline__ void move_column(const Table<K>& t, int i, int b, int64_t col) {
  const char* src = t.src[i] + (int64_t)b * t.source * t.src_pitch[i] + col * (int64_t)sizeof(U);
  char* dst = t.dst[i] + (int64_t)b * t.rows * t.dst_pitch[i] + col * (int64_t)sizeof(U);
  const int64_t* par = t.parents + (int64_t)b * t.pb;
  for (int j0 = 0; j0 < t.rows; j0 += R) {  // in place there is one round: rows <= R
    // where each row comes from, before any is loaded, so that all loads are in flight together (1.5 GB of a model's
    // cache: 253 us, row by row 313); neighbours that continue the same beam, as often in sorted candidates, share one (0.6 GB
    // of forks: 104 us, each for itself 116)
    U v[R];
    uint32_t moved = 0, same = 0;
    int from[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int64_t f = j0 + j < t.rows ? par[(j0 + j) * t.pk] : 0;
      from[j] = f >= 0 && f < t.source ? (int)f : -1;
      if (j0 + j < t.rows && !(t.in_place && f == j0 + j)) moved |= 1u << j;
      if (j > 0 && from[j] == from[j - 1] && (moved >> (j - 1) & 1)) same |= 1u << j;
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
      v[j] = U{};
      if ((moved & ~same) >> j & 1 && from[j] >= 0) v[j] = *reinterpret_cast<const U*>(src + from[j] * t.src_pitch[i]);
    }
#pragma unroll
    for (int j = 1; j < R; ++j)
      if (same >> j & 1) v[j] = v[j - 1];
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (moved >> j & 1) *reinterpret_cast<U*>(dst + (int64_t)(j0 + j) * t.dst_pitch[i]) = v[j];
  }
}

// R: rows that a thread holds at a time
template <int R, int K>
__global__ void __launch_bounds__(kThreads) reorder_kernel(const __grid_constant__ Table<K> t) {
  for (uint32_t part = blockIdx.x; part < t.parts; part += gridDim.x) {
    int lo = 0, hi = t.count - 1;  // the part's tensor: the last one that begins at or before it
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (t.first[mid] <= part) lo = mid;
      else hi = mid - 1;
    }
    const uint32_t blocks = (uint32_t)((t.units[lo] + kThreads - 1) / kThreads), at = part - t.first[lo];
    const int b = (int)(at / blocks);
    const int64_t col = (int64_t)(at % blocks) * kThreads + threadIdx.x;
    if (col >= t.units[lo]) continue;
    if (t.log_unit[lo] == 4) move_column<R, uint4>(t, lo, b, col);
    else if (t.log_unit[lo] == 2) move_column<R, uint32_t>(t, lo, b, col);
    else move_column<R, uint8_t>(t, lo, b, col);
  }
}

template <int R, int K>
int launch(const ReorderArgs& a, cudaStream_t s) {
  int sms = 0;
  M3_TRY(device_sm_count(&sms));
  Table<K> t;
  t.parents = a.parents; t.pb = a.pb; t.pk = a.pk;
  t.batch = (int)a.batch; t.source = (int)a.source; t.rows = (int)a.rows;
  t.in_place = a.in_place;
  t.count = 0;
  t.parts = 0;
  auto flush = [&]() -> int {
    if (t.parts == 0) return M3_OK;
    const unsigned grid = (unsigned)std::min<int64_t>(t.parts, (int64_t)sms * 64);
    reorder_kernel<R, K><<<grid, kThreads, 0, s>>>(t);
    t.count = 0;
    t.parts = 0;
    return check_launch("reorder_kernel");
  };
  for (int64_t i = 0; i < a.count; ++i) {
    if (a.row_bytes[i] == 0) continue;
    const uint64_t any = reinterpret_cast<uintptr_t>(a.src[i]) | reinterpret_cast<uintptr_t>(a.dst[i]) |
                         (uint64_t)a.row_bytes[i] | (uint64_t)a.src_pitch[i] | (uint64_t)a.dst_pitch[i];
    const int lg = (any & 15) == 0 ? 4 : (any & 3) == 0 ? 2 : 0;
    const int64_t units = a.row_bytes[i] >> lg, parts = a.batch * ((units + kThreads - 1) / kThreads);
    if (parts >= (int64_t(1) << 31)) return fail(M3_ERR_UNSUPPORTED, "reorder_states: tensor too large");
    if (t.count == K || (int64_t)t.parts + parts >= (int64_t(1) << 32)) M3_TRY(flush());
    const int c = t.count++;
    t.src[c] = static_cast<const char*>(a.src[i]);
    t.dst[c] = static_cast<char*>(a.dst[i]);
    t.src_pitch[c] = a.src_pitch[i];
    t.dst_pitch[c] = a.dst_pitch[i];
    t.units[c] = units;
    t.log_unit[c] = (uint8_t)lg;
    t.first[c] = t.parts;
    t.parts += (uint32_t)parts;
  }
  return flush();
}

template <int K>
int by_rows(const ReorderArgs& a, cudaStream_t s) {
  if (a.rows <= 4) return launch<4, K>(a, s);
  if (a.rows <= 8 || !a.in_place) return launch<8, K>(a, s);
  if (a.rows <= 16) return launch<16, K>(a, s);
  return launch<32, K>(a, s);
}

}  // namespace

int launch_reorder_states(const ReorderArgs& a, cudaStream_t s) {
  if (a.count <= kFew) return by_rows<kFew>(a, s);
  return by_rows<kMany>(a, s);
}

}  // namespace m3
