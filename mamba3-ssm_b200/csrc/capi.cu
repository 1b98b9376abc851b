// extern "C" entry points of libmamba3_b200: argument validation, dispatch to the
// kernels, and the thread-local error string. Nothing here allocates device memory.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <limits>
#include <mutex>
#include <string>
#include <vector>

#include "argmax.cuh"
#include "beam.cuh"
#include "causal_conv.cuh"
#include "decode_step.cuh"
#include "grad_clip.cuh"
#include "m3_common.cuh"
#include "mimo_scan.cuh"
#include "prologue.cuh"
#include "rmsnorm.cuh"
#include "selective_scan.cuh"
#include "siso_chunk.cuh"
#include "siso_scan.cuh"
#include "token_loss.cuh"

namespace m3 {

static thread_local std::string g_last_error;

void set_error(const std::string& msg) { g_last_error = msg; }

int fail(int code, const std::string& msg) {
  g_last_error = msg;
  return code;
}

int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(M3_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  return M3_OK;
}

int current_device(int* dev) {
  cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return fail(M3_ERR_CUDA, std::string("cudaGetDevice: ") + cudaGetErrorString(e));
  if (*dev < 0 || *dev >= kMaxDevices) return fail(M3_ERR_UNSUPPORTED, "device ordinal beyond the supported range");
  return M3_OK;
}

int device_sm_count(int* sms) {
  static std::atomic<int> cache[kMaxDevices];
  int dev = 0;
  M3_TRY(current_device(&dev));
  int n = cache[dev].load(std::memory_order_acquire);
  if (n <= 0) {
    cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess || n <= 0)
      return fail(M3_ERR_CUDA, std::string("multiprocessor count: ") + cudaGetErrorString(e));
    cache[dev].store(n, std::memory_order_release);  // concurrent first callers store the same value
  }
  *sms = n;
  return M3_OK;
}

int ensure_dynamic_smem(const void* kernel, size_t bytes, std::atomic<bool>* done) {
  int dev = 0;
  M3_TRY(current_device(&dev));
  if (done[dev].load(std::memory_order_acquire)) return M3_OK;
  // idempotent: two threads that both get here set the same attribute twice
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return fail(M3_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
  done[dev].store(true, std::memory_order_release);
  return M3_OK;
}

int kernel_residency(const void* kernel, int threads, size_t smem, LaunchCache* c, int* resident) {
  int dev = 0;
  M3_TRY(current_device(&dev));
  const long long want = (long long)smem;
  const long long w = c->word[dev].load(std::memory_order_acquire);
  if (w > 0 && (w >> 32) == want) {
    *resident = (int)(w & 0xffffffffLL);
    return M3_OK;
  }
  // the opt-in only ever grows, so a launch of a larger size on another host thread never
  // finds it lowered under it
  long long cur = c->smem_max[dev].load(std::memory_order_acquire);
  while (want > cur) {
    if (c->smem_max[dev].compare_exchange_weak(cur, want)) {
      cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)want);
      if (e != cudaSuccess) return fail(M3_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
      break;
    }
  }
  // all of the unified L1 / shared array as shared memory: the CTAs that fit are then set by
  // registers and shared memory, not by the carveout (a hint; its failure is not an error)
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100) != cudaSuccess)
    cudaGetLastError();
  int per_sm = 0, sms = 0;
  cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem);
  if (e != cudaSuccess) return fail(M3_ERR_CUDA, std::string("occupancy query: ") + cudaGetErrorString(e));
  M3_TRY(device_sm_count(&sms));
  const int n = std::max(1, per_sm * sms);
  c->word[dev].store((want << 32) | (long long)n, std::memory_order_release);
  *resident = n;
  return M3_OK;
}

// Fixed scratch of the allocation-free SISO backward (m3_siso_scan_bwd_noalloc): room for
// the per-position workspace of up to M3_NOALLOC_MAX_POSITIONS (batch * heads * seqlen)
// positions, 4 bytes each (8 MiB). Lives in every GPU that loads the library, for the
// lifetime of the process, and is shared by all calls on that GPU.
static __device__ __align__(256) float g_noalloc_scratch[M3_NOALLOC_MAX_POSITIONS];

namespace {

constexpr unsigned kAnyFloat = (1u << M3_FLOAT32) | (1u << M3_BFLOAT16) | (1u << M3_FLOAT16);
constexpr unsigned kF32 = 1u << M3_FLOAT32;

std::string shape_str(const m3_tensor* t) {
  std::string s = "(";
  for (int i = 0; i < t->ndim; ++i) s += std::to_string(t->shape[i]) + (i + 1 < t->ndim ? "," : "");
  return s + ")";
}

bool present(const m3_tensor* t) { return t != nullptr && t->data != nullptr; }

int check_device_ptr(const void* p, const char* name) {
  cudaPointerAttributes attr;
  cudaError_t e = cudaPointerGetAttributes(&attr, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": not a CUDA pointer (" + cudaGetErrorString(e) + ")");
  }
  if (attr.type != cudaMemoryTypeDevice && attr.type != cudaMemoryTypeManaged)
    return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": host memory is not accepted (no CPU path)");
  return M3_OK;
}

// shape must match `shape` (entries < 0 are free); dtype in `mask`; innermost stride 1
// unless the dim has extent 1; `contig` requires the full row-major layout.
int check(const m3_tensor* t, const char* name, int ndim, const int64_t* shape, unsigned mask,
          bool contig, bool optional, bool devcheck) {
  if (!present(t)) {
    if (optional) return M3_OK;
    return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": missing");
  }
  if (t->ndim != ndim)
    return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": expected " + std::to_string(ndim) +
                                             " dims, got " + std::to_string(t->ndim));
  for (int i = 0; i < ndim; ++i)
    if (shape[i] >= 0 && t->shape[i] != shape[i]) {
      std::string want = "(";
      for (int j = 0; j < ndim; ++j) want += (shape[j] >= 0 ? std::to_string(shape[j]) : std::string("*")) + (j + 1 < ndim ? "," : "");
      return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": shape " + shape_str(t) + " != " + want + ")");
    }
  if (t->dtype < 0 || t->dtype > 2 || !(mask & (1u << t->dtype)))
    return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": unsupported dtype " + std::to_string(t->dtype));
  int64_t n = 1;
  for (int i = 0; i < ndim; ++i) n *= t->shape[i];
  if (n == 0) return M3_OK;  // empty views carry arbitrary strides and are never dereferenced
  if (ndim > 0 && t->shape[ndim - 1] > 1 && t->stride[ndim - 1] != 1)
    return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": innermost dimension must be contiguous");
  if (contig) {
    int64_t st = 1;
    for (int i = ndim - 1; i >= 0; --i) {
      if (t->shape[i] > 1 && t->stride[i] != st)
        return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": must be contiguous");
      st *= t->shape[i];
    }
  }
  for (int i = 0; i < ndim; ++i)
    if (t->stride[i] < 0) return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": negative stride");
  if (devcheck) return check_device_ptr(t->data, name);
  return M3_OK;
}

// strides of dims (0,1,2) of a 4-d view
Str3 s3(const m3_tensor* t) { return Str3{t->stride[0], t->stride[1], t->stride[2]}; }
Str3 s3_scal(const m3_tensor* t) { return Str3{t->stride[0], t->stride[1], t->stride[2]}; }
Str4 s4(const m3_tensor* t) { return Str4{t->stride[0], t->stride[1], t->stride[2], t->stride[3]}; }

template <typename T>
T* fptr(const m3_tensor* t) { return present(t) ? reinterpret_cast<T*>(t->data) : nullptr; }

int memset_async(void* p, size_t bytes, cudaStream_t s, const char* what) {
  if (!p || bytes == 0) return M3_OK;
  cudaError_t e = cudaMemsetAsync(p, 0, bytes, s);
  if (e != cudaSuccess) return fail(M3_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  return M3_OK;
}

int copy_or_zero(void* dst, const void* src, size_t bytes, cudaStream_t s, const char* what) {
  if (!dst || bytes == 0) return M3_OK;
  cudaError_t e = src ? cudaMemcpyAsync(dst, src, bytes, cudaMemcpyDeviceToDevice, s) : cudaMemsetAsync(dst, 0, bytes, s);
  if (e != cudaSuccess) return fail(M3_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  return M3_OK;
}

// Shared checks of the scan operands. bc_ndim 4 (SISO) or 5 (MIMO).
int check_scan_inputs(const m3_tensor* x, const m3_tensor* B, const m3_tensor* C, const m3_tensor* ADT,
                      const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D, int bc_ndim,
                      int64_t* Bn, int64_t* L, int64_t* H, int64_t* P, int64_t* Ds, int64_t* R) {
  if (!present(x)) return fail(M3_ERR_INVALID_ARGUMENT, "x: missing");
  if (x->ndim != 4) return fail(M3_ERR_INVALID_ARGUMENT, "x: expected (B, L, H, P)");
  *Bn = x->shape[0]; *L = x->shape[1]; *H = x->shape[2]; *P = x->shape[3];
  if (!present(B) || B->ndim != bc_ndim) return fail(M3_ERR_INVALID_ARGUMENT, bc_ndim == 4 ? "B: expected (B, L, H, D)" : "B: expected (B, L, R, H, D)");
  *Ds = B->shape[bc_ndim - 1];
  *R = bc_ndim == 5 ? B->shape[2] : 1;
  const bool empty = (*Bn) * (*L) * (*H) * (*P) == 0;
  const int64_t xs[4] = {*Bn, *L, *H, *P};
  M3_TRY(check(x, "x", 4, xs, kAnyFloat, false, false, !empty));
  if (bc_ndim == 4) {
    const int64_t bs[4] = {*Bn, *L, *H, *Ds};
    M3_TRY(check(B, "B", 4, bs, kAnyFloat, false, false, !empty));
    M3_TRY(check(C, "C", 4, bs, 1u << B->dtype, false, false, !empty));
  } else {
    const int64_t bs[5] = {*Bn, *L, *R, *H, *Ds};
    M3_TRY(check(B, "B", 5, bs, kAnyFloat, false, false, !empty));
    M3_TRY(check(C, "C", 5, bs, 1u << B->dtype, false, false, !empty));
  }
  const int64_t ss[3] = {*Bn, *L, *H};
  M3_TRY(check(ADT, "ADT", 3, ss, kF32, false, false, false));
  M3_TRY(check(DT, "DT", 3, ss, kF32, false, false, false));
  M3_TRY(check(trap, "trap", 3, ss, kF32, false, false, false));
  const int64_t hs[1] = {*H};
  if (!present(D) || D->ndim != 1 || D->shape[0] != *H || D->dtype != M3_FLOAT32)
    return fail(M3_ERR_INVALID_ARGUMENT, "D: expected (H) float32");
  (void)hs;
  if (*Ds <= 0 && !empty) return fail(M3_ERR_INVALID_ARGUMENT, "B: d_state must be positive");
  return M3_OK;
}

}  // namespace
}  // namespace m3

using namespace m3;

extern "C" {

int m3_abi_version(void) { return M3_ABI_VERSION; }

const char* m3_last_error_string(void) { return g_last_error.c_str(); }

int m3_siso_scan_fwd(const m3_tensor* x, const m3_tensor* B, const m3_tensor* C, const m3_tensor* ADT,
                     const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D, const m3_tensor* h0,
                     const m3_tensor* bx0, m3_tensor* y, m3_tensor* h_last, m3_tensor* bx_last, void* stream) {
  int64_t Bn, L, H, P, Ds, R;
  M3_TRY(check_scan_inputs(x, B, C, ADT, DT, trap, D, 4, &Bn, &L, &H, &P, &Ds, &R));
  const int64_t xs[4] = {Bn, L, H, P}, st[4] = {Bn, H, P, Ds};
  const bool empty = Bn * L * H * P == 0;
  M3_TRY(check(y, "y", 4, xs, 1u << x->dtype, false, false, !empty));
  M3_TRY(check(h0, "h0", 4, st, kF32, true, true, false));
  M3_TRY(check(bx0, "bx0", 4, st, kF32, true, true, false));
  M3_TRY(check(h_last, "h_last", 4, st, kF32, true, true, false));
  M3_TRY(check(bx_last, "bx_last", 4, st, kF32, true, true, false));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (Bn * H * P * Ds == 0) return M3_OK;
  if (L == 0) {
    const size_t bytes = sizeof(float) * Bn * H * P * Ds;
    M3_TRY(copy_or_zero(fptr<void>(h_last), fptr<void>(h0), bytes, s, "h_last"));
    return copy_or_zero(fptr<void>(bx_last), fptr<void>(bx0), bytes, s, "bx_last");
  }
  if (Bn > INT32_MAX || L > INT32_MAX || H > INT32_MAX || P > 65535)
    return fail(M3_ERR_UNSUPPORTED, "siso scan: dimension too large");
  SisoParams p{};
  p.Bn = (int)Bn; p.L = (int)L; p.H = (int)H; p.P = (int)P; p.D = (int)Ds;
  p.x = x->data; p.sx = s3(x);
  p.Bm = B->data; p.sB = s3(B);
  p.Cm = C->data; p.sC = s3(C);
  p.adt = fptr<const float>(ADT); p.sadt = s3_scal(ADT);
  p.dt = fptr<const float>(DT); p.sdt = s3_scal(DT);
  p.trap = fptr<const float>(trap); p.strap = s3_scal(trap);
  p.Dskip = fptr<const float>(D); p.sD = D->stride[0];
  p.h0 = fptr<const float>(h0); p.bx0 = fptr<const float>(bx0);
  p.y = y->data; p.sy = s3(y);
  p.h_last = fptr<float>(h_last); p.bx_last = fptr<float>(bx_last);
  if (siso_chunk_supported(p, x->dtype, B->dtype)) return launch_siso_fwd_chunked(p, x->dtype, B->dtype, s);
  return launch_siso_fwd_recurrent(p, x->dtype, B->dtype, s);
}

// Bytes of the workspace the chunked tensor-core backward needs: the forward's chunk states
// (recomputed inside m3_siso_scan_bwd) followed by three per-position scratch arrays.
static size_t chunked_bwd_ws_bytes(int64_t Bn, int64_t L, int64_t H) {
  const size_t ks = (siso_chunk_kstate_bytes(Bn, L, H) + 255) & ~size_t(255);
  return ks + siso_chunk_bwd_scratch_bytes(Bn, L, H);
}

size_t m3_siso_scan_bwd_workspace_size(int64_t batch, int64_t seqlen, int64_t nheads, int64_t headdim,
                                       int64_t dstate) {
  const size_t rec = sizeof(float) * (size_t)(batch * nheads * seqlen);
  // headdim 64 / d_state 128 or 64 may take the chunked path (bf16); size for it
  if (headdim == 64 && (dstate == 128 || dstate == 64)) {
    const size_t ch = chunked_bwd_ws_bytes(batch, seqlen, nheads);
    return ch > rec ? ch : rec;
  }
  return rec;
}

size_t m3_siso_scan_kstates_size(int64_t batch, int64_t seqlen, int64_t nheads, int64_t headdim,
                                 int64_t dstate, int x_dtype, int bc_dtype) {
  if (headdim != 64 || (dstate != 128 && dstate != 64) || x_dtype != M3_BFLOAT16 || bc_dtype != M3_BFLOAT16 || seqlen <= 0 ||
      batch * nheads <= 0)
    return 0;
  return siso_chunk_kstate_bytes(batch, seqlen, nheads);
}

size_t m3_siso_scan_bwd_kstates_workspace_size(int64_t batch, int64_t seqlen, int64_t nheads) {
  return siso_chunk_bwd_scratch_bytes(batch, seqlen, nheads);
}

namespace m3 {
namespace {
// Shared argument checks and parameter fill of the SISO backward entries. Returns M3_OK
// with *done set when nothing is left to launch (empty shapes).
int prep_siso_bwd(SisoParams& p, const m3_tensor* x, const m3_tensor* B, const m3_tensor* C, const m3_tensor* ADT,
                  const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D, const m3_tensor* h0,
                  const m3_tensor* bx0, const m3_tensor* dy, m3_tensor* dx, m3_tensor* dB, m3_tensor* dC,
                  m3_tensor* dADT, m3_tensor* dDT, m3_tensor* dtrap, m3_tensor* dD, m3_tensor* dh0,
                  m3_tensor* dbx0, cudaStream_t s, bool* done) {
  *done = false;
  int64_t Bn, L, H, P, Ds, R;
  M3_TRY(check_scan_inputs(x, B, C, ADT, DT, trap, D, 4, &Bn, &L, &H, &P, &Ds, &R));
  const bool empty = Bn * L * H * P == 0;
  const int64_t xs[4] = {Bn, L, H, P}, bs[4] = {Bn, L, H, Ds}, st[4] = {Bn, H, P, Ds}, ss[3] = {Bn, L, H}, hs[1] = {H};
  M3_TRY(check(h0, "h0", 4, st, kF32, true, true, false));
  M3_TRY(check(bx0, "bx0", 4, st, kF32, true, true, false));
  M3_TRY(check(dy, "dy", 4, xs, 1u << x->dtype, false, false, !empty));
  M3_TRY(check(dx, "dx", 4, xs, 1u << x->dtype, false, false, !empty));
  M3_TRY(check(dB, "dB", 4, bs, 1u << B->dtype, false, false, !empty));
  M3_TRY(check(dC, "dC", 4, bs, 1u << B->dtype, false, false, !empty));
  M3_TRY(check(dADT, "dADT", 3, ss, kF32, false, false, false));
  M3_TRY(check(dDT, "dDT", 3, ss, kF32, false, false, false));
  M3_TRY(check(dtrap, "dtrap", 3, ss, kF32, false, false, false));
  M3_TRY(check(dD, "dD", 1, hs, kF32, true, false, false));
  M3_TRY(check(dh0, "dh0", 4, st, kF32, true, true, false));
  M3_TRY(check(dbx0, "dbx0", 4, st, kF32, true, true, false));
  M3_TRY(memset_async(dD->data, sizeof(float) * H, s, "dD"));
  if (Bn * H * P * Ds == 0) {
    *done = true;
    return M3_OK;
  }
  if (L == 0) {
    const size_t bytes = sizeof(float) * Bn * H * P * Ds;
    M3_TRY(copy_or_zero(fptr<void>(dh0), nullptr, bytes, s, "dh0"));
    M3_TRY(copy_or_zero(fptr<void>(dbx0), nullptr, bytes, s, "dbx0"));
    *done = true;
    return M3_OK;
  }
  if (Bn > INT32_MAX || L > INT32_MAX || H > INT32_MAX || P > 65535)
    return fail(M3_ERR_UNSUPPORTED, "siso scan: dimension too large");
  p = SisoParams{};
  p.Bn = (int)Bn; p.L = (int)L; p.H = (int)H; p.P = (int)P; p.D = (int)Ds;
  p.x = x->data; p.sx = s3(x);
  p.Bm = B->data; p.sB = s3(B);
  p.Cm = C->data; p.sC = s3(C);
  p.adt = fptr<const float>(ADT); p.sadt = s3_scal(ADT);
  p.dt = fptr<const float>(DT); p.sdt = s3_scal(DT);
  p.trap = fptr<const float>(trap); p.strap = s3_scal(trap);
  p.Dskip = fptr<const float>(D); p.sD = D->stride[0];
  p.h0 = fptr<const float>(h0); p.bx0 = fptr<const float>(bx0);
  p.dy = dy->data; p.sdy = s3(dy);
  p.dx = dx->data; p.sdx = s3(dx);
  p.dB = dB->data; p.sdB = s3(dB);
  p.dC = dC->data; p.sdC = s3(dC);
  p.dadt = fptr<float>(dADT); p.sdadt = s3_scal(dADT);
  p.ddt = fptr<float>(dDT); p.sddt = s3_scal(dDT);
  p.dtrap = fptr<float>(dtrap); p.sdtrap = s3_scal(dtrap);
  p.dD = fptr<float>(dD);
  p.dh0 = fptr<float>(dh0); p.dbx0 = fptr<float>(dbx0);
  return M3_OK;
}
}  // namespace
}  // namespace m3

int m3_siso_scan_bwd(const m3_tensor* x, const m3_tensor* B, const m3_tensor* C, const m3_tensor* ADT,
                     const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D, const m3_tensor* h0,
                     const m3_tensor* bx0, const m3_tensor* dy, m3_tensor* dx, m3_tensor* dB, m3_tensor* dC,
                     m3_tensor* dADT, m3_tensor* dDT, m3_tensor* dtrap, m3_tensor* dD, m3_tensor* dh0,
                     m3_tensor* dbx0, void* workspace, size_t workspace_bytes, void* stream) {
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  SisoParams p;
  bool done = false;
  M3_TRY(prep_siso_bwd(p, x, B, C, ADT, DT, trap, D, h0, bx0, dy, dx, dB, dC, dADT, dDT, dtrap, dD, dh0, dbx0, s,
                       &done));
  if (done) return M3_OK;
  const size_t need = sizeof(float) * (size_t)p.Bn * p.H * p.L;
  if (workspace == nullptr || workspace_bytes < need)
    return fail(M3_ERR_WORKSPACE, "siso backward: workspace of " + std::to_string(need) + " bytes required");
  // chunked tensor-core path: recompute the forward's chunk states into the workspace, then
  // the reverse-chunk kernel (taken when the workspace has room for both)
  if (siso_chunk_bwd_supported(p, x->dtype, B->dtype) && workspace_bytes >= chunked_bwd_ws_bytes(p.Bn, p.L, p.H) &&
      (reinterpret_cast<uintptr_t>(workspace) & 255) == 0) {
    const size_t ks = (siso_chunk_kstate_bytes(p.Bn, p.L, p.H) + 255) & ~size_t(255);
    SisoParams f = p;
    f.y = nullptr; f.sy = Str3{0, 0, 0};
    f.h_last = nullptr; f.bx_last = nullptr;
    f.kstates = workspace;
    M3_TRY(launch_siso_fwd_chunked(f, x->dtype, B->dtype, s));
    p.kstates = workspace;
    return launch_siso_bwd_chunked(p, reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ks), s);
  }
  p.q = reinterpret_cast<float*>(workspace);
  return launch_siso_bwd_recurrent(p, x->dtype, B->dtype, s);
}

int m3_siso_scan_fwd_kstates(const m3_tensor* x, const m3_tensor* B, const m3_tensor* C, const m3_tensor* ADT,
                             const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D, const m3_tensor* h0,
                             const m3_tensor* bx0, m3_tensor* y, m3_tensor* h_last, m3_tensor* bx_last,
                             void* kstates, size_t kstates_bytes, void* stream) {
  int64_t Bn, L, H, P, Ds, R;
  M3_TRY(check_scan_inputs(x, B, C, ADT, DT, trap, D, 4, &Bn, &L, &H, &P, &Ds, &R));
  const size_t need = m3_siso_scan_kstates_size(Bn, L, H, P, Ds, x->dtype, B->dtype);
  if (need == 0) return fail(M3_ERR_UNSUPPORTED, "siso scan: no chunk states for this shape / dtype");
  if (kstates == nullptr || kstates_bytes < need || (reinterpret_cast<uintptr_t>(kstates) & 255) != 0)
    return fail(M3_ERR_WORKSPACE, "siso scan: kstates of " + std::to_string(need) + " bytes (256-byte aligned) required");
  const int64_t xs[4] = {Bn, L, H, P}, st[4] = {Bn, H, P, Ds};
  M3_TRY(check(y, "y", 4, xs, 1u << x->dtype, false, false, true));
  M3_TRY(check(h0, "h0", 4, st, kF32, true, true, false));
  M3_TRY(check(bx0, "bx0", 4, st, kF32, true, true, false));
  M3_TRY(check(h_last, "h_last", 4, st, kF32, true, true, false));
  M3_TRY(check(bx_last, "bx_last", 4, st, kF32, true, true, false));
  if (Bn > INT32_MAX || L > INT32_MAX || H > INT32_MAX) return fail(M3_ERR_UNSUPPORTED, "siso scan: dimension too large");
  SisoParams p{};
  p.Bn = (int)Bn; p.L = (int)L; p.H = (int)H; p.P = (int)P; p.D = (int)Ds;
  p.x = x->data; p.sx = s3(x);
  p.Bm = B->data; p.sB = s3(B);
  p.Cm = C->data; p.sC = s3(C);
  p.adt = fptr<const float>(ADT); p.sadt = s3_scal(ADT);
  p.dt = fptr<const float>(DT); p.sdt = s3_scal(DT);
  p.trap = fptr<const float>(trap); p.strap = s3_scal(trap);
  p.Dskip = fptr<const float>(D); p.sD = D->stride[0];
  p.h0 = fptr<const float>(h0); p.bx0 = fptr<const float>(bx0);
  p.y = y->data; p.sy = s3(y);
  p.h_last = fptr<float>(h_last); p.bx_last = fptr<float>(bx_last);
  p.kstates = kstates;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (!siso_chunk_supported(p, x->dtype, B->dtype))
    return fail(M3_ERR_UNSUPPORTED, "siso scan: inputs not eligible for the chunked kernel (alignment / strides)");
  return launch_siso_fwd_chunked(p, x->dtype, B->dtype, s);
}

int m3_siso_scan_bwd_kstates(const m3_tensor* x, const m3_tensor* B, const m3_tensor* C, const m3_tensor* ADT,
                             const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D, const m3_tensor* h0,
                             const m3_tensor* bx0, const m3_tensor* dy, m3_tensor* dx, m3_tensor* dB,
                             m3_tensor* dC, m3_tensor* dADT, m3_tensor* dDT, m3_tensor* dtrap, m3_tensor* dD,
                             m3_tensor* dh0, m3_tensor* dbx0, const void* kstates, size_t kstates_bytes,
                             void* workspace, size_t workspace_bytes, void* stream) {
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  SisoParams p;
  bool done = false;
  M3_TRY(prep_siso_bwd(p, x, B, C, ADT, DT, trap, D, h0, bx0, dy, dx, dB, dC, dADT, dDT, dtrap, dD, dh0, dbx0, s,
                       &done));
  if (done) return M3_OK;
  const size_t kneed = m3_siso_scan_kstates_size(p.Bn, p.L, p.H, p.P, p.D, x->dtype, B->dtype);
  if (kneed == 0 || !siso_chunk_bwd_supported(p, x->dtype, B->dtype))
    return fail(M3_ERR_UNSUPPORTED, "siso backward: inputs not eligible for the chunked kernel");
  if (kstates == nullptr || kstates_bytes < kneed || (reinterpret_cast<uintptr_t>(kstates) & 255) != 0)
    return fail(M3_ERR_INVALID_ARGUMENT, "siso backward: kstates of " + std::to_string(kneed) + " bytes required");
  const size_t need = siso_chunk_bwd_scratch_bytes(p.Bn, p.L, p.H);
  if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)
    return fail(M3_ERR_WORKSPACE, "siso backward: workspace of " + std::to_string(need) + " bytes required");
  p.kstates = const_cast<void*>(kstates);
  return launch_siso_bwd_chunked(p, reinterpret_cast<float*>(workspace), s);
}

// Device address of g_noalloc_scratch, looked up once per device with that device
// current (host code cannot use the symbol itself as a device pointer).
static float* noalloc_scratch_for_current_device() {
  static std::mutex mu;
  static float* addr[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return nullptr;
  }
  std::lock_guard<std::mutex> lock(mu);
  if (!addr[dev]) {
    void* p = nullptr;
    cudaError_t e = cudaGetSymbolAddress(&p, g_noalloc_scratch);
    if (e != cudaSuccess) {
      fail(M3_ERR_CUDA, std::string("cudaGetSymbolAddress(noalloc scratch): ") + cudaGetErrorString(e));
      return nullptr;
    }
    addr[dev] = static_cast<float*>(p);
  }
  return addr[dev];
}

int m3_siso_scan_bwd_noalloc(const m3_tensor* x, const m3_tensor* B, const m3_tensor* C, const m3_tensor* ADT,
                             const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D, const m3_tensor* h0,
                             const m3_tensor* bx0, const m3_tensor* dy, m3_tensor* dx, m3_tensor* dB,
                             m3_tensor* dC, m3_tensor* dADT, m3_tensor* dDT, m3_tensor* dtrap, m3_tensor* dD,
                             m3_tensor* dh0, m3_tensor* dbx0, void* stream) {
  if (!present(x) || x->ndim != 4) return fail(M3_ERR_INVALID_ARGUMENT, "x: expected (B, L, H, P)");
  const int64_t positions = x->shape[0] * x->shape[1] * x->shape[2];
  if (positions > (int64_t)M3_NOALLOC_MAX_POSITIONS)
    return fail(M3_ERR_WORKSPACE, "siso backward (no-alloc): batch*heads*seqlen = " + std::to_string(positions) +
                                      " exceeds the fixed scratch of " + std::to_string(M3_NOALLOC_MAX_POSITIONS) +
                                      " positions; use m3_siso_scan_bwd with a caller workspace");
  float* scratch = nullptr;
  if (positions > 0) {
    scratch = noalloc_scratch_for_current_device();
    if (!scratch) return M3_ERR_CUDA;
  }
  // every position of the scratch that the kernels read is written first in the same call,
  // so nothing needs clearing between calls
  return m3_siso_scan_bwd(x, B, C, ADT, DT, trap, D, h0, bx0, dy, dx, dB, dC, dADT, dDT, dtrap, dD, dh0, dbx0,
                          scratch, sizeof(float) * (size_t)M3_NOALLOC_MAX_POSITIONS, stream);
}

static int fill_mimo(MimoParams& p, const m3_tensor* x, const m3_tensor* B, const m3_tensor* C,
                     const m3_tensor* ADT, const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D,
                     const m3_tensor* mimo_x, const m3_tensor* mimo_o, const m3_tensor* h0,
                     const m3_tensor* bx0, int64_t* dims) {
  int64_t Bn, L, H, P, Ds, R;
  M3_TRY(check_scan_inputs(x, B, C, ADT, DT, trap, D, 5, &Bn, &L, &H, &P, &Ds, &R));
  const int64_t ms[3] = {H, R, P}, st[3] = {Bn, H, Ds};
  M3_TRY(check(mimo_x, "mimo_x", 3, ms, kF32, false, false, false));
  M3_TRY(check(mimo_o, "mimo_o", 3, ms, kF32, false, false, false));
  M3_TRY(check(h0, "h0", 3, st, kF32, true, true, false));
  M3_TRY(check(bx0, "bx0", 3, st, kF32, true, true, false));
  if (Bn > INT32_MAX || L > INT32_MAX || H > INT32_MAX || P > 65535 || R > 8)
    return fail(M3_ERR_UNSUPPORTED, "mimo scan: dimension too large (rank must be <= 8)");
  p.Bn = (int)Bn; p.L = (int)L; p.H = (int)H; p.P = (int)P; p.D = (int)Ds; p.R = (int)R;
  p.x = x->data; p.sx = s3(x);
  p.Bm = B->data; p.sB = s4(B);
  p.Cm = C->data; p.sC = s4(C);
  p.adt = fptr<const float>(ADT); p.sadt = s3_scal(ADT);
  p.dt = fptr<const float>(DT); p.sdt = s3_scal(DT);
  p.trap = fptr<const float>(trap); p.strap = s3_scal(trap);
  p.Dskip = fptr<const float>(D); p.sD = D->stride[0];
  p.mimo_x = fptr<const float>(mimo_x); p.smx_h = mimo_x->stride[0]; p.smx_r = mimo_x->stride[1];
  p.mimo_o = fptr<const float>(mimo_o); p.smo_h = mimo_o->stride[0]; p.smo_r = mimo_o->stride[1];
  p.h0 = fptr<const float>(h0); p.bx0 = fptr<const float>(bx0);
  dims[0] = Bn; dims[1] = L; dims[2] = H; dims[3] = P; dims[4] = Ds; dims[5] = R;
  return M3_OK;
}

int m3_mimo_scan_fwd(const m3_tensor* x, const m3_tensor* B, const m3_tensor* C, const m3_tensor* ADT,
                     const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D, const m3_tensor* mimo_x,
                     const m3_tensor* mimo_o, const m3_tensor* h0, const m3_tensor* bx0, m3_tensor* y,
                     m3_tensor* h_last, m3_tensor* bx_last, void* stream) {
  MimoParams p{};
  int64_t d[6];
  M3_TRY(fill_mimo(p, x, B, C, ADT, DT, trap, D, mimo_x, mimo_o, h0, bx0, d));
  const int64_t xs[4] = {d[0], d[1], d[2], d[3]}, st[3] = {d[0], d[2], d[4]};
  const bool empty = d[0] * d[1] * d[2] * d[3] == 0;
  M3_TRY(check(y, "y", 4, xs, 1u << x->dtype, false, false, !empty));
  M3_TRY(check(h_last, "h_last", 3, st, kF32, true, true, false));
  M3_TRY(check(bx_last, "bx_last", 3, st, kF32, true, true, false));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (d[0] * d[2] * d[4] == 0) return M3_OK;
  if (d[1] == 0 || d[3] == 0) {
    const size_t bytes = sizeof(float) * d[0] * d[2] * d[4];
    if (d[1] == 0) {
      M3_TRY(copy_or_zero(fptr<void>(h_last), fptr<void>(h0), bytes, s, "h_last"));
      return copy_or_zero(fptr<void>(bx_last), fptr<void>(bx0), bytes, s, "bx_last");
    }
  }
  p.y = y->data; p.sy = s3(y);
  p.h_last = fptr<float>(h_last); p.bx_last = fptr<float>(bx_last);
  return launch_mimo(p, x->dtype, B->dtype, false, s);
}

size_t m3_mimo_scan_fwd_workspace_size(int64_t batch, int64_t seqlen, int64_t nheads, int64_t dstate) {
  if (batch < 0 || seqlen < 0 || nheads < 0 || dstate < 0) return 0;
  return mimo_fwd_workspace_bytes(batch, seqlen, nheads, dstate);
}

int m3_mimo_scan_fwd_ws(const m3_tensor* x, const m3_tensor* B, const m3_tensor* C, const m3_tensor* ADT,
                        const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D, const m3_tensor* mimo_x,
                        const m3_tensor* mimo_o, const m3_tensor* h0, const m3_tensor* bx0, m3_tensor* y,
                        m3_tensor* h_last, m3_tensor* bx_last, void* workspace, size_t workspace_bytes,
                        void* stream) {
  MimoParams p{};
  int64_t d[6];
  M3_TRY(fill_mimo(p, x, B, C, ADT, DT, trap, D, mimo_x, mimo_o, h0, bx0, d));
  const int64_t xs[4] = {d[0], d[1], d[2], d[3]}, st[3] = {d[0], d[2], d[4]};
  const bool empty = d[0] * d[1] * d[2] * d[3] == 0;
  M3_TRY(check(y, "y", 4, xs, 1u << x->dtype, false, false, !empty));
  M3_TRY(check(h_last, "h_last", 3, st, kF32, true, true, false));
  M3_TRY(check(bx_last, "bx_last", 3, st, kF32, true, true, false));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (d[0] * d[2] * d[4] == 0) return M3_OK;
  if (d[1] == 0 || d[3] == 0) {
    const size_t bytes = sizeof(float) * d[0] * d[2] * d[4];
    if (d[1] == 0) {
      M3_TRY(copy_or_zero(fptr<void>(h_last), fptr<void>(h0), bytes, s, "h_last"));
      return copy_or_zero(fptr<void>(bx_last), fptr<void>(bx0), bytes, s, "bx_last");
    }
  }
  const size_t need = mimo_fwd_workspace_bytes(d[0], d[1], d[2], d[4]);
  if (!workspace || workspace_bytes < need)
    return fail(M3_ERR_WORKSPACE, "workspace: need " + std::to_string(need) + " bytes");
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(M3_ERR_INVALID_ARGUMENT, "workspace: not 16-byte aligned");
  M3_TRY(check_device_ptr(workspace, "workspace"));
  p.y = y->data; p.sy = s3(y);
  p.h_last = fptr<float>(h_last); p.bx_last = fptr<float>(bx_last);
  return launch_mimo_fwd_chunked(p, x->dtype, B->dtype, workspace, s);
}

size_t m3_mimo_scan_bwd_workspace_size(int64_t batch, int64_t seqlen, int64_t nheads, int64_t headdim,
                                       int64_t dstate, int64_t rank) {
  return sizeof(float) * mimo_bwd_workspace_floats(batch, seqlen, nheads, headdim, dstate, rank);
}

static int mimo_bwd_common(const m3_tensor* x, const m3_tensor* B, const m3_tensor* C, const m3_tensor* ADT,
                           const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D, const m3_tensor* mimo_x,
                           const m3_tensor* mimo_o, const m3_tensor* h0, const m3_tensor* bx0, const m3_tensor* dy,
                           m3_tensor* dx, m3_tensor* dB, m3_tensor* dC, m3_tensor* dADT, m3_tensor* dDT,
                           m3_tensor* dtrap, m3_tensor* dD, m3_tensor* dmimo_x, m3_tensor* dmimo_o, m3_tensor* dh0,
                           m3_tensor* dbx0, const void* fwd_workspace, size_t fwd_workspace_bytes, void* workspace,
                           size_t workspace_bytes, void* stream) {
  MimoParams p{};
  int64_t d[6];
  M3_TRY(fill_mimo(p, x, B, C, ADT, DT, trap, D, mimo_x, mimo_o, h0, bx0, d));
  const int64_t Bn = d[0], L = d[1], H = d[2], P = d[3], Ds = d[4], R = d[5];
  const bool empty = Bn * L * H * P == 0;
  const int64_t xs[4] = {Bn, L, H, P}, bs[5] = {Bn, L, R, H, Ds}, ss[3] = {Bn, L, H}, hs[1] = {H},
                ms[3] = {H, R, P}, st[3] = {Bn, H, Ds};
  M3_TRY(check(dy, "dy", 4, xs, 1u << x->dtype, false, false, !empty));
  M3_TRY(check(dx, "dx", 4, xs, 1u << x->dtype, false, false, !empty));
  M3_TRY(check(dB, "dB", 5, bs, 1u << B->dtype, false, false, !empty));
  M3_TRY(check(dC, "dC", 5, bs, 1u << B->dtype, false, false, !empty));
  M3_TRY(check(dADT, "dADT", 3, ss, kF32, false, false, false));
  M3_TRY(check(dDT, "dDT", 3, ss, kF32, false, false, false));
  M3_TRY(check(dtrap, "dtrap", 3, ss, kF32, false, false, false));
  M3_TRY(check(dD, "dD", 1, hs, kF32, true, false, false));
  M3_TRY(check(dmimo_x, "dmimo_x", 3, ms, kF32, true, false, false));
  M3_TRY(check(dmimo_o, "dmimo_o", 3, ms, kF32, true, false, false));
  M3_TRY(check(dh0, "dh0", 3, st, kF32, true, true, false));
  M3_TRY(check(dbx0, "dbx0", 3, st, kF32, true, true, false));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  M3_TRY(memset_async(dD->data, sizeof(float) * H, s, "dD"));
  M3_TRY(memset_async(dmimo_x->data, sizeof(float) * H * R * P, s, "dmimo_x"));
  M3_TRY(memset_async(dmimo_o->data, sizeof(float) * H * R * P, s, "dmimo_o"));
  if (Bn * H * Ds == 0) return M3_OK;
  if (L == 0) {
    const size_t bytes = sizeof(float) * Bn * H * Ds;
    M3_TRY(copy_or_zero(fptr<void>(dh0), nullptr, bytes, s, "dh0"));
    return copy_or_zero(fptr<void>(dbx0), nullptr, bytes, s, "dbx0");
  }
  if (workspace && reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return fail(M3_ERR_INVALID_ARGUMENT, "mimo backward: workspace not 16-byte aligned");
  if (fwd_workspace && reinterpret_cast<uintptr_t>(fwd_workspace) % 16 != 0)
    return fail(M3_ERR_INVALID_ARGUMENT, "mimo backward: forward workspace not 16-byte aligned");
  p.dy = dy->data; p.sdy = s3(dy);
  p.dx = dx->data; p.sdx = s3(dx);
  p.dB = dB->data; p.sdB = s4(dB);
  p.dC = dC->data; p.sdC = s4(dC);
  p.dadt = fptr<float>(dADT); p.sdadt = s3_scal(dADT);
  p.ddt = fptr<float>(dDT); p.sddt = s3_scal(dDT);
  p.dtrap = fptr<float>(dtrap); p.sdtrap = s3_scal(dtrap);
  p.dD = fptr<float>(dD);
  p.dmx = fptr<float>(dmimo_x); p.dmo = fptr<float>(dmimo_o);
  p.dh0 = fptr<float>(dh0); p.dbx0 = fptr<float>(dbx0);
  if (fwd_workspace) {
    M3_TRY(check_device_ptr(fwd_workspace, "fwd_workspace"));
    const int rc = launch_mimo_bwd_fused(p, x->dtype, B->dtype, fwd_workspace, fwd_workspace_bytes, workspace,
                                         workspace_bytes, s);
    if (rc != M3_ERR_UNSUPPORTED) return rc;
  }
  const size_t need = m3_mimo_scan_bwd_workspace_size(Bn, L, H, P, Ds, R);
  if (need == 0) return fail(M3_ERR_UNSUPPORTED, "mimo backward: shapes too large for shared memory");
  if (workspace == nullptr || workspace_bytes < need)
    return fail(M3_ERR_WORKSPACE, "mimo backward: workspace of " + std::to_string(need) + " bytes required");
  p.work = reinterpret_cast<float*>(workspace);
  return launch_mimo(p, x->dtype, B->dtype, true, s);
}

int m3_mimo_scan_bwd(const m3_tensor* x, const m3_tensor* B, const m3_tensor* C, const m3_tensor* ADT,
                     const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D, const m3_tensor* mimo_x,
                     const m3_tensor* mimo_o, const m3_tensor* h0, const m3_tensor* bx0, const m3_tensor* dy,
                     m3_tensor* dx, m3_tensor* dB, m3_tensor* dC, m3_tensor* dADT, m3_tensor* dDT,
                     m3_tensor* dtrap, m3_tensor* dD, m3_tensor* dmimo_x, m3_tensor* dmimo_o, m3_tensor* dh0,
                     m3_tensor* dbx0, void* workspace, size_t workspace_bytes, void* stream) {
  return mimo_bwd_common(x, B, C, ADT, DT, trap, D, mimo_x, mimo_o, h0, bx0, dy, dx, dB, dC, dADT, dDT, dtrap, dD,
                         dmimo_x, dmimo_o, dh0, dbx0, nullptr, 0, workspace, workspace_bytes, stream);
}

size_t m3_mimo_scan_bwd_ws_workspace_size(int64_t batch, int64_t seqlen, int64_t nheads, int64_t headdim,
                                          int64_t dstate, int64_t rank) {
  if (batch < 0 || seqlen < 0 || nheads < 0 || headdim < 0 || dstate < 0 || rank < 0) return 0;
  return std::max(m3_mimo_scan_bwd_workspace_size(batch, seqlen, nheads, headdim, dstate, rank),
                  mimo_bwd_fused_workspace_bytes(batch, seqlen, nheads, dstate));
}

int m3_mimo_scan_bwd_ws(const m3_tensor* x, const m3_tensor* B, const m3_tensor* C, const m3_tensor* ADT,
                        const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* D, const m3_tensor* mimo_x,
                        const m3_tensor* mimo_o, const m3_tensor* h0, const m3_tensor* bx0, const m3_tensor* dy,
                        m3_tensor* dx, m3_tensor* dB, m3_tensor* dC, m3_tensor* dADT, m3_tensor* dDT,
                        m3_tensor* dtrap, m3_tensor* dD, m3_tensor* dmimo_x, m3_tensor* dmimo_o, m3_tensor* dh0,
                        m3_tensor* dbx0, const void* fwd_workspace, size_t fwd_workspace_bytes, void* workspace,
                        size_t workspace_bytes, void* stream) {
  return mimo_bwd_common(x, B, C, ADT, DT, trap, D, mimo_x, mimo_o, h0, bx0, dy, dx, dB, dC, dADT, dDT, dtrap, dD,
                         dmimo_x, dmimo_o, dh0, dbx0, fwd_workspace, fwd_workspace_bytes, workspace, workspace_bytes,
                         stream);
}

static int step_common(bool mimo, const m3_layer_dims* dims, const m3_tensor* zxbcdt, const m3_tensor* dt_bias,
                       const m3_tensor* B_bias, const m3_tensor* C_bias, const m3_tensor* B_norm_w,
                       const m3_tensor* C_norm_w, const m3_tensor* Dskip, const m3_tensor* mimo_x,
                       const m3_tensor* mimo_o, const m3_tensor* angle_in, const m3_tensor* ssm_in,
                       const m3_tensor* bx_in, m3_tensor* angle_out, m3_tensor* ssm_out, m3_tensor* bx_out,
                       m3_tensor* y_gated, void* stream) {
  if (!dims) return fail(M3_ERR_INVALID_ARGUMENT, "dims: missing");
  const int64_t H = dims->nheads, P = dims->headdim, Ds = dims->d_state, G = dims->ngroups,
                R = mimo ? dims->mimo_rank : 1, S = dims->num_rope_angles, di = dims->d_inner;
  if (H <= 0 || P <= 0 || Ds <= 0 || G <= 0 || R <= 0 || S < 0 || di != H * P || dims->rope_split != 2 * S ||
      dims->rope_split > Ds || (G != 1 && G != H))
    return fail(M3_ERR_INVALID_ARGUMENT, "dims: inconsistent layer dimensions");
  if (!mimo && dims->mimo_rank != 1) return fail(M3_ERR_INVALID_ARGUMENT, "dims: SISO step needs mimo_rank 1");
  if (!present(zxbcdt) || zxbcdt->ndim != 2) return fail(M3_ERR_INVALID_ARGUMENT, "zxbcdt: expected (batch, d_in_proj)");
  const int64_t Bn = zxbcdt->shape[0];
  const int64_t dproj = 2 * di + 2 * Ds * G * R + 3 * H + S;
  const int64_t zs[2] = {Bn, dproj}, ys[2] = {Bn, di}, h1[1] = {H}, hrd[3] = {H, R, Ds}, d1[1] = {Ds},
                hrp[3] = {H, R, P}, as[3] = {Bn, H, S};
  M3_TRY(check(zxbcdt, "zxbcdt", 2, zs, kAnyFloat, false, false, Bn > 0));
  M3_TRY(check(y_gated, "y_gated", 2, ys, 1u << zxbcdt->dtype, false, false, false));
  M3_TRY(check(dt_bias, "dt_bias", 1, h1, kF32, true, false, false));
  M3_TRY(check(B_bias, "B_bias", 3, hrd, kF32, true, false, false));
  M3_TRY(check(C_bias, "C_bias", 3, hrd, kF32, true, false, false));
  M3_TRY(check(B_norm_w, "B_norm_w", 1, d1, kF32, true, false, false));
  M3_TRY(check(C_norm_w, "C_norm_w", 1, d1, kF32, true, false, false));
  M3_TRY(check(Dskip, "D", 1, h1, kF32, true, false, false));
  if (mimo) {
    M3_TRY(check(mimo_x, "mimo_x", 3, hrp, kF32, true, false, false));
    M3_TRY(check(mimo_o, "mimo_o", 3, hrp, kF32, true, false, false));
  }
  if (S > 0) {
    M3_TRY(check(angle_in, "angle_in", 3, as, kF32, true, false, false));
    M3_TRY(check(angle_out, "angle_out", 3, as, kF32, true, false, false));
  }
  if (mimo) {
    const int64_t st[3] = {Bn, H, Ds};
    M3_TRY(check(ssm_in, "ssm_in", 3, st, kF32, true, false, false));
    M3_TRY(check(bx_in, "bx_in", 3, st, kF32, true, false, false));
    M3_TRY(check(ssm_out, "ssm_out", 3, st, kF32, true, false, false));
    M3_TRY(check(bx_out, "bx_out", 3, st, kF32, true, false, false));
  } else {
    const int64_t st[4] = {Bn, H, P, Ds};
    M3_TRY(check(ssm_in, "ssm_in", 4, st, kF32, true, false, false));
    M3_TRY(check(bx_in, "bx_in", 4, st, kF32, true, false, false));
    M3_TRY(check(ssm_out, "ssm_out", 4, st, kF32, true, false, false));
    M3_TRY(check(bx_out, "bx_out", 4, st, kF32, true, false, false));
  }
  if (Bn == 0) return M3_OK;
  if (!mimo) {
    for (const m3_tensor* t : {ssm_in, bx_in, (const m3_tensor*)ssm_out, (const m3_tensor*)bx_out})
      if (reinterpret_cast<uintptr_t>(t->data) % 16 != 0)
        return fail(M3_ERR_INVALID_ARGUMENT, "siso step: state buffers must be 16-byte aligned");
  }
  StepParams p{};
  p.Bn = (int)Bn; p.H = (int)H; p.P = (int)P; p.D = (int)Ds; p.R = (int)R; p.G = (int)G; p.S = (int)S;
  p.split = dims->rope_split; p.d_inner = (int)di; p.A_floor = dims->A_floor; p.eps = dims->norm_eps;
  p.zxbcdt = zxbcdt->data; p.s_row = zxbcdt->stride[0];
  p.dt_bias = fptr<const float>(dt_bias);
  p.B_bias = fptr<const float>(B_bias); p.C_bias = fptr<const float>(C_bias);
  p.B_norm_w = fptr<const float>(B_norm_w); p.C_norm_w = fptr<const float>(C_norm_w);
  p.Dskip = fptr<const float>(Dskip);
  p.mimo_x = mimo ? fptr<const float>(mimo_x) : nullptr;
  p.mimo_o = mimo ? fptr<const float>(mimo_o) : nullptr;
  p.angle_in = S > 0 ? fptr<const float>(angle_in) : nullptr;
  p.angle_out = S > 0 ? fptr<float>(angle_out) : nullptr;
  p.ssm_in = fptr<const float>(ssm_in); p.ssm_out = fptr<float>(ssm_out);
  p.bx_in = fptr<const float>(bx_in); p.bx_out = fptr<float>(bx_out);
  p.y = y_gated->data; p.s_y = y_gated->stride[0];
  return launch_step(p, zxbcdt->dtype, mimo, reinterpret_cast<cudaStream_t>(stream));
}

int m3_siso_step(const m3_layer_dims* dims, const m3_tensor* zxbcdt, const m3_tensor* dt_bias, const m3_tensor* B_bias,
                 const m3_tensor* C_bias, const m3_tensor* B_norm_w, const m3_tensor* C_norm_w, const m3_tensor* Dskip,
                 const m3_tensor* angle_in, const m3_tensor* ssm_in, const m3_tensor* bx_in, m3_tensor* angle_out,
                 m3_tensor* ssm_out, m3_tensor* bx_out, m3_tensor* y_gated, void* stream) {
  return step_common(false, dims, zxbcdt, dt_bias, B_bias, C_bias, B_norm_w, C_norm_w, Dskip, nullptr, nullptr,
                     angle_in, ssm_in, bx_in, angle_out, ssm_out, bx_out, y_gated, stream);
}

int m3_mimo_step(const m3_layer_dims* dims, const m3_tensor* zxbcdt, const m3_tensor* dt_bias, const m3_tensor* B_bias,
                 const m3_tensor* C_bias, const m3_tensor* B_norm_w, const m3_tensor* C_norm_w, const m3_tensor* Dskip,
                 const m3_tensor* mimo_x, const m3_tensor* mimo_o, const m3_tensor* angle_in, const m3_tensor* ssm_in,
                 const m3_tensor* bx_in, m3_tensor* angle_out, m3_tensor* ssm_out, m3_tensor* bx_out,
                 m3_tensor* y_gated, void* stream) {
  return step_common(true, dims, zxbcdt, dt_bias, B_bias, C_bias, B_norm_w, C_norm_w, Dskip, mimo_x, mimo_o,
                     angle_in, ssm_in, bx_in, angle_out, ssm_out, bx_out, y_gated, stream);
}


int m3_rmsnorm(const m3_tensor* x, const m3_tensor* residual, const m3_tensor* weight, float eps,
               m3_tensor* out, m3_tensor* residual_out, void* stream) {
  if (!present(x) || x->ndim < 1) return fail(M3_ERR_INVALID_ARGUMENT, "x: missing or 0-d");
  const int nd = x->ndim;
  const int64_t d = x->shape[nd - 1];
  int64_t rows = 1;
  for (int i = 0; i < nd - 1; ++i) rows *= x->shape[i];
  const bool empty = rows * d == 0;
  // every operand: (..., d) whose leading dims collapse into rows of one stride
  auto rows_of = [&](const m3_tensor* t, const char* name, bool optional, unsigned mask, int64_t* srow) -> int {
    if (!present(t)) {
      if (optional) return M3_OK;
      return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": missing");
    }
    M3_TRY(check(t, name, nd, x->shape, mask, false, false, !empty));
    if (empty) return M3_OK;
    for (int i = 0; i + 2 < nd; ++i)
      if (t->shape[i] > 1 && t->stride[i] != t->stride[i + 1] * t->shape[i + 1])
        return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": leading dims must collapse into rows");
    *srow = nd >= 2 ? t->stride[nd - 2] : d;
    return M3_OK;
  };
  NormParams p{};
  p.rows = rows; p.d = d; p.eps = eps;
  M3_TRY(rows_of(x, "x", false, kAnyFloat, &p.sx));
  M3_TRY(rows_of(residual, "residual", true, 1u << x->dtype, &p.sres));
  M3_TRY(rows_of(out, "out", false, 1u << x->dtype, &p.sout));
  M3_TRY(rows_of(residual_out, "residual_out", true, 1u << x->dtype, &p.shout));
  const int64_t ws[1] = {d};
  M3_TRY(check(weight, "weight", 1, ws, kAnyFloat, true, false, !empty));
  if (present(residual_out) && !present(residual))
    return fail(M3_ERR_INVALID_ARGUMENT, "residual_out: given without residual");
  if (present(residual_out) && present(out) && residual_out->data == out->data && !empty)
    return fail(M3_ERR_INVALID_ARGUMENT, "out: must not alias residual_out");
  p.x = x->data; p.res = present(residual) ? residual->data : nullptr;
  p.w = weight->data; p.out = out->data; p.hout = present(residual_out) ? residual_out->data : nullptr;
  return launch_rmsnorm(p, x->dtype, weight->dtype, reinterpret_cast<cudaStream_t>(stream));
}


int m3_argmax_rows(const m3_tensor* logits, m3_tensor* out, void* stream) {
  if (!present(logits) || logits->ndim < 1) return fail(M3_ERR_INVALID_ARGUMENT, "logits: missing or 0-d");
  if (!present(out)) return fail(M3_ERR_INVALID_ARGUMENT, "out: missing");
  const int nd = logits->ndim;
  const int64_t n = logits->shape[nd - 1];
  int64_t rows = 1;
  for (int i = 0; i < nd - 1; ++i) rows *= logits->shape[i];
  M3_TRY(check(logits, "logits", nd, logits->shape, kAnyFloat, false, false, rows * n > 0));
  if (n <= 0 && rows > 0) return fail(M3_ERR_INVALID_ARGUMENT, "logits: empty last dimension");
  for (int i = 0; i + 2 < nd; ++i)
    if (logits->shape[i] > 1 && logits->stride[i] != logits->stride[i + 1] * logits->shape[i + 1])
      return fail(M3_ERR_INVALID_ARGUMENT, "logits: leading dims must collapse into rows");
  if (out->dtype != M3_INT64) return fail(M3_ERR_INVALID_ARGUMENT, "out: expected int64");
  int64_t on = 1, expect = 1;
  for (int i = out->ndim - 1; i >= 0; --i) {
    if (out->shape[i] > 1 && out->stride[i] != expect)
      return fail(M3_ERR_INVALID_ARGUMENT, "out: must be contiguous");
    expect *= out->shape[i];
    on *= out->shape[i];
  }
  if (on != rows) return fail(M3_ERR_INVALID_ARGUMENT, "out: one element per logits row expected");
  if (rows == 0) return M3_OK;
  M3_TRY(check_device_ptr(out->data, "out"));
  const int64_t sx = nd >= 2 ? logits->stride[nd - 2] : n;
  return launch_argmax_rows(logits->data, logits->dtype, rows, n, sx, static_cast<int64_t*>(out->data),
                            reinterpret_cast<cudaStream_t>(stream));
}

int m3_device_timeouts(int reset, int* flag_out) {
  if (!flag_out) return fail(M3_ERR_INVALID_ARGUMENT, "flag_out: missing");
  int f = 0, b = 0, m = 0, q = 0, t = 0;
  M3_TRY(chunk_error_word(reset != 0, &f));
  M3_TRY(chunk_bwd_error_word(reset != 0, &b));
  M3_TRY(mimo_error_word(reset != 0, &m));
  M3_TRY(prologue_error_word(reset != 0, &q));
  M3_TRY(token_error_word(reset != 0, &t));
  *flag_out = f | b | m | q | t;
  return M3_OK;
}


int m3_layer_prologue(const m3_layer_dims* dims, const m3_tensor* zxbcdt, const m3_tensor* dt_bias,
                      const m3_tensor* B_bias, const m3_tensor* C_bias, const m3_tensor* B_norm_w,
                      const m3_tensor* C_norm_w, const m3_tensor* angle0, m3_tensor* B_proj, m3_tensor* C_proj,
                      m3_tensor* ADT, m3_tensor* DT, m3_tensor* trap, m3_tensor* angles, void* stream) {
  if (!dims) return fail(M3_ERR_INVALID_ARGUMENT, "dims: missing");
  const int64_t H = dims->nheads, P = dims->headdim, Ds = dims->d_state, G = dims->ngroups,
                R = dims->mimo_rank, S = dims->num_rope_angles, di = dims->d_inner;
  if (H <= 0 || P <= 0 || Ds <= 0 || G <= 0 || R <= 0 || S < 0 || di != H * P || dims->rope_split != 2 * S ||
      dims->rope_split > Ds || (G != 1 && G != H))
    return fail(M3_ERR_INVALID_ARGUMENT, "dims: inconsistent layer dimensions");
  if (!present(zxbcdt) || zxbcdt->ndim != 3) return fail(M3_ERR_INVALID_ARGUMENT, "zxbcdt: expected (batch, seqlen, d_in_proj)");
  const int64_t Bn = zxbcdt->shape[0], L = zxbcdt->shape[1];
  const int64_t dproj = 2 * di + 2 * Ds * G * R + 3 * H + S;
  const bool empty = Bn * L == 0;
  const int64_t zs[3] = {Bn, L, dproj}, bs[5] = {Bn, L, R, H, Ds}, ss[3] = {Bn, L, H}, as[4] = {Bn, L, H, S},
                h1[1] = {H}, hrd[3] = {H, R, Ds}, d1[1] = {Ds};
  M3_TRY(check(zxbcdt, "zxbcdt", 3, zs, kAnyFloat, false, false, !empty));
  // B_proj and C_proj: both present, or both absent (angles and step scalars only)
  const bool with_bc = present(B_proj) || present(C_proj);
  if (with_bc) {
    M3_TRY(check(B_proj, "B_proj", 5, bs, kAnyFloat, true, false, !empty));
    M3_TRY(check(C_proj, "C_proj", 5, bs, 1u << B_proj->dtype, true, false, !empty));
  }
  M3_TRY(check(ADT, "ADT", 3, ss, kF32, true, false, false));
  M3_TRY(check(DT, "DT", 3, ss, kF32, true, false, false));
  M3_TRY(check(trap, "trap", 3, ss, kF32, true, false, false));
  M3_TRY(check(angles, "angles", 4, as, kF32, true, S == 0, false));
  M3_TRY(check(dt_bias, "dt_bias", 1, h1, kF32, true, false, false));
  M3_TRY(check(B_bias, "B_bias", 3, hrd, kF32, true, false, false));
  M3_TRY(check(C_bias, "C_bias", 3, hrd, kF32, true, false, false));
  M3_TRY(check(B_norm_w, "B_norm_w", 1, d1, kF32, true, false, false));
  M3_TRY(check(C_norm_w, "C_norm_w", 1, d1, kF32, true, false, false));
  const int64_t a0s[3] = {Bn, H, S};
  M3_TRY(check(angle0, "angle0", 3, a0s, kF32, true, true, false));
  if (empty) return M3_OK;
  if (Bn > INT32_MAX || L > INT32_MAX) return fail(M3_ERR_UNSUPPORTED, "prologue: dimension too large");
  PrologueParams p{};
  p.Bn = (int)Bn; p.L = (int)L; p.H = (int)H; p.P = (int)P; p.D = (int)Ds; p.R = (int)R; p.G = (int)G;
  p.S = (int)S; p.split = dims->rope_split; p.d_inner = (int)di; p.A_floor = dims->A_floor; p.eps = dims->norm_eps;
  p.zx = zxbcdt->data; p.s_zb = zxbcdt->stride[0]; p.s_zl = zxbcdt->stride[1];
  p.dt_bias = fptr<const float>(dt_bias);
  p.B_bias = fptr<const float>(B_bias); p.C_bias = fptr<const float>(C_bias);
  p.B_norm_w = fptr<const float>(B_norm_w); p.C_norm_w = fptr<const float>(C_norm_w);
  p.Bp = with_bc ? B_proj->data : nullptr;
  p.Cp = with_bc ? C_proj->data : nullptr;
  p.ADT = fptr<float>(ADT); p.DT = fptr<float>(DT); p.trap = fptr<float>(trap); p.angles = fptr<float>(angles);
  p.angle0 = S > 0 ? fptr<const float>(angle0) : nullptr;
  return launch_prologue(p, zxbcdt->dtype, with_bc ? B_proj->dtype : zxbcdt->dtype,
                         reinterpret_cast<cudaStream_t>(stream));
}

int m3_mimo_layer_scan_fwd(const m3_layer_dims* dims, const m3_tensor* zxbcdt, const m3_tensor* ADT,
                           const m3_tensor* DT, const m3_tensor* trap, const m3_tensor* angles,
                           const m3_tensor* B_bias, const m3_tensor* C_bias, const m3_tensor* B_norm_w,
                           const m3_tensor* C_norm_w, const m3_tensor* D, const m3_tensor* mimo_x,
                           const m3_tensor* mimo_o, const m3_tensor* h0, const m3_tensor* bx0, int32_t gate,
                           m3_tensor* out, m3_tensor* h_last, m3_tensor* bx_last, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (!dims) return fail(M3_ERR_INVALID_ARGUMENT, "dims: missing");
  const int64_t H = dims->nheads, P = dims->headdim, Ds = dims->d_state, G = dims->ngroups,
                R = dims->mimo_rank, S = dims->num_rope_angles, di = dims->d_inner;
  if (H <= 0 || P <= 0 || Ds <= 0 || G <= 0 || R <= 0 || S < 0 || di != H * P || dims->rope_split != 2 * S ||
      dims->rope_split > Ds || (G != 1 && G != H))
    return fail(M3_ERR_INVALID_ARGUMENT, "dims: inconsistent layer dimensions");
  if (gate != 0 && gate != 1) return fail(M3_ERR_INVALID_ARGUMENT, "gate: must be 0 or 1");
  if (!present(zxbcdt) || zxbcdt->ndim != 3) return fail(M3_ERR_INVALID_ARGUMENT, "zxbcdt: expected (batch, seqlen, d_in_proj)");
  const int64_t Bn = zxbcdt->shape[0], L = zxbcdt->shape[1];
  const int64_t dproj = 2 * di + 2 * Ds * G * R + 3 * H + S;
  const bool empty = Bn * L == 0;
  const int64_t zs[3] = {Bn, L, dproj}, ss[3] = {Bn, L, H}, as[4] = {Bn, L, H, S}, h1[1] = {H},
                hrd[3] = {H, R, Ds}, d1[1] = {Ds}, ms[3] = {H, R, P}, st[3] = {Bn, H, Ds}, ys[4] = {Bn, L, H, P};
  M3_TRY(check(zxbcdt, "zxbcdt", 3, zs, kAnyFloat, false, false, !empty));
  M3_TRY(check(ADT, "ADT", 3, ss, kF32, false, false, false));
  M3_TRY(check(DT, "DT", 3, ss, kF32, false, false, false));
  M3_TRY(check(trap, "trap", 3, ss, kF32, false, false, false));
  M3_TRY(check(angles, "angles", 4, as, kF32, true, S == 0, false));
  M3_TRY(check(B_bias, "B_bias", 3, hrd, kF32, true, false, false));
  M3_TRY(check(C_bias, "C_bias", 3, hrd, kF32, true, false, false));
  M3_TRY(check(B_norm_w, "B_norm_w", 1, d1, kF32, true, false, false));
  M3_TRY(check(C_norm_w, "C_norm_w", 1, d1, kF32, true, false, false));
  M3_TRY(check(D, "D", 1, h1, kF32, false, false, false));
  M3_TRY(check(mimo_x, "mimo_x", 3, ms, kF32, false, false, false));
  M3_TRY(check(mimo_o, "mimo_o", 3, ms, kF32, false, false, false));
  M3_TRY(check(h0, "h0", 3, st, kF32, true, true, false));
  M3_TRY(check(bx0, "bx0", 3, st, kF32, true, true, false));
  M3_TRY(check(out, "out", 4, ys, 1u << zxbcdt->dtype, false, false, !empty));
  M3_TRY(check(h_last, "h_last", 3, st, kF32, true, true, false));
  M3_TRY(check(bx_last, "bx_last", 3, st, kF32, true, true, false));
  if (G != 1) return fail(M3_ERR_UNSUPPORTED, "mimo layer scan: one B / C group only");
  if (Bn > INT32_MAX || L > INT32_MAX || H > INT32_MAX || P > 65535 || R > 8)
    return fail(M3_ERR_UNSUPPORTED, "mimo layer scan: dimension too large (rank must be <= 8)");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (Bn * H * Ds == 0) return M3_OK;
  if (L == 0) {
    const size_t bytes = sizeof(float) * Bn * H * Ds;
    M3_TRY(copy_or_zero(fptr<void>(h_last), fptr<void>(h0), bytes, s, "h_last"));
    return copy_or_zero(fptr<void>(bx_last), fptr<void>(bx0), bytes, s, "bx_last");
  }
  const size_t need = mimo_fwd_workspace_bytes(Bn, L, H, Ds);
  if (!workspace || workspace_bytes < need)
    return fail(M3_ERR_WORKSPACE, "workspace: need " + std::to_string(need) + " bytes");
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(M3_ERR_INVALID_ARGUMENT, "workspace: not 16-byte aligned");
  M3_TRY(check_device_ptr(workspace, "workspace"));
  MimoParams p{};
  p.Bn = (int)Bn; p.L = (int)L; p.H = (int)H; p.P = (int)P; p.D = (int)Ds; p.R = (int)R;
  p.adt = fptr<const float>(ADT); p.sadt = s3_scal(ADT);
  p.dt = fptr<const float>(DT); p.sdt = s3_scal(DT);
  p.trap = fptr<const float>(trap); p.strap = s3_scal(trap);
  p.Dskip = fptr<const float>(D); p.sD = D->stride[0];
  p.mimo_x = fptr<const float>(mimo_x); p.smx_h = mimo_x->stride[0]; p.smx_r = mimo_x->stride[1];
  p.mimo_o = fptr<const float>(mimo_o); p.smo_h = mimo_o->stride[0]; p.smo_r = mimo_o->stride[1];
  p.h0 = fptr<const float>(h0); p.bx0 = fptr<const float>(bx0);
  p.y = out->data; p.sy = s3(out);
  p.h_last = fptr<float>(h_last); p.bx_last = fptr<float>(bx_last);
  MimoGrpParams q{};
  q.zx = zxbcdt->data; q.s_zb = zxbcdt->stride[0]; q.s_zl = zxbcdt->stride[1];
  q.dtype = zxbcdt->dtype;
  q.angles = S > 0 ? fptr<const float>(angles) : nullptr;
  q.B_bias = fptr<const float>(B_bias); q.C_bias = fptr<const float>(C_bias);
  q.B_norm_w = fptr<const float>(B_norm_w); q.C_norm_w = fptr<const float>(C_norm_w);
  q.eps = dims->norm_eps;
  q.S = (int)S;
  q.gate = gate;
  return launch_mimo_layer_fwd(p, q, workspace, s);
}

size_t m3_layer_prologue_bwd_workspace_size(const m3_layer_dims* dims, int64_t batch, int64_t seqlen) {
  if (!dims || batch < 0 || seqlen < 0) return 0;
  return prologue_bwd_workspace_bytes(batch, seqlen, dims->nheads, dims->num_rope_angles, dims->mimo_rank,
                                      dims->d_state);
}

int m3_layer_prologue_bwd(const m3_layer_dims* dims, const m3_tensor* zxbcdt, const m3_tensor* dt_bias,
                          const m3_tensor* B_bias, const m3_tensor* C_bias, const m3_tensor* B_norm_w,
                          const m3_tensor* C_norm_w, const m3_tensor* DT, const m3_tensor* angles,
                          const m3_tensor* dB_proj, const m3_tensor* dC_proj, const m3_tensor* dADT,
                          const m3_tensor* dDT, const m3_tensor* dtrap, m3_tensor* d_zxbcdt, m3_tensor* d_dt_bias,
                          m3_tensor* d_B_bias, m3_tensor* d_C_bias, m3_tensor* d_B_norm_w, m3_tensor* d_C_norm_w,
                          void* workspace, size_t workspace_bytes, void* stream) {
  if (!dims) return fail(M3_ERR_INVALID_ARGUMENT, "dims: missing");
  const int64_t H = dims->nheads, P = dims->headdim, Ds = dims->d_state, G = dims->ngroups,
                R = dims->mimo_rank, S = dims->num_rope_angles, di = dims->d_inner;
  if (H <= 0 || P <= 0 || Ds <= 0 || G <= 0 || R <= 0 || S < 0 || di != H * P || dims->rope_split != 2 * S ||
      dims->rope_split > Ds || (G != 1 && G != H))
    return fail(M3_ERR_INVALID_ARGUMENT, "dims: inconsistent layer dimensions");
  if (!present(zxbcdt) || zxbcdt->ndim != 3) return fail(M3_ERR_INVALID_ARGUMENT, "zxbcdt: expected (batch, seqlen, d_in_proj)");
  const int64_t Bn = zxbcdt->shape[0], L = zxbcdt->shape[1];
  const int64_t dproj = 2 * di + 2 * Ds * G * R + 3 * H + S;
  const bool empty = Bn * L == 0;
  const int64_t zs[3] = {Bn, L, dproj}, bs[5] = {Bn, L, R, H, Ds}, ss[3] = {Bn, L, H}, as[4] = {Bn, L, H, S},
                h1[1] = {H}, hrd[3] = {H, R, Ds}, d1[1] = {Ds};
  M3_TRY(check(zxbcdt, "zxbcdt", 3, zs, kAnyFloat, false, false, !empty));
  M3_TRY(check(d_zxbcdt, "d_zxbcdt", 3, zs, 1u << zxbcdt->dtype, false, false, !empty));
  M3_TRY(check(dB_proj, "dB_proj", 5, bs, kAnyFloat, true, false, !empty));
  M3_TRY(check(dC_proj, "dC_proj", 5, bs, 1u << dB_proj->dtype, true, false, !empty));
  M3_TRY(check(DT, "DT", 3, ss, kF32, true, false, false));
  M3_TRY(check(dADT, "dADT", 3, ss, kF32, true, false, false));
  M3_TRY(check(dDT, "dDT", 3, ss, kF32, true, false, false));
  M3_TRY(check(dtrap, "dtrap", 3, ss, kF32, true, false, false));
  M3_TRY(check(angles, "angles", 4, as, kF32, true, S == 0, false));
  M3_TRY(check(dt_bias, "dt_bias", 1, h1, kF32, true, false, false));
  M3_TRY(check(B_bias, "B_bias", 3, hrd, kF32, true, false, false));
  M3_TRY(check(C_bias, "C_bias", 3, hrd, kF32, true, false, false));
  M3_TRY(check(B_norm_w, "B_norm_w", 1, d1, kF32, true, false, false));
  M3_TRY(check(C_norm_w, "C_norm_w", 1, d1, kF32, true, false, false));
  M3_TRY(check(d_dt_bias, "d_dt_bias", 1, h1, kF32, true, false, false));
  M3_TRY(check(d_B_bias, "d_B_bias", 3, hrd, kF32, true, false, false));
  M3_TRY(check(d_C_bias, "d_C_bias", 3, hrd, kF32, true, false, false));
  M3_TRY(check(d_B_norm_w, "d_B_norm_w", 1, d1, kF32, true, false, false));
  M3_TRY(check(d_C_norm_w, "d_C_norm_w", 1, d1, kF32, true, false, false));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (empty) {
    // no positions: every parameter gradient is zero
    M3_TRY(memset_async(d_dt_bias->data, sizeof(float) * H, s, "d_dt_bias"));
    M3_TRY(memset_async(d_B_bias->data, sizeof(float) * H * R * Ds, s, "d_B_bias"));
    M3_TRY(memset_async(d_C_bias->data, sizeof(float) * H * R * Ds, s, "d_C_bias"));
    M3_TRY(memset_async(d_B_norm_w->data, sizeof(float) * Ds, s, "d_B_norm_w"));
    return memset_async(d_C_norm_w->data, sizeof(float) * Ds, s, "d_C_norm_w");
  }
  if (Bn > INT32_MAX || L > INT32_MAX) return fail(M3_ERR_UNSUPPORTED, "prologue backward: dimension too large");
  const size_t need = prologue_bwd_workspace_bytes(Bn, L, H, S, R, Ds);
  if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)
    return fail(M3_ERR_WORKSPACE, "prologue backward: workspace of " + std::to_string(need) + " bytes required");
  PrologueBwdParams p{};
  p.Bn = (int)Bn; p.L = (int)L; p.H = (int)H; p.P = (int)P; p.D = (int)Ds; p.R = (int)R; p.G = (int)G;
  p.S = (int)S; p.split = dims->rope_split; p.d_inner = (int)di; p.A_floor = dims->A_floor; p.eps = dims->norm_eps;
  p.zx = zxbcdt->data; p.s_zb = zxbcdt->stride[0]; p.s_zl = zxbcdt->stride[1];
  p.dzx = d_zxbcdt->data; p.s_dzb = d_zxbcdt->stride[0]; p.s_dzl = d_zxbcdt->stride[1];
  p.dt_bias = fptr<const float>(dt_bias);
  p.B_bias = fptr<const float>(B_bias); p.C_bias = fptr<const float>(C_bias);
  p.B_norm_w = fptr<const float>(B_norm_w); p.C_norm_w = fptr<const float>(C_norm_w);
  p.angles = fptr<const float>(angles); p.DT = fptr<const float>(DT);
  p.dBp = dB_proj->data; p.dCp = dC_proj->data;
  p.dADT = fptr<const float>(dADT); p.dDT = fptr<const float>(dDT); p.dtrap = fptr<const float>(dtrap);
  p.dB_bias = fptr<float>(d_B_bias); p.dC_bias = fptr<float>(d_C_bias);
  p.dB_norm_w = fptr<float>(d_B_norm_w); p.dC_norm_w = fptr<float>(d_C_norm_w);
  p.ddt_bias = fptr<float>(d_dt_bias);
  return launch_prologue_bwd(p, reinterpret_cast<float*>(workspace), zxbcdt->dtype, dB_proj->dtype, s);
}

int m3_silu_gate_bwd(const m3_tensor* y, const m3_tensor* z, const m3_tensor* dout, m3_tensor* dy, m3_tensor* dz,
                     void* stream) {
  if (!present(y) || y->ndim != 4) return fail(M3_ERR_INVALID_ARGUMENT, "y: expected (B, L, H, P)");
  const int64_t* sh = y->shape;
  const bool empty = sh[0] * sh[1] * sh[2] * sh[3] == 0;
  M3_TRY(check(y, "y", 4, sh, kAnyFloat, false, false, !empty));
  M3_TRY(check(z, "z", 4, sh, 1u << y->dtype, false, false, !empty));
  M3_TRY(check(dout, "dout", 4, sh, 1u << y->dtype, false, false, !empty));
  M3_TRY(check(dy, "dy", 4, sh, 1u << y->dtype, false, false, !empty));
  M3_TRY(check(dz, "dz", 4, sh, 1u << y->dtype, false, false, !empty));
  if (empty) return M3_OK;
  if (sh[1] > INT32_MAX || sh[2] > INT32_MAX || sh[3] > INT32_MAX)
    return fail(M3_ERR_UNSUPPORTED, "gate backward: dimension too large");
  GateBwdParams p{};
  p.rows = sh[0] * sh[1] * sh[2];
  p.L = (int)sh[1]; p.H = (int)sh[2]; p.P = (int)sh[3];
  p.y = y->data; p.sy = s3(y);
  p.z = z->data; p.sz = s3(z);
  p.dout = dout->data; p.sd = s3(dout);
  p.dy = dy->data; p.sdy = s3(dy);
  p.dz = dz->data; p.sdz = s3(dz);
  return launch_gate_bwd(p, y->dtype, z->dtype, dout->dtype, reinterpret_cast<cudaStream_t>(stream));
}

int m3_silu_gate(const m3_tensor* y, const m3_tensor* z, m3_tensor* out, void* stream) {
  if (!present(y) || y->ndim != 4) return fail(M3_ERR_INVALID_ARGUMENT, "y: expected (B, L, H, P)");
  const int64_t* sh = y->shape;
  const bool empty = sh[0] * sh[1] * sh[2] * sh[3] == 0;
  M3_TRY(check(y, "y", 4, sh, kAnyFloat, false, false, !empty));
  M3_TRY(check(z, "z", 4, sh, kAnyFloat, false, false, !empty));
  M3_TRY(check(out, "out", 4, sh, kAnyFloat, false, false, !empty));
  if (empty) return M3_OK;
  if (sh[1] > INT32_MAX || sh[2] > INT32_MAX || sh[3] > INT32_MAX) return fail(M3_ERR_UNSUPPORTED, "gate: dimension too large");
  GateParams p{};
  p.rows = sh[0] * sh[1] * sh[2]; p.L = (int)sh[1]; p.H = (int)sh[2]; p.P = (int)sh[3];
  p.y = y->data; p.sy = s3(y); p.z = z->data; p.sz = s3(z); p.out = out->data; p.so = s3(out);
  return launch_gate(p, y->dtype, z->dtype, out->dtype, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"

// ------------------------------------------------------------------------------------
// token losses
// ------------------------------------------------------------------------------------
namespace m3 {
namespace {

// A (batch, seqlen) operand of the token losses: one dtype, any strides.
template <typename T>
int map2(const m3_tensor* t, const char* name, int dtype, const int64_t* bt, bool optional, bool devcheck,
         Map2<T>* out) {
  *out = Map2<T>{nullptr, 0, 0};
  if (!present(t)) {
    if (optional) return M3_OK;
    return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": missing");
  }
  if (t->ndim != 2 || t->shape[0] != bt[0] || t->shape[1] != bt[1])
    return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": expected (batch, seqlen) = (" + std::to_string(bt[0]) +
                                             "," + std::to_string(bt[1]) + ")");
  if (t->dtype != dtype)
    return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": unsupported dtype " + std::to_string(t->dtype));
  if (t->stride[0] < 0 || t->stride[1] < 0)
    return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": negative stride");
  if (devcheck) {
    if (reinterpret_cast<uintptr_t>(t->data) % sizeof(T) != 0)
      return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": address not aligned to its elements");
    M3_TRY(check_device_ptr(t->data, name));
  }
  *out = Map2<T>{static_cast<T*>(t->data), t->stride[0], t->stride[1]};
  return M3_OK;
}

// Vector and element accesses need addresses that are multiples of the element's size.
int aligned(const m3_tensor* t, const char* name, size_t bytes) {
  if (!present(t) || reinterpret_cast<uintptr_t>(t->data) % bytes == 0) return M3_OK;
  return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": address not aligned to " + std::to_string(bytes) + " bytes");
}

// The rows that every token loss reads; *empty: there is no position. policy: its scale is one float.
int token_rows(const m3_tensor* logits, const m3_tensor* tokens, const m3_tensor* mask, double temperature,
               int64_t ignore_index, bool policy, TokenRows* p, bool* empty) {
  if (!present(logits)) return fail(M3_ERR_INVALID_ARGUMENT, "logits: missing");
  if (logits->ndim != 3) return fail(M3_ERR_INVALID_ARGUMENT, "logits: expected (batch, seqlen, vocabulary)");
  const int64_t* sh = logits->shape;
  if (sh[0] < 0 || sh[1] < 0 || sh[2] <= 0) return fail(M3_ERR_INVALID_ARGUMENT, "logits: empty vocabulary");
  if (sh[1] > INT32_MAX || sh[2] > INT32_MAX / 2 || (sh[0] > 0 && sh[1] > INT32_MAX / 8 / sh[0]))
    return fail(M3_ERR_UNSUPPORTED, "logits: dimension too large");
  *empty = sh[0] * sh[1] == 0;
  M3_TRY(check(logits, "logits", 3, sh, kAnyFloat, false, false, !*empty));
  if (!*empty) M3_TRY(aligned(logits, "logits", dtype_size(logits->dtype)));
  if (!(temperature > 1e-6 && temperature < 1e6))
    return fail(M3_ERR_INVALID_ARGUMENT, "temperature: expected a number between 1e-6 and 1e6");
  M3_TRY(map2(tokens, "tokens", M3_INT64, sh, false, !*empty, &p->tok));
  M3_TRY(map2(mask, "mask", M3_UINT8, sh, true, !*empty, &p->mask));
  p->logits = logits->data;
  p->sb = logits->stride[0]; p->st = logits->stride[1];
  p->R = sh[0] * sh[1]; p->T = (int)sh[1]; p->V = (int)sh[2];
  p->ignore = ignore_index;
  p->scale = 1.0 / temperature;
  // c in two floats, the upper one rounded down so that the lower one is positive; or in one,
  // rounded to the nearest, the lower one then the smallest number that keeps -inf from NaN (with
  // a product less in the kernels instead, one of them needs more registers than it has)
  const double c = p->scale * 1.44269504088896340736;
  float hi = (float)c;
  if (!policy && (double)hi >= c) hi = std::nextafterf(hi, 0.f);
  p->c_hi = hi;
  p->c_lo = policy ? std::numeric_limits<float>::min() : (float)(c - (double)hi);
  return M3_OK;
}

// One f32 value on the device, 0-d or of one element.
int scalar_out(const m3_tensor* t, const char* name, bool optional) {
  if (!present(t) && optional) return M3_OK;
  const int64_t one[1] = {1};
  return check(t, name, present(t) && t->ndim == 0 ? 0 : 1, one, kF32, true, false, true);
}

int workspace_ok(const void* ws, size_t have, size_t need, const char* what) {
  if (ws == nullptr || have < need || (reinterpret_cast<uintptr_t>(ws) & 15) != 0)
    return fail(M3_ERR_WORKSPACE, std::string(what) + ": workspace of " + std::to_string(need) + " bytes required");
  return M3_OK;
}

}  // namespace
}  // namespace m3

extern "C" {

int m3_token_logprobs(const m3_tensor* logits, const m3_tensor* tokens, const m3_tensor* mask, double temperature,
                      int64_t ignore_index, m3_tensor* logprobs, m3_tensor* stats, void* stream) {
  TokenRows p{};
  bool empty = false;
  M3_TRY(token_rows(logits, tokens, mask, temperature, ignore_index, false, &p, &empty));
  const int64_t bt[3] = {logits->shape[0], logits->shape[1], 2};
  M3_TRY(check(logprobs, "logprobs", 2, bt, kF32, true, false, !empty));
  M3_TRY(check(stats, "stats", 3, bt, kF32, true, true, !empty));
  if (!empty) M3_TRY(aligned(stats, "stats", 8));
  if (empty) return M3_OK;
  return launch_token_logprobs(p, logits->dtype, fptr<float>(logprobs), fptr<float2>(stats),
                               reinterpret_cast<cudaStream_t>(stream));
}

size_t m3_policy_loss_workspace_size(int64_t batch, int64_t seqlen) {
  if (batch < 0 || seqlen < 0) return 0;
  return policy_workspace_bytes(batch, batch * seqlen);
}

int m3_policy_loss(const m3_tensor* logits, const m3_tensor* tokens, const m3_tensor* mask,
                   const m3_tensor* old_logprobs, const m3_tensor* advantages, const m3_tensor* ref_logprobs,
                   double temperature, int64_t ignore_index, double clip_low, double clip_high, double kl_coef,
                   int by_sequence, m3_tensor* loss, m3_tensor* kl, m3_tensor* clip_fraction, m3_tensor* logprobs,
                   m3_tensor* dlogits, void* workspace, size_t workspace_bytes, void* stream) {
  TokenRows p{};
  bool empty = false;
  M3_TRY(token_rows(logits, tokens, mask, temperature, ignore_index, true, &p, &empty));
  const int64_t* sh = logits->shape;
  const int64_t bt[2] = {sh[0], sh[1]};
  if (!(clip_low >= 0 && clip_low <= 1)) return fail(M3_ERR_INVALID_ARGUMENT, "clip_low: expected a number from 0 to 1");
  if (!(clip_high >= 0)) return fail(M3_ERR_INVALID_ARGUMENT, "clip_high: expected a number from 0 on");
  if (!(kl_coef >= 0 && std::isfinite(kl_coef))) return fail(M3_ERR_INVALID_ARGUMENT, "kl_coef: expected a finite number from 0 on");
  if (by_sequence != 0 && by_sequence != 1) return fail(M3_ERR_INVALID_ARGUMENT, "by_sequence: expected 0 or 1");
  PolicyArgs a{};
  M3_TRY(map2(old_logprobs, "old_logprobs", M3_FLOAT32, sh, false, !empty, &a.old_logp));
  M3_TRY(map2(advantages, "advantages", M3_FLOAT32, sh, false, !empty, &a.adv));
  M3_TRY(map2(ref_logprobs, "ref_logprobs", M3_FLOAT32, sh, true, !empty, &a.ref));
  M3_TRY(check(logprobs, "logprobs", 2, bt, kF32, true, false, !empty));
  M3_TRY(check(dlogits, "dlogits", 3, sh, 1u << logits->dtype, false, true, !empty));
  if (!empty) M3_TRY(aligned(dlogits, "dlogits", dtype_size(logits->dtype)));
  M3_TRY(scalar_out(loss, "loss", false));
  M3_TRY(scalar_out(kl, "kl", false));
  M3_TRY(scalar_out(clip_fraction, "clip_fraction", false));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (empty) {
    M3_TRY(memset_async(loss->data, sizeof(float), s, "loss"));
    M3_TRY(memset_async(kl->data, sizeof(float), s, "kl"));
    return memset_async(clip_fraction->data, sizeof(float), s, "clip_fraction");
  }
  M3_TRY(workspace_ok(workspace, workspace_bytes, policy_workspace_bytes(sh[0], p.R), "policy loss"));
  a.clip_lo = 1.0 - clip_low; a.clip_hi = 1.0 + clip_high; a.kl_coef = kl_coef; a.by_sequence = by_sequence;
  const bool grad = present(dlogits);
  return launch_policy_loss(p, logits->dtype, a, sh[0], fptr<float>(loss), fptr<float>(kl),
                            fptr<float>(clip_fraction), fptr<float>(logprobs), fptr<void>(dlogits),
                            grad ? dlogits->stride[0] : 0, grad ? dlogits->stride[1] : 0, workspace, s);
}

size_t m3_preference_loss_workspace_size(int64_t batch, int64_t seqlen) {
  if (batch < 0 || seqlen < 0) return 0;
  return preference_workspace_bytes(batch, batch * seqlen);
}

int m3_preference_loss(const m3_tensor* logits, const m3_tensor* tokens, const m3_tensor* mask,
                       const m3_tensor* ref_logprobs, double temperature, int64_t ignore_index, double beta,
                       double label_smoothing, m3_tensor* loss, m3_tensor* rewards, m3_tensor* logprobs,
                       void* workspace, size_t workspace_bytes, void* stream) {
  TokenRows p{};
  bool empty = false;
  M3_TRY(token_rows(logits, tokens, mask, temperature, ignore_index, false, &p, &empty));
  const int64_t* sh = logits->shape;
  if (sh[0] % 2 != 0 || sh[0] == 0)
    return fail(M3_ERR_INVALID_ARGUMENT, "logits: an even number of sequences expected, chosen before rejected");
  if (!(beta >= 0 && std::isfinite(beta))) return fail(M3_ERR_INVALID_ARGUMENT, "beta: expected a finite number from 0 on");
  if (!(label_smoothing >= 0 && label_smoothing <= 1))
    return fail(M3_ERR_INVALID_ARGUMENT, "label_smoothing: expected a number from 0 to 1");
  const int64_t bt[2] = {sh[0], sh[1]};
  Map2<const float> ref;
  M3_TRY(map2(ref_logprobs, "ref_logprobs", M3_FLOAT32, sh, true, !empty, &ref));
  M3_TRY(scalar_out(loss, "loss", false));
  M3_TRY(check(rewards, "rewards", 1, bt, kF32, true, false, true));
  M3_TRY(check(logprobs, "logprobs", 2, bt, kF32, true, false, !empty));
  M3_TRY(workspace_ok(workspace, workspace_bytes, preference_workspace_bytes(sh[0], p.R), "preference loss"));
  return launch_preference_loss(p, logits->dtype, ref, beta, label_smoothing, sh[0] / 2, fptr<float>(loss),
                                fptr<float>(rewards), fptr<float>(logprobs), workspace, reinterpret_cast<cudaStream_t>(stream));
}

namespace m3 {
namespace {
// The gradient of a loss from its workspace.
int loss_grad(const m3_tensor* logits, const m3_tensor* tokens, const m3_tensor* mask, const m3_tensor* up,
              double temperature, int64_t ignore_index, bool keep_if_one, m3_tensor* dlogits, const void* workspace,
              size_t workspace_bytes, bool policy, cudaStream_t s) {
  TokenRows p{};
  bool empty = false;
  M3_TRY(token_rows(logits, tokens, mask, temperature, ignore_index, policy, &p, &empty));
  const int64_t* sh = logits->shape;
  M3_TRY(check(dlogits, "dlogits", 3, sh, 1u << logits->dtype, false, false, !empty));
  if (!empty) M3_TRY(aligned(dlogits, "dlogits", dtype_size(logits->dtype)));
  M3_TRY(scalar_out(up, "up", true));
  if (empty) return M3_OK;
  const size_t need = policy ? policy_workspace_bytes(sh[0], p.R) : preference_workspace_bytes(sh[0], p.R);
  M3_TRY(workspace_ok(workspace, workspace_bytes, need, policy ? "policy loss" : "preference loss"));
  const Map2<const float> coef = policy ? policy_coef(workspace, p) : preference_coef(workspace, p);
  return launch_token_grad(p, logits->dtype, workspace_stats(workspace), coef, fptr<const float>(up), keep_if_one,
                           dlogits->data, dlogits->stride[0], dlogits->stride[1], s);
}
}  // namespace
}  // namespace m3

int m3_policy_loss_grad(const m3_tensor* logits, const m3_tensor* tokens, const m3_tensor* mask, const m3_tensor* up,
                        double temperature, int64_t ignore_index, int keep_if_one, m3_tensor* dlogits,
                        const void* workspace, size_t workspace_bytes, void* stream) {
  if (keep_if_one != 0 && keep_if_one != 1) return fail(M3_ERR_INVALID_ARGUMENT, "keep_if_one: expected 0 or 1");
  return loss_grad(logits, tokens, mask, up, temperature, ignore_index, keep_if_one != 0, dlogits, workspace,
                   workspace_bytes, true, reinterpret_cast<cudaStream_t>(stream));
}

int m3_preference_loss_grad(const m3_tensor* logits, const m3_tensor* tokens, const m3_tensor* mask,
                            const m3_tensor* up, double temperature, int64_t ignore_index, m3_tensor* dlogits,
                            const void* workspace, size_t workspace_bytes, void* stream) {
  return loss_grad(logits, tokens, mask, up, temperature, ignore_index, false, dlogits, workspace, workspace_bytes,
                   false, reinterpret_cast<cudaStream_t>(stream));
}

int m3_token_logprobs_grad(const m3_tensor* logits, const m3_tensor* tokens, const m3_tensor* mask,
                           const m3_tensor* stats, const m3_tensor* dlogprobs, double temperature,
                           int64_t ignore_index, m3_tensor* dlogits, void* stream) {
  TokenRows p{};
  bool empty = false;
  M3_TRY(token_rows(logits, tokens, mask, temperature, ignore_index, false, &p, &empty));
  const int64_t* sh = logits->shape;
  const int64_t bt[3] = {sh[0], sh[1], 2};
  Map2<const float> c;
  M3_TRY(check(stats, "stats", 3, bt, kF32, true, false, !empty));
  if (!empty) M3_TRY(aligned(stats, "stats", 8));
  M3_TRY(map2(dlogprobs, "dlogprobs", M3_FLOAT32, sh, false, !empty, &c));
  M3_TRY(check(dlogits, "dlogits", 3, sh, 1u << logits->dtype, false, false, !empty));
  if (!empty) M3_TRY(aligned(dlogits, "dlogits", dtype_size(logits->dtype)));
  if (empty) return M3_OK;
  return launch_token_grad(p, logits->dtype, fptr<const float2>(stats), c, nullptr, false, dlogits->data,
                           dlogits->stride[0], dlogits->stride[1], reinterpret_cast<cudaStream_t>(stream));
}

size_t m3_clip_grads_workspace_size(int64_t count) { return count < 0 ? 0 : clip_grads_workspace_bytes(count); }

int m3_clip_grads(int64_t count, const void* const* grads, const int64_t* numel, const int32_t* dtypes,
                  void* const* outs, const int32_t* out_dtypes, int largest, double max_norm, double scale,
                  m3_tensor* norm, void* workspace, size_t workspace_bytes, void* stream) try {
  if (count < 0 || (count > 0 && (!grads || !numel || !dtypes)))
    return fail(M3_ERR_INVALID_ARGUMENT, "grads: missing");
  if (outs && !out_dtypes) return fail(M3_ERR_INVALID_ARGUMENT, "out_dtypes: missing");
  if (largest != 0 && largest != 1) return fail(M3_ERR_INVALID_ARGUMENT, "largest: expected 0 or 1");
  if (!(max_norm >= 0)) return fail(M3_ERR_INVALID_ARGUMENT, "max_norm: expected a number from 0 on");
  if (!(scale > 0 && std::isfinite(scale))) return fail(M3_ERR_INVALID_ARGUMENT, "scale: expected a positive finite number");
  bool in_place = true;  // outs that are the gradients themselves count as that too
  if (outs)
    for (int64_t i = 0; i < count && in_place; ++i) in_place = outs[i] == grads[i] && out_dtypes[i] == dtypes[i];
  const bool norm_alone = !outs && scale == 1.0 && std::isinf(max_norm);
  // what is written (and, with outs, what is read) as address ranges, to find overlaps; in place
  // with scale 1 and no bound nothing but NaN is written, to all of the gradients
  struct Range { uintptr_t lo, hi; bool written; int64_t index; };
  const bool writes = !in_place || scale != 1.0 || !std::isinf(max_norm);
  int64_t first = -1;  // tensor with elements
  std::vector<Range> ranges;
  if (writes) ranges.reserve((size_t)count * (outs ? 2 : 1));
  for (int64_t i = 0; i < count; ++i) {
    auto name = [&](const char* what) { return std::string(what) + "[" + std::to_string(i) + "]"; };
    if (numel[i] < 0) return fail(M3_ERR_INVALID_ARGUMENT, name("numel") + ": negative");
    if (dtypes[i] < 0 || dtypes[i] > M3_FLOAT16) return fail(M3_ERR_INVALID_ARGUMENT, name("grads") + ": unsupported dtype");
    if (outs && out_dtypes[i] != dtypes[i] && out_dtypes[i] != M3_FLOAT32)
      return fail(M3_ERR_INVALID_ARGUMENT, name("outs") + ": dtype must be the gradient's own or float32");
    if (numel[i] == 0) continue;
    if (!grads[i] || (outs && !outs[i])) return fail(M3_ERR_INVALID_ARGUMENT, name("grads") + ": missing");
    const uintptr_t g = reinterpret_cast<uintptr_t>(grads[i]), o = outs ? reinterpret_cast<uintptr_t>(outs[i]) : g;
    const size_t gs = dtype_size(dtypes[i]), os = outs ? dtype_size(out_dtypes[i]) : gs;
    if (g % gs != 0 || o % os != 0) return fail(M3_ERR_INVALID_ARGUMENT, name("grads") + ": not aligned to its elements");
    if (first < 0) first = i;
    if (!writes) continue;
    ranges.push_back(Range{o, o + os * (size_t)numel[i], true, i});
    if (outs && !(o == g && os == gs)) ranges.push_back(Range{g, g + gs * (size_t)numel[i], false, i});
  }
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
  // sorted by their starts, a range meets an earlier one exactly if it begins before the
  // furthest end so far (of the written ones, or of any where it is written itself)
  uintptr_t end_any = 0, end_written = 0;
  for (const Range& r : ranges) {
    if (r.lo < (r.written ? end_any : end_written))
      return fail(M3_ERR_INVALID_ARGUMENT, "grads[" + std::to_string(r.index) + "]: shares memory with another tensor of the call");
    end_any = std::max(end_any, r.hi);
    if (r.written) end_written = std::max(end_written, r.hi);
  }
  // one address of each kind is looked up: hundreds would cost more than the launches
  if (first >= 0) {
    M3_TRY(check_device_ptr(grads[first], "grads"));
    if (outs) M3_TRY(check_device_ptr(outs[first], "outs"));
  }
  M3_TRY(scalar_out(norm, "norm", false));
  if (count > 0) M3_TRY(workspace_ok(workspace, workspace_bytes, clip_grads_workspace_bytes(count), "clip_grads"));
  ClipArgs a{count, grads, numel, dtypes, outs, out_dtypes, largest != 0, max_norm, scale, in_place, norm_alone,
             fptr<float>(norm)};
  return launch_clip_grads(a, workspace, reinterpret_cast<cudaStream_t>(stream));
} catch (const std::exception& e) {
  return fail(M3_ERR_INVALID_ARGUMENT, std::string("clip_grads: ") + e.what());
}

}  // extern "C"

// ------------------------------------------------------------------------------------
// selective scan, causal convolution
// ------------------------------------------------------------------------------------
namespace m3 {
namespace {

constexpr int64_t kMaxGrid = 65535;

// Multiprocessors of the current device; 148 where there is none (workspace sizes asked for on a host).
int sms_here() {
  int n = 0;
  if (device_sm_count(&n) != M3_OK) {
    cudaGetLastError();
    n = 148;
  }
  return n;
}

// What a tensor of the call's other float type may be: u's own dtype or fp32.
unsigned own_or_f32(const m3_tensor* t) { return (1u << t->dtype) | kF32; }

int flag(int v, const char* name) {
  return v == 0 || v == 1 ? M3_OK : fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": expected 0 or 1");
}

int elem_aligned(const m3_tensor* t, const char* name) {
  if (!present(t)) return M3_OK;
  return aligned(t, name, t->dtype == M3_INT64 ? 8 : dtype_size(t->dtype));
}

// check() with the address on a boundary of its elements
int operand(const m3_tensor* t, const char* name, int ndim, const int64_t* shape, unsigned mask, bool contig, bool optional,
            bool devcheck) {
  M3_TRY(check(t, name, ndim, shape, mask, contig, optional, devcheck));
  return devcheck ? elem_aligned(t, name) : M3_OK;
}

// An optional (batch) i64 tensor, contiguous.
int lengths_ok(const m3_tensor* t, int64_t batch, bool devcheck, const int64_t** out) {
  *out = nullptr;
  if (!present(t)) return M3_OK;
  if (t->ndim != 1 || t->shape[0] != batch || t->dtype != M3_INT64 || (batch > 1 && t->stride[0] != 1))
    return fail(M3_ERR_INVALID_ARGUMENT, "lengths: expected (batch) int64, contiguous");
  if (devcheck) {
    M3_TRY(check_device_ptr(t->data, "lengths"));
    M3_TRY(elem_aligned(t, "lengths"));
  }
  *out = static_cast<const int64_t*>(t->data);
  return M3_OK;
}

int conv_operands(const m3_tensor* x, int xdims, const m3_tensor* weight, const m3_tensor* bias, int silu, int64_t* taps) {
  if (!present(x) || x->ndim != xdims)
    return fail(M3_ERR_INVALID_ARGUMENT, xdims == 3 ? "x: expected (batch, seqlen, channels)" : "x: expected (batch, channels)");
  const int64_t E = x->shape[xdims - 1], batch = x->shape[0], L = xdims == 3 ? x->shape[1] : 1;
  if (batch < 0 || L < 0 || E < 0) return fail(M3_ERR_INVALID_ARGUMENT, "x: negative extent");
  if (L > INT32_MAX / 2 || E > INT32_MAX / 8 || (xdims == 3 && batch > kMaxGrid))
    return fail(M3_ERR_UNSUPPORTED, "x: dimension too large");
  M3_TRY(operand(x, "x", xdims, x->shape, kAnyFloat, false, false, batch * L * E > 0));
  if (!present(weight) || weight->ndim != 2) return fail(M3_ERR_INVALID_ARGUMENT, "weight: expected (channels, taps)");
  *taps = weight->shape[1];
  if (*taps < 2 || *taps > 4) return fail(M3_ERR_UNSUPPORTED, "weight: 2, 3 or 4 taps expected, got " + std::to_string(*taps));
  const int64_t ws[2] = {E, *taps};
  M3_TRY(operand(weight, "weight", 2, ws, own_or_f32(x), false, false, E > 0));
  M3_TRY(operand(bias, "bias", 1, ws, 1u << weight->dtype, true, true, E > 0));
  return flag(silu, "silu");
}

int conv_params(const m3_tensor* x, const m3_tensor* weight, const m3_tensor* bias, const m3_tensor* initial,
                const m3_tensor* lengths, int silu, ConvParams* p, int64_t* taps) {
  M3_TRY(conv_operands(x, 3, weight, bias, silu, taps));
  const int64_t batch = x->shape[0], L = x->shape[1], E = x->shape[2], is[3] = {batch, *taps - 1, E};
  M3_TRY(operand(initial, "initial", 3, is, 1u << x->dtype, false, true, batch * E > 0));
  M3_TRY(lengths_ok(lengths, batch, batch > 0, &p->lengths));
  p->x = x->data; p->xb = x->stride[0]; p->xl = x->stride[1];
  p->w = weight->data; p->we = weight->stride[0];
  p->bias = fptr<const void>(bias);
  p->w_f32 = weight->dtype == M3_FLOAT32;
  p->init = fptr<const void>(initial);
  p->ib = present(initial) ? initial->stride[0] : 0; p->il = present(initial) ? initial->stride[1] : 0;
  p->silu = silu != 0;
  p->batch = (int)batch; p->L = (int)L; p->E = (int)E;
  return M3_OK;
}

Seq seq(const m3_tensor* t) { return present(t) ? Seq{t->data, t->stride[0], t->stride[1]} : Seq{nullptr, 0, 0}; }

// Everything that the scan's forward and backward read; *empty: no channel of any sequence.
int selective_params(const m3_tensor* u, const m3_tensor* delta, const m3_tensor* A, const m3_tensor* B, const m3_tensor* C,
                     const m3_tensor* D, const m3_tensor* z, const m3_tensor* delta_bias, const m3_tensor* initial,
                     const m3_tensor* lengths, int softplus, SelScanParams* p, bool* empty) {
  if (!present(u) || u->ndim != 3) return fail(M3_ERR_INVALID_ARGUMENT, "u: expected (batch, seqlen, channels)");
  const int64_t batch = u->shape[0], L = u->shape[1], E = u->shape[2];
  if (batch < 0 || L < 0 || E < 0) return fail(M3_ERR_INVALID_ARGUMENT, "u: negative extent");
  const bool some = batch * L * E > 0;
  *empty = batch * E == 0;
  M3_TRY(operand(u, "u", 3, u->shape, kAnyFloat, false, false, some));
  M3_TRY(operand(delta, "delta", 3, u->shape, own_or_f32(u), false, false, some));
  M3_TRY(operand(z, "z", 3, u->shape, 1u << u->dtype, false, true, some));
  if (!present(A) || A->ndim != 2) return fail(M3_ERR_INVALID_ARGUMENT, "A: expected (channels, d_state)");
  const int64_t N = A->shape[1], an[2] = {E, N};
  if (N < 1) return fail(M3_ERR_INVALID_ARGUMENT, "A: d_state must be positive");
  if (N > kSelMaxStates) return fail(M3_ERR_UNSUPPORTED, "A: d_state above " + std::to_string(kSelMaxStates));
  M3_TRY(operand(A, "A", 2, an, kF32, true, false, E > 0));
  if (!present(B) || B->ndim != 4) return fail(M3_ERR_INVALID_ARGUMENT, "B: expected (batch, seqlen, groups, d_state)");
  const int64_t G = B->shape[2], bs[4] = {batch, L, G, N};
  if (G < 1 || E % G != 0) return fail(M3_ERR_INVALID_ARGUMENT, "B: the channels must divide into its groups");
  M3_TRY(operand(B, "B", 4, bs, own_or_f32(u), false, false, batch * L > 0));
  M3_TRY(operand(C, "C", 4, bs, 1u << B->dtype, false, false, batch * L > 0));
  M3_TRY(operand(D, "D", 1, an, kF32, true, true, E > 0));
  M3_TRY(operand(delta_bias, "delta_bias", 1, an, kF32, true, true, E > 0));
  const int64_t hs[3] = {batch, E, N};
  M3_TRY(operand(initial, "initial", 3, hs, kF32, true, true, !*empty));
  M3_TRY(lengths_ok(lengths, batch, batch > 0, &p->lengths));
  M3_TRY(flag(softplus, "softplus"));
  if (batch > kMaxGrid || L > INT32_MAX / 2 || E > INT32_MAX / (2 * kSelMaxStates) || batch * L * G > INT64_C(1) << 36)
    return fail(M3_ERR_UNSUPPORTED, "u: dimension too large");
  p->u = seq(u); p->delta = seq(delta); p->z = seq(z); p->B = seq(B); p->C = seq(C);
  p->Bg = B->stride[2]; p->Cg = C->stride[2];
  p->delta_f32 = delta->dtype == M3_FLOAT32; p->bc_f32 = B->dtype == M3_FLOAT32;
  p->A = fptr<const float>(A); p->D = fptr<const float>(D); p->bias = fptr<const float>(delta_bias);
  p->softplus = softplus != 0;
  p->h0 = fptr<const float>(initial);
  p->batch = (int)batch; p->L = (int)L; p->E = (int)E; p->N = (int)N; p->G = (int)G;
  return M3_OK;
}

SelScanParams selective_sizes(int64_t batch, int64_t seqlen, int64_t channels, int64_t d_state, int64_t groups) {
  SelScanParams p{};
  p.batch = (int)batch; p.L = (int)seqlen; p.E = (int)channels; p.N = (int)d_state; p.G = (int)groups;
  return p;
}

bool selective_sizes_ok(int64_t batch, int64_t seqlen, int64_t channels, int64_t d_state, int64_t groups) {
  return batch >= 0 && seqlen >= 0 && channels >= 0 && d_state >= 1 && d_state <= kSelMaxStates && groups >= 1 &&
         batch <= kMaxGrid && seqlen <= INT32_MAX / 2 && channels <= INT32_MAX / (2 * kSelMaxStates);
}

}  // namespace
}  // namespace m3

extern "C" {

int m3_causal_conv(const m3_tensor* x, const m3_tensor* weight, const m3_tensor* bias, const m3_tensor* initial,
                   const m3_tensor* lengths, int silu, m3_tensor* y, m3_tensor* last, void* stream) {
  ConvParams p{};
  int64_t taps = 0;
  M3_TRY(conv_params(x, weight, bias, initial, lengths, silu, &p, &taps));
  const int64_t ls[3] = {p.batch, taps - 1, p.E};
  const bool some = (int64_t)p.batch * p.E > 0;
  M3_TRY(operand(y, "y", 3, x->shape, 1u << x->dtype, false, false, some && p.L > 0));
  M3_TRY(operand(last, "last", 3, ls, 1u << x->dtype, true, true, some));
  if (!some) return M3_OK;
  p.y = y->data; p.yb = y->stride[0]; p.yl = y->stride[1];
  p.last = fptr<void>(last);
  return launch_conv_fwd(p, (int)taps, x->dtype, reinterpret_cast<cudaStream_t>(stream));
}

size_t m3_causal_conv_bwd_workspace_size(int64_t batch, int64_t seqlen, int64_t channels, int64_t taps) {
  if (batch < 0 || seqlen < 0 || channels < 0 || taps < 2 || taps > 4) return 0;
  return conv_bwd_workspace(batch, seqlen, channels, (int)taps);
}

int m3_causal_conv_bwd(const m3_tensor* x, const m3_tensor* weight, const m3_tensor* bias, const m3_tensor* initial,
                       const m3_tensor* lengths, int silu, const m3_tensor* dy, const m3_tensor* dlast, m3_tensor* dx,
                       m3_tensor* dweight, m3_tensor* dbias, m3_tensor* dinitial, void* workspace, size_t workspace_bytes,
                       void* stream) {
  ConvParams p{};
  ConvGrads g{};
  int64_t taps = 0;
  M3_TRY(conv_params(x, weight, bias, initial, lengths, silu, &p, &taps));
  const int64_t ls[3] = {p.batch, taps - 1, p.E}, wsz[2] = {p.E, taps};
  const bool some = (int64_t)p.batch * p.E > 0;
  const unsigned xt = 1u << x->dtype, wt = 1u << weight->dtype;
  M3_TRY(operand(dy, "dy", 3, x->shape, xt, false, false, some && p.L > 0));
  M3_TRY(operand(dx, "dx", 3, x->shape, xt, false, false, some && p.L > 0));
  M3_TRY(operand(dlast, "dlast", 3, ls, xt, false, true, some));
  M3_TRY(operand(dweight, "dweight", 2, wsz, wt, true, false, p.E > 0));
  M3_TRY(operand(dbias, "dbias", 1, wsz, wt, true, true, p.E > 0));
  M3_TRY(operand(dinitial, "dinitial", 3, ls, xt, true, true, some));
  if (p.E == 0) return M3_OK;
  const size_t need = conv_bwd_workspace(p.batch, p.L, p.E, (int)taps);
  if (need > 0) M3_TRY(workspace_ok(workspace, workspace_bytes, need, "causal_conv_bwd"));
  g.dy = dy->data; g.dyb = dy->stride[0]; g.dyl = dy->stride[1];
  g.dlast = fptr<const void>(dlast);
  g.dlb = present(dlast) ? dlast->stride[0] : 0; g.dll = present(dlast) ? dlast->stride[1] : 0;
  g.dx = dx->data; g.dxb = dx->stride[0]; g.dxl = dx->stride[1];
  g.dw = dweight->data;
  g.dbias = fptr<void>(dbias);
  g.dinit = fptr<void>(dinitial);
  return launch_conv_bwd(p, g, (int)taps, x->dtype, workspace, reinterpret_cast<cudaStream_t>(stream));
}

int m3_causal_conv_step(m3_tensor* state, const m3_tensor* x, const m3_tensor* weight, const m3_tensor* bias, int silu,
                        m3_tensor* y, void* stream) {
  int64_t taps = 0;
  M3_TRY(conv_operands(x, 2, weight, bias, silu, &taps));
  const int64_t batch = x->shape[0], E = x->shape[1], ss[3] = {batch, taps - 1, E};
  const bool some = batch * E > 0;
  M3_TRY(operand(state, "state", 3, ss, 1u << x->dtype, false, false, some));
  M3_TRY(operand(y, "y", 2, x->shape, 1u << x->dtype, true, false, some));
  if (!some) return M3_OK;
  // rows of E elements, one after the other in either order of sequences and rows
  const int64_t sb = state->stride[0], sl = state->stride[1], rows = taps - 1;
  const bool apart = batch == 1 ? rows == 1 || sl >= E
                     : rows == 1 ? sb >= E
                                 : (sl >= E && sb >= (rows - 1) * sl + E) || (sb >= E && sl >= (batch - 1) * sb + E);
  if (!apart) return fail(M3_ERR_INVALID_ARGUMENT, "state: rows overlap");
  ConvStepParams p{state->data, state->stride[0], state->stride[1], x->data, x->stride[0], weight->data, weight->stride[0],
                   fptr<const void>(bias), weight->dtype == M3_FLOAT32, silu != 0, y->data, batch, (int)E, false};
  return launch_conv_step(p, (int)taps, x->dtype, reinterpret_cast<cudaStream_t>(stream));
}

size_t m3_selective_scan_workspace_size(int64_t batch, int64_t seqlen, int64_t channels, int64_t d_state, int64_t groups) {
  if (!selective_sizes_ok(batch, seqlen, channels, d_state, groups)) return 0;
  return sel_scan_fwd_workspace(selective_sizes(batch, seqlen, channels, d_state, groups), sms_here());
}

size_t m3_selective_scan_states_size(int64_t batch, int64_t seqlen, int64_t channels, int64_t d_state) {
  if (!selective_sizes_ok(batch, seqlen, channels, d_state, 1)) return 0;
  return sel_scan_save_bytes(batch, seqlen, channels, (int)d_state);
}

size_t m3_selective_scan_bwd_workspace_size(int64_t batch, int64_t seqlen, int64_t channels, int64_t d_state, int64_t groups) {
  if (!selective_sizes_ok(batch, seqlen, channels, d_state, groups)) return 0;
  return sel_scan_bwd_workspace(selective_sizes(batch, seqlen, channels, d_state, groups), sms_here());
}

int m3_selective_scan(const m3_tensor* u, const m3_tensor* delta, const m3_tensor* A, const m3_tensor* B, const m3_tensor* C,
                      const m3_tensor* D, const m3_tensor* z, const m3_tensor* delta_bias, const m3_tensor* initial,
                      const m3_tensor* lengths, int softplus, m3_tensor* y, m3_tensor* last, void* states,
                      size_t states_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  SelScanParams p{};
  bool empty = false;
  M3_TRY(selective_params(u, delta, A, B, C, D, z, delta_bias, initial, lengths, softplus, &p, &empty));
  const int64_t hs[3] = {p.batch, p.E, p.N};
  M3_TRY(operand(y, "y", 3, u->shape, 1u << u->dtype, false, false, !empty && p.L > 0));
  M3_TRY(operand(last, "last", 3, hs, kF32, true, true, !empty));
  if (empty) return M3_OK;
  const size_t need = sel_scan_fwd_workspace(p, sms_here());
  if (need > 0) M3_TRY(workspace_ok(workspace, workspace_bytes, need, "selective_scan"));
  if (states != nullptr)
    M3_TRY(workspace_ok(states, states_bytes, sel_scan_save_bytes(p.batch, p.L, p.E, p.N), "selective_scan states"));
  p.y = seq(y);
  p.h_last = fptr<float>(last);
  p.save = static_cast<float*>(states);
  return launch_sel_scan_fwd(p, u->dtype, workspace, reinterpret_cast<cudaStream_t>(stream));
}

int m3_selective_scan_bwd(const m3_tensor* u, const m3_tensor* delta, const m3_tensor* A, const m3_tensor* B,
                          const m3_tensor* C, const m3_tensor* D, const m3_tensor* z, const m3_tensor* delta_bias,
                          const m3_tensor* initial, const m3_tensor* lengths, int softplus, const m3_tensor* dy,
                          const m3_tensor* dlast, m3_tensor* du, m3_tensor* ddelta, m3_tensor* dA, m3_tensor* dB,
                          m3_tensor* dC, m3_tensor* dD, m3_tensor* dz, m3_tensor* ddelta_bias, m3_tensor* dinitial,
                          const void* states, size_t states_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  SelScanParams p{};
  SelScanGrads g{};
  bool empty = false;
  M3_TRY(selective_params(u, delta, A, B, C, D, z, delta_bias, initial, lengths, softplus, &p, &empty));
  const bool some = !empty && p.L > 0;
  const unsigned ut = 1u << u->dtype;
  const int64_t hs[3] = {p.batch, p.E, p.N}, an[2] = {p.E, p.N};
  M3_TRY(operand(dy, "dy", 3, u->shape, ut, false, false, some));
  M3_TRY(operand(dlast, "dlast", 3, hs, kF32, true, true, !empty));
  M3_TRY(operand(du, "du", 3, u->shape, ut, false, false, some));
  M3_TRY(operand(ddelta, "ddelta", 3, u->shape, 1u << delta->dtype, false, false, some));
  M3_TRY(operand(dz, "dz", 3, u->shape, ut, false, !present(z), some));
  M3_TRY(operand(dA, "dA", 2, an, kF32, true, false, p.E > 0));
  M3_TRY(operand(dB, "dB", 4, B->shape, 1u << B->dtype, true, false, some));
  M3_TRY(operand(dC, "dC", 4, B->shape, 1u << B->dtype, true, false, some));
  M3_TRY(operand(dD, "dD", 1, an, kF32, true, true, p.E > 0));
  M3_TRY(operand(ddelta_bias, "ddelta_bias", 1, an, kF32, true, true, p.E > 0));
  M3_TRY(operand(dinitial, "dinitial", 3, hs, kF32, true, true, !empty));
  if (p.E == 0) return M3_OK;
  if (some) M3_TRY(workspace_ok(states, states_bytes, sel_scan_save_bytes(p.batch, p.L, p.E, p.N), "selective_scan states"));
  const size_t need = sel_scan_bwd_workspace(p, sms_here());
  if (need > 0) M3_TRY(workspace_ok(workspace, workspace_bytes, need, "selective_scan_bwd"));
  p.save = static_cast<float*>(const_cast<void*>(states));
  g.dy = seq(dy); g.du = seq(du); g.ddelta = seq(ddelta); g.dz = seq(dz);
  g.dstate = fptr<const float>(dlast);
  g.dA = fptr<float>(dA); g.dD = fptr<float>(dD); g.dbias = fptr<float>(ddelta_bias);
  g.dB = dB->data; g.dC = dC->data;
  g.dh0 = fptr<float>(dinitial);
  return launch_sel_scan_bwd(p, g, u->dtype, workspace, reinterpret_cast<cudaStream_t>(stream));
}

int m3_selective_step(m3_tensor* state, const m3_tensor* u, const m3_tensor* delta, const m3_tensor* A, const m3_tensor* B,
                      const m3_tensor* C, const m3_tensor* D, const m3_tensor* z, const m3_tensor* delta_bias, int softplus,
                      m3_tensor* y, void* stream) {
  if (!present(u) || u->ndim != 2) return fail(M3_ERR_INVALID_ARGUMENT, "u: expected (batch, channels)");
  const int64_t batch = u->shape[0], E = u->shape[1];
  if (batch < 0 || E < 0) return fail(M3_ERR_INVALID_ARGUMENT, "u: negative extent");
  const bool some = batch * E > 0;
  M3_TRY(operand(u, "u", 2, u->shape, kAnyFloat, false, false, some));
  M3_TRY(operand(delta, "delta", 2, u->shape, own_or_f32(u), false, false, some));
  M3_TRY(operand(z, "z", 2, u->shape, 1u << u->dtype, false, true, some));
  if (!present(A) || A->ndim != 2) return fail(M3_ERR_INVALID_ARGUMENT, "A: expected (channels, d_state)");
  const int64_t N = A->shape[1], an[2] = {E, N}, hs[3] = {batch, E, N};
  if (N < 1) return fail(M3_ERR_INVALID_ARGUMENT, "A: d_state must be positive");
  if (N > kSelMaxStates) return fail(M3_ERR_UNSUPPORTED, "A: d_state above " + std::to_string(kSelMaxStates));
  M3_TRY(operand(A, "A", 2, an, kF32, true, false, some));
  if (!present(B) || B->ndim != 3) return fail(M3_ERR_INVALID_ARGUMENT, "B: expected (batch, groups, d_state)");
  const int64_t G = B->shape[1], bs[3] = {batch, G, N};
  if (G < 1 || E % G != 0) return fail(M3_ERR_INVALID_ARGUMENT, "B: the channels must divide into its groups");
  M3_TRY(operand(B, "B", 3, bs, own_or_f32(u), false, false, some));
  M3_TRY(operand(C, "C", 3, bs, 1u << B->dtype, false, false, some));
  M3_TRY(operand(D, "D", 1, an, kF32, true, true, some));
  M3_TRY(operand(delta_bias, "delta_bias", 1, an, kF32, true, true, some));
  M3_TRY(operand(state, "state", 3, hs, kF32, false, false, some));
  if (some && E > 1 && state->stride[1] != N)
    return fail(M3_ERR_INVALID_ARGUMENT, "state: each sequence's part must be contiguous");
  if (some && batch > 1 && state->stride[0] < E * N) return fail(M3_ERR_INVALID_ARGUMENT, "state: sequences overlap");
  M3_TRY(operand(y, "y", 2, u->shape, 1u << u->dtype, false, false, some));
  M3_TRY(flag(softplus, "softplus"));
  if (E > INT32_MAX / (2 * kSelMaxStates) || batch > (INT64_C(1) << 36) / std::max<int64_t>(1, E))
    return fail(M3_ERR_UNSUPPORTED, "u: dimension too large");
  if (!some) return M3_OK;
  SelStepParams p{};
  p.u = u->data; p.delta = delta->data; p.z = fptr<const void>(z); p.B = B->data; p.C = C->data; p.y = y->data;
  p.su = u->stride[0]; p.sd = delta->stride[0]; p.sz = present(z) ? z->stride[0] : 0;
  p.sB = B->stride[0]; p.sC = C->stride[0]; p.sBg = B->stride[1]; p.sCg = C->stride[1]; p.sy = y->stride[0];
  p.delta_f32 = delta->dtype == M3_FLOAT32; p.bc_f32 = B->dtype == M3_FLOAT32;
  p.A = fptr<const float>(A); p.D = fptr<const float>(D); p.bias = fptr<const float>(delta_bias);
  p.softplus = softplus != 0;
  p.state = fptr<float>(state); p.sstate = state->stride[0];
  p.batch = batch; p.E = (int)E; p.N = (int)N; p.G = (int)G;
  return launch_sel_step(p, u->dtype, reinterpret_cast<cudaStream_t>(stream));
}

// ------------------------------------------------------------------------------------
// beam search
// ------------------------------------------------------------------------------------
size_t m3_beam_select_workspace_size(int64_t batch, int64_t beams, int64_t vocabulary, int64_t num, int dtype) {
  if (batch < 0 || beams < 1 || beams > kMaxBeams || vocabulary < 1 || vocabulary > kMaxVocab || num < 1 ||
      num > kMaxCandidates || dtype < 0 || dtype > M3_FLOAT16)
    return 0;
  return beam_workspace_bytes(batch, (int)beams, (int)vocabulary, (int)num, dtype, sms_here());
}

int m3_beam_select(const m3_tensor* logits, const m3_tensor* scores, const m3_tensor* finished, int64_t end_token,
                   m3_tensor* out_scores, m3_tensor* parents, m3_tensor* tokens, void* workspace, size_t workspace_bytes,
                   void* stream) {
  if (!present(logits) || logits->ndim != 3) return fail(M3_ERR_INVALID_ARGUMENT, "logits: expected (batch, beams, vocabulary)");
  const int64_t batch = logits->shape[0], K = logits->shape[1], V = logits->shape[2];
  if (batch < 0 || K < 1 || V < 1) return fail(M3_ERR_INVALID_ARGUMENT, "logits: no beam or no token");
  if (K > kMaxBeams) return fail(M3_ERR_UNSUPPORTED, "logits: more than " + std::to_string(kMaxBeams) + " beams");
  if (V > kMaxVocab || batch * K > kMaxGrid) return fail(M3_ERR_UNSUPPORTED, "logits: dimension too large");
  M3_TRY(operand(logits, "logits", 3, logits->shape, kAnyFloat, false, false, batch > 0));
  Map2<const float> sc;
  Map2<const uint8_t> fin;
  M3_TRY(map2(scores, "scores", M3_FLOAT32, logits->shape, false, batch > 0, &sc));
  M3_TRY(map2(finished, "finished", M3_UINT8, logits->shape, true, batch > 0, &fin));
  if (end_token < 0 || end_token >= V) return fail(M3_ERR_INVALID_ARGUMENT, "end_token: outside the vocabulary");
  if (!present(out_scores) || out_scores->ndim != 2) return fail(M3_ERR_INVALID_ARGUMENT, "out_scores: expected (batch, num)");
  const int64_t num = out_scores->shape[1], os[2] = {batch, num};
  if (num < 1 || num > K * V) return fail(M3_ERR_INVALID_ARGUMENT, "out_scores: 1 to beams * vocabulary candidates expected");
  if (num > kMaxCandidates) return fail(M3_ERR_UNSUPPORTED, "out_scores: more than " + std::to_string(kMaxCandidates) + " candidates");
  M3_TRY(operand(out_scores, "out_scores", 2, os, kF32, true, false, batch > 0));
  for (const m3_tensor* t : {static_cast<const m3_tensor*>(parents), static_cast<const m3_tensor*>(tokens)}) {
    const char* name = t == parents ? "parents" : "tokens";
    if (!present(t) || t->dtype != M3_INT64 || t->ndim != 2 || t->shape[0] != batch || t->shape[1] != num ||
        (num > 1 && t->stride[1] != 1) || (batch > 1 && t->stride[0] != num))
      return fail(M3_ERR_INVALID_ARGUMENT, std::string(name) + ": expected (batch, num) int64, contiguous");
    if (batch > 0) {
      M3_TRY(check_device_ptr(t->data, name));
      M3_TRY(elem_aligned(t, name));
    }
  }
  if (batch == 0) return M3_OK;
  const size_t need = beam_workspace_bytes(batch, (int)K, (int)V, (int)num, logits->dtype, sms_here());
  if (need > 0) M3_TRY(workspace_ok(workspace, workspace_bytes, need, "beam_select"));
  BeamParams p{};
  p.logits = logits->data; p.lb = logits->stride[0]; p.lk = logits->stride[1];
  p.scores = sc.p; p.sb = sc.sb; p.sk = sc.st;
  p.finished = fin.p; p.fb = fin.sb; p.fk = fin.st;
  p.batch = batch; p.beams = (int)K; p.V = (int)V; p.num = (int)num; p.end_token = (int)end_token;
  p.out_scores = fptr<float>(out_scores); p.parents = fptr<int64_t>(parents); p.tokens = fptr<int64_t>(tokens);
  return launch_beam_select(p, logits->dtype, workspace, reinterpret_cast<cudaStream_t>(stream));
}

int m3_reorder_states(int64_t count, const void* const* src, void* const* dst, const int64_t* row_bytes,
                      const int64_t* src_pitch, const int64_t* dst_pitch, int64_t source_rows, const m3_tensor* parents,
                      void* stream) try {
  if (count < 0 || (count > 0 && (!src || !row_bytes || !src_pitch || (dst && !dst_pitch))))
    return fail(M3_ERR_INVALID_ARGUMENT, "states: missing");
  if (!present(parents) || parents->ndim != 2 || parents->dtype != M3_INT64)
    return fail(M3_ERR_INVALID_ARGUMENT, "parents: expected (batch, rows) int64");
  const int64_t batch = parents->shape[0], T = parents->shape[1], S = source_rows;
  if (parents->stride[0] < 0 || parents->stride[1] < 0) return fail(M3_ERR_INVALID_ARGUMENT, "parents: negative stride");
  if (S < 0 || batch < 0 || T < 0 || S > INT32_MAX || batch > INT32_MAX || T > INT32_MAX)
    return fail(M3_ERR_INVALID_ARGUMENT, "parents: sizes out of range");
  if (!dst && S != T) return fail(M3_ERR_INVALID_ARGUMENT, "parents: in place, as many rows as the source has expected");
  if (!dst && T > kMaxBeams)
    return fail(M3_ERR_UNSUPPORTED, "parents: more than " + std::to_string(kMaxBeams) + " rows of a group in place");
  // what is read and written: rows of `bytes` every `pitch` bytes from lo to hi
  struct Range { uintptr_t lo, hi; int64_t bytes, pitch, index; bool written; };
  std::vector<Range> ranges, open;
  ranges.reserve((size_t)count * (dst ? 2 : 1));
  const bool some = batch > 0 && T > 0;
  int64_t first = -1;
  for (int64_t i = 0; i < count; ++i) {
    auto name = [&](const char* what) { return std::string(what) + "[" + std::to_string(i) + "]"; };
    if (row_bytes[i] < 0) return fail(M3_ERR_INVALID_ARGUMENT, name("row_bytes") + ": negative");
    if (row_bytes[i] == 0 || !some) continue;
    auto add = [&](const void* p, int64_t pitch, int64_t rows, bool written, const char* what) {
      if (!p) return fail(M3_ERR_INVALID_ARGUMENT, name(what) + ": missing");
      if (rows > 1 && pitch < row_bytes[i]) return fail(M3_ERR_INVALID_ARGUMENT, name(what) + ": rows overlap");
      const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
      ranges.push_back(Range{lo, lo + (uintptr_t)((rows - 1) * pitch + row_bytes[i]), row_bytes[i], pitch, i, written});
      return (int)M3_OK;
    };
    if (S > 0) M3_TRY(add(src[i], src_pitch[i], batch * S, dst == nullptr, "states"));
    if (dst) M3_TRY(add(dst[i], dst_pitch[i], batch * T, true, "out"));
    if (first < 0) first = i;
  }
  // ranges that meet may still be rows of one pitch that lie between each other, as views of a pool do
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
  for (const Range& r : ranges) {
    open.erase(std::remove_if(open.begin(), open.end(), [&](const Range& o) { return o.hi <= r.lo; }), open.end());
    for (const Range& o : open) {
      if (!o.written && !r.written) continue;
      const uintptr_t d = o.pitch > 0 ? (r.lo - o.lo) % (uintptr_t)o.pitch : 0;
      if (o.pitch != r.pitch || d < (uintptr_t)o.bytes || d + (uintptr_t)r.bytes > (uintptr_t)o.pitch)
        return fail(M3_ERR_INVALID_ARGUMENT, "states[" + std::to_string(r.index) + "]: shares memory with another tensor of the call");
    }
    open.push_back(r);
  }
  if (first < 0) return M3_OK;
  M3_TRY(check_device_ptr(parents->data, "parents"));
  M3_TRY(elem_aligned(parents, "parents"));
  if (S > 0) M3_TRY(check_device_ptr(src[first], "states"));
  if (dst) M3_TRY(check_device_ptr(dst[first], "out"));
  ReorderArgs a{count, src, dst ? dst : const_cast<void* const*>(src), row_bytes, src_pitch, dst ? dst_pitch : src_pitch, static_cast<const int64_t*>(parents->data),
                parents->stride[0], parents->stride[1], batch, S, T, dst == nullptr};
  return launch_reorder_states(a, reinterpret_cast<cudaStream_t>(stream));
} catch (const std::exception& e) {
  return fail(M3_ERR_INVALID_ARGUMENT, std::string("reorder_states: ") + e.what());
}

}  // extern "C"
