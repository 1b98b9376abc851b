// Global norm of many gradient tensors, and their scaling and clipping.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <cuda_runtime.h>

namespace m3 {

struct ClipArgs {
  int64_t count;
  const void* const* grads;    // host array of device pointers
  const int64_t* numel;
  const int32_t* dtypes;       // of the gradients
  void* const* outs;           // null: in place
  const int32_t* out_dtypes;
  bool largest;                // the largest magnitude in place of the 2-norm
  double max_norm, scale;
  bool in_place;               // outs are null or the gradients themselves
  bool norm_alone;             // nothing is written but the norm
  float* norm;                 // device, one value
};

size_t clip_grads_workspace_bytes(int64_t count);
int launch_clip_grads(const ClipArgs& a, void* ws, cudaStream_t s);

}  // namespace m3
