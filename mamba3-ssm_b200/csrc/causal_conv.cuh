// Short depthwise causal convolution: parameters of the launches (causal_conv.cu).
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <cuda_runtime.h>

namespace m3 {

struct ConvParams {
  const void* x; int64_t xb, xl;        // (batch, length, E), element strides of batch and length
  const void* w; int64_t we;            // (E, taps), stride of the channels
  const void* bias;                     // (E), w's type; may be null
  bool w_f32;                           // w and bias in fp32, else in x's type
  const void* init; int64_t ib, il;     // (batch, taps - 1, E): rows in front of the first; may be null
  const int64_t* lengths;               // (batch), may be null
  bool silu;
  void* y; int64_t yb, yl;
  void* last;                           // (batch, taps - 1, E) contiguous: the last rows; may be null
  int batch, L, E;
  int run;                              // rows that a warp walks
  bool vec;                             // a lane's channels are moved at once
};

struct ConvGrads {
  const void* dy; int64_t dyb, dyl;
  const void* dlast; int64_t dlb, dll;  // gradient of the last rows, may be null
  void* dx; int64_t dxb, dxl;
  void* dw;                             // (E, taps) contiguous, w's type
  void* dbias;                          // (E), w's type; may be null
  void* dinit;                          // (batch, taps - 1, E) contiguous, may be null
  float* part;                          // (parts, taps + 1, E)
};

struct ConvStepParams {
  void* state; int64_t sb, sl;          // (batch, taps - 1, E), in place
  const void* x; int64_t xb;
  const void* w; int64_t we;
  const void* bias;
  bool w_f32, silu;
  void* y;                              // (batch, E) contiguous
  int64_t batch; int E;
  bool vec;                             // a lane's channels are moved at once
};

int launch_conv_fwd(ConvParams p, int taps, int dtype, cudaStream_t s);
size_t conv_bwd_workspace(int64_t batch, int64_t L, int64_t E, int taps);
int launch_conv_bwd(ConvParams p, ConvGrads g, int taps, int dtype, void* ws, cudaStream_t s);
int launch_conv_step(ConvStepParams p, int taps, int dtype, cudaStream_t s);

}  // namespace m3
