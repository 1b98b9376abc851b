// Beam search: selection over beams and vocabulary (beam_select.cu) and the moves of the beams'
// states (reorder_states.cu).
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <cuda_runtime.h>

namespace m3 {

constexpr int kMaxBeams = 32;       // of one prompt
constexpr int kMaxCandidates = 64;  // selected of one prompt
constexpr int kMaxVocab = 1 << 24;

struct BeamParams {
  const void* logits; int64_t lb, lk;    // (batch, beams, V), element strides
  const float* scores; int64_t sb, sk;   // (batch, beams)
  const uint8_t* finished; int64_t fb, fk;  // (batch, beams), may be null
  int64_t batch;
  int beams, V, num, end_token;
  float* out_scores;                     // (batch, num) contiguous, as are the next two
  int64_t* parents;
  int64_t* tokens;
};

size_t beam_workspace_bytes(int64_t batch, int beams, int V, int num, int dtype, int sms);
int launch_beam_select(const BeamParams& p, int dtype, void* ws, cudaStream_t s);

struct ReorderArgs {
  int64_t count;               // tensors
  const void* const* src;
  void* const* dst;            // dst[i] == src[i]: in place
  const int64_t* row_bytes;
  const int64_t* src_pitch;    // bytes from row to row
  const int64_t* dst_pitch;
  const int64_t* parents; int64_t pb, pk;  // (batch, rows), element strides
  int64_t batch, source, rows; // rows of a group at the source and of its parents
  bool in_place;
};

int launch_reorder_states(const ReorderArgs& a, cudaStream_t s);

}  // namespace m3
