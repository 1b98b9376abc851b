// Book-keeping of a warp that copies rows piece by piece, one mbarrier a piece whose phase a copy
// completes. Plain integers, so that it also compiles for the host.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define M3_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define M3_HOST_DEVICE inline
#endif

namespace m3 {

struct CopyRounds {
  uint32_t round = 0;   // the present row
  uint32_t issued = 0;  // its pieces whose copy is under way

  M3_HOST_DEVICE void issue(int piece) { issued |= 1u << piece; }
  // to the next row, of which nothing is under way yet
  M3_HOST_DEVICE void next() {
    ++round;
    issued = 0;
  }
  // Whether the piece was copied at all, and the parity of the phase that its last copy completes:
  // of the present row, or of the one before.
  M3_HOST_DEVICE bool copied(int piece) const { return round > 0 || (issued >> piece & 1) != 0; }
  M3_HOST_DEVICE uint32_t last_phase(int piece) const {
    return ((issued >> piece & 1) != 0 ? round : round + 1) & 1;
  }
};

}  // namespace m3
