// Shared-memory staging of the tensor-core kernels' epilogues.
#pragma once

#include "tc.cuh"

namespace mb {

constexpr int XG_STG = 2048;                     // row staging of one epilogue warp

// Row staging of the epilogue: a warp's 32 rows x 64 bytes, 16-byte piece c of row r at piece c ^ (r / 2 % 4), so that a
// lane's access to its own row and the warp's access to eight whole row segments are both free of bank conflicts.
__device__ __forceinline__ uint32_t xg_stg(uint32_t stg, int row, int c) {
  return stg + row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
}
struct XgLane {
  uint32_t own[4], seg[4];                       // staging addresses: this lane's row, piece c; row 8 i + l / 4, piece l % 4
};
__device__ __forceinline__ XgLane xg_lane(uint32_t stg) {
  const int lane = threadIdx.x & 31;
  XgLane a;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a.own[i] = xg_stg(stg, lane, i);
    a.seg[i] = xg_stg(stg, 8 * i + (lane >> 2), lane & 3);
  }
  return a;
}

}  // namespace mb
