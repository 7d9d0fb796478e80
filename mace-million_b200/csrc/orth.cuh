// Orthogonalised matrices: what the kernel over the whole GPU (orth.cu) and the one on the chip (orth_small.cu) share.
#pragma once

#include "dtypes.cuh"

namespace mb {

constexpr int OR_STEPS = 16;                      // most steps
constexpr float OR_SA = 4096.f, OR_SB = 256.f;    // scales of the fp16 planes of A and of b A + c A A
constexpr unsigned long long OR_WAIT = 2000000000ull;

struct OrPoly {
  int32_t steps;
  float a[OR_STEPS], b[OR_STEPS], c[OR_STEPS];
  float s, inv_s;                                 // scale of X
  double eps;
};

// Whether orth_small_launch takes the shape; out: bf16 [batch][m][n]
bool orth_small(int64_t batch, int32_t m, int32_t n);
int orth_small_launch(const void* g, int64_t ldb, int64_t ldg, void* out, int64_t batch, int32_t m, int32_t n, const OrPoly& poly,
                      int32_t dtype, cudaStream_t st);

}  // namespace mb
