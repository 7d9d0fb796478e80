// Orthogonalised matrices: what the kernel over the whole GPU (orth.cu) and the one on the chip (orth_small.cu) share.
#pragma once

#include "dtypes.cuh"

namespace mb {

constexpr int OR_STEPS = 16;                      // most steps
constexpr float OR_SA = 4096.f, OR_SB = 256.f;    // scales of the fp16 planes of A and of b A + c A A
constexpr double OR_GROW = 8.0;
constexpr unsigned long long OR_WAIT = 2000000000ull;

struct OrPoly {
  int32_t steps;
  float a[OR_STEPS], b[OR_STEPS], c[OR_STEPS];
  uint32_t grow;                                  // bit k: what step k leaves in weak directions still grows by more than OR_GROW
  float s, inv_s;                                 // scale of X
  double eps;
};

// a X + e X + (the products' part), for a diagonal entry e of b A + c A A; GROW: e times X as the products read it
template <bool GROW>
__device__ __forceinline__ float or_update(float ca, float e, float x, float acc) {
  return GROW ? fmaf(ca, x, fmaf(e, __half2float(__float2half_rn(x)), acc)) : fmaf(ca + e, x, acc);
}

// Whether orth_small_launch takes the shape; out: bf16 [batch][m][n]
bool orth_small(int64_t batch, int32_t m, int32_t n);
int orth_small_launch(const void* g, int64_t ldb, int64_t ldg, void* out, int64_t batch, int32_t m, int32_t n, const OrPoly& poly,
                      int32_t dtype, cudaStream_t st);

}  // namespace mb
