// What the norms share.
#pragma once

#include "dtypes.cuh"

namespace mb {

// dw[j] = sum over nb rows of partial[row][0][j], db[j] = of partial[row][1][j] (d columns, type ptype, either may be null), in a
// fixed order
int col_sums(const float* partial, int nb, int32_t d, void* dw, void* db, int ptype, cudaStream_t st);

}  // namespace mb
