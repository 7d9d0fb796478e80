// Expert products: what the planning / data-movement kernels (experts.cu) and the tensor-core kernel
// (experts_gemm.cu) share.
#pragma once

#include "dtypes.cuh"

namespace mb {

// Layout of a plan (int32 words) for R slots and E experts.  The slots of one expert become consecutive rows, padded to
// whole tiles of XP_BM rows, so that a tile belongs to one expert.
constexpr int XP_BM = 128;                       // rows of a tile
constexpr int XP_CHUNK = 2048;                   // slots per block of the counting and placing kernels
struct XPlan {
  int64_t R;
  int32_t E, nblk;
  int64_t tiles;                                 // most tiles there can be
  int64_t o_seg, o_cnt, o_order, o_tile, o_pair, o_row, o_slot, o_hist, words;
};
// header words: 0 = tiles in use, 1 = status bits, 2 = pairs of tiles in use
inline XPlan xplan(int64_t R, int32_t E) {
  XPlan p;
  p.R = R;
  p.E = E;
  p.nblk = (int32_t)((R + XP_CHUNK - 1) / XP_CHUNK);
  p.tiles = R / XP_BM + (R < E ? R : E);
  p.o_seg = 8;                                   // [E + 1] first row of each expert
  p.o_cnt = p.o_seg + E + 1;                     // [E] slots of each expert
  p.o_order = p.o_cnt + E;                       // [E] experts, most slots first (ties: lowest index)
  p.o_tile = p.o_order + E;                      // [tiles] expert of each tile
  p.o_pair = p.o_tile + p.tiles;                 // [tiles] first tile of each pair of an expert's tiles
  p.o_row = p.o_pair + p.tiles;                  // [tiles * XP_BM] slot of each row, -1 = padding
  p.o_slot = p.o_row + p.tiles * XP_BM;          // [R] row of each slot, -1 = no expert
  p.o_hist = p.o_slot + R;                       // [E][nblk] scratch
  p.words = p.o_hist + (int64_t)E * p.nblk;
  return p;
}

enum { XG_FWD = 0, XG_DGRAD = 1, XG_WGRAD = 2 };

// One launch of the tensor-core kernel.  Operands are 16-bit planes (fp32 data: three bf16 planes; WGRAD with `split`: two of
// b, and of a where the data is fp16).
//   FWD    rows of `a` [planes][rows][lda] (expert-sorted), b = w [planes][E][O][ldb]: C[row][o] = sum_d a[row][d] w[e][o][d]
//   DGRAD  the same rows with width O, b = w: C[row][d] = sum_o a[row][o] w[e][o][d]
//   WGRAD  a [planes][rows][lda] (width M = O), b [planes][rows][ldb] (width N = D): C[e][o][d] = sum over e's rows
struct XGemm {
  int mode, dtype;
  const void *a, *b;
  int64_t rows, lda, ldb;                        // rows per plane; strides in elements, multiples of 8
  int32_t E, M, N, K;                            // WGRAD: M = O, N = D; else N, K of the product
  const int32_t* plan;
  XPlan lay;
  const float* scale;                            // per slot, or null
  void* out;                                     // FWD / DGRAD: [slots][ldo] (null: only dgpart); WGRAD: [E][M][N]
  int64_t ldo;
  int32_t out32;                                 // FWD / DGRAD: the rows leave in fp32 whatever dtype is (to be summed)
  int32_t split;                                 // WGRAD of 16-bit data: operands in bf16 planes
  int32_t kc;                                    // WGRAD: K blocks of a part (xgemm_kc)
  float* parts;                                  // WGRAD: xgemm_parts partial sums [M][N] (null: there are none)
  int32_t* pre;                                  // WGRAD with parts: [E + 1] scratch
  // DGRAD: dgpart[2 x n tile + half][slot] = partial <x, C> of the slot's x row (null: off)
  const void* x;
  int64_t ldx;
  int32_t kdiv;                                  // slot / kdiv = row of x
  float* dgpart;
};
int xgemm_n_tiles(int64_t N, int dtype);
int xgemm_kc(int64_t E, int64_t M, int64_t N, int64_t slots, int dtype);
int64_t xgemm_parts(int64_t E, int64_t slots, int kc);
int xgemm_launch(const XGemm& g, cudaStream_t st);

}  // namespace mb
