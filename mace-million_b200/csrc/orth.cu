// Orthogonalised matrices by Newton-Schulz products, for the updates of an optimiser (a batch of matrices [m][n]):
//   X = G / (|G|_F + eps);  per step  A = X X^T,  X <- a X + (b A + c A A) X   (m <= n; else A = X^T X, products from the right)
// so every singular value s moves to a s + b s^3 + c s^5, towards one.  The result is bf16.
//
// Products are tcgen05 kind::f16 with fp32 accumulators, on fp16 operands, which have three bits more than bf16.  Everything is bounded, and
// powers of two scale it into fp16's range: a polynomial whose values pass 3.5 (or 200 in b s^2 + c s^4) for the singular values that
// reach it, taken 2% larger, is refused, so X's entries are at most 3.5 (times 2^14 at most: 57,344 of 65,504), A's 12.8 (times 4096: 52,300)
// and those of b A + c A A 200 (times 256: 51,200).  What is rounded, and why that is enough (fp64 simulation and
// measurement, Frobenius error before the last rounding 2e-4 to 1.2e-3, of a bf16 result that rounds by 1.7e-3; 2e-3 for 2 x 2 matrices, the
// worst of millions of which was 1.6% off, where no errors average out):
//  * X itself stays in fp32, and the term a X is taken from that.  An error added to X grows by up to a^steps (485) in its weak
//    directions: with X in fp16 a matrix of rank 8 over noise was 0.04 off.
//  * The products read X rounded to fp16.  An error of the left factor (A, B = b A + c A A) multiplies X, and the polar factor of
//    (1 + E) X differs by |E| whatever the singular values; what B X loses lies in the strong directions, which do not grow.  That
//    holds for the whole of B: its diagonal alone has weak directions, too, so while they still grow by more than 8 (OR_GROW; the
//    first three of five steps) the diagonal's term takes the same rounded X.  With the fp32 X there 4 x 64 matrices of rank 1 over
//    noise of 1e-3 were 2.7% off, now 0.1%; 16 x 128 1.6% and 0.08%.  In the last steps the fp32 X is better (random 128 x 512 4.6e-4
//    in every step, 7.9e-4 in the last two, 1.2e-3 in none).
//  * The diagonals of A and of b A + c A A dominate them and stay apart in fp32: A = A1 + D gives A A = A1 A1 + A1 D + D A1 + D D, and
//    the diagonal of the second multiplies X in the epilogue.  In the planes they cost 2 to 9 times the error.
//  * The tensor cores truncate when they add: a diagonal loses 1e-7 of itself per 16 terms, 4e-4 at MB_ORTH_MAX_DIM.
//
// A and A A are symmetric: only tiles that reach the diagonal or lie above it are multiplied, and stored to both places.
// The fp32 X lies in pieces of 32 x 32 in the order in which the epilogue's lanes hold them (its reads and writes are whole
// 512 bytes, in place); the fp16 planes that TMA reads are row-major and are written through shared memory in 64-byte rows.
// One cooperative kernel runs all steps: persistent CTAs, one per SM, 3 phases a step with a barrier over the grid between them
// (separate launches cost a pipeline's fill and drain each).  Warp 0 loads with TMA, warp 1 issues, warps 4-11 drain one of two
// accumulators.  Tall matrices are not transposed: their Gram product reads both operands MN-major.  Two small kernels before
// it take the norm (sums of squares in fp64) and split G into the planes.
// Every wait is bounded; after one expires the grid stops and the tiles of the result that have none are NaN.
//
// Measured on a B200 (5 steps, bf16 matrices, all launches; rates count half of the symmetric products): 4096 x 4096 1.17 ms
// (1.17 PFLOP/s; 2 or 4 rounds of tiles a phase for 1.8 and 3.5 rounds' worth, and a drain and a barrier of 15 us at each of 15 phases'
// ends), 2048 x 2048 238 us, 1024 x 1024 121 us and 3 of 515 x 1023 134 us: 8 to 9 us a phase, of which 3 are products, 2 the drain, 3 the
// stores' way to memory and the grid's barrier, 1 the first loads; 16 of 1024 x 1024 560 us (X, its planes, A and B are 190 MB, more
// than L2 holds).
#include <cuda.h>

#include <type_traits>

#include "dtypes.cuh"
#include "epilogue.cuh"
#include "orth.cuh"
#include "tc.cuh"
#include "tensor_map.cuh"

namespace mb {

constexpr int OR_EPI0 = 4, OR_EPI = 8, OR_THREADS = 32 * (OR_EPI0 + OR_EPI), OR_BK = 64,
              OR_WORDS = 1 + 3 * OR_STEPS;
constexpr int OR_BOX = 64 * OR_BK * 2;            // bytes of one 64 x 64 box: operands are loaded in those
constexpr int OR_PARTS = 256;                     // most partial sums of squares of a matrix

enum { OR_GRAM = 0, OR_SQUARE = 1, OR_UPDATE = 2 };
struct OrPhase {
  int32_t bn, ti, tj, per, nk, a_mn, b_mn, tri;   // columns of a tile, tiles, per matrix, K blocks; operands' layouts
  int32_t M, N, bm;                               // bm: rows of a tile
};
struct OrArgs {
  int32_t m, n, r, batch, tall, stages, stage_bytes, vec_out;
  int32_t ci, cj;                                 // pieces of X along rows and columns
  int64_t ldx, ldr, px, pr, pc;                   // row strides of the planes, elements of a matrix in them and in the pieces
  OrPoly poly;
  OrPhase ph[3];
  f16 *hi[2], *A, *B;
  float* X;
  float *d, *e;                                   // diagonals [batch][r]
  bf16* out;
  unsigned* words;                                // failed, then the CTAs that are through with each phase
};

// ------------------------------------------------------------------------------------------------ norm and planes
template <typename T>
__global__ void __launch_bounds__(256) k_orth_norm(const T* g, int64_t ldb, int64_t ldg, int32_t m, int32_t n, bool vec,
                                                   double* part, unsigned* words) {
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < OR_WORDS) words[threadIdx.x] = 0u;
  constexpr int V = kVec<T>;
  const T* p = g + blockIdx.y * ldb;
  double s = 0.0;
  const int w = vec ? n / V : n;                  // accesses of a row
  const int64_t all = (int64_t)m * w, step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += step) {
    const int64_t row = i / w, c = i - row * w;
    if (vec) {
      float f[V];
      load_v<T, V>(p + row * ldg + c * V, f);
#pragma unroll
      for (int q = 0; q < V; ++q) s = fma((double)f[q], (double)f[q], s);
    } else {
      const double f = to_f(p[row * ldg + c]);
      s = fma(f, f, s);
    }
  }
  __shared__ double red[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int q = 1; q < 8; ++q) s += red[q];
    part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = s;
  }
}

// X = S G / (|G| + eps): pieces of 32 x 32 in fp32 and the fp16 plane; a warp per piece, a lane holds eight columns of four rows
template <typename T>
__global__ void __launch_bounds__(256) k_orth_split(const T* g, int64_t ldb, int64_t ldg, bool vec, const double* part, int np,
                                                    const OrArgs a) {
  __shared__ double red[8];
  double s = (int)threadIdx.x < np ? part[(int64_t)blockIdx.y * np + threadIdx.x] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
  for (int q = 0; q < 8; ++q) s += red[q];
  const float scale = (float)((double)a.poly.s / (sqrt(s) + a.poly.eps));
  const int lane = threadIdx.x & 31, c8 = (lane & 3) * 8;
  const T* p = g + blockIdx.y * ldb;
  f16* h = a.hi[0] + blockIdx.y * a.px;
  float* X = a.X + blockIdx.y * a.pc;
  const int pieces = a.ci * a.cj;
  for (int t = blockIdx.x * 8 + (threadIdx.x >> 5); t < pieces; t += gridDim.x * 8) {
    const int r0 = t / a.cj * 32, c = t % a.cj * 32 + c8;
    float4* x = reinterpret_cast<float4*>(X + (int64_t)t * 1024);
    float f[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = r0 + 8 * i + (lane >> 2);
      const T* q = p + row * ldg + c;
#pragma unroll
      for (int k = 0; k < 8; ++k) f[i][k] = 0.f;
      if (row >= a.m) continue;
      if (vec && c + 8 <= a.n) {
        if constexpr (sizeof(T) == 4) {
          float u[4], v[4];
          load_v<T, 4>(q, u);
          load_v<T, 4>(q + 4, v);
#pragma unroll
          for (int k = 0; k < 4; ++k) f[i][k] = u[k], f[i][4 + k] = v[k];
        } else {
          load_v<T, 8>(q, f[i]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c + k < a.n) f[i][k] = to_f(q[k]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 2);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[i][k] *= scale;
      x[c8 / 4 * 32 + r] = make_float4(f[i][0], f[i][1], f[i][2], f[i][3]);
      x[(c8 / 4 + 1) * 32 + r] = make_float4(f[i][4], f[i][5], f[i][6], f[i][7]);
      if (r0 + r < a.m && c < a.n) *reinterpret_cast<uint4*>(h + (r0 + r) * a.ldx + c) = pack16<f16>(f[i]);
    }
  }
}

// ------------------------------------------------------------------------------------------------ the steps
struct OrBars {
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2], phase;
  uint32_t tmem;
  int failed, never;                              // never: a flag that stays 0
};
struct OrMaps {
  CUtensorMap a[2][3], b[2][3];                   // operands of each phase, by the parity of the step
};
struct OrTile {
  int b, m0, n0;
};
__device__ __forceinline__ OrTile or_tile(const OrPhase& p, int t) {
  OrTile o;
  o.b = t / p.per;
  t -= o.b * p.per;
  int i;
  if (p.tri) {                                    // row of tiles i starts at the tile that holds its diagonal
    i = 0;
    for (int left = p.tj; t >= left; ++i) {
      t -= left;
      left = p.tj - (i + 1) * p.bm / p.bn;
    }
    t += i * p.bm / p.bn;
  } else {
    i = t / p.tj;
    t -= i * p.tj;
  }
  o.m0 = i * p.bm;
  o.n0 = t * p.bn;
  return o;
}

__device__ __forceinline__ unsigned ld_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// Waits until every CTA is through with the phase (each phase counts for itself: CTAs without tiles run ahead); false on a failure
// anywhere or when the limit is over.  For a whole warp.
__device__ __forceinline__ bool or_wait(const OrArgs& g, int phase) {
  unsigned long long t0 = 0;
  for (unsigned it = 0;; ++it) {
    if (__all_sync(0xffffffffu, ld_acquire(g.words + 1 + phase) >= gridDim.x)) break;
    if ((it & 15u) == 15u && __any_sync(0xffffffffu, ld_acquire(g.words))) return false;
    if ((it & 255u) == 255u) {
      const unsigned long long now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      if (__any_sync(0xffffffffu, now - t0 > OR_WAIT)) return false;
    }
  }
  asm volatile("fence.proxy.async;" ::: "memory");  // what others stored is read by TMA
  return true;
}

// Writes the 32 x 32 values that a warp holds (lane = row) through shared memory in 64-byte rows: rows [0, rows) and columns
// [0, nc) of dst.  PAD: the memory goes on to whole pieces of eight columns; else vec says that rows of eight are aligned.
template <typename OUT, bool PAD>
__device__ __forceinline__ void or_put(const float (&v)[32], const XgLane& a, uint32_t stg, OUT* dst, int64_t ld, int rows, int nc,
                                       bool vec) {
  const int lane = threadIdx.x & 31, c8 = (lane & 3) * 8;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float f[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = v[8 * c + q];
    sts128(a.own[c], pack16<OUT>(f));
  }
  __syncwarp();
  if (PAD || (vec && nc == 32)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 2);
      if (r < rows && c8 < nc) *reinterpret_cast<uint4*>(dst + r * ld + c8) = lds128(a.seg[i]);
    }
  } else {
    for (int r = 0; r < rows; ++r)
      if (lane < nc) {
        const uint16_t u = lds16(xg_stg(stg, r, lane / 8) + 2 * (lane & 7));
        dst[r * ld + lane] = *reinterpret_cast<const OUT*>(&u);
      }
  }
  __syncwarp();
}

template <int CG>
__global__ void __launch_bounds__(OR_THREADS, 1)
    k_orth(const __grid_constant__ OrMaps maps, const __grid_constant__ OrArgs g) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* stg0 = smem + g.stages * g.stage_bytes;
  OrBars& B = *reinterpret_cast<OrBars*>(stg0 + OR_EPI * XG_STG);
  volatile int* failed = &B.failed;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = CG == 2 ? (int)cluster_ctarank() : 0, cta = blockIdx.x / CG, ctas = gridDim.x / CG;
  if (warp == 1) {
    tmem_alloc<CG>(&B.tmem, 512);
    if (lane == 0) {
      for (int s = 0; s < 8; ++s) {
        mbar_init(&B.full[s], 1);
        mbar_init(&B.empty[s], 1);
      }
      for (int a = 0; a < 2; ++a) {
        mbar_init(&B.acc_full[a], 1);
        mbar_init(&B.acc_empty[a], OR_EPI * CG);
      }
      mbar_init(&B.phase, 1);
      B.failed = B.never = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();          // the peer's barriers are initialised
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = B.tmem;
  const int phases = 3 * g.poly.steps;

  // Warps 0 and 1 go through their loops as a whole with uniform values, and everything of a phase is in registers: parameters
  // behind asm with a memory clobber are read again each time.
  if (warp == 0) {
    // ------------------------------------------------------------------------------------------ loads
    const uint32_t lead = elect_lane();
    const int stages = g.stages, stage_bytes = g.stage_bytes;
    const uint32_t smem0 = smem_u32(smem), full0 = smem_u32(B.full), empty0 = smem_u32(B.empty);
    const uint32_t target = CG == 2 ? mapa_u32(full0, 0) : full0;
    int s = 0;
    uint32_t par = 1;                             // parity of the ring's free places
    bool ok = true, wrapped = false;
    for (int ph = 0; ok && ph < phases; ++ph) {
      const OrPhase p = g.ph[ph % 3];
      const int tiles = g.batch * p.per, nk = p.nk, bh = p.bn / CG;   // bh: columns of B that this CTA loads
      const CUtensorMap *ma = &maps.a[(ph / 3) & 1][ph % 3], *mb = &maps.b[(ph / 3) & 1][ph % 3];
      const uint32_t bytes = CG * (uint32_t)(2 + bh / 64) * OR_BOX;
      const int adx = p.a_mn ? 0 : OR_BK, ady = p.a_mn ? OR_BK : 0, bdx = p.b_mn ? 0 : OR_BK, bdy = p.b_mn ? OR_BK : 0;
      OrTile w{};
      if (cta < tiles) w = or_tile(p, cta);       // before the wait, not after it
      if (ph > 0) {
        ok = or_wait(g, ph - 1);
        if (!ok) *failed = 1;
        if (lead) mbar_arrive(&B.phase);          // the epilogue may read what the phase before wrote
      }
      for (int t = cta; ok && t < tiles; t += ctas) {
        // coordinates: K-major (k, row, 0, matrix), MN-major (0, k, column / 64, matrix)
        const int m0 = w.m0 + rank * 128, n0 = w.n0 + rank * bh;
        int ax = 0, ay = p.a_mn ? 0 : m0, bx = 0, by = p.b_mn ? 0 : n0;
        const int az = p.a_mn ? m0 / 64 : 0, bz = p.b_mn ? n0 / 64 : 0;
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait_warp(empty0 + 8 * s, par, OR_WAIT, failed)) {
            *failed = 1;
            ok = false;
            break;
          }
          const uint32_t a = smem0 + s * stage_bytes;
          // both CTAs' bytes arrive at the first one's barrier
          mbar_arrive_tx_lead(rank == 0 ? lead : 0u, full0 + 8 * s, bytes);
          tma_load_4d_lead<CG>(lead, a, ma, ax, ay, az, w.b, target + 8 * s);
          tma_load_4d_lead<CG>(lead, a + 2 * OR_BOX, mb, bx, by, bz, w.b, target + 8 * s);
          ax += adx;
          ay += ady;
          bx += bdx;
          by += bdy;
          if (++s == stages) s = 0, par ^= 1, wrapped = true;
        }
        if (t + ctas < tiles) w = or_tile(p, t + ctas);
      }
    }
    if (!ok && rank == 0)                         // copies in flight land before the block ends (bounded)
      for (int q = 0; q < stages; ++q) {          // places before s: this round's, the others: the round before
        if (q >= s && !wrapped) break;
        mbar_wait_ns(&B.full[q], q < s ? par ^ 1 : par, OR_WAIT);
      }
  } else if (warp == 1) {
    // ------------------------------------------------------------------------------------------ MMA issue
    if (rank == 0) {
      const uint32_t lead = elect_lane();
      const int stages = g.stages, stage_bytes = g.stage_bytes;
      const uint32_t smem0 = smem_u32(smem), full0 = smem_u32(B.full), empty0 = smem_u32(B.empty);
      const uint32_t acc_full0 = smem_u32(B.acc_full), acc_empty0 = smem_u32(B.acc_empty);
      int s = 0, acc = 0;
      uint32_t par = 0, acc_par = 1, last_bar = 0, last_par = 0;
      bool ok = true;
      for (int ph = 0; ok && ph < phases; ++ph) {
        const OrPhase p = g.ph[ph % 3];
        const int tiles = g.batch * p.per, nk = p.nk;
        const uint32_t idesc = f16_idesc(128 * CG, p.bn, false, p.a_mn, p.b_mn);
        // 16 K elements are 32 bytes of a K-major row, or two 8-row atoms of an MN-major operand
        const uint64_t a_base = p.a_mn ? sw128_desc_mn(smem0, OR_BOX) : sw128_desc(smem0);
        const uint64_t b_base = p.b_mn ? sw128_desc_mn(smem0 + 2 * OR_BOX, OR_BOX) : sw128_desc(smem0 + 2 * OR_BOX);
        const uint32_t a_lo = (uint32_t)a_base, a_hi = (uint32_t)(a_base >> 32), b_lo = (uint32_t)b_base, b_hi = (uint32_t)(b_base >> 32);
        const int a_step = (p.a_mn ? 2048 : 32) >> 4, b_step = (p.b_mn ? 2048 : 32) >> 4;
        for (int t = cta; ok && t < tiles; t += ctas) {
          if (!mbar_wait_warp(acc_empty0 + 8 * acc, acc_par, OR_WAIT, failed)) {
            *failed = 1;
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t d = tmem + acc * 256;
          bool here = false;                      // the next K block, looked for while this one's products are issued
          for (int kb = 0; kb < nk; ++kb) {
            // the first wait of a phase includes the grid's barrier
            if (!here && !mbar_wait_warp(full0 + 8 * s, par, 2 * OR_WAIT, failed)) {
              *failed = 1;
              ok = false;
              break;
            }
            const uint32_t off = (uint32_t)(s * stage_bytes) >> 4, ad = a_lo + off, bd = b_lo + off;
            last_bar = empty0 + 8 * s;
            last_par = par;
            if (++s == stages) s = 0, par ^= 1;
            here = kb + 1 < nk && mbar_over_warp(full0 + 8 * s, par);
#pragma unroll
            for (int kk = 0; kk < OR_BK / 16; ++kk)
              mma_f16_ss_lead<CG>(lead, d, ad + kk * a_step, a_hi, bd + kk * b_step, b_hi, idesc, (kb | kk) ? 1u : 0u);
            mma_commit_lead<CG>(lead, last_bar);
          }
          if (!ok) break;
          mma_commit_lead<CG>(lead, acc_full0 + 8 * acc);
          last_bar = acc_full0 + 8 * acc;
          last_par = acc_par ^ 1;
          acc ^= 1;
          if (acc == 0) acc_par ^= 1;
        }
      }
      if (*failed && last_bar) mbar_wait_warp(last_bar, last_par, OR_WAIT, &B.never);
    }
  } else if (warp >= OR_EPI0) {
    // ------------------------------------------------------------------------------------------ epilogue
    const int q4 = warp & 3, hf = (warp - OR_EPI0) >> 2;
    const uint32_t stg = smem_u32(stg0) + (warp - OR_EPI0) * XG_STG;
    const XgLane at = xg_lane(stg);
    int tc = 0;
    bool lost = false;                            // warp-uniform
    for (int ph = 0; ph < phases; ++ph) {
      const int kind = ph % 3, step = ph / 3;
      const OrPhase p = g.ph[kind];
      const int tiles = g.batch * p.per, hw = p.bn / 2;
      const bool last = ph == phases - 1;
      const float ca = g.poly.a[step], cb = g.poly.b[step], cc = g.poly.c[step];
      if (ph > 0 && !lost) lost = !mbar_wait_warp(smem_u32(&B.phase), (ph - 1) & 1, 2 * OR_WAIT, failed);
      // after a failure only the result's tiles are gone through (every warp takes part in every phase's block barrier)
      for (int t = lost && !last ? tiles : cta; t < tiles; t += ctas, ++tc) {
        const OrTile w = or_tile(p, t);
        const int acc = tc & 1, i0 = w.m0 + rank * 128 + q4 * 32, i = i0 + lane, rows = p.M - i0 < 32 ? p.M - i0 : 32;
        float4 nx[8];                             // the next piece of X, or in the first four of A, on its way
        float dn = 0.f;                           // and the diagonal's entry of this lane's column
        const float* dvec = (kind == OR_UPDATE ? g.e : g.d) + (int64_t)w.b * g.r;
        const float di = !lost && (kind == OR_SQUARE || (kind == OR_UPDATE && !g.tall)) && lane < rows ? __ldcg(dvec + i) : 0.f;
        auto fetch = [&](int c) {
          const int j0 = w.n0 + hf * hw + c;
          if (lost || rows <= 0 || j0 >= p.N) return;
          if (kind == OR_SQUARE || (kind == OR_UPDATE && g.tall)) dn = j0 + lane < p.N ? __ldcg(dvec + j0 + lane) : 0.f;
          if (kind == OR_UPDATE) {
            const float4* x = reinterpret_cast<const float4*>(g.X + w.b * g.pc + ((int64_t)(i0 >> 5) * g.cj + (j0 >> 5)) * 1024);
#pragma unroll
            for (int q = 0; q < 8; ++q) nx[q] = __ldcg(x + 32 * q + lane);
          } else if (kind == OR_SQUARE) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int r = 8 * q + (lane >> 2), c8 = (lane & 3) * 8;
              nx[q] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (r < rows && j0 + c8 < p.N)
                nx[q] = __ldcg(reinterpret_cast<const float4*>(g.A + w.b * g.pr + (i0 + r) * g.ldr + j0 + c8));
            }
          }
        };
        fetch(0);
        if (!lost) lost = !mbar_wait_warp(smem_u32(&B.acc_full[acc]), (tc >> 1) & 1, 3 * OR_WAIT, failed);
        if (lost) {
          *failed = 1;
          if (!last) break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int c = 0; c < hw; c += 32) {
          const int j0 = w.n0 + hf * hw + c, nc = p.N - j0 < 32 ? p.N - j0 : 32;   // columns here (<= 0: none)
          const bool some = nc > 0 && rows > 0;   // warp-uniform
          uint32_t u[32];
          if (!lost) {
            tmem_ld32(tmem + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * 256 + hf * hw + c), u);
            tmem_wait_ld();
            if (c + 32 >= hw) {                   // the accumulator is free
              asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
              __syncwarp();
              if (lane == 0) {
                if constexpr (CG == 2)
                  mbar_arrive_remote(mapa_u32(smem_u32(&B.acc_empty[acc]), 0));
                else
                  mbar_arrive(&B.acc_empty[acc]);
              }
            }
          }
          if (!some) continue;
          float v[32];
          if (kind == OR_UPDATE) {
            if (lost) {
#pragma unroll
              for (int x = 0; x < 32; ++x) v[x] = __int_as_float(0x7fc00000);
            } else {
#pragma unroll
              for (int q = 0; q < 8; ++q) v[4 * q] = nx[q].x, v[4 * q + 1] = nx[q].y, v[4 * q + 2] = nx[q].z, v[4 * q + 3] = nx[q].w;
              const float el = dn;
              if (c + 32 < hw) fetch(c + 32);
              auto update = [&](auto grow) {
                constexpr bool GROW = decltype(grow)::value;
                if (g.tall) {
#pragma unroll
                  for (int x = 0; x < 32; ++x)
                    v[x] = or_update<GROW>(ca, __shfl_sync(0xffffffffu, el, x), v[x], __uint_as_float(u[x]) * (1.f / OR_SB));
                } else {
#pragma unroll
                  for (int x = 0; x < 32; ++x) v[x] = or_update<GROW>(ca, di, v[x], __uint_as_float(u[x]) * (1.f / OR_SB));
                }
              };
              if (g.poly.grow >> step & 1)
                update(std::true_type());
              else
                update(std::false_type());
            }
            if (last) {
#pragma unroll
              for (int x = 0; x < 32; ++x) v[x] *= g.poly.inv_s;
              or_put<bf16, false>(v, at, stg, g.out + ((int64_t)w.b * g.m + i0) * g.n + j0, g.n, rows, nc, g.vec_out);
            } else {
              float4* x = reinterpret_cast<float4*>(g.X + w.b * g.pc + ((int64_t)(i0 >> 5) * g.cj + (j0 >> 5)) * 1024);
#pragma unroll
              for (int q = 0; q < 8; ++q) __stcg(x + 32 * q + lane, make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]));
              or_put<f16, true>(v, at, stg, g.hi[(step & 1) ^ 1] + w.b * g.px + i0 * g.ldx + j0, g.ldx, rows, nc, true);
            }
          } else {
            f16* dst = (kind == OR_GRAM ? g.A : g.B) + w.b * g.pr;
            float* diag = (kind == OR_GRAM ? g.d : g.e) + (int64_t)w.b * g.r;
            const bool on = i0 == j0;             // the diagonal runs through this piece: column x = lane
            float dia = 0.f;
            if (kind == OR_GRAM) {
              const float sc = g.poly.inv_s * g.poly.inv_s * OR_SA;
#pragma unroll
              for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(u[x]) * sc;
            } else {
              // b a1 + c (a1 (d_i + d_j) + sq), all times SB: a1's plane is SA a1, the accumulator SA^2 sq
              const float k2 = cc * (OR_SB / OR_SA), k1 = fmaf(k2, di, cb * (OR_SB / OR_SA)), k3 = cc * (OR_SB / (OR_SA * OR_SA));
              const float dl = k2 * dn;
#pragma unroll
              for (int q = 0; q < 4; ++q) sts128(at.seg[q], *reinterpret_cast<const uint4*>(&nx[q]));
              __syncwarp();
              if (c + 32 < hw) fetch(c + 32);
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float f[8];
                unpack16(lds128(at.own[q]), f, f16());
#pragma unroll
                for (int x = 0; x < 8; ++x)
                  v[8 * q + x] = fmaf(f[x], k1 + __shfl_sync(0xffffffffu, dl, 8 * q + x), __uint_as_float(u[8 * q + x]) * k3);
              }
              __syncwarp();
            }
            if (on) {
#pragma unroll
              for (int x = 0; x < 32; ++x)
                if (x == lane) dia = v[x], v[x] = 0.f;
              if (lane < rows)
                diag[i] = kind == OR_GRAM ? dia * (1.f / OR_SA) : fmaf(cb, di, fmaf(cc * di, di, dia * (1.f / OR_SB)));
            }
            or_put<f16, true>(v, at, stg, dst + i0 * g.ldr + j0, g.ldr, rows, nc, true);
            // and to the other side of the diagonal, where no tile is computed
            if (i0 < j0 / p.bm * p.bm / p.bn * p.bn) {
#pragma unroll
              for (int x = 0; x < 32; ++x)
                sts16(xg_stg(stg, x, lane >> 3) + 2 * (lane & 7), __half_as_ushort(__float2half_rn(v[x])));
              __syncwarp();
              const int c8 = (lane & 3) * 8;
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int x = 8 * q + (lane >> 2);
                if (x < nc && c8 < rows) *reinterpret_cast<uint4*>(dst + (j0 + x) * g.ldr + i0 + c8) = lds128(at.seg[q]);
              }
              __syncwarp();
            }
          }
        }
      }
      if (!last) {                                // this CTA's part of the phase is in memory
        asm volatile("bar.sync 1, %0;" ::"n"(32 * OR_EPI) : "memory");
        if (tid == 32 * OR_EPI0) {
          if (*failed)                            // and nobody gets past this phase
            atomicExch(g.words, 1u);
          else
            asm volatile("fence.acq_rel.gpu;\n\tred.release.gpu.global.add.u32 [%0], 1;" ::"l"(g.words + 1 + ph) : "memory");
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();          // no CTA leaves while its peer can still signal it or read its operands
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_dealloc<CG>(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------------ host side
struct OrLayout {
  int64_t ldx, ldr, px, pr, pc, hi, plane, X, A, B, d, e, part, words, bytes;
};
static OrLayout or_layout(int64_t batch, int64_t m, int64_t n) {
  OrLayout l{};
  const int64_t r = m < n ? m : n;
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  l.ldx = (n + 63) / 64 * 64;                     // MN-major boxes read 64 columns, whatever lies behind the last
  l.ldr = (r + 7) / 8 * 8;
  l.px = m * l.ldx;
  l.pr = r * l.ldr;
  l.plane = up(batch * l.px * 2);
  l.pc = ((m + 31) / 32) * ((n + 31) / 32) * 1024;
  l.hi = 0;                                       // two planes
  l.X = 2 * l.plane;
  l.A = l.X + up(batch * l.pc * 4);
  l.B = l.A + up(batch * l.pr * 2);
  l.d = l.B + up(batch * l.pr * 2);
  l.e = l.d + up(batch * r * 4);
  l.part = l.e + up(batch * r * 4);
  l.words = l.part + up(batch * OR_PARTS * 8);
  l.bytes = l.words + 256;
  return l;
}

// Tiles of a phase: the width whose rounds over the CTAs (or pairs) take least.  A K block takes about 540, 320 or 230 cycles at
// 256, 128 and 64 columns (of one CTA; pairs' tiles are twice as high), and a tile's start and drain as much as ten.
static void or_cut(OrPhase& p, int64_t batch, int M, int N, int K, bool tri, int cg) {
  p.M = M;
  p.N = N;
  p.bm = 128 * cg;
  p.nk = (K + OR_BK - 1) / OR_BK;
  p.tri = tri;
  p.ti = (M + p.bm - 1) / p.bm;
  const int units = sm_count() / cg;
  double least = 0.0;
  for (int bn = 256; bn >= 64 * cg; bn /= 2) {
    const int tj = (N + bn - 1) / bn;
    int64_t per = 0;
    for (int i = 0; i < p.ti; ++i) per += tri ? tj - i * p.bm / bn : tj;
    const double cost = (double)((batch * per + units - 1) / units) * (p.nk + 10) * (bn == 256 ? 540 : bn == 128 ? 320 : 230);
    if (bn == 256 || cost < least) {
      least = cost;
      p.bn = bn;
      p.tj = tj;
      p.per = (int)per;
    }
  }
}

template <typename T>
static int orth_go(const void* gp, int64_t ldb, int64_t ldg, const OrArgs& a, double* part, cudaStream_t st) {
  constexpr int V = kVec<T>;
  const bool vec = a.n % V == 0 && ldg % V == 0 && ldb % V == 0 && aligned16(gp);
  const int64_t work = ((int64_t)a.m * a.n + 8 * 256 - 1) / (8 * 256), fill = (4 * (int64_t)sm_count() + a.batch - 1) / a.batch;
  int64_t np = work < fill ? work : fill;
  if (np > OR_PARTS) np = OR_PARTS;
  k_orth_norm<T><<<dim3((unsigned)np, a.batch), 256, 0, st>>>((const T*)gp, ldb, ldg, a.m, a.n, vec, part, a.words);
  if (int rc = check_launch("orthogonalize (norm)")) return rc;
  const bool vec8 = ldg % V == 0 && ldb % V == 0 && aligned16(gp);
  const int64_t pieces = ((int64_t)a.ci * a.cj + 7) / 8;
  k_orth_split<T><<<dim3((unsigned)(pieces < 2 * fill ? pieces : 2 * fill), a.batch), 256, 0, st>>>((const T*)gp, ldb, ldg, vec8, part,
                                                                                             (int)np, a);
  return check_launch("orthogonalize (planes)");
}

template <int CG>
static int orth_steps(OrArgs& a, int r, int len, cudaStream_t st) {
  or_cut(a.ph[OR_GRAM], a.batch, r, r, len, true, CG);
  or_cut(a.ph[OR_SQUARE], a.batch, r, r, r, true, CG);
  or_cut(a.ph[OR_UPDATE], a.batch, a.m, a.n, r, false, CG);
  a.ph[OR_GRAM].a_mn = a.ph[OR_GRAM].b_mn = a.tall;
  a.ph[OR_UPDATE].b_mn = !a.tall;
  int64_t most = 0;
  int bn = 64;
  for (const OrPhase& p : a.ph) {
    const int64_t tiles = (int64_t)a.batch * p.per;
    if (tiles > most) most = tiles;
    if (p.bn > bn) bn = p.bn;
  }
  if (most > 0x7fffffff) {
    set_error("orthogonalize: too many tiles (%lld)", (long long)most);
    return MB_E_ARG;
  }
  a.stage_bytes = (2 + bn / CG / 64) * OR_BOX;
  a.stages = 196608 / a.stage_bytes < 8 ? 196608 / a.stage_bytes : 8;
  OrMaps maps;
  for (int q = 0; q < 2; ++q)
    for (int kind = 0; kind < 3; ++kind)
      for (int side = 0; side < 2; ++side) {
        const bool is_x = kind == OR_GRAM || (kind == OR_UPDATE && (side == 0) == a.tall), mn = side ? a.ph[kind].b_mn : a.ph[kind].a_mn;
        const void* p = is_x ? a.hi[q] : kind == OR_SQUARE ? a.A : a.B;
        const int64_t cols = is_x ? a.n : r, rows = is_x ? a.m : r, ld = is_x ? a.ldx : a.ldr, pm = is_x ? a.px : a.pr;
        const int across = side ? a.ph[kind].bn / CG : 128;
        const int64_t dk[4] = {cols, rows, 1, a.batch}, sk[3] = {ld, pm, pm}, dm[4] = {64, rows, (cols + 63) / 64, a.batch},
                      sm[3] = {ld, 64, pm};
        const int bk[4] = {OR_BK, across, 1, 1}, bm[4] = {64, OR_BK, across / 64, 1};
        if (int rc = tensor_map("orthogonalize", side ? &maps.b[q][kind] : &maps.a[q][kind], CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, 4, p,
                                mn ? dm : dk, mn ? sm : sk, mn ? bm : bk))
          return rc;
      }
  static int ready_dev = -1;
  int dev = 0;
  constexpr int SMEM = 196608 + OR_EPI * XG_STG + 256 + 1024;
  if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("orthogonalize (device)");
  if (ready_dev != dev) {
    if (cudaFuncSetAttribute(k_orth<CG>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) {
      set_error("orthogonalize: cannot reserve %d bytes of shared memory", SMEM);
      return MB_E_CUDA;
    }
    ready_dev = dev;
  }
  const int units = sm_count() / CG;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(most < units ? most : units) * CG);
  cfg.blockDim = dim3(OR_THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = CG;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CG;
  cudaLaunchKernelEx(&cfg, k_orth<CG>, maps, a);
  return check_launch("orthogonalize");
}

// Pairs of CTAs halve the bytes that an SM fetches of one operand: for long sums.  One CTA / pairs: 4096 x 4096 1281 / 1166 us,
// 2048 x 2048 251 / 240, 1500 x 8192 539 / 459, 1500 x 1500 207 / 195; 1300 x 1300 182 / 197, 1280 x 4096 245 / 258, 1024 x 1024 124 / 151, 16 of
// them 645 / 667, 4 of 1500 x 700 189 / 197.  Around the limit it is the rounds of tiles that decide: 1400 x 1400 178 / 193, but 4 of them
// 406 / 373, 16 of them 1400 / 1327 and 4 of 1200 x 1200 311 / 293.
static bool or_pairs(int64_t r) { return r >= 1400; }

}  // namespace mb

using namespace mb;

extern "C" int mace_b200_orthogonalize_workspace(int64_t batch, int32_t m, int32_t n, int64_t* bytes) {
  if (batch < 0 || batch > 65535 || m < 1 || n < 1 || m > MB_ORTH_MAX_DIM || n > MB_ORTH_MAX_DIM || !bytes) {
    set_error("orthogonalize: bad sizes (batch %lld, %d x %d; at most 65535 matrices, sides of %d)", (long long)batch, m, n,
              MB_ORTH_MAX_DIM);
    return MB_E_ARG;
  }
  *bytes = orth_small(batch, m, n) ? 0 : or_layout(batch, m, n).bytes;
  return 0;
}

extern "C" int mace_b200_orthogonalize(const void* gp, int64_t ldb, int64_t ldg, void* out, void* workspace, int64_t batch, int32_t m,
                                       int32_t n, const double* coefficients, int32_t steps, double eps, int32_t dtype,
                                       void* stream) {
  int64_t need = 0;
  if (int rc = mace_b200_orthogonalize_workspace(batch, m, n, &need)) return rc;
  if (steps < 1 || steps > OR_STEPS || !coefficients || !(eps >= 1e-30 && eps < 1e30) || !dtype_ok(dtype) || ldg < n) {
    set_error("orthogonalize: bad arguments (steps %d of 1 .. %d, eps %g, type %d, row stride %lld)", steps, OR_STEPS, eps, dtype,
              (long long)ldg);
    return MB_E_ARG;
  }
  // the largest singular value that a step can give, from those that the step before can: fp16 planes hold values up to 3.5
  double top = 1.0;
  for (int k = 0; k < steps; ++k) {
    const double *c = coefficients + 3 * k, in = top * 1.02;
    double most = 0.0, left = 0.0;
    for (int i = 0; i <= 1024; ++i) {
      const double s = in * i / 1024.0, q = s * s * (c[1] + c[2] * s * s), v = s * (c[0] + q);
      if (!(fabs(v) <= 1e30)) most = 1e30;       // NaN, too
      most = fabs(v) > most ? fabs(v) : most;
      left = fabs(q) > left ? fabs(q) : left;
    }
    if (!(most <= 3.5 && left <= 200.0)) {
      set_error("orthogonalize: the polynomial of step %d reaches %g (at most 3.5)", k, most);
      return MB_E_ARG;
    }
    top = most;
  }
  if (batch == 0) return 0;
  if (!gp || !out || (need > 0 && !workspace)) {
    set_error("orthogonalize: null pointer");
    return MB_E_ARG;
  }
  if (sm_count() < 1) {
    set_error("orthogonalize: no CUDA device");
    return MB_E_CUDA;
  }
  OrPoly poly{};
  poly.steps = steps;
  poly.eps = eps;
  for (int k = 0; k < steps; ++k) {
    poly.a[k] = (float)coefficients[3 * k];
    poly.b[k] = (float)coefficients[3 * k + 1];
    poly.c[k] = (float)coefficients[3 * k + 2];
  }
  double grows = 1.0;                             // of what the steps from k + 1 on do to weak directions
  for (int k = steps - 1; k >= 0; --k) {
    if (grows > OR_GROW) poly.grow |= 1u << k;
    grows *= fabs(coefficients[3 * k]);
  }
  // X's scale: a power of two near the inverse of its first entries, 2^14 at most (values up to 3.5 stay below 65504)
  int ex = 0;
  while (ex < 14 && (double)(1 << (ex + 1)) * (1 << (ex + 1)) <= (double)m * n) ++ex;
  poly.s = (float)(1 << ex);
  poly.inv_s = 1.f / poly.s;
  if (orth_small(batch, m, n)) return orth_small_launch(gp, ldb, ldg, out, batch, m, n, poly, dtype, (cudaStream_t)stream);
  const OrLayout l = or_layout(batch, m, n);
  char* ws = (char*)workspace;
  OrArgs a{};
  a.m = m; a.n = n; a.r = m < n ? m : n; a.batch = (int)batch; a.tall = m > n;
  a.ldx = l.ldx; a.ldr = l.ldr; a.px = l.px; a.pr = l.pr;
  a.poly = poly;
  for (int q = 0; q < 2; ++q) a.hi[q] = (f16*)(ws + l.hi + q * l.plane);
  a.X = (float*)(ws + l.X);
  a.ci = (m + 31) / 32;
  a.cj = (n + 31) / 32;
  a.pc = l.pc;
  a.A = (f16*)(ws + l.A); a.B = (f16*)(ws + l.B);
  a.d = (float*)(ws + l.d); a.e = (float*)(ws + l.e);
  a.out = (bf16*)out;
  a.vec_out = n % 8 == 0 && aligned16(out);
  a.words = (unsigned*)(ws + l.words);
  const int r = a.r, len = m < n ? n : m;
  double* part = (double*)(ws + l.part);
  cudaStream_t st = (cudaStream_t)stream;
  int rc = dtype == MB_F32    ? orth_go<float>(gp, ldb, ldg, a, part, st)
           : dtype == MB_BF16 ? orth_go<bf16>(gp, ldb, ldg, a, part, st)
                              : orth_go<f16>(gp, ldb, ldg, a, part, st);
  if (rc) return rc;
  return or_pairs(r) ? orth_steps<2>(a, r, len, st) : orth_steps<1>(a, r, len, st);
}
