// Orthogonalised matrices by Newton-Schulz products, for the updates of an optimiser (a batch of matrices [m][n]):
//   X = G / (|G|_F + eps);  per step  A = X X^T,  X <- a X + (b A + c A A) X   (m <= n; else A = X^T X, products from the right)
// so every singular value s moves to a s + b s^3 + c s^5, towards one.  The result is bf16.
//
// Products are tcgen05 kind::f16 with fp32 accumulators, on fp16 operands: everything is bounded (|X| <= 2, so powers of two
// scale it into fp16's range) and fp16 has three bits more than bf16.  What is rounded, and why that is enough (fp64 simulation and
// measurement, Frobenius error before the last rounding 2e-4 to 7e-4, of a bf16 result that rounds by 1.7e-3):
//  * X lies in two fp16 planes (x = hi + lo / 2048, 22 bits).  An error added to X grows by up to a^steps (485) in its weak
//    directions: one plane was 0.04 off for a matrix of rank 8 over noise.
//  * The products read hi alone.  An error of the left factor (A, b A + c A A) multiplies X, and the polar factor of (1 + E) X
//    differs by |E| whatever the singular values; lo's part of B X lies in the strong directions, which do not grow.
//  * The diagonals of A and of b A + c A A dominate them and stay apart in fp32: A = A1 + D gives A A = A1 A1 + A1 D + D A1 + D D, and
//    the diagonal of the second multiplies X in the epilogue.  In the planes they cost 2 to 9 times the error.
//  * The tensor cores truncate when they add: a diagonal loses 1e-7 of itself per 16 terms, 4e-4 at MB_ORTH_MAX_DIM.
//
// A and A A are symmetric: only tiles that reach the diagonal or lie above it are multiplied, and stored to both places.
// One cooperative kernel runs all steps: persistent CTAs, one per SM, 3 phases a step with a barrier over the grid between them
// (separate launches cost a pipeline's fill and drain each).  Warp 0 loads with TMA, warp 1 issues, warps 4-11 drain one of two
// accumulators.  Tall matrices are not transposed: their Gram product reads both operands MN-major.  Two small kernels before
// it take the norm (sums of squares in fp64) and split G into the planes.
// Every wait is bounded; after one expires the grid stops and the tiles of the result that have none are NaN.
#include <cuda.h>

#include <type_traits>

#include "dtypes.cuh"
#include "tc.cuh"
#include "tensor_map.cuh"

namespace mb {

constexpr int OR_EPI0 = 4, OR_EPI = 8, OR_THREADS = 32 * (OR_EPI0 + OR_EPI), OR_BK = 64, OR_STEPS = 16,
              OR_WORDS = 1 + 3 * OR_STEPS;
constexpr int OR_BOX = 64 * OR_BK * 2;            // bytes of one 64 x 64 box: operands are loaded in those
constexpr unsigned long long OR_WAIT = 2000000000ull;
constexpr int OR_PARTS = 256;                     // most partial sums of squares of a matrix
constexpr float OR_LO = 2048.f, OR_SA = 4096.f, OR_SB = 256.f;   // scales of the lo plane, of A and of b A + c A A

enum { OR_GRAM = 0, OR_SQUARE = 1, OR_UPDATE = 2 };
struct OrPhase {
  int32_t bn, ti, tj, per, nk, a_mn, b_mn, tri;   // columns of a tile, tiles, per matrix, K blocks; operands' layouts
  int32_t M, N;
};
struct OrArgs {
  int32_t m, n, r, batch, steps, tall, stages, stage_bytes, vec_out;
  int64_t ldx, ldr, px, pr;                       // row strides of the planes, elements of a matrix in them
  float ca[OR_STEPS], cb[OR_STEPS], cc[OR_STEPS];
  float s, inv_s;                                 // scale of the hi plane
  OrPhase ph[3];
  f16 *hi[2], *lo[2], *A, *B;
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

__device__ __forceinline__ void or_split(float x, float& hi, float& lo) {
  hi = to_f(from_f<f16>(x));
  lo = (x - hi) * OR_LO;
}

// Planes of S G / (|G| + eps); a thread writes eight columns
template <typename T>
__global__ void __launch_bounds__(256) k_orth_split(const T* g, int64_t ldb, int64_t ldg, int32_t m, int32_t n, bool vec,
                                                    const double* part, int np, double S, double eps, f16* hi, f16* lo,
                                                    int64_t ldx, int64_t px) {
  __shared__ double red[8];
  double s = (int)threadIdx.x < np ? part[(int64_t)blockIdx.y * np + threadIdx.x] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
  for (int q = 0; q < 8; ++q) s += red[q];
  const float scale = (float)(S / (sqrt(s) + eps));
  const T* p = g + blockIdx.y * ldb;
  f16 *h = hi + blockIdx.y * px, *l = lo + blockIdx.y * px;
  const int w = (n + 7) / 8;
  const int64_t all = (int64_t)m * w, step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += step) {
    const int64_t row = i / w;
    const int c = (int)(i - row * w) * 8;
    const T* q = p + row * ldg + c;
    float f[8], a[8], b[8];
    if (vec && c + 8 <= n) {
      if constexpr (sizeof(T) == 4) {
        float u[4], v[4];
        load_v<T, 4>(q, u);
        load_v<T, 4>(q + 4, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = u[j], f[4 + j] = v[j];
      } else {
        load_v<T, 8>(q, f);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = c + j < n ? to_f(q[j]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) or_split(f[j] * scale, a[j], b[j]);
    *reinterpret_cast<uint4*>(h + row * ldx + c) = pack16<f16>(a);
    *reinterpret_cast<uint4*>(l + row * ldx + c) = pack16<f16>(b);
  }
}

// ------------------------------------------------------------------------------------------------ the steps
struct OrBars {
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2];
  uint32_t tmem;
  int failed;
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
      left = p.tj - (i + 1) * 128 / p.bn;
    }
    t += i * 128 / p.bn;
  } else {
    i = t / p.tj;
    t -= i * p.tj;
  }
  o.m0 = i * 128;
  o.n0 = t * p.bn;
  return o;
}

__device__ __forceinline__ unsigned ld_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// Waits until every CTA is through with the phase (each phase counts for itself: CTAs without tiles run ahead); false on a failure
// anywhere or when the limit is over
__device__ __forceinline__ bool or_wait(const OrArgs& g, int phase) {
  unsigned long long t0 = 0;
  for (unsigned it = 0;; ++it) {
    if (ld_acquire(g.words + 1 + phase) >= gridDim.x) break;
    if ((it & 15u) == 15u && ld_acquire(g.words)) return false;
    if ((it & 255u) == 255u) {
      const unsigned long long now = globaltimer_ns();
      if (t0 == 0)
        t0 = now;
      else if (now - t0 > OR_WAIT)
        return false;
    }
  }
  asm volatile("fence.proxy.async;" ::: "memory");  // what others stored is read by TMA
  return true;
}

__device__ __forceinline__ void or_load32(const f16* p, uint4 (&u)[4], int n) {   // 32 elements in memory of 8 at a time
#pragma unroll
  for (int q = 0; q < 4; ++q) u[q] = 8 * q < n ? __ldcg(reinterpret_cast<const uint4*>(p) + q) : make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ float or_half(const uint4 (&u)[4], int i) {
  const uint4& v = u[i / 8];
  const uint32_t w = i / 2 % 4 == 0 ? v.x : i / 2 % 4 == 1 ? v.y : i / 2 % 4 == 2 ? v.z : v.w;
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return i & 1 ? f.y : f.x;
}
__device__ __forceinline__ void or_store32(f16* p, const float (&v)[32], int n) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (8 * q < n) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = v[8 * q + i];
      *(reinterpret_cast<uint4*>(p) + q) = pack16<f16>(f);
    }
}

__global__ void __launch_bounds__(OR_THREADS, 1)
    k_orth(const __grid_constant__ CUtensorMap map_x0, const __grid_constant__ CUtensorMap map_x1,
           const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ OrArgs g) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  OrBars& B = *reinterpret_cast<OrBars*>(smem + g.stages * g.stage_bytes);
  volatile int* failed = &B.failed;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x, ctas = gridDim.x;
  if (warp == 1) {
    tmem_alloc<1>(&B.tmem, 512);
    if (lane == 0) {
      for (int s = 0; s < 8; ++s) {
        mbar_init(&B.full[s], 1);
        mbar_init(&B.empty[s], 1);
      }
      for (int a = 0; a < 2; ++a) {
        mbar_init(&B.acc_full[a], 1);
        mbar_init(&B.acc_empty[a], OR_EPI);
      }
      B.failed = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = B.tmem;
  const int phases = 3 * g.steps;

  if (warp == 0) {
    // ------------------------------------------------------------------------------------------ loads
    if (lane == 0) {
      int seq = 0;
      bool ok = true;
      for (int ph = 0; ok && ph < phases; ++ph) {
        const OrPhase& p = g.ph[ph % 3];
        const int tiles = g.batch * p.per;
        const CUtensorMap* mx = (ph / 3) & 1 ? &map_x1 : &map_x0;
        const int kind = ph % 3;
        const CUtensorMap *ma = kind == OR_GRAM ? mx : kind == OR_SQUARE ? &map_a : g.tall ? mx : &map_b;
        const CUtensorMap *mbp = kind == OR_GRAM ? mx : kind == OR_SQUARE ? &map_a : g.tall ? &map_b : mx;
        const uint32_t bytes = (uint32_t)(2 + p.bn / 64) * OR_BOX;
        bool waited = ph == 0;
        for (int t = cta; ok && t < tiles; t += ctas) {
          const OrTile w = or_tile(p, t);
          if (!waited) {
            if (!or_wait(g, ph - 1)) {
              *failed = 1;
              ok = false;
              break;
            }
            waited = true;
          }
          for (int kb = 0; kb < p.nk; ++kb, ++seq) {
            const int s = seq % g.stages;
            if (*failed || !mbar_wait_ns(&B.empty[s], ((seq / g.stages) & 1) ^ 1, OR_WAIT)) {
              *failed = 1;
              ok = false;
              break;
            }
            const uint32_t bar = smem_u32(&B.full[s]), a = smem_u32(smem + s * g.stage_bytes), b = a + 2 * OR_BOX;
            mbar_arrive_tx(&B.full[s], bytes);
            const int k0 = kb * OR_BK;
#pragma unroll
            for (int q = 0; q < 2; ++q)
              tma_load_3d<1>(a + q * OR_BOX, ma, p.a_mn ? w.m0 + 64 * q : k0, p.a_mn ? k0 : w.m0 + 64 * q, w.b, bar);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (64 * q < p.bn)
                tma_load_3d<1>(b + q * OR_BOX, mbp, p.b_mn ? w.n0 + 64 * q : k0, p.b_mn ? k0 : w.n0 + 64 * q, w.b, bar);
          }
        }
      }
      if (!ok)                                    // copies in flight land before the block ends (bounded)
        for (int q = seq - g.stages < 0 ? 0 : seq - g.stages; q < seq; ++q)
          mbar_wait_ns(&B.full[q % g.stages], (q / g.stages) & 1, OR_WAIT);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------------------------------ MMA issue
    if (lane == 0) {
      int seq = 0, tc = 0;
      bool ok = true;
      uint64_t* last_bar = nullptr;
      uint32_t last_par = 0;
      for (int ph = 0; ok && ph < phases; ++ph) {
        const OrPhase& p = g.ph[ph % 3];
        const int tiles = g.batch * p.per;
        const uint32_t idesc = f16_idesc(128, p.bn, false, p.a_mn, p.b_mn);
        for (int t = cta; ok && t < tiles; t += ctas, ++tc) {
          const int acc = tc & 1;
          // the first wait of a phase includes the grid's barrier: the loads' limit, then this one's
          if (*failed || !mbar_wait_ns(&B.acc_empty[acc], ((tc >> 1) & 1) ^ 1, OR_WAIT)) {
            *failed = 1;
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          for (int kb = 0; kb < p.nk; ++kb, ++seq) {
            const int s = seq % g.stages;
            if (!mbar_wait_ns(&B.full[s], (seq / g.stages) & 1, 2 * OR_WAIT)) {
              *failed = 1;
              ok = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t a = smem_u32(smem + s * g.stage_bytes), b = a + 2 * OR_BOX;
#pragma unroll
            for (int kk = 0; kk < OR_BK / 16; ++kk) {
              const uint64_t ad = p.a_mn ? sw128_desc_mn(a + kk * 2048, OR_BOX) : sw128_desc(a + kk * 32);
              const uint64_t bd = p.b_mn ? sw128_desc_mn(b + kk * 2048, OR_BOX) : sw128_desc(b + kk * 32);
              mma_f16_ss<1>(tmem + acc * 256, ad, bd, idesc, (kb | kk) ? 1u : 0u);
            }
            mma_commit_to<1>(&B.empty[s]);
            last_bar = &B.empty[s];
            last_par = (seq / g.stages) & 1;
          }
          if (!ok) break;
          mma_commit_to<1>(&B.acc_full[acc]);
          last_bar = &B.acc_full[acc];
          last_par = (tc >> 1) & 1;
        }
      }
      if (*failed && last_bar) mbar_wait_ns(last_bar, last_par, OR_WAIT);
    }
  } else if (warp >= OR_EPI0) {
    // ------------------------------------------------------------------------------------------ epilogue
    const int q4 = warp & 3, hf = (warp - OR_EPI0) >> 2;
    int tc = 0;
    bool lost = false;                            // warp-uniform
    for (int ph = 0; ph < phases; ++ph) {
      const OrPhase& p = g.ph[ph % 3];
      const int kind = ph % 3, step = ph / 3, tiles = g.batch * p.per, hw = p.bn / 2;
      const bool last = ph == phases - 1;
      bool waited = ph == 0 || kind == OR_GRAM;   // the Gram phase's epilogue reads nothing
      // after a failure only the result's tiles are gone through (every warp takes part in every phase's block barrier)
      for (int t = lost && !last ? tiles : cta; t < tiles; t += ctas, ++tc) {
        const OrTile w = or_tile(p, t);
        const int acc = tc & 1, i = w.m0 + q4 * 32 + lane;
        if (!waited && !lost) {
          lost = !__all_sync(0xffffffffu, lane != 0 || or_wait(g, ph - 1));
          waited = true;
        }
        if (!lost)
          lost = __shfl_sync(0xffffffffu, *failed, 0) ||
                 !__all_sync(0xffffffffu, mbar_wait_ns(&B.acc_full[acc], (tc >> 1) & 1, 3 * OR_WAIT));
        if (lost) {
          *failed = 1;
          if (!last) break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int c = 0; c < hw; c += 32) {
          const int j0 = w.n0 + hf * hw + c, nc = p.N - j0 < 32 ? p.N - j0 : 32;   // columns here (<= 0: none)
          uint32_t u[32];
          float v[32];
          if (!lost) {
            tmem_ld32(tmem + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * 256 + hf * hw + c), u);
            tmem_wait_ld();
            if (c + 32 >= hw) {                   // the accumulator is free
              asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
              __syncwarp();
              if (lane == 0) mbar_arrive(&B.acc_empty[acc]);
            }
          }
          if (nc <= 0 || i >= p.M) continue;      // (no warp-collective operation below)
          if (kind == OR_UPDATE) {
            const int64_t at = w.b * g.px + i * g.ldx + j0;
            const int from = step & 1, to = from ^ 1;
            const float ca = g.ca[step];
            const float* e = g.e + (int64_t)w.b * g.r;
            uint4 h4[4], l4[4];
            if (!lost) {
              or_load32(g.hi[from] + at, h4, nc);
              or_load32(g.lo[from] + at, l4, nc);
            }
            const float ei = !lost && !g.tall ? ca + __ldcg(e + i) : 0.f;
#pragma unroll
            for (int x = 0; x < 32; ++x) {
              if (lost) {
                v[x] = __int_as_float(0x7fc00000);
                continue;
              }
              const float f = g.tall ? (x < nc ? ca + __ldcg(e + j0 + x) : 0.f) : ei;
              const float old = fmaf(or_half(l4, x), 1.f / OR_LO, or_half(h4, x));
              v[x] = fmaf(f, old, __uint_as_float(u[x]) * (1.f / OR_SB));
            }
            if (last) {
              bf16* o = g.out + ((int64_t)w.b * g.m + i) * g.n + j0;
              const bool vec = g.vec_out && nc == 32;
#pragma unroll
              for (int x = 0; x < 32; ++x) v[x] *= g.inv_s;
              if (vec) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  float f[8];
#pragma unroll
                  for (int x = 0; x < 8; ++x) f[x] = v[8 * q + x];
                  *(reinterpret_cast<uint4*>(o) + q) = pack16<bf16>(f);
                }
              } else {
#pragma unroll
                for (int x = 0; x < 32; ++x)
                  if (x < nc) o[x] = from_f<bf16>(v[x]);
              }
            } else {
              float lo[32];
#pragma unroll
              for (int x = 0; x < 32; ++x) {
                float h;
                or_split(v[x], h, lo[x]);
                v[x] = h;
              }
              or_store32(g.hi[to] + at, v, nc);
              or_store32(g.lo[to] + at, lo, nc);
            }
          } else {
            f16* dst = (kind == OR_GRAM ? g.A : g.B) + w.b * g.pr;
            float* diag = (kind == OR_GRAM ? g.d : g.e) + (int64_t)w.b * g.r;
            if (kind == OR_GRAM) {
              const float sc = g.inv_s * g.inv_s;
#pragma unroll
              for (int x = 0; x < 32; ++x) {
                const float a = __uint_as_float(u[x]) * sc;
                if (j0 + x == i) diag[i] = a;
                v[x] = j0 + x == i ? 0.f : a * OR_SA;
              }
            } else {
              const float cb = g.cb[step], cc = g.cc[step];
              const float* d = g.d + (int64_t)w.b * g.r;
              uint4 a4[4];
              or_load32(g.A + w.b * g.pr + i * g.ldr + j0, a4, nc);
              const float di = __ldcg(d + i);
#pragma unroll
              for (int x = 0; x < 32; ++x) {
                const float dj = x < nc ? __ldcg(d + j0 + x) : 0.f, a1 = or_half(a4, x) * (1.f / OR_SA);
                const float sq = __uint_as_float(u[x]) * (1.f / (OR_SA * OR_SA));
                if (j0 + x == i) {
                  diag[i] = fmaf(cb, di, cc * fmaf(di, di, sq));
                  v[x] = 0.f;
                } else {
                  v[x] = fmaf(cb, a1, cc * fmaf(a1, di + dj, sq)) * OR_SB;
                }
              }
            }
            if (j0 >= w.m0 + 128) {               // above the diagonal
              or_store32(dst + i * g.ldr + j0, v, nc);
#pragma unroll
              for (int x = 0; x < 32; ++x)
                if (x < nc) dst[(j0 + x) * g.ldr + i] = from_f<f16>(v[x]);
            } else {
#pragma unroll
              for (int x = 0; x < 32; ++x)
                if (x < nc && j0 + x >= i) {
                  dst[i * g.ldr + j0 + x] = from_f<f16>(v[x]);
                  dst[(j0 + x) * g.ldr + i] = from_f<f16>(v[x]);
                }
            }
          }
        }
      }
      if (!last) {                                // this CTA's part of the phase is in memory
        asm volatile("fence.proxy.async;" ::: "memory");
        __threadfence();
        asm volatile("bar.sync 1, %0;" ::"n"(32 * OR_EPI) : "memory");
        if (tid == 32 * OR_EPI0) {
          if (*failed)                            // and nobody gets past this phase
            atomicExch(g.words, 1u);
          else
            asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(g.words + 1 + ph) : "memory");
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_dealloc<1>(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------------ host side
struct OrLayout {
  int64_t ldx, ldr, px, pr, hi, plane, A, B, d, e, part, words, bytes;
};
static OrLayout or_layout(int64_t batch, int64_t m, int64_t n) {
  OrLayout l{};
  const int64_t r = m < n ? m : n;
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  l.ldx = (n + 7) / 8 * 8;
  l.ldr = (r + 7) / 8 * 8;
  l.px = m * l.ldx;
  l.pr = r * l.ldr;
  l.plane = up(batch * l.px * 2);
  l.hi = 0;                                       // hi0, hi1, lo0, lo1
  l.A = 4 * l.plane;
  l.B = l.A + up(batch * l.pr * 2);
  l.d = l.B + up(batch * l.pr * 2);
  l.e = l.d + up(batch * r * 4);
  l.part = l.e + up(batch * r * 4);
  l.words = l.part + up(batch * OR_PARTS * 8);
  l.bytes = l.words + 256;
  return l;
}

// Tiles of a phase: the widest that leave every SM one, 64 columns at least
static void or_cut(OrPhase& p, int64_t batch, int M, int N, int K, bool tri) {
  p.M = M;
  p.N = N;
  p.nk = (K + OR_BK - 1) / OR_BK;
  p.tri = tri;
  p.ti = (M + 127) / 128;
  for (p.bn = 256;; p.bn /= 2) {
    p.tj = (N + p.bn - 1) / p.bn;
    p.per = 0;
    for (int i = 0; i < p.ti; ++i) p.per += tri ? p.tj - i * 128 / p.bn : p.tj;
    if (p.bn == 64 || batch * p.per >= sm_count()) return;
  }
}

template <typename T>
static int orth_go(const void* gp, int64_t ldb, int64_t ldg, OrArgs& a, const OrLayout& l, char* ws, double eps, cudaStream_t st) {
  constexpr int V = kVec<T>;
  const bool vec = a.n % V == 0 && ldg % V == 0 && ldb % V == 0 && aligned16(gp);
  const int64_t work = ((int64_t)a.m * a.n + 8 * 256 - 1) / (8 * 256), fill = (4 * (int64_t)sm_count() + a.batch - 1) / a.batch;
  int64_t np = work < fill ? work : fill;
  if (np > OR_PARTS) np = OR_PARTS;
  double* part = (double*)(ws + l.part);
  k_orth_norm<T><<<dim3((unsigned)np, a.batch), 256, 0, st>>>((const T*)gp, ldb, ldg, a.m, a.n, vec, part, a.words);
  if (int rc = check_launch("orthogonalize (norm)")) return rc;
  const bool vec8 = ldg % V == 0 && ldb % V == 0 && aligned16(gp);
  k_orth_split<T><<<dim3((unsigned)(work < fill ? work : fill), a.batch), 256, 0, st>>>(
      (const T*)gp, ldb, ldg, a.m, a.n, vec8, part, (int)np, (double)a.s, eps, a.hi[0], a.lo[0], l.ldx, l.px);
  return check_launch("orthogonalize (planes)");
}

}  // namespace mb

using namespace mb;

extern "C" int mace_b200_orthogonalize_workspace(int64_t batch, int32_t m, int32_t n, int64_t* bytes) {
  if (batch < 0 || batch > 65535 || m < 1 || n < 1 || m > MB_ORTH_MAX_DIM || n > MB_ORTH_MAX_DIM || !bytes) {
    set_error("orthogonalize: bad sizes (batch %lld, %d x %d; at most 65535 matrices, sides of %d)", (long long)batch, m, n,
              MB_ORTH_MAX_DIM);
    return MB_E_ARG;
  }
  *bytes = or_layout(batch, m, n).bytes;
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
  if (!gp || !out || !workspace) {
    set_error("orthogonalize: null pointer");
    return MB_E_ARG;
  }
  if (sm_count() < 1) {
    set_error("orthogonalize: no CUDA device");
    return MB_E_CUDA;
  }
  const OrLayout l = or_layout(batch, m, n);
  char* ws = (char*)workspace;
  OrArgs a{};
  a.m = m; a.n = n; a.r = m < n ? m : n; a.batch = (int)batch; a.steps = steps; a.tall = m > n;
  a.ldx = l.ldx; a.ldr = l.ldr; a.px = l.px; a.pr = l.pr;
  for (int k = 0; k < steps; ++k) {
    a.ca[k] = (float)coefficients[3 * k];
    a.cb[k] = (float)coefficients[3 * k + 1];
    a.cc[k] = (float)coefficients[3 * k + 2];
  }
  // hi's scale: a power of two near the inverse of X's first entries, 2^14 at most (values up to 3.5 stay below 65504)
  int ex = 0;
  while (ex < 14 && (double)(1 << (ex + 1)) * (1 << (ex + 1)) <= (double)m * n) ++ex;
  a.s = (float)(1 << ex);
  a.inv_s = 1.f / a.s;
  for (int q = 0; q < 2; ++q) {
    a.hi[q] = (f16*)(ws + l.hi + q * l.plane);
    a.lo[q] = (f16*)(ws + l.hi + (2 + q) * l.plane);
  }
  a.A = (f16*)(ws + l.A); a.B = (f16*)(ws + l.B);
  a.d = (float*)(ws + l.d); a.e = (float*)(ws + l.e);
  a.out = (bf16*)out;
  a.vec_out = n % 8 == 0 && aligned16(out);
  a.words = (unsigned*)(ws + l.words);
  const int r = a.r, len = m < n ? n : m;
  or_cut(a.ph[OR_GRAM], batch, r, r, len, true);
  or_cut(a.ph[OR_SQUARE], batch, r, r, r, true);
  or_cut(a.ph[OR_UPDATE], batch, m, n, r, false);
  a.ph[OR_GRAM].a_mn = a.ph[OR_GRAM].b_mn = a.tall;
  a.ph[OR_UPDATE].b_mn = !a.tall;
  int64_t most = 0;
  int bn = 64;
  for (const OrPhase& p : a.ph) {
    if (batch * p.per > most) most = batch * p.per;
    if (p.bn > bn) bn = p.bn;
  }
  if (most > 0x7fffffff) {
    set_error("orthogonalize: too many tiles (%lld)", (long long)most);
    return MB_E_ARG;
  }
  a.stage_bytes = (2 + bn / 64) * OR_BOX;
  a.stages = 196608 / a.stage_bytes < 8 ? 196608 / a.stage_bytes : 8;
  cudaStream_t st = (cudaStream_t)stream;
  int rc = dtype == MB_F32    ? orth_go<float>(gp, ldb, ldg, a, l, ws, eps, st)
           : dtype == MB_BF16 ? orth_go<bf16>(gp, ldb, ldg, a, l, ws, eps, st)
                              : orth_go<f16>(gp, ldb, ldg, a, l, ws, eps, st);
  if (rc) return rc;
  CUtensorMap mx[2], ma, mbm;
  const int box[3] = {64, 64, 1};
  const int64_t dx[3] = {n, m, batch}, sx[2] = {l.ldx, l.px}, dr[3] = {r, r, batch}, sr[2] = {l.ldr, l.pr};
  for (int q = 0; q < 2; ++q)
    if ((rc = tensor_map("orthogonalize", &mx[q], CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, 3, a.hi[q], dx, sx, box))) return rc;
  if ((rc = tensor_map("orthogonalize", &ma, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, 3, a.A, dr, sr, box))) return rc;
  if ((rc = tensor_map("orthogonalize", &mbm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, 3, a.B, dr, sr, box))) return rc;
  static int ready_dev = -1;
  int dev = 0;
  constexpr int SMEM = 196608 + 256 + 1024;
  if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("orthogonalize (device)");
  if (ready_dev != dev) {
    if (cudaFuncSetAttribute(k_orth, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) {
      set_error("orthogonalize: cannot reserve %d bytes of shared memory", SMEM);
      return MB_E_CUDA;
    }
    ready_dev = dev;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(most < sm_count() ? most : sm_count()));
  cfg.blockDim = dim3(OR_THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, k_orth, mx[0], mx[1], ma, mbm, a);
  return check_launch("orthogonalize");
}
