// The three expert products on the 5th-generation tensor cores (tcgen05 kind::f16, fp32 accumulators in TMEM):
//   FWD    C[row][o] = sum_d x[row][d] W[e][o][d]        both operands K-major
//   DGRAD  C[row][d] = sum_o dy[row][o] W[e][o][d]       W is MN-major (its rows run along N)
//   WGRAD  C[e][o][d] = sum over e's rows dy[row][o] x[row][d]   both MN-major, K = the expert's rows
// Rows are sorted by expert and padded to 128, so a 128-row tile (FWD, DGRAD) or a 64-row K block (WGRAD) has one expert,
// and no matrix is transposed in memory: the MN-major operands are read as they lie.
// fp32 data comes as three bf16 planes; the products of the planes whose ranks add up to at most 2 (six of nine, small
// ones first) accumulate in the same fp32 accumulator, the rest is below 2^-24 of the result.
//
// Persistent CTA, one per SM: warp 0 loads tiles with TMA (SWIZZLE_128B) into a ring of stages, warp 1 issues the MMAs
// (128 x BN x 16) into one of two TMEM accumulators, warps 2-5 drain the other one (one row per lane), scale the row by
// its slot's weight and write it to the slot's place in the output.  Every wait is bounded: on expiry the kernel sets
// MB_ST_TC_TIMEOUT in the plan's status word, drains its copies and MMAs, frees its TMEM and returns.
#include <cuda.h>

#include "experts.cuh"
#include "tc.cuh"

namespace mb {

constexpr int XG_BM = XP_BM, XG_BK = 64, XG_THREADS = 192;
constexpr unsigned long long XG_WAIT_NS = 2000000000ull;   // a tile takes microseconds

constexpr int XG_STG = 4096;                     // row staging of one epilogue warp
template <int BN>
struct XgCfg {
  static constexpr int A_BYTES = XG_BM * XG_BK * 2, B_BYTES = BN * XG_BK * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 196608 / STAGE;              // 192 KB ring: 4 stages at BN = 256, 6 at 128
  static constexpr int TMEM = 2 * BN;
  static constexpr int SMEM = STAGES * STAGE + 4 * XG_STG + 256 + 1024;   // + row staging, barriers, alignment slack
};

struct XgParams {
  int32_t E, M, N, K, tn, tm, np;                // tn / tm: tiles along N, along M (WGRAD)
  int32_t split;                                 // WGRAD: parts of an expert's rows
  int64_t rows;                                  // rows per plane of the sorted operands
  int32_t w_rows;                                // E (planes of w follow each other)
  const int32_t* plan;
  XPlan lay;
  const float* scale;
  void* out;
  int64_t ldo;
  const void* x;
  int64_t ldx;
  int32_t kdiv;
  float* dgpart;
};

struct XgBars {
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2];
  uint32_t tmem;
  int failed;
};

// planes of A and B multiplied in pass p (of 6): small products first
__device__ __forceinline__ int xg_plane_a(int p) { return (0x021010 >> (4 * (5 - p))) & 0xF; }
__device__ __forceinline__ int xg_plane_b(int p) { return (0x201100 >> (4 * (5 - p))) & 0xF; }

// Row staging of the epilogue: a warp's 32 rows x 128 bytes, 16-byte piece c of row r at piece c ^ (r % 8), so that a lane's
// access to its own row and the warp's access to four whole row segments are both free of bank conflicts.
__device__ __forceinline__ uint4* xg_stg(unsigned char* stg, int row, int c) {
  return reinterpret_cast<uint4*>(stg + row * 128 + ((c ^ (row & 7)) << 4));
}

// OUT: element type of the output (T, or float for partial sums)
template <int MODE, typename T, typename OUT, int BN>
__global__ void __launch_bounds__(XG_THREADS, 1)
    k_expert_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const XgParams g) {
  using C = XgCfg<BN>;
  constexpr bool A_MN = MODE == XG_WGRAD, B_MN = MODE != XG_FWD;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  XgBars& B = *reinterpret_cast<XgBars*>(smem + C::STAGES * C::STAGE + 4 * XG_STG);
  volatile int* failed = &B.failed;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&B.tmem)),
                 "r"(C::TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    if (lane == 0) {
      for (int s = 0; s < C::STAGES; ++s) {
        mbar_init(&B.full[s], 1);
        mbar_init(&B.empty[s], 1);
      }
      for (int a = 0; a < 2; ++a) {
        mbar_init(&B.acc_full[a], 1);
        mbar_init(&B.acc_empty[a], 128);
      }
      B.failed = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = B.tmem;
  const int32_t* plan = g.plan;
  const int tiles = MODE == XG_WGRAD ? g.split * g.E * g.tm * g.tn : plan[0] * g.tn;

  // This CTA's n-th tile.  WGRAD: experts come longest first and odd rounds run backwards over the CTAs, so that every CTA
  // gets about the same number of K blocks.
  auto tile_at = [&](int n) {
    const int t = n * gridDim.x + (MODE == XG_WGRAD && (n & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
    return t;
  };
  const int rounds = (tiles + gridDim.x - 1) / gridDim.x;
  // tile -> (expert, first row of A / first output row, first column, K blocks)
  struct Tile {
    int e, m0, n0, r0, nk, se;
  };
  auto tile_of = [&](int t) {
    Tile o;
    const int m = t / g.tn;
    o.n0 = (t - m * g.tn) * BN;
    if constexpr (MODE == XG_WGRAD) {
      const int sr = m / g.tm, part = sr / g.E;
      o.e = plan[g.lay.o_order + sr - part * g.E];
      o.m0 = (m - sr * g.tm) * XG_BM;
      o.se = part * g.E + o.e;
      const int nk = (plan[g.lay.o_cnt + o.e] + XG_BK - 1) / XG_BK;
      const int k0 = (int)((int64_t)nk * part / g.split);
      o.r0 = plan[g.lay.o_seg + o.e] + k0 * XG_BK;
      o.nk = (int)((int64_t)nk * (part + 1) / g.split) - k0;
    } else {
      o.e = plan[g.lay.o_tile + m];
      o.m0 = o.r0 = m * XG_BM;
      o.nk = (g.K + XG_BK - 1) / XG_BK;
    }
    return o;
  };
  const int p0 = g.np == 3 ? 0 : 5;              // passes over the planes: p0 .. 5

  if (warp == 0) {
    // ------------------------------------------------------------------------------------------ loads
    if (lane == 0) {
      int seq = 0;
      bool ok = true;
      for (int r = 0; ok && r < rounds; ++r) {
        const int t = tile_at(r);
        if (t >= tiles) break;                     // only in the last round
        const Tile w = tile_of(t);
        for (int p = p0; ok && p < 6; ++p) {
          const int pa = xg_plane_a(p), pb = xg_plane_b(p);
          for (int kb = 0; kb < w.nk; ++kb, ++seq) {
            const int s = seq % C::STAGES;
            if (*failed || !mbar_wait_ns(&B.empty[s], ((seq / C::STAGES) & 1) ^ 1, XG_WAIT_NS)) {
              *failed = 1;
              ok = false;
              break;
            }
            const uint32_t a = smem_u32(smem + s * C::STAGE), b = a + C::A_BYTES;
            uint64_t* bar = &B.full[s];
            mbar_arrive_tx(bar, C::STAGE);
            const int k0 = kb * XG_BK;
            if constexpr (MODE == XG_WGRAD) {
#pragma unroll
              for (int c = 0; c < XG_BM / 64; ++c)
                tma_load_2d(a + c * 8192, &map_a, w.m0 + 64 * c, (int)(pa * g.rows) + w.r0 + k0, bar);
#pragma unroll
              for (int c = 0; c < BN / 64; ++c)
                tma_load_2d(b + c * 8192, &map_b, w.n0 + 64 * c, (int)(pb * g.rows) + w.r0 + k0, bar);
            } else {
              tma_load_2d(a, &map_a, k0, (int)(pa * g.rows) + w.m0, bar);
              if constexpr (MODE == XG_FWD) {
                tma_load_3d(b, &map_b, k0, w.n0, pb * g.w_rows + w.e, bar);
              } else {
#pragma unroll
                for (int c = 0; c < BN / 64; ++c)
                  tma_load_3d(b + c * 8192, &map_b, w.n0 + 64 * c, k0, pb * g.w_rows + w.e, bar);
              }
            }
          }
        }
      }
      // after a timeout: the copies already issued land before the block ends (bounded)
      if (!ok)
        for (int q = seq - C::STAGES < 0 ? 0 : seq - C::STAGES; q < seq; ++q)
          mbar_wait_ns(&B.full[q % C::STAGES], (q / C::STAGES) & 1, XG_WAIT_NS);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------------------------------ MMA issue
    if (lane == 0) {
      constexpr uint32_t idesc = f16_idesc(XG_BM, BN, !std::is_same<T, f16>::value, A_MN, B_MN);
      int seq = 0, tc = 0;
      bool ok = true;
      uint64_t* last_bar = nullptr;
      uint32_t last_par = 0;
      for (int r = 0; ok && r < rounds; ++r) {
        const int t = tile_at(r);
        if (t >= tiles) break;
        const Tile w = tile_of(t);
        if (w.nk == 0) continue;
        const int acc = tc & 1;
        if (*failed || !mbar_wait_ns(&B.acc_empty[acc], ((tc >> 1) & 1) ^ 1, XG_WAIT_NS)) {
          *failed = 1;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem + (uint32_t)(acc * BN);
        const int total = w.nk * (6 - p0);
        for (int kb = 0; kb < total; ++kb, ++seq) {
          const int s = seq % C::STAGES;
          if (!mbar_wait_ns(&B.full[s], (seq / C::STAGES) & 1, XG_WAIT_NS)) {
            *failed = 1;
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t a = smem_u32(smem + s * C::STAGE), b = a + C::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < XG_BK / 16; ++kk) {
            // 16 K elements: 32 bytes along a K-major row, two 8-row atoms of an MN-major operand
            const uint64_t ad = A_MN ? sw128_desc_mn(a + kk * 2048, 8192) : sw128_desc(a + kk * 32);
            const uint64_t bd = B_MN ? sw128_desc_mn(b + kk * 2048, 8192) : sw128_desc(b + kk * 32);
            mma_f16_ss(d, ad, bd, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
          }
          mma_commit(&B.empty[s]);
          last_bar = &B.empty[s];
          last_par = (seq / C::STAGES) & 1;
        }
        if (!ok) break;
        mma_commit(&B.acc_full[acc]);
        last_bar = &B.acc_full[acc];
        last_par = (tc >> 1) & 1;
        ++tc;
      }
      // after a timeout: wait (bounded) for the MMAs already issued before the TMEM is freed
      if (*failed && last_bar) mbar_wait_ns(last_bar, last_par, XG_WAIT_NS);
    }
  } else {
    // ------------------------------------------------------------------------------------------ epilogue
    // One row per lane out of TMEM; rows pass through shared memory in pieces of 128 bytes so that global accesses are
    // whole 128-byte segments of four rows (one row per lane: 32 scattered 16-byte pieces per access, which held a tile
    // for longer than its products at K <= 1024).
    const int q4 = warp & 3, row = q4 * 32 + lane;
    unsigned char* stg = smem + C::STAGES * C::STAGE + (warp - 2) * XG_STG;
    constexpr int NC = 128 / (int)sizeof(OUT);     // columns of a piece
    constexpr int XV = kVec<T>;
    const int r8 = lane >> 3, c8 = lane & 7;       // this lane's row (of four) and 16-byte piece in whole-segment accesses
    const bool vec = g.ldo % kVec<OUT> == 0 && (reinterpret_cast<uintptr_t>(g.out) & 15) == 0;
    const bool xvec = MODE == XG_DGRAD && g.ldx % XV == 0 && (reinterpret_cast<uintptr_t>(g.x) & 15) == 0;
    int tc = 0;
    // every exit decision is warp-uniform: the loop body holds warp-collective tcgen05.ld.sync.aligned
    for (int r = 0; r < rounds; ++r) {
      if (__shfl_sync(0xffffffffu, *failed, 0)) break;
      const int t = tile_at(r);
      if (t >= tiles) break;
      const Tile w = tile_of(t);
      OUT* dst = nullptr;
      float sc = 1.f, dot = 0.f;
      const T* xr = nullptr;
      int slot = -1;
      if constexpr (MODE == XG_WGRAD) {
        if (w.m0 + row < g.M) dst = (OUT*)g.out + ((int64_t)w.se * g.M + w.m0 + row) * g.ldo + w.n0;
      } else {
        slot = plan[g.lay.o_row + w.m0 + row];
        if (slot >= 0) {
          if (g.out) dst = (OUT*)g.out + (int64_t)slot * g.ldo + w.n0;
          if (g.scale) sc = g.scale[slot];
          if (MODE == XG_DGRAD && g.dgpart) xr = (const T*)g.x + (int64_t)(slot / g.kdiv) * g.ldx + w.n0;
        }
      }
      const int acc = tc & 1, nc = g.N - w.n0 < BN ? g.N - w.n0 : BN;
      // the x rows' pieces for the dot products, loaded one piece ahead (and the first before the wait)
      uint4 xq[MODE == XG_DGRAD ? 8 : 1];
      auto fetch_x = [&](int h) {
        const int n = nc - h * NC < NC ? nc - h * NC : NC;
#pragma unroll
        for (int i = 0; i < (MODE == XG_DGRAD ? 8 : 0); ++i) {
          const T* xp =
              reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<uintptr_t>(xr), 4 * i + r8));
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (xp) {
            xp += h * NC + c8 * XV;
            if (xvec && (c8 + 1) * XV <= n) {
              v = *reinterpret_cast<const uint4*>(xp);
            } else {
              float f[XV];
#pragma unroll
              for (int q = 0; q < XV; ++q) f[q] = c8 * XV + q < n ? to_f(xp[q]) : 0.f;
              v = pack16<T>(f);
            }
          }
          xq[i] = v;
        }
      };
      if (MODE == XG_DGRAD && g.dgpart) fetch_x(0);
      if (w.nk > 0) {
        if (!__all_sync(0xffffffffu, mbar_wait_ns(&B.acc_full[acc], (tc >> 1) & 1, XG_WAIT_NS))) {
          *failed = 1;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
#pragma unroll 1
      for (int h = 0; h * NC < nc; ++h) {
        const int n = nc - h * NC < NC ? nc - h * NC : NC;
        uint32_t u[NC];
        if (w.nk > 0) {
          const uint32_t ta = tmem + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * BN + NC * h);
#pragma unroll
          for (int q = 0; q < NC / 32; ++q) tmem_ld32(ta + 32 * q, *reinterpret_cast<uint32_t(*)[32]>(u + 32 * q));
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < NC; ++i) u[i] = 0u;
        }
        if constexpr (MODE == XG_DGRAD) {          // dot += <x row, row> over this piece's columns
          if (g.dgpart) {
            // a piece of 128 bytes of x holds as many columns as one of the output: T = OUT here
#pragma unroll
            for (int i = 0; i < (MODE == XG_DGRAD ? 8 : 0); ++i) *xg_stg(stg, 4 * i + r8, c8) = xq[i];
            if ((h + 1) * NC < nc) fetch_x(h + 1);
            __syncwarp();
            // one short chain per vector, added up as a tree: the rounding of 256 terms in a row would show
            float part[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              float f[XV];
              unpack16(*xg_stg(stg, lane, c), f, T());
              part[c] = 0.f;
#pragma unroll
              for (int q = 0; q < XV; ++q) part[c] = fmaf(f[q], __uint_as_float(u[c * XV + q]), part[c]);
            }
            dot += ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
            __syncwarp();
          }
        }
        if (MODE == XG_WGRAD || g.out) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float f[kVec<OUT>];
#pragma unroll
            for (int q = 0; q < kVec<OUT>; ++q) {
              const float v = __uint_as_float(u[c * kVec<OUT> + q]);
              f[q] = MODE == XG_WGRAD ? v : v * sc;
            }
            *xg_stg(stg, lane, c) = pack16<OUT>(f);
          }
          __syncwarp();
          if (vec && n == NC) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              OUT* p = reinterpret_cast<OUT*>(__shfl_sync(0xffffffffu, reinterpret_cast<uintptr_t>(dst), 4 * i + r8));
              if (p) *reinterpret_cast<uint4*>(p + h * NC + c8 * kVec<OUT>) = *xg_stg(stg, 4 * i + r8, c8);
            }
          } else {                                 // odd strides and the last columns: one row at a time, lanes along it
#pragma unroll 4
            for (int r = 0; r < 32; ++r) {
              OUT* p = reinterpret_cast<OUT*>(__shfl_sync(0xffffffffu, reinterpret_cast<uintptr_t>(dst), r));
#pragma unroll
              for (int q = 0; q < NC / 32; ++q) {
                const int c = lane + 32 * q;
                if (p && c < n)
                  p[h * NC + c] = reinterpret_cast<const OUT*>(xg_stg(stg, r, c / kVec<OUT>))[c % kVec<OUT>];
              }
            }
          }
          __syncwarp();
        }
      }
      if (MODE == XG_DGRAD && xr) g.dgpart[(int64_t)(w.n0 / BN) * g.lay.R + slot] = dot;
      if (w.nk > 0) {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive(&B.acc_empty[acc]);
        ++tc;
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (tid == 0 && *failed) atomicOr((unsigned*)plan + 1, (unsigned)MB_ST_TC_TIMEOUT);
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------ host side
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeTiled)p;
  }();
  return fn;
}

// Tensor map of a 16-bit tensor, dimensions inner to outer, SWIZZLE_128B boxes 64 elements wide
static int xg_map(CUtensorMap* m, bool is_bf16, int rank, const void* p, const int64_t* dims, const int64_t* strides,
                  const int* box) {
  EncodeTiled enc = encode_tiled();
  if (!enc) {
    set_error("expert_linear: the driver has no cuTensorMapEncodeTiled");
    return MB_E_CUDA;
  }
  cuuint64_t d[3], s[2];
  cuuint32_t b[3], es[3] = {1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    d[i] = (cuuint64_t)dims[i];
    b[i] = (cuuint32_t)box[i];
    if (i) s[i - 1] = (cuuint64_t)strides[i - 1] * 2;
  }
  const CUresult rc = enc(m, is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                          const_cast<void*>(p), d, s, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) {
    set_error("expert_linear: cuTensorMapEncodeTiled failed (%d)", (int)rc);
    return MB_E_CUDA;
  }
  return 0;
}

static int xg_bn(int64_t N) { return N <= 128 ? 128 : 256; }
int xgemm_n_tiles(int mode, int64_t N) {
  (void)mode;
  return (int)((N + xg_bn(N) - 1) / xg_bn(N));
}

// Parts of each expert's rows in WGRAD: enough tiles for four per SM when there are few, with at least 16 K blocks left
// in an average part (below that the partial sums cost more than the idle SMs)
int xgemm_split(int64_t E, int64_t M, int64_t N, int64_t slots, int planes) {
  const int64_t tiles = E * ((M + XG_BM - 1) / XG_BM) * ((N + xg_bn(N) - 1) / xg_bn(N));
  const int64_t blocks = slots / E / XG_BK * (planes == 3 ? 6 : 1);
  int64_t s = 4 * (int64_t)sm_count() / tiles;
  if (s > blocks / 16) s = blocks / 16;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

template <int MODE, typename T, typename OUT, int BN>
static int xg_go(const XGemm& x, cudaStream_t st) {
  using C = XgCfg<BN>;
  static int ready_dev = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("expert_linear (device)");
  auto kern = k_expert_gemm<MODE, T, OUT, BN>;
  if (ready_dev != dev) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) {
      set_error("expert_linear: cannot reserve %d bytes of shared memory", C::SMEM);
      return MB_E_CUDA;
    }
    ready_dev = dev;
  }
  const bool is_bf16 = !std::is_same<T, f16>::value;
  const int np = x.dtype == MB_F32 ? 3 : 1;
  CUtensorMap ma, mbm;
  {
    const int64_t dims[2] = {x.lda, np * x.rows}, str[1] = {x.lda};
    const int box[2] = {64, MODE == XG_WGRAD ? XG_BK : XG_BM};
    if (int rc = xg_map(&ma, is_bf16, 2, x.a, dims, str, box)) return rc;
  }
  if (MODE == XG_WGRAD) {
    const int64_t dims[2] = {x.ldb, np * x.rows}, str[1] = {x.ldb};
    const int box[2] = {64, XG_BK};
    if (int rc = xg_map(&mbm, is_bf16, 2, x.b, dims, str, box)) return rc;
  } else {
    const int64_t O = MODE == XG_FWD ? x.N : x.K;
    const int64_t dims[3] = {x.ldb, O, (int64_t)np * x.E}, str[2] = {x.ldb, x.ldb * O};
    const int box[3] = {64, MODE == XG_FWD ? BN : XG_BK, 1};
    if (int rc = xg_map(&mbm, is_bf16, 3, x.b, dims, str, box)) return rc;
  }
  XgParams g{};
  g.E = x.E; g.M = x.M; g.N = x.N; g.K = x.K; g.np = np;
  g.tn = (x.N + BN - 1) / BN;
  g.tm = (x.M + XG_BM - 1) / XG_BM;
  g.rows = x.rows; g.w_rows = x.E;
  g.plan = x.plan; g.lay = x.lay; g.scale = x.scale;
  g.out = x.out; g.ldo = x.ldo;
  g.split = x.split > 1 ? x.split : 1;
  g.x = x.x; g.ldx = x.ldx; g.kdiv = x.kdiv; g.dgpart = x.dgpart;
  const int64_t most = MODE == XG_WGRAD ? (int64_t)g.split * x.E * g.tm * g.tn : x.lay.tiles * g.tn;
  if (most > 0x7fffffff || np * x.rows > 0x7fffffff) {
    set_error("expert_linear: too many tiles (%lld) or rows (%lld)", (long long)most, (long long)(np * x.rows));
    return MB_E_ARG;
  }
  if (most == 0) return 0;
  const int sms = sm_count();
  kern<<<(unsigned)(most < sms ? most : sms), XG_THREADS, C::SMEM, st>>>(ma, mbm, g);
  return check_launch("expert_linear");
}

template <int MODE, typename T>
static int xg_bn_any(const XGemm& x, cudaStream_t st) {
  if constexpr (MODE == XG_WGRAD)
    if (x.split > 1) return xg_bn(x.N) == 128 ? xg_go<MODE, T, float, 128>(x, st) : xg_go<MODE, T, float, 256>(x, st);
  return xg_bn(x.N) == 128 ? xg_go<MODE, T, T, 128>(x, st) : xg_go<MODE, T, T, 256>(x, st);
}

template <int MODE>
static int xg_type(const XGemm& x, cudaStream_t st) {
  if (x.dtype == MB_F32) return xg_bn_any<MODE, float>(x, st);
  return x.dtype == MB_BF16 ? xg_bn_any<MODE, bf16>(x, st) : xg_bn_any<MODE, f16>(x, st);
}

int xgemm_launch(const XGemm& x, cudaStream_t st) {
  if (x.mode == XG_FWD) return xg_type<XG_FWD>(x, st);
  return x.mode == XG_DGRAD ? xg_type<XG_DGRAD>(x, st) : xg_type<XG_WGRAD>(x, st);
}

int sm_count() {
  static int dev_known = -1, sms = 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev != dev_known) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    sms = n;
    dev_known = dev;
  }
  return sms;
}

}  // namespace mb
