// The three expert products on the 5th-generation tensor cores (tcgen05 kind::f16, fp32 accumulators in TMEM):
//   FWD    C[row][o] = sum_d x[row][d] W[e][o][d]        both operands K-major
//   DGRAD  C[row][d] = sum_o dy[row][o] W[e][o][d]       W is MN-major (its rows run along N)
//   WGRAD  C[e][o][d] = sum over e's rows dy[row][o] x[row][d]   both MN-major, K = the expert's rows
// Rows are sorted by expert and padded to 128, so a 128-row tile (FWD, DGRAD) or a 64-row K block (WGRAD) has one expert,
// and no matrix is transposed in memory: the MN-major operands are read as they lie.
// fp32 data comes as three bf16 planes; a stage holds all three of both operands.  The product of the first planes has an
// accumulator of its own, and the five others whose ranks add up to at most 2 share another; the rest is below 2^-24 of
// the sum of the absolute products.
// WGRAD with routing weights multiplies rows by fp32 weights of any size: x g comes as two bf16 planes (2^-16 of it, and the
// exponents of fp32), and fp16 dy as two, which hold it exactly.  The product of the second planes is left out (2^-18).
// One plane in the type itself was 1.4 times as far off as one rounding, and left the range of fp16 (x g above 65,504,
// or below 6e-5) where the gradient does not.
// The tensor cores truncate when they add to an fp32 accumulator.  Sums of one sign lose 1e-7 of themselves for each 16-wide
// step (measured: 2.5e-3 after 25,000 steps), products of either sign less (a deviation of 3.2e-6 after 192 steps, 4.7e-7
// after 32).  Where the result leaves in fp32 (fp32 data, and the gradient of the routing weights) an accumulator therefore
// takes a few K blocks at most, and the chunks are added in registers with rounding to nearest (7e-7 for sums of one sign).
// 16-bit results take up to xg_acc_long K blocks in one accumulator.  Longer sums are cut: WGRAD into parts that are added in
// fp32 afterwards, FWD and DGRAD into chunks in registers.
//
// Persistent CTAs, one per SM.  Warp 0 loads tiles with TMA (SWIZZLE_128B) into a ring of stages, warp 1 issues the MMAs
// into one of two TMEM accumulators, warps 4-11 drain the other one (a lane holds half a row).  CG = 2: a cluster of two
// CTAs works on a 256-row tile (cta_group::2, each CTA holds its 128 rows of A and half of B's columns), which halves the
// B bytes a CTA fetches.
// The N tile is the smallest multiple of 64 that cuts N into ceil(N / 256) tiles.
// WGRAD cuts an expert's rows into parts of kc K blocks when there are few tiles; parts of an expert with several are
// added up afterwards in their order.  Items come longest expert first and odd rounds run backwards over the CTAs, so
// that every CTA gets about the same number of K blocks.
// Every wait is bounded: on expiry the kernel sets MB_ST_TC_TIMEOUT in the plan's status word, fills the tiles that it has no
// result for with NaN, drains its copies and MMAs, frees its TMEM and returns.
//
// What bounds it (B200; copy 6.5 TB/s, cuBLAS bf16 1.64 PFLOP/s in a burst and 1.37 sustained): 262,144 slots on 64 experts,
// 1024 -> 2048 bf16, pairs: forward 833 us, dx alone about 780, dW without weights 815 (1.32, 1.4, 1.35 PFLOP/s): the
// operands' way from L2 into shared memory (11 TB/s).  With rows that leave in fp32 (k > 1): forward 951, dx with the gradient of
// the weights 1044: their bytes.  dW with weights 1436 (1.53 PFLOP/s of its two products): the MMAs.  48,000 slots on 16
// experts, 512 -> 515 fp16, k = 2: 41 / 66 / 88 us: 8 or 9 K blocks a tile, and the drain of a tile takes about as long.
// 16,384 slots on 89 experts, 128 -> 512 fp32: 25 / 34 / 30 us: two or three rounds of short tiles and the latency of their first
// loads.
#include <cuda.h>

#include <type_traits>

#include "experts.cuh"
#include "tc.cuh"

namespace mb {

constexpr int XG_BM = XP_BM, XG_BK = 64, XG_EPI_WARPS = 8, XG_EPI0 = 4, XG_THREADS = 32 * (XG_EPI0 + XG_EPI_WARPS);
// Registers of a thread in the first four warps and in the epilogue's, where the latter hold half a row of 256 columns:
// 128 x 72 + 256 x 216 = 384 x 168, what the block is launched with
constexpr int XG_REGS = 168, XG_REGS_LOW = 72, XG_REGS_HIGH = 216;
static_assert(32 * (XG_EPI0 * XG_REGS_LOW + XG_EPI_WARPS * XG_REGS_HIGH) <= XG_THREADS * XG_REGS, "registers");
// Limit of every wait (a tile takes microseconds), and whether the first load of CTA 0 goes missing once:
// mace_b200_expert_test_hooks sets them, so that a test drives the timeout path without any fault.
__device__ unsigned long long g_xg_wait_ns = 2000000000ull;
__device__ int g_xg_skip_load = 0;
constexpr int XG_STG = 2048;                     // row staging of one epilogue warp
// Most K blocks of an accumulator whose result leaves in fp32: of fp32 data, of 16-bit data, and where each CTA has one tile
// at most (its drains cost nothing then).  Gradients of the routing weights from 16-bit data, 2,048 columns: error 7e-7 at
// 12, 4.8e-7 at 8; 65,536 x 4 slots, 1024 -> 2048: dx with them 80 us longer at 8.
constexpr int XG_ACC_K = 8, XG_ACC_K16 = 12, XG_ACC_K1 = 4;
// and of one whose result leaves in 16 bits: sums of one sign lose 5.2e-5 over 8,192 terms of fp16 (rounding: 2.1e-4), 1e-4 over
// 16,384 of bf16 (rounding: 1.6e-3)
__host__ __device__ constexpr int xg_acc_long(int dtype) { return dtype == MB_F16 ? 128 : 256; }

// T: element type; BN: most columns of a tile that a CTA (of CG) holds operands and accumulators for; SPL: XGemm::split
template <typename T, int BN, int CG, bool SPL>
struct XgCfg {
  static constexpr bool F32 = sizeof(T) == 4, AS_BF16 = SPL || !std::is_same<T, f16>::value;
  static constexpr int PA = F32 ? 3 : SPL && std::is_same<T, f16>::value ? 2 : 1, PB = F32 ? 3 : SPL ? 2 : 1;   // planes
  static constexpr int PRODS = PA == 3 ? 6 : PA + PB - 1;    // products of planes: ranks that add up to 2 (fp32) or 1 at most
  static constexpr int A_BYTES = XG_BM * XG_BK * 2, B_BYTES = BN / CG * XG_BK * 2;
  static constexpr int STAGE = PA * A_BYTES + PB * B_BYTES;
  static constexpr int STAGES = 196608 / STAGE;
  static constexpr int ACC = F32 ? 2 * BN : BN;              // TMEM columns of an accumulator (fp32: both of them)
  static constexpr int TMEM = 2 * ACC;
  // WGRAD, per expert, longest first: first item [E + 1], expert, first row, K blocks
  static constexpr int PRE = (4 * MB_PLAN_MAX_EXPERTS + 1) * 4 + 252;
  static constexpr int SMEM = STAGES * STAGE + XG_EPI_WARPS * XG_STG + PRE + 256 + 1024;   // + barriers, alignment slack
  static_assert(STAGES >= 2 && STAGES <= 8 && SMEM <= 227 * 1024 && TMEM <= 512 && PRE % 256 == 0, "shared memory");
};

struct XgParams {
  int32_t E, M, N, K, bn, tn, tm, kc;            // bn columns a tile, tn / tm tiles along N / M (WGRAD), kc see above
  int64_t rows;                                  // rows per plane of the sorted operands
  const int32_t* plan;
  XPlan lay;
  const float* scale;
  void* out;
  float* parts;
  int32_t* pre;
  int64_t ldo;
  int32_t out32;
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

struct XgTile {
  int e, m0, n0, r0, nk, ck;                     // expert; first row, column; first K row (WGRAD); K blocks, of a chunk
  int part;                                      // WGRAD: >= 0: the item's place in the partial sums
  bool rows_ok;                                  // FWD / DGRAD: this CTA's rows belong to the expert
};

// Row staging of the epilogue: a warp's 32 rows x 64 bytes, 16-byte piece c of row r at piece c ^ (r / 2 % 4), so that a
// lane's access to its own row and the warp's access to eight whole row segments are both free of bank conflicts.
__device__ __forceinline__ uint32_t xg_stg(uint32_t stg, int row, int c) {
  return stg + row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
}
// element i of a staged piece
template <typename OUT>
__device__ __forceinline__ OUT xg_elem(uint32_t piece, int i) {
  if constexpr (sizeof(OUT) == 4) {
    return __uint_as_float(lds32(piece + 4 * i));
  } else {
    const uint16_t u = lds16(piece + 2 * i);
    return *reinterpret_cast<const OUT*>(&u);
  }
}

// 16-byte piece l % 4 of the rows 8 i + l / 4 (i = 0 .. 3) is what lane l of a warp moves between shared and global memory;
// row[i] is the row's place there, -1: none.
template <typename T>
__device__ __forceinline__ void xg_fetch(uint4 (&xq)[4], const int (&row)[4], const T* x, int64_t ldx, bool xvec, int left) {
  constexpr int XV = kVec<T>;
  const int c = (threadIdx.x & 3) * XV;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (row[i] >= 0 && c < left) {
      const T* xp = x + row[i] * ldx + c;
      if (xvec && c + XV <= left) {
        u = *reinterpret_cast<const uint4*>(xp);
      } else {
        float f[XV];
#pragma unroll
        for (int q = 0; q < XV; ++q) f[q] = c + q < left ? to_f(xp[q]) : 0.f;
        u = pack16<T>(f);
      }
    }
    xq[i] = u;
  }
}

// Writes 32 columns of the rows that the lanes of a warp hold (v, one row per lane), scaled, through shared memory in pieces
// of 64 bytes: global accesses are whole sectors of eight rows (one row per lane would be 32 scattered 16-byte pieces per
// access, and held a tile for longer than its products at K <= 1024).  out: first column; left: columns that exist.
// Everything that does not change from piece to piece is in XgLane.
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

template <typename OUT>
__device__ __forceinline__ void xg_emit32(const float* v, const XgLane& a, uint32_t stg, const int (&row)[4], OUT* out,
                                          int64_t ldo, bool vec, float sc, int left) {
  constexpr int NC = 64 / (int)sizeof(OUT), OV = kVec<OUT>;   // columns of a piece, of a vector
  const int lane = threadIdx.x & 31, c4 = lane & 3;
  const bool whole = vec && left >= 32;
#pragma unroll
  for (int h = 0; h < 32 / NC; ++h) {
    const int n = left - h * NC;
    if (n <= 0) break;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float f[OV];
#pragma unroll
      for (int q = 0; q < OV; ++q) f[q] = v[h * NC + c * OV + q] * sc;
      sts128(a.own[c], pack16<OUT>(f));
    }
    __syncwarp();
    if (whole) {
      OUT* p = out + h * NC + c4 * OV;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (row[i] >= 0) *reinterpret_cast<uint4*>(p + row[i] * ldo) = lds128(a.seg[i]);
    } else if (vec) {
      const int mine = n - c4 * OV;              // columns of this lane's piece
      OUT* p = out + h * NC + c4 * OV;
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        const int at = i == 0 ? row[0] : i == 1 ? row[1] : i == 2 ? row[2] : row[3];
        const uint32_t s = xg_stg(stg, 8 * i + (lane >> 2), c4);
        if (at < 0) continue;
        if (mine >= OV)
          *reinterpret_cast<uint4*>(p + at * ldo) = lds128(s);
        else
          for (int q = 0; q < mine; ++q) p[at * ldo + q] = xg_elem<OUT>(s, q);
      }
    } else {                                     // odd strides: one row at a time (two of 16 columns), lanes along it
      constexpr int RP = 32 / NC;
#pragma unroll 1
      for (int r = 0; r < 32; r += RP) {
        const int rr = r + lane / NC, c = lane % NC, i = r >> 3;
        const int mine = i == 0 ? row[0] : i == 1 ? row[1] : i == 2 ? row[2] : row[3];
        const int at = __shfl_sync(0xffffffffu, mine, (rr & 7) * 4);
        if (at >= 0 && c < n) out[at * ldo + h * NC + c] = xg_elem<OUT>(xg_stg(stg, rr, c / OV), c % OV);
      }
    }
    __syncwarp();
  }
}

// Scalar products of the columns of the lanes' rows that a piece of x (64 bytes a row, in xq by xg_fetch) covers
template <typename T>
__device__ __forceinline__ float xg_dot(const float* v, const XgLane& a, const uint4 (&xq)[4]) {
  constexpr int XV = kVec<T>;
#pragma unroll
  for (int i = 0; i < 4; ++i) sts128(a.seg[i], xq[i]);
  __syncwarp();
  float part[4];                                 // short chains, added up as a tree
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float f[XV];
    unpack16(lds128(a.own[c]), f, T());
    part[c] = 0.f;
#pragma unroll
    for (int q = 0; q < XV; ++q) part[c] = fmaf(f[q], v[c * XV + q], part[c]);
  }
  __syncwarp();
  return (part[0] + part[1]) + (part[2] + part[3]);
}

// DOT: DGRAD with dgpart; LONG: FWD or DGRAD of 16-bit data with K of more than xg_acc_long blocks
template <int MODE, typename T, int BN, int CG, bool DOT, bool SPL, bool LONG>
__global__ void __launch_bounds__(XG_THREADS, 1)
    k_expert_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const XgParams g) {
  using C = XgCfg<T, BN, CG, SPL>;
  constexpr bool A_MN = MODE == XG_WGRAD, B_MN = MODE != XG_FWD;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* stg0 = smem + C::STAGES * C::STAGE;
  int* pre = reinterpret_cast<int*>(stg0 + XG_EPI_WARPS * XG_STG);
  XgBars& B = *reinterpret_cast<XgBars*>(stg0 + XG_EPI_WARPS * XG_STG + C::PRE);
  volatile int* failed = &B.failed;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = CG == 2 ? (int)cluster_ctarank() : 0, cta = blockIdx.x / CG, ctas = gridDim.x / CG;
  const int32_t* plan = g.plan;
  const unsigned long long wait_ns = *(volatile unsigned long long*)&g_xg_wait_ns;

  if (warp == 1) {
    tmem_alloc<CG>(&B.tmem, C::TMEM);
    if (lane == 0) {
      for (int s = 0; s < C::STAGES; ++s) {
        mbar_init(&B.full[s], 1);
        mbar_init(&B.empty[s], 1);
      }
      for (int a = 0; a < 2; ++a) {
        mbar_init(&B.acc_full[a], 1);
        mbar_init(&B.acc_empty[a], XG_EPI_WARPS * CG);
      }
      B.failed = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  int *by_ex = pre + g.E + 1, *by_row = by_ex + g.E, *by_nk = by_row + g.E;
  if (MODE == XG_WGRAD && warp == 0) {
    int run = 0;
    for (int e0 = 0; e0 < g.E; e0 += 32) {
      const int e = e0 + lane;
      int n = 0;
      if (e < g.E) {
        const int ex = plan[g.lay.o_order + e], nk = (plan[g.lay.o_cnt + ex] + XG_BK - 1) / XG_BK;
        n = nk <= g.kc ? 1 : (nk + g.kc - 1) / g.kc;
        by_ex[e] = ex;
        by_row[e] = plan[g.lay.o_seg + ex];
        by_nk[e] = nk;
      }
      int inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (e < g.E) pre[e] = run + inc - n;
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) pre[g.E] = run;
    __syncwarp();
    if (g.pre && blockIdx.x == 0)
      for (int e = lane; e <= g.E; e += 32) g.pre[e] = pre[e];
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();         // the peer's barriers are initialised
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = B.tmem;
  const int tiles = MODE == XG_WGRAD ? pre[g.E] * g.tm * g.tn : plan[CG == 2 ? 2 : 0] * g.tn;
  const int rounds = (tiles + ctas - 1) / ctas;
  constexpr bool CHUNKS = sizeof(T) == 4 || DOT || LONG;
  auto tile_at = [&](int n) { return n * ctas + (MODE == XG_WGRAD && (n & 1) ? ctas - 1 - cta : cta); };
  auto tile_of = [&](int t) {
    XgTile o;
    const int m = t / g.tn;
    o.n0 = (t - m * g.tn) * g.bn;
    o.part = -1;
    o.rows_ok = true;
    if constexpr (MODE == XG_WGRAD) {
      const int item = m / g.tm;
      o.m0 = (m - item * g.tm) * (XG_BM * CG) + rank * XG_BM;
      int lo = 0, hi = g.E - 1;                  // last expert whose first item is <= item
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (pre[mid] <= item)
          lo = mid;
        else
          hi = mid - 1;
      }
      o.e = by_ex[lo];
      const int nk = by_nk[lo], parts = pre[lo + 1] - pre[lo], q = item - pre[lo];
      const int k0 = (int)((int64_t)nk * q / parts);
      o.r0 = by_row[lo] + k0 * XG_BK;
      o.nk = (int)((int64_t)nk * (q + 1) / parts) - k0;
      if (parts > 1) o.part = item;
    } else {
      const int tile = CG == 2 ? plan[g.lay.o_pair + m] : m;
      o.e = plan[g.lay.o_tile + tile];
      o.m0 = (tile + rank) * XG_BM;
      o.r0 = 0;
      if (CG == 2 && rank == 1) o.rows_ok = o.m0 < plan[g.lay.o_seg + o.e + 1];
      o.nk = (g.K + XG_BK - 1) / XG_BK;
    }
    o.ck = o.nk;                                 // K blocks of one accumulator: even chunks
    if constexpr (CHUNKS) {
      constexpr int LONGEST = xg_acc_long(std::is_same<T, f16>::value ? MB_F16 : MB_BF16);
      const int most = LONG ? LONGEST : rounds == 1 ? XG_ACC_K1 : C::F32 ? XG_ACC_K : XG_ACC_K16;
      const int n = (o.nk + most - 1) / most;
      if (n > 1) o.ck = (o.nk + n - 1) / n;
    }
    return o;
  };
  const int bh = g.bn / CG;                      // columns of B that this CTA loads
  constexpr bool SPLIT = DOT && BN == 256;       // registers move from the first four warps to the epilogue's

  if (warp < XG_EPI0) {
  if constexpr (SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(XG_REGS_LOW));
  if (warp == 0) {
    // ------------------------------------------------------------------------------------------ loads
    if (lane == 0) {
      int seq = 0;
      bool ok = true;
      const uint32_t b_bytes = B_MN ? (uint32_t)((bh + 63) / 64) * 8192u : (uint32_t)bh * 128u;
      const uint32_t bytes = CG * (C::PA * C::A_BYTES + C::PB * b_bytes);
      XgTile next{};
      if (tile_at(0) < tiles) next = tile_of(tile_at(0));
      for (int r = 0; ok && r < rounds; ++r) {
        if (tile_at(r) >= tiles) break;          // only in the last round
        const XgTile w = next;
        if (tile_at(r + 1) < tiles) next = tile_of(tile_at(r + 1));   // its table look-ups overlap this tile
        for (int kb = 0; kb < w.nk; ++kb, ++seq) {
          const int s = seq % C::STAGES;
          if (*failed || !mbar_wait_ns(&B.empty[s], ((seq / C::STAGES) & 1) ^ 1, wait_ns)) {
            *failed = 1;
            ok = false;
            break;
          }
          if (seq == 0 && blockIdx.x == 0 && *(volatile int*)&g_xg_skip_load && atomicExch(&g_xg_skip_load, 0)) continue;
          const uint32_t bar = CG == 2 ? mapa_u32(smem_u32(&B.full[s]), 0) : smem_u32(&B.full[s]);
          if (rank == 0) mbar_arrive_tx(&B.full[s], bytes);   // both CTAs' bytes arrive at the first one's barrier
          const int k0 = kb * XG_BK;
#pragma unroll
          for (int p = 0; p < (C::PA > C::PB ? C::PA : C::PB); ++p) {
            const uint32_t a = smem_u32(smem + s * C::STAGE) + p * C::A_BYTES;
            const uint32_t b = smem_u32(smem + s * C::STAGE) + C::PA * C::A_BYTES + p * C::B_BYTES;
            const int row0 = (int)(p * g.rows);
            if constexpr (MODE == XG_WGRAD) {
              if (p < C::PA)
#pragma unroll
                for (int c = 0; c < XG_BM / 64; ++c)
                  tma_load_2d<CG>(a + c * 8192, &map_a, w.m0 + 64 * c, row0 + w.r0 + k0, bar);
#pragma unroll
              for (int c = 0; c < BN / CG / 64; ++c)
                if (c * 64 < bh) tma_load_2d<CG>(b + c * 8192, &map_b, w.n0 + rank * bh + 64 * c, row0 + w.r0 + k0, bar);
            } else {
              tma_load_2d<CG>(a, &map_a, k0, row0 + w.m0, bar);
              if constexpr (MODE == XG_FWD)
                tma_load_3d<CG>(b, &map_b, k0, w.n0 + rank * bh, p * g.E + w.e, bar);
              else
#pragma unroll
                for (int c = 0; c < BN / CG / 64; ++c)
                  if (c * 64 < bh) tma_load_3d<CG>(b + c * 8192, &map_b, w.n0 + rank * bh + 64 * c, k0, p * g.E + w.e, bar);
            }
          }
        }
      }
      // after a timeout: the copies already issued land before the block ends (bounded; a pair's land at rank 0)
      if (!ok && rank == 0)
        for (int q = seq - C::STAGES < 0 ? 0 : seq - C::STAGES; q < seq; ++q)
          mbar_wait_ns(&B.full[q % C::STAGES], (q / C::STAGES) & 1, wait_ns);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------------------------------ MMA issue
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = f16_idesc(XG_BM * CG, g.bn, C::AS_BF16, A_MN, B_MN);
      int seq = 0, tc = 0;
      bool ok = true;
      uint64_t* last_bar = nullptr;
      uint32_t last_par = 0;
      for (int r = 0; ok && r < rounds; ++r) {
        const int t = tile_at(r);
        if (t >= tiles) break;
        const XgTile w = tile_of(t);
        for (int kb0 = 0; ok && kb0 < w.nk; kb0 += w.ck, ++tc) {
          const int acc = tc & 1, kb1 = w.nk - kb0 > w.ck ? kb0 + w.ck : w.nk;
          if (*failed || !mbar_wait_ns(&B.acc_empty[acc], ((tc >> 1) & 1) ^ 1, wait_ns)) {
            *failed = 1;
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t d = tmem + (uint32_t)(acc * C::ACC);
          for (int kb = kb0; kb < kb1; ++kb, ++seq) {
            const int s = seq % C::STAGES;
            if (!mbar_wait_ns(&B.full[s], (seq / C::STAGES) & 1, wait_ns)) {
              *failed = 1;
              ok = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t a0 = smem_u32(smem + s * C::STAGE), b0 = a0 + C::PA * C::A_BYTES;
#pragma unroll
            for (int p = 0; p < C::PRODS; ++p) {
              // planes (a, b), small products first.  fp32: (0,2) (2,0) (1,1) (0,1) (1,0), then (0,0) in the other
              // accumulator; split: (1,0) of fp16, (0,1), (0,0)
              constexpr int PA3[6] = {0, 2, 1, 0, 1, 0}, PB3[6] = {2, 0, 1, 1, 0, 0};
              const int left = C::PRODS - 1 - p;
              const int pa = C::F32 ? PA3[p] : left == 2 ? 1 : 0, pb = C::F32 ? PB3[p] : left == 1 ? 1 : 0;
              const uint32_t a = a0 + pa * C::A_BYTES, b = b0 + pb * C::B_BYTES;
              const bool second = C::F32 && p < 5;
              const uint32_t dp = second ? d + BN : d;
#pragma unroll
              for (int kk = 0; kk < XG_BK / 16; ++kk) {
                // 16 K elements: 32 bytes along a K-major row, two 8-row atoms of an MN-major operand
                const uint64_t ad = A_MN ? sw128_desc_mn(a + kk * 2048, 8192) : sw128_desc(a + kk * 32);
                const uint64_t bd = B_MN ? sw128_desc_mn(b + kk * 2048, 8192) : sw128_desc(b + kk * 32);
                mma_f16_ss<CG>(dp, ad, bd, idesc, (kb > kb0 || kk > 0 || (p > 0 && second == (C::F32 && p - 1 < 5))) ? 1u : 0u);
              }
            }
            mma_commit_to<CG>(&B.empty[s]);
            last_bar = &B.empty[s];
            last_par = (seq / C::STAGES) & 1;
          }
          if (!ok) break;
          mma_commit_to<CG>(&B.acc_full[acc]);
          last_bar = &B.acc_full[acc];
          last_par = (tc >> 1) & 1;
        }
      }
      // after a timeout: wait (bounded) for the MMAs already issued before the TMEM is freed
      if (*failed && last_bar) mbar_wait_ns(last_bar, last_par, wait_ns);
    }
  }
  } else {
    // ------------------------------------------------------------------------------------------ epilogue
    if constexpr (SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(XG_REGS_HIGH));
    // warp w reads TMEM lanes 32 (w % 4) .., one row per lane, and the first or second half of the tile's columns
    const int q4 = warp & 3, row = q4 * 32 + lane, hf = (warp - XG_EPI0) >> 2, hw = g.bn / 2;
    const uint32_t stg = smem_u32(stg0) + (warp - XG_EPI0) * XG_STG;
    const bool vec = g.ldo % kVec<T> == 0 && (reinterpret_cast<uintptr_t>(g.out) & 15) == 0;
    const bool xvec = MODE == XG_DGRAD && g.ldx % kVec<T> == 0 && (reinterpret_cast<uintptr_t>(g.x) & 15) == 0;
    const XgLane at = xg_lane(stg);
    constexpr int NG = BN / 64;                    // groups of 32 columns in a half row
    constexpr int XC = 32 * 2 / (int)sizeof(T);    // columns of x in a fetch (64 bytes)
    int tc = 0;
    // after a wait that expired the rest of this CTA's tiles is filled with NaN; the flag is warp-uniform (the loop body holds
    // the warp-collective tcgen05.ld.sync.aligned)
    bool lost = false;
    for (int r = 0; r < rounds; ++r) {
      const int t = tile_at(r);
      if (t >= tiles) break;
      const XgTile w = tile_of(t);
      const int n0 = w.n0 + hf * hw, nc = g.N - n0 < hw ? g.N - n0 : hw;   // nc <= 0: nothing in this half
      int slot = -1, orow[4], xrow[4];
      float sc = 1.f, dot = 0.f;
      T* out = (T*)g.out + n0;
      float* pout = nullptr;                       // fp32 results of 16-bit data; WGRAD: partial sums
      int64_t ldo = g.ldo;
      if constexpr (MODE != XG_WGRAD) {            // in flight during the wait
        if (sizeof(T) == 2 && g.out32) pout = (float*)g.out + n0;
        slot = w.rows_ok ? plan[g.lay.o_row + w.m0 + row] : -1;
        if (slot >= 0 && g.scale) sc = g.scale[slot];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          orow[i] = __shfl_sync(0xffffffffu, slot, 8 * i + (lane >> 2));
          xrow[i] = DOT && orow[i] >= 0 ? orow[i] / g.kdiv : -1;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          orow[i] = w.m0 + q4 * 32 + 8 * i + (lane >> 2);
          if (orow[i] >= g.M) orow[i] = -1;
        }
        out += (int64_t)w.e * g.M * ldo;
        if (w.part >= 0) {
          ldo = g.N;
          pout = g.parts + (int64_t)w.part * g.M * ldo + n0;
        }
      }
      const T* x = (const T*)g.x + n0;
      uint4 xq[2][4];                              // pieces of x, two ahead (the first before the wait)
      if constexpr (DOT) {
        xg_fetch<T>(xq[0], xrow, x, g.ldx, xvec, nc);
        xg_fetch<T>(xq[1], xrow, x + XC, g.ldx, xvec, nc - XC);
      }
      auto wait = [&](int acc) {
        const bool got = !__shfl_sync(0xffffffffu, *failed, 0) &&
                         __all_sync(0xffffffffu, mbar_wait_ns(&B.acc_full[acc], (tc >> 1) & 1, wait_ns));
        if (!got) *failed = 1;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        return got;
      };
      auto release = [&](int acc) {                // one arrival per warp
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2)
            mbar_arrive_cluster(mapa_u32(smem_u32(&B.acc_empty[acc]), 0));
          else
            mbar_arrive(&B.acc_empty[acc]);
        }
      };
      auto load32 = [&](int acc, int q, float* v, bool add) {   // columns [32 q, + 32) of the half row
        const uint32_t ta = tmem + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * C::ACC + hf * hw + 32 * q);
        uint32_t u[32];
        tmem_ld32(ta, u);
        if constexpr (C::F32) {
          uint32_t u2[32];
          tmem_ld32(ta + BN, u2);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) + __uint_as_float(u2[i]));
        } else {
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = add ? v[i] + __uint_as_float(u[i]) : __uint_as_float(u[i]);
      };
      auto emit = [&](int q, const float* v) {
        if ((MODE == XG_WGRAD || sizeof(T) == 2) && pout)
          xg_emit32<float>(v, at, stg, orow, pout + 32 * q, ldo, ldo % 4 == 0, sc, nc - 32 * q);
        else
          xg_emit32<T>(v, at, stg, orow, out + 32 * q, ldo, vec, sc, nc - 32 * q);
      };
      if constexpr (!CHUNKS) {                     // one accumulator: 32 columns at a time straight from TMEM
        const int acc = tc & 1;
        if (w.nk > 0 && !lost) lost = !wait(acc);
        const bool have = w.nk > 0 && !lost;
        if (w.nk > 0 && lost) sc = __int_as_float(0x7fc00000);
#pragma unroll 1
        for (int q = 0; 32 * q < nc; ++q) {
          float v[32];
          if (have) {
            load32(acc, q, v, false);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.f;
          }
          if (have && 32 * (q + 1) >= nc) release(acc);
          emit(q, v);
        }
        if (have && nc <= 0) release(acc);
        if (w.nk > 0) ++tc;
      } else {                                     // chunks of K: their sum stays in registers
        float v[NG][32];
#pragma unroll
        for (int q = 0; q < NG; ++q)
#pragma unroll
          for (int i = 0; i < 32; ++i) v[q][i] = 0.f;
        for (int kb0 = 0; kb0 < w.nk; kb0 += w.ck, ++tc) {
          const int acc = tc & 1;
          if (!lost) lost = !wait(acc);
          if (lost) break;
#pragma unroll
          for (int q = 0; q < NG; ++q)
            if (32 * q < nc) load32(acc, q, v[q], true);
          release(acc);
        }
        if (w.nk > 0 && lost) sc = dot = __int_as_float(0x7fc00000);
        if constexpr (DOT) {
#pragma unroll
          for (int h = 0; h < 32 * NG / XC; ++h) {
            if (h * XC >= nc) break;
            dot += xg_dot<T>(&v[h * XC / 32][h * XC % 32], at, xq[h & 1]);
            const int c = (h + 2) * XC;
            if (c < nc) xg_fetch<T>(xq[h & 1], xrow, x + c, g.ldx, xvec, nc - c);
          }
        }
#pragma unroll
        for (int q = 0; q < NG; ++q)
          if (32 * q < nc && (!DOT || g.out)) emit(q, v[q]);
      }
      if (DOT && slot >= 0) g.dgpart[(int64_t)(2 * (w.n0 / g.bn) + hf) * g.lay.R + slot] = dot;
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (tid == 0 && *failed) atomicOr((unsigned*)plan + 1, (unsigned)MB_ST_TC_TIMEOUT);
  if constexpr (CG == 2) cluster_sync();         // no CTA leaves while its peer can still signal it or read its operands
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_dealloc<CG>(tmem, C::TMEM);
  }
}

// dW of the experts whose rows were cut into parts: the sum of the parts, in their order.  Block row y: expert order[y].
template <typename T>
__global__ void __launch_bounds__(256) k_parts_sum(const float* parts, const int32_t* pre, const int32_t* order, int64_t n,
                                                   bool vec, T* out) {
  const int first = pre[blockIdx.y], np = pre[blockIdx.y + 1] - first;
  if (np < 2) return;                            // written by the product itself
  T* o = out + (int64_t)order[blockIdx.y] * n;
  const float* p = parts + (int64_t)first * n;
  const int64_t step = (int64_t)gridDim.x * 256, i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t n4 = vec ? n / 4 : 0;
  for (int64_t i = i0; i < n4; i += step) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int q = 0; q < np; ++q) {
      const float4 v = *reinterpret_cast<const float4*>(p + q * n + 4 * i);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<float4*>(o + 4 * i) = s;
    else
      *reinterpret_cast<uint2*>(o + 4 * i) = make_uint2(pack2(s.x, s.y, T()), pack2(s.z, s.w, T()));
  }
  for (int64_t i = 4 * n4 + i0; i < n; i += step) {
    float s = 0.f;
    for (int q = 0; q < np; ++q) s += p[q * n + i];
    o[i] = from_f<T>(s);
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

// Widest tile: three planes of two operands fill a stage at 128 columns
static int xg_bn_max(int64_t N, int dtype) { return dtype == MB_F32 || N <= 128 ? 128 : 256; }
int xgemm_n_tiles(int64_t N, int dtype) {
  const int bn = xg_bn_max(N, dtype);
  return (int)((N + bn - 1) / bn);
}

// K blocks of a part in WGRAD: whole experts when that makes four or more rounds of tiles, else parts that make about
// that many, of at least 8 K blocks (below that the partial sums' traffic outweighs the idle SMs); for 16-bit data no more
// than an accumulator takes
int xgemm_kc(int64_t E, int64_t M, int64_t N, int64_t slots, int dtype) {
  const int64_t per = ((M + XG_BM - 1) / XG_BM) * xgemm_n_tiles(N, dtype), want = 4 * (int64_t)sm_count();
  const int64_t blocks = slots / XG_BK;          // K blocks of all experts
  const int64_t most = dtype == MB_F32 ? 0x3fffffff : xg_acc_long(dtype);
  if (E * per >= want) return (int)most;
  const int64_t kc = blocks * per / want, least = dtype == MB_F32 ? 4 : 8;
  return (int)(kc < least ? least : kc < most ? kc : most);
}
// Most partial sums there can be.  The m experts with more than kc K blocks have more than 64 kc slots each, and come first
// among the items; ceil(nk / kc) <= (nk - 1) / kc + 1 parts each, and their nk add up to slots / 64 + m at most.
int64_t xgemm_parts(int64_t E, int64_t slots, int kc) {
  const int64_t blocks = (slots + XG_BK - 1) / XG_BK, m = blocks / kc < E ? blocks / kc : E;
  return blocks / kc + m;
}

template <int MODE, typename T, int BN, int CG, bool DOT, bool SPL, bool LONG>
static int xg_go(const XGemm& x, cudaStream_t st) {
  using C = XgCfg<T, BN, CG, SPL>;
  static int ready_dev = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("expert_linear (device)");
  auto kern = k_expert_gemm<MODE, T, BN, CG, DOT, SPL, LONG>;
  if (ready_dev != dev) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) {
      set_error("expert_linear: cannot reserve %d bytes of shared memory", C::SMEM);
      return MB_E_CUDA;
    }
    cudaFuncAttributes at{};
    if (DOT && BN == 256 && (cudaFuncGetAttributes(&at, kern) != cudaSuccess || at.numRegs < XG_REGS)) {
      set_error("expert_linear: launched with %d registers a thread, %d are needed", at.numRegs, XG_REGS);
      return MB_E_CUDA;
    }
    ready_dev = dev;
  }
  XgParams g{};
  g.E = x.E; g.M = x.M; g.N = x.N; g.K = x.K;
  g.tn = (x.N + BN - 1) / BN;
  g.bn = (int)(((x.N + g.tn - 1) / g.tn + 63) / 64 * 64);
  g.tm = (x.M + XG_BM * CG - 1) / (XG_BM * CG);
  g.kc = x.kc;
  const bool is_bf16 = C::AS_BF16;
  CUtensorMap ma, mbm;
  {
    const int64_t dims[2] = {x.lda, C::PA * x.rows}, str[1] = {x.lda};
    const int box[2] = {64, MODE == XG_WGRAD ? XG_BK : XG_BM};
    if (int rc = xg_map(&ma, is_bf16, 2, x.a, dims, str, box)) return rc;
  }
  if (MODE == XG_WGRAD) {
    const int64_t dims[2] = {x.ldb, C::PB * x.rows}, str[1] = {x.ldb};
    const int box[2] = {64, XG_BK};
    if (int rc = xg_map(&mbm, is_bf16, 2, x.b, dims, str, box)) return rc;
  } else {
    const int64_t O = MODE == XG_FWD ? x.N : x.K;
    const int64_t dims[3] = {x.ldb, O, (int64_t)C::PB * x.E}, str[2] = {x.ldb, x.ldb * O};
    const int box[3] = {64, MODE == XG_FWD ? g.bn / CG : XG_BK, 1};
    if (int rc = xg_map(&mbm, is_bf16, 3, x.b, dims, str, box)) return rc;
  }
  g.rows = x.rows;
  g.plan = x.plan; g.lay = x.lay; g.scale = x.scale;
  g.out = x.out; g.ldo = x.ldo; g.out32 = x.out32;
  g.parts = x.parts; g.pre = x.pre;
  g.x = x.x; g.ldx = x.ldx; g.kdiv = x.kdiv; g.dgpart = x.dgpart;
  const int64_t items = MODE == XG_WGRAD ? (xgemm_parts(x.E, x.lay.R, x.kc) + x.E) * g.tm : x.lay.tiles;
  if (items * g.tn > 0x7fffffff || C::PB * x.rows > 0x7fffffff) {
    set_error("expert_linear: too many tiles (%lld) or rows (%lld)", (long long)(items * g.tn), (long long)(C::PB * x.rows));
    return MB_E_ARG;
  }
  if (items == 0) return 0;
  const int sms = sm_count() / CG;
  const int grid = (int)(items * g.tn < sms ? items * g.tn : sms) * CG;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(XG_THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CG > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kern, ma, mbm, g);
  if (int rc = check_launch("expert_linear")) return rc;
  if (MODE == XG_WGRAD && x.parts) {
    const int64_t n = (int64_t)x.M * x.N;
    const bool vec = n % 4 == 0 && aligned16(x.out);
    const int64_t bx = (n / (vec ? 4 : 1) + 255) / 256, most = 16 * (int64_t)sm_count() / x.E + 1;
    k_parts_sum<T><<<dim3((unsigned)(bx < most ? bx : most), x.E), 256, 0, st>>>(x.parts, x.pre, x.plan + x.lay.o_order, n,
                                                                               vec, (T*)x.out);
    return check_launch("expert_linear (parts)");
  }
  return 0;
}

// Pairs of CTAs pay with long K loops, full 256-row tiles and several rounds of them.  B200, one CTA / pairs: forward
// 262,144 slots on 64 experts, 1024 -> 2048 853 / 821 us, its dx 878 / 766, its dW 950 / 842, with its row moves and weights
// 2335 / 1974 (bf16) and 3138 / 2884 (fp16); 48,000 slots on 40 experts, 1024 -> 1024, dW with weights 303 / 247, but dx with
// their gradient 154 / 173; 48,000 slots on 16 experts, 512 -> 515 (8 K blocks; 5 or 3 row tiles of dW) forward 36 / 43 us, dW
// 49 / 55; 65,536 slots on 128 experts, 512 -> 256 (two tiles an expert) forward and sum 60 / 69 us.
static bool xg_pairs(const XGemm& x) {
  const int64_t rows = x.lay.R / x.E, tn = xgemm_n_tiles(x.N, x.dtype);
  const int64_t blocks = x.mode == XG_WGRAD ? rows / XG_BK : x.K / XG_BK;
  const int64_t m = x.mode == XG_WGRAD ? x.M : rows, tiles = x.E * ((m + 255) / 256) * tn;
  const int64_t waste = x.mode == XG_WGRAD ? (m + 255) / 256 * 256 - m : 128;
  return blocks >= 16 && 8 * waste <= m && tiles >= 8 * (int64_t)(sm_count() / 2);
}

template <int MODE, typename T, bool DOT, bool SPL>
static int xg_bn_any(const XGemm& x, cudaStream_t st) {
  // for accuracy: the sum over the chunks takes registers that 256 columns do not leave (20,000 rows to 1024 columns, bf16
  // 16,384 wide 746 us, 16,448 wide 916)
  if constexpr (sizeof(T) == 2 && MODE != XG_WGRAD && !DOT)
    if (x.K > xg_acc_long(x.dtype) * XG_BK) return xg_go<MODE, T, 128, 1, DOT, SPL, true>(x, st);
  if constexpr (sizeof(T) == 2)
    if (xg_bn_max(x.N, x.dtype) == 256)
      return xg_pairs(x) ? xg_go<MODE, T, 256, 2, DOT, SPL, false>(x, st) : xg_go<MODE, T, 256, 1, DOT, SPL, false>(x, st);
  return xg_go<MODE, T, 128, 1, DOT, SPL, false>(x, st);
}

template <int MODE, typename T>
static int xg_form(const XGemm& x, cudaStream_t st) {
  if constexpr (MODE == XG_DGRAD)
    if (x.dgpart) return xg_bn_any<MODE, T, true, false>(x, st);
  if constexpr (MODE == XG_WGRAD && sizeof(T) == 2)
    if (x.split) return xg_bn_any<MODE, T, false, true>(x, st);
  return xg_bn_any<MODE, T, false, false>(x, st);
}

template <int MODE>
static int xg_type(const XGemm& x, cudaStream_t st) {
  if (x.dtype == MB_F32) return xg_form<MODE, float>(x, st);
  return x.dtype == MB_BF16 ? xg_form<MODE, bf16>(x, st) : xg_form<MODE, f16>(x, st);
}

int xgemm_launch(const XGemm& x, cudaStream_t st) {
  if (x.mode == XG_FWD) return xg_type<XG_FWD>(x, st);
  return x.mode == XG_DGRAD ? xg_type<XG_DGRAD>(x, st) : xg_type<XG_WGRAD>(x, st);
}

}  // namespace mb

extern "C" int mace_b200_expert_test_hooks(uint64_t wait_ns, int32_t skip_one_load) {
  using namespace mb;
  if (wait_ns == 0) {
    set_error("expert_test_hooks: wait_ns must be positive");
    return MB_E_ARG;
  }
  const unsigned long long w = wait_ns;
  const int k = skip_one_load ? 1 : 0;
  if (cudaMemcpyToSymbol(g_xg_wait_ns, &w, sizeof(w)) != cudaSuccess ||
      cudaMemcpyToSymbol(g_xg_skip_load, &k, sizeof(k)) != cudaSuccess) {
    set_error("expert_test_hooks: cudaMemcpyToSymbol failed");
    return MB_E_CUDA;
  }
  return 0;
}

namespace mb {

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
