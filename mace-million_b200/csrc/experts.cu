// Products with per-token experts: slot s = (t, j) of a token's k choices goes through the matrix W[experts[s]].
//   z_s = W_e x_t (or x_s),   out_t = sum_j g_tj z_tj  (or out_s = z_s without weights)
//   dx_t = sum_j g_tj W_e^T dy_t,  dW_e = sum over e's slots of g_s dy_t x_t^T,  dg_s = <dy_t, W_e x_t> = <x_t, W_e^T dy_t>
// This file holds the plan (slots sorted by expert), the few-slots form, and the kernels that move rows: scatter into
// expert order, sum of a token's rows.  The products themselves are in experts_gemm.cu.
//
// fp32 operands become three bf16 planes, x = h + m + l with h = bf16(x), m = bf16(x - h), l = bf16(x - h - m): the 24 bits
// of the mantissa for values above 2^-109 (the planes end at 2^-133, so smaller ones lose low bits).  The planes of a finite
// value are finite; an infinite one has a NaN among them.
#include "experts.cuh"
#include "tc.cuh"

namespace mb {

// ------------------------------------------------------------------------------------------------ plan
// Stable counting sort of the slots by expert.  Every warp counts its run of slots per expert, prefix sums over the warps
// (and blocks) and over the experts' padded segments give each (warp, expert) its first row, and the warp places its slots
// in order (ranks inside a warp by ballots): the rows of an expert keep the slots' order, and no result depends on a
// schedule.  Slots with expert -1 get no row; other values outside [0, E) set MB_ST_BAD_EXPERT and get none either.
// Up to XP_CLUSTER_SLOTS it is one launch: a cluster of 8 CTAs that exchange their counts through distributed shared
// memory, one CTA up to 4096 slots; above, three launches over all SMs.  Latency bounds both (B200, one launch / three):
// 200 slots, 8 experts 5.5 / 7.6 us; 16,384, 89 experts 11.6 / 13.2; 65,536, 16 experts 9.5 / 9.3; 131,072, 16 experts
// 14.6 / 10.2; 262,144, 64 experts 29 / 15.

__device__ __forceinline__ int xp_expert(const int32_t* experts, int64_t s, int64_t end, int E, bool& bad) {
  if (s >= end) return -1;
  const int e = experts[s];
  bad |= e < -1 || e >= E;
  return e >= 0 && e < E ? e : -1;
}

// inclusive sum over the warp's lanes
__device__ __forceinline__ int warp_prefix(int v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int q = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += q;
  }
  return v;
}

// seg[e] = first row of expert e, pair[e] = its first pair of tiles, for e <= E, by one warp
__device__ __forceinline__ void xp_segments(int E, const int* cnt, int* seg, int* pair) {
  const int lane = threadIdx.x & 31;
  int run = 0, prun = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int e = e0 + lane;
    const int tiles = e < E ? (cnt[e] + XP_BM - 1) / XP_BM : 0, pairs = (tiles + 1) / 2;
    const int inc = warp_prefix(tiles), pinc = warp_prefix(pairs);
    if (e < E) {
      seg[e] = (run + inc - tiles) * XP_BM;
      pair[e] = prun + pinc - pairs;
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
    prun += __shfl_sync(0xffffffffu, pinc, 31);
  }
  if (lane == 0) {
    seg[E] = run * XP_BM;
    pair[E] = prun;
  }
}

// The plan's tables, by block `b` of `nb` (whole blocks; the experts e = b, b + nb, .. warp by warp)
__device__ __forceinline__ void xp_tables(const XPlan& p, int32_t* plan, const int* cnt, const int* seg, const int* pair,
                                          int b, int nb) {
  const int lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  if (b == 0 && threadIdx.x == 0) {
    plan[0] = seg[p.E] / XP_BM;
    plan[2] = pair[p.E];
    plan[p.o_seg + p.E] = seg[p.E];
  }
  for (int e = b + nb * (threadIdx.x >> 5); e < p.E; e += nb * nw) {
    const int c = cnt[e], r0 = seg[e], r1 = seg[e + 1];
    int rank = 0;                                // experts with more slots, or as many and a lower index
    for (int i = lane; i < p.E; i += 32) rank += cnt[i] > c || (cnt[i] == c && i < e);
    rank = __reduce_add_sync(0xffffffffu, rank);
    if (lane == 0) {
      plan[p.o_seg + e] = r0;
      plan[p.o_cnt + e] = c;
      plan[p.o_order + rank] = e;
    }
    for (int t = r0 / XP_BM + lane; t < r1 / XP_BM; t += 32) plan[p.o_tile + t] = e;
    for (int i = lane; i < pair[e + 1] - pair[e]; i += 32) plan[p.o_pair + pair[e] + i] = r0 / XP_BM + 2 * i;
    for (int r = r0 + c + lane; r < r1; r += 32) plan[p.o_row + r] = -1;
  }
}

// Lanes of the warp with the same expert, by one ballot per bit of the index (-1 counts as E); match_any takes a step per
// distinct value and made the plan of 262,144 slots on 64 experts three times as long
__device__ __forceinline__ unsigned same_expert(int e, int E) {
  const int v = e < 0 ? E : e;
  unsigned m = 0xffffffffu;
  for (int b = 1; b <= E; b <<= 1) {
    const unsigned on = __ballot_sync(0xffffffffu, v & b);
    m &= v & b ? on : ~on;
  }
  return m;
}

// Counts of the slots [s0, end) per expert into mine[E] (zeroed), by one warp; eight loads in flight
__device__ __forceinline__ void xp_count(const int32_t* experts, int64_t s0, int64_t end, int E, int* mine) {
  const int lane = threadIdx.x & 31;
  bool bad = false;
  for (; s0 < end; s0 += 256) {
    int ev[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) ev[q] = xp_expert(experts, s0 + 32 * q + lane, end, E, bad);
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (ev[q] >= 0) atomicAdd(&mine[ev[q]], 1);
  }
}

// Places the slots [s0, end); next[e] = next row of expert e for this warp, advanced here
__device__ __forceinline__ void xp_place(const int32_t* experts, const XPlan& p, int32_t* plan, int64_t s0, int64_t end,
                                         int* next) {
  const int lane = threadIdx.x & 31;
  bool bad = false;
  for (; s0 < end; s0 += 256) {
    int ev[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) ev[q] = xp_expert(experts, s0 + 32 * q + lane, end, p.E, bad);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int64_t s = s0 + 32 * q + lane;
      const int e = ev[q];
      const unsigned same = same_expert(e, p.E);
      const int first = __ffs(same) - 1;
      int at = 0;
      if (e >= 0 && lane == first) {
        at = next[e];
        next[e] = at + __popc(same);
      }
      at = __shfl_sync(0xffffffffu, at, first) + __popc(same & ((1u << lane) - 1));
      if (e >= 0) plan[p.o_row + at] = (int)s;
      if (s < end) plan[p.o_slot + s] = e >= 0 ? at : -1;
      __syncwarp();
    }
  }
  if (bad) atomicOr((unsigned*)plan + 1, (unsigned)MB_ST_BAD_EXPERT);
}

// One launch: CL CTAs of 32 warps (a cluster when CL > 1), each warp `per` slots.
// Shared memory: total[E], seg[E + 1], pair[E + 1], own[E], next[32][E].
constexpr int64_t XP_CLUSTER_SLOTS = 1 << 16;
template <int CL>
__global__ void __launch_bounds__(1024) k_plan_one(const int32_t* experts, const XPlan p, int32_t* plan, int64_t per) {
  extern __shared__ int sm[];
  const int E = p.E, tid = threadIdx.x, warp = tid >> 5;
  int *total = sm, *seg = total + E, *pair = seg + E + 1, *own = pair + E + 1, *next = own + E;
  const int rank = CL > 1 ? (int)cluster_ctarank() : 0;
  for (int i = tid; i < 32 * E; i += 1024) next[i] = 0;
  if (rank == 0 && tid == 0) plan[1] = 0;        // status: set below, after the first barrier
  __syncthreads();
  const int64_t s0 = ((int64_t)rank * 32 + warp) * per;
  const int64_t end = s0 + per < p.R ? s0 + per : p.R;
  xp_count(experts, s0, end, E, next + warp * E);
  __syncthreads();
  for (int e = tid; e < E; e += 1024) {          // first slot of each warp within the CTA's run of the expert
    int run = 0;
#pragma unroll 8
    for (int w = 0; w < 32; ++w) {
      const int c = next[w * E + e];
      next[w * E + e] = run;
      run += c;
    }
    own[e] = run;
  }
  if constexpr (CL > 1)
    cluster_sync();
  else
    __syncthreads();
  for (int e = tid; e < E; e += 1024) {
    int all = 0, before = 0;
    if constexpr (CL > 1) {
#pragma unroll
      for (int q = 0; q < CL; ++q) {
        const int c = ld_cluster_s32(mapa_u32(smem_u32(own + e), q));
        before += q < rank ? c : 0;
        all += c;
      }
    } else {
      all = own[e];
    }
    total[e] = all;
    pair[e] = before;                            // until the segments are known
  }
  __syncthreads();
  for (int i = tid; i < 32 * E; i += 1024) next[i] += pair[i % E];
  __syncthreads();
  if (warp == 0) xp_segments(E, total, seg, pair);
  __syncthreads();
  for (int i = tid; i < 32 * E; i += 1024) next[i] += seg[i % E];
  __syncthreads();
  xp_place(experts, p, plan, s0, end, next + warp * E);
  xp_tables(p, plan, total, seg, pair, rank, CL);
  if constexpr (CL > 1) cluster_sync();          // no CTA leaves while another can still read its counts
}

// Three launches, for more slots: XP_CHUNK slots per block, hist[e][block] in the plan
__global__ void __launch_bounds__(256) k_plan_count(const int32_t* experts, const XPlan p, int32_t* plan) {
  extern __shared__ int next[];                  // [8][E]
  for (int i = threadIdx.x; i < 8 * p.E; i += 256) next[i] = 0;
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  const int64_t s0 = (int64_t)blockIdx.x * XP_CHUNK + warp * (XP_CHUNK / 8);
  const int64_t end = s0 + XP_CHUNK / 8 < p.R ? s0 + XP_CHUNK / 8 : p.R;
  xp_count(experts, s0, end, p.E, next + warp * p.E);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += 256) {
    int run = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) run += next[w * p.E + e];
    plan[p.o_hist + (int64_t)e * p.nblk + blockIdx.x] = run;
  }
}

__global__ void __launch_bounds__(1024) k_plan_scan(const XPlan p, int32_t* plan) {
  extern __shared__ int sm[];
  int *cnt = sm, *seg = cnt + p.E, *pair = seg + p.E + 1;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) plan[1] = 0;
  for (int e = threadIdx.x >> 5; e < p.E; e += 32) {
    int32_t* h = plan + p.o_hist + (int64_t)e * p.nblk;
    int run = 0;
    for (int b0 = 0; b0 < p.nblk; b0 += 32) {
      const int v = b0 + lane < p.nblk ? h[b0 + lane] : 0, inc = warp_prefix(v);
      if (b0 + lane < p.nblk) h[b0 + lane] = run + inc - v;
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) cnt[e] = run;
  }
  __syncthreads();
  if (threadIdx.x < 32) xp_segments(p.E, cnt, seg, pair);
  __syncthreads();
  xp_tables(p, plan, cnt, seg, pair, 0, 1);
}

__global__ void __launch_bounds__(256) k_plan_place(const int32_t* experts, const XPlan p, int32_t* plan) {
  extern __shared__ int next[];                  // [8][E]
  for (int i = threadIdx.x; i < 8 * p.E; i += 256) next[i] = 0;
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  const int64_t s0 = (int64_t)blockIdx.x * XP_CHUNK + warp * (XP_CHUNK / 8);
  const int64_t end = s0 + XP_CHUNK / 8 < p.R ? s0 + XP_CHUNK / 8 : p.R;
  xp_count(experts, s0, end, p.E, next + warp * p.E);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += 256) {
    int run = plan[p.o_seg + e] + plan[p.o_hist + (int64_t)e * p.nblk + blockIdx.x];
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const int c = next[w * p.E + e];
      next[w * p.E + e] = run;
      run += c;
    }
  }
  __syncthreads();
  xp_place(experts, p, plan, s0, end, next + warp * p.E);
}

template <int CL>
static int plan_one(const int32_t* experts, const XPlan& p, int32_t* plan, cudaStream_t st) {
  static int ready_dev = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("expert_plan (device)");
  if (ready_dev != dev) {
    const int most = (4 * MB_PLAN_MAX_EXPERTS + 2 + 32 * MB_PLAN_MAX_EXPERTS) * 4;
    if (cudaFuncSetAttribute(k_plan_one<CL>, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess) {
      set_error("expert_plan: cannot reserve %d bytes of shared memory", most);
      return MB_E_CUDA;
    }
    ready_dev = dev;
  }
  const int64_t per = (p.R + 32 * CL * 32 - 1) / (32 * CL * 32) * 32;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(CL);
  cfg.blockDim = dim3(1024);
  cfg.dynamicSmemBytes = (4 * p.E + 2 + 32 * p.E) * 4;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CL;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CL > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, k_plan_one<CL>, experts, p, plan, per);
  return check_launch("expert_plan");
}

// ------------------------------------------------------------------------------------------------ row movement
// bytes [at, at + 16) of eight words, at = 0 .. 16 and even
__device__ __forceinline__ uint4 take16(uint32_t (&w)[8], unsigned at) {
  if (at & 16) return make_uint4(w[4], w[5], w[6], w[7]);
  if (at & 8)
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  if (at & 4)
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  const unsigned sh = (at & 2) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], sh), __funnelshift_r(w[1], w[2], sh), __funnelshift_r(w[2], w[3], sh),
                    __funnelshift_r(w[3], w[4], sh));
}

// 16 bytes at any even address: two aligned vectors and a shift.  [lo, hi): the bytes that may be read; where an aligned
// vector would leave them the bytes come one element at a time.
__device__ __forceinline__ uint4 load16_any(const uint16_t* p, const char* lo, const char* hi) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  const unsigned s = (unsigned)(a & 15);
  const char* base = reinterpret_cast<const char*>(a - s);
  if (s == 0) return *reinterpret_cast<const uint4*>(p);
  if (base < lo || base + 32 > hi) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  const uint4 u = reinterpret_cast<const uint4*>(base)[0], v = reinterpret_cast<const uint4*>(base)[1];
  uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
  return take16(w, s);
}

// 8 columns [c, c + 8) of a row of d elements as floats (0 beyond d); vec: 16-byte loads are aligned
__device__ __forceinline__ void load8(const float* row, int c, int d, bool vec, const char*, const char*, float (&f)[8]) {
  if (vec && c + 8 <= d) {
    load_p<float, 8>(row + c, f);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = c + q < d ? row[c + q] : 0.f;
  }
}
// the same of 16-bit elements, as they are
template <typename T>
__device__ __forceinline__ uint4 load8_raw(const T* row, int c, int d, bool vec, const char* lo, const char* hi) {
  if (c + 8 <= d)
    return vec ? *reinterpret_cast<const uint4*>(row + c)
               : load16_any(reinterpret_cast<const uint16_t*>(row + c), lo, hi);
  const uint16_t* r = reinterpret_cast<const uint16_t*>(row);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = (c + 2 * i < d ? (uint32_t)r[c + 2 * i] : 0u) | ((c + 2 * i + 1 < d ? (uint32_t)r[c + 2 * i + 1] : 0u) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Writes 8 columns as one vector of each of NP bf16 planes.  The first plane of a finite value is finite: above the largest
// bf16 (3.3895e38) rounding to nearest would give infinity, so it is that one, and the next plane has the rest.
// CUT: the first of two planes is cut off instead of rounded, and the second is never zero beside it (2^-24 of it where
// nothing is left): both have the sign of the value, so an infinite bf16 dy times both is that infinity.  (fp16 dy has planes
// of its own, the first one finite; rounded planes of either sign lose less in long accumulators.)
constexpr float BF16_MAX = 3.38953138925153547590470800371487867e+38f;   // (2 - 2^-7) 2^127
template <int NP, bool CUT>
__device__ __forceinline__ void store_planes(uint16_t* dst, int64_t plane, int64_t at, const float (&f)[8]) {
  float r[8], h[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) r[q] = f[q];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if (p == 0) {
        h[q] = fminf(fmaxf(r[q], -BF16_MAX), BF16_MAX);
        if (CUT) h[q] = __uint_as_float(__float_as_uint(h[q]) & 0xFFFF0000u);
      } else {
        h[q] = CUT && r[q] == 0.f ? h[q] * 0x1p-24f : r[q];
      }
    }
    const uint4 u = pack16<bf16>(h);
    *reinterpret_cast<uint4*>(dst + p * plane + at) = u;
    if (p + 1 == NP) break;
    unpack16(u, h, bf16());
#pragma unroll
    for (int q = 0; q < 8; ++q) r[q] -= h[q];
  }
}

// One job of k_rows_move; a launch runs up to XMOVES side by side, each on its own blocks (few launches: every one costs a
// small call more than its work).
struct XMove {
  int kind;                                      // MOVE_*
  int planes;                                    // fp32 data: 3 bf16 planes; 16-bit data: 1, the elements as they are, or 2 bf16 planes
  int d, dp, kdiv, vec;
  unsigned block0, blocks;                       // first block and number of blocks
  int64_t rows, lds, plane;
  const void* src;
  const char *lo, *hi;                           // the source's first and last byte + 1
  const float* scale;                            // not with one plane
  void* out;
};
enum {
  // out[row of slot] = scale[slot] src[slot / kdiv], in planes, for the slots with an expert: each source row is read once
  // and written to its kdiv rows (in expert order the rows of a token are far apart, and a gather would read it kdiv times)
  MOVE_SCATTER = 0,
  MOVE_STAGE = 1,                                // out[row] = src[row] in planes
  MOVE_PAD = 2,                                  // out[row] = 0 in planes for the rows that pad the experts' segments
  MOVE_ZERO = 3,                                 // out[slot] = 0 for slots without an expert (elements of T)
};                                               // columns between d and dp are written as zeros
constexpr int XMOVES = 7;                        // backward: dy (fp16 with weights: twice), x, their padding, W, rows without an expert
struct XMoves {
  XMove m[XMOVES];
  int n;
  __host__ void add(const XMove& j) {
    if (n < XMOVES) m[n] = j;
    ++n;                                         // x_moves refuses more than XMOVES
  }
};

// Narrow rows share a warp (lpr lanes a row, a power of two); wide ones take several passes, four vectors in flight.
template <typename T>
__global__ void __launch_bounds__(256, 4) k_rows_move(const XMoves mv, const int32_t* plan, const XPlan p) {
  int q = 0;
  while (q + 1 < mv.n && blockIdx.x >= mv.m[q + 1].block0) ++q;
  const XMove& m = mv.m[q];
  const int lane = threadIdx.x & 31, nv = m.dp / 8;
  const int64_t warp0 = (int64_t)(blockIdx.x - m.block0) * 8 + (threadIdx.x >> 5), warps = (int64_t)m.blocks * 8;
  if (m.kind == MOVE_ZERO) {                     // 32 slots a warp; the whole warp zeros a row
    for (int64_t r0 = warp0 * 32; r0 < m.rows; r0 += warps * 32) {
      unsigned todo = __ballot_sync(0xffffffffu, r0 + lane < m.rows && plan[p.o_slot + r0 + lane] < 0);
      for (; todo; todo &= todo - 1) {
        T* o = (T*)m.out + (r0 + __ffs(todo) - 1) * m.d;
        for (int c = lane; c < m.d; c += 32) o[c] = from_f<T>(0.f);
      }
    }
    return;
  }
  uint16_t* out = (uint16_t*)m.out;
  if (m.kind == MOVE_PAD) {                      // candidate i: row i % 128 of the last tile of expert i / 128
    for (int64_t i = warp0; i < m.rows; i += warps) {
      const int e = (int)(i / XP_BM), c = plan[p.o_cnt + e] % XP_BM, r = (int)(i % XP_BM);
      if (c == 0 || r < c) continue;
      const int64_t row = plan[p.o_seg + e + 1] - XP_BM + r;
      for (int pl = 0; pl < m.planes; ++pl)
        for (int v = lane; v < nv; v += 32)
          *reinterpret_cast<uint4*>(out + pl * m.plane + row * m.dp + 8 * v) = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  int lpr = 1;
  while (lpr < 32 && lpr < nv) lpr *= 2;
  const int rpw = 32 / lpr, sub = lane & (lpr - 1);
  const bool scatter = m.kind == MOVE_SCATTER;
  const int32_t* slot_row = plan + p.o_slot;
  const int copies = scatter ? m.kdiv : 1;
  for (int64_t row = warp0 * rpw + lane / lpr; row < m.rows; row += warps * rpw) {
    const T* s = (const T*)m.src + row * m.lds;
    if constexpr (sizeof(T) == 2) {
      const bool whole = m.vec && m.d == m.dp;   // every piece is an aligned vector
      for (int c0 = sub * 8; c0 < m.dp; c0 += 32 * lpr) {
        uint4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = c0 + i * 8 * lpr;
          if (c < m.dp) u[i] = whole ? *reinterpret_cast<const uint4*>(s + c) : load8_raw<T>(s, c, m.d, m.vec != 0, m.lo, m.hi);
        }
        for (int j = 0; j < copies; ++j) {
          const int64_t to = scatter ? slot_row[row * copies + j] : row;
          if (to < 0) continue;
          uint16_t* o = out + to * m.dp + c0;
          if (m.planes == 2) {                     // x with its weight; dy (fp16), exact in two rounded planes
            const float g = m.scale ? m.scale[row * copies + j] : 1.f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (c0 + i * 8 * lpr < m.dp) {
                float f[8];
                unpack16(u[i], f, T());
#pragma unroll
                for (int x = 0; x < 8; ++x) f[x] *= g;
                store_planes<2, std::is_same<T, bf16>::value>(o, m.plane, i * 8 * lpr, f);
              }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (c0 + i * 8 * lpr < m.dp) *reinterpret_cast<uint4*>(o + i * 8 * lpr) = u[i];
          }
        }
      }
    } else {
      for (int c = sub * 8; c < m.dp; c += 8 * lpr) {
        float f[8];
        load8(s, c, m.d, m.vec != 0, m.lo, m.hi, f);
        for (int j = 0; j < copies; ++j) {
          const int64_t to = scatter ? slot_row[row * copies + j] : row;
          if (to < 0) continue;
          float v[8];
          const float g = m.scale ? m.scale[row * copies + j] : 1.f;
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = f[x] * g;
          store_planes<3, false>(out, m.plane, to * m.dp + c, v);
        }
      }
    }
  }
}

// V fp32 values as loaded
template <int V>
struct RawF {
  uint4 u[V / 4];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) u[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void add_to(float (&s)[V]) const {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      s[4 * i] += __uint_as_float(u[i].x), s[4 * i + 1] += __uint_as_float(u[i].y);
      s[4 * i + 2] += __uint_as_float(u[i].z), s[4 * i + 3] += __uint_as_float(u[i].w);
    }
  }
};

// Blocks [0, sum_blocks): out[t] = sum over the token's k slots (in their order) of buf[slot], skipping slots without an
// expert; a thread adds one vector of a token's rows, four loads in flight; ldb is padded to whole vectors.  The rows are
// fp32 whatever the type of out: one rounding of the sum, and a row need not fit fp16 where the sum does (65,536 x 4 rows of
// 2,048 361 us, 6.7 TB/s).
// The other blocks: dg[slot] = sum of its nparts partial products (0 without an expert).
template <typename T, int V>
__global__ void __launch_bounds__(256) k_rows_sum(const float* buf, int64_t ldb, T* out, int64_t tokens, int k, int d,
                                                  const int32_t* slot_row, unsigned sum_blocks, const float* dgpart,
                                                  int nparts, float* dg) {
  if (blockIdx.x >= sum_blocks) {
    const int64_t R = tokens * k, step = (int64_t)(gridDim.x - sum_blocks) * 256;
    for (int64_t s = (int64_t)(blockIdx.x - sum_blocks) * 256 + threadIdx.x; s < R; s += step) {
      float v = 0.f;
      if (slot_row[s] >= 0)
        for (int q = 0; q < nparts; ++q) v += dgpart[q * R + s];
      dg[s] = v;
    }
    return;
  }
  if constexpr (V == 1) {                        // odd widths: a warp per token, aligned loads, stores shifted into place
    constexpr int VV = kVec<T>;
    const int lane = threadIdx.x & 31;
    for (int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); t < tokens; t += (int64_t)sum_blocks * 8) {
      T* o = out + t * d;
      const int sh = (int)(reinterpret_cast<uintptr_t>(o) & 15);
      const float* p = buf + t * k * ldb;
      const int32_t* row = slot_row + t * k;
      uint32_t c[4] = {0u, 0u, 0u, 0u};            // the last lane's vector of the pass before
      for (int n0 = 0; n0 * VV - sh / (int)sizeof(T) < d; n0 += 32) {
        const int n = n0 + lane;
        float s[VV];
#pragma unroll
        for (int q = 0; q < VV; ++q) s[q] = 0.f;
        if (n * VV < d)
          for (int j0 = 0; j0 < k; j0 += 4) {
            RawF<VV> r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              r[j].zero();
              if (j0 + j < k && row[j0 + j] >= 0) r[j].load(p + (j0 + j) * ldb + n * VV);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j].add_to(s);
          }
        const uint4 u = pack16<T>(s);
        // bytes [16 - sh, 32 - sh) of the neighbour's vector and this one go to the aligned address 16 n - sh
        uint32_t w[8] = {c[0], c[1], c[2], c[3], u.x, u.y, u.z, u.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t up = __shfl_up_sync(0xffffffffu, w[4 + q], 1);
          if (lane > 0) w[q] = up;
          c[q] = __shfl_sync(0xffffffffu, w[4 + q], 31);
        }
        const uint4 v = take16(w, 16 - sh);
        const int e0 = n * VV - sh / (int)sizeof(T);   // first element of the store
        if (e0 >= 0 && e0 + VV <= d) {
          *reinterpret_cast<uint4*>(o + e0) = v;
        } else {
          const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int q = 0; q < VV; ++q) {
            if (e0 + q < 0 || e0 + q >= d) continue;
            if constexpr (sizeof(T) == 4) {
              o[e0 + q] = __uint_as_float(vw[q]);
            } else {
              const uint16_t h = (uint16_t)(vw[q / 2] >> (16 * (q & 1)));
              reinterpret_cast<uint16_t*>(o)[e0 + q] = h;
            }
          }
        }
      }
    }
  } else {
    const unsigned nv = d / V;
    const int64_t total = tokens * nv, step = (int64_t)sum_blocks * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
      const int64_t t = total >> 32 ? i / nv : (unsigned)i / nv;
      const int c = (int)(i - t * nv) * V;
      float s[V];
#pragma unroll
      for (int q = 0; q < V; ++q) s[q] = 0.f;
      const float* p = buf + t * k * ldb + c;
      const int32_t* row = slot_row + t * k;
      for (int j0 = 0; j0 < k; j0 += 4) {
        RawF<V> r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          r[j].zero();
          if (j0 + j < k && row[j0 + j] >= 0) r[j].load(p + (j0 + j) * ldb);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j].add_to(s);
      }
      store_v<T, V>(out + t * d + c, s);
    }
  }
}

// ------------------------------------------------------------------------------------------------ few slots
// out[t][o] = sum_j g_tj <W[e_tj][o], x> without a plan: L lanes per (token, output), the rows of W of four choices side
// by side in flight.  Bound by the bytes of W (4 of 64 experts, 1024 x 1024 bf16: one token 5.8 us, 16 tokens 134 MB in
// 25 us, 5.3 TB/s); a row of W that several tokens use comes from L2 after the first.
// SLOTS: out[slot][o] = <W[e][o], x>, L lanes per (slot, output).
template <typename T, int V, int L, bool SLOTS>
__global__ void __launch_bounds__(128) k_expert_few(const T* x, int64_t ldx, int kx, const T* w, const int32_t* experts,
                                                    const float* g, T* out, int k, int E, int d, int o_n) {
  const int lane = threadIdx.x & 31, sub = lane & (L - 1);
  const int o = (blockIdx.x * 4 + (threadIdx.x >> 5)) * (32 / L) + lane / L;
  const bool live = o < o_n;
  const int64_t t = blockIdx.y;
  const int n = SLOTS ? 1 : k;
  constexpr int J = SLOTS ? 1 : 4;
  float total = 0.f;
  for (int j0 = 0; j0 < n; j0 += J) {
    const T *wr[J], *xr[J];
    float acc[J];
#pragma unroll
    for (int q = 0; q < J; ++q) {
      const int64_t s = SLOTS ? t : t * k + j0 + q;
      const int e = j0 + q < n ? experts[s] : -1;
      wr[q] = live && e >= 0 && e < E ? w + ((int64_t)e * o_n + o) * d : nullptr;
      xr[q] = x + s / kx * ldx;
      acc[q] = 0.f;
    }
#pragma unroll 4
    for (int c = sub * V; c < d; c += L * V) {
      float b[V];
#pragma unroll
      for (int q = 0; q < J; ++q) {
        if (!wr[q]) continue;
        float a[V];
        load_v<T, V>(wr[q] + c, a);
        load_v<T, V>(xr[q] + c, b);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[q] = fmaf(a[i], b[i], acc[q]);
      }
    }
#pragma unroll
    for (int q = 0; q < J; ++q) {
#pragma unroll
      for (int h = L / 2; h > 0; h >>= 1) acc[q] += __shfl_xor_sync(0xffffffffu, acc[q], h);
      if (wr[q]) total += SLOTS ? acc[q] : g[t * k + j0 + q] * acc[q];
    }
  }
  if (sub == 0 && live) out[t * o_n + o] = from_f<T>(total);
}

// ------------------------------------------------------------------------------------------------ host side
static inline int pad8(int d) { return (d + 7) / 8 * 8; }

struct XShape {
  int64_t T, R;
  int32_t k, E, D, O, dtype, np, Dp, Op;
  XPlan lay;
  int64_t rows;
};

static int x_shape(const char* who, XShape& s, int64_t T, int32_t k, int32_t E, int32_t D, int32_t O, int32_t dtype) {
  if (T < 0 || k < 1 || E < 1 || E > MB_PLAN_MAX_EXPERTS || D < 1 || O < 1 || D > (1 << 24) || O > (1 << 24) ||
      T > (int64_t)(1 << 29) / k) {
    set_error("%s: bad sizes (tokens %lld, k %d, experts %d (at most %d), widths %d -> %d, at most 2^29 slots)", who,
              (long long)T, k, E, MB_PLAN_MAX_EXPERTS, D, O);
    return MB_E_ARG;
  }
  if (!dtype_ok(dtype)) {
    set_error("%s: unsupported type %d", who, dtype);
    return MB_E_ARG;
  }
  if (sm_count() < 1) {
    set_error("%s: no CUDA device", who);
    return MB_E_CUDA;
  }
  s.T = T; s.k = k; s.R = T * k; s.E = E; s.D = D; s.O = O; s.dtype = dtype;
  s.np = dtype == MB_F32 ? 3 : 1;
  s.Dp = pad8(D);
  s.Op = pad8(O);
  s.lay = xplan(s.R, E);
  s.rows = s.lay.tiles * XP_BM;
  return 0;
}

struct XWork {                                   // workspace cursor: byte offsets, 256-byte aligned
  int64_t used = 0;
  int64_t take(int64_t bytes) {
    const int64_t at = used;
    used += (bytes + 255) / 256 * 256;
    return at;
  }
};

struct XFwd {
  int64_t xs = 0, ws = -1, y = -1, bytes = 0;
};
// the 16-bit matrices can be read as they are when their rows are whole 16-byte vectors
static bool w_direct(const XShape& s, const void* w) { return s.dtype != MB_F32 && s.D % 8 == 0 && aligned16(w); }

static XFwd x_fwd_layout(const XShape& s, bool combine, bool direct) {
  XWork c;
  XFwd f;
  f.xs = c.take((int64_t)s.np * s.rows * s.Dp * 2);
  if (!direct) f.ws = c.take((int64_t)s.np * s.E * s.O * s.Dp * 2);
  if (combine && s.k > 1) f.y = c.take(s.R * s.Op * 4);
  f.bytes = c.used;
  return f;
}

struct XBwd {
  int64_t xs = -1, dys = -1, dyw = -1, ws = -1, dxb = -1, dgp = -1, parts = -1, pre = -1, bytes = 0;
  int kc = 0;
  bool split = false;                            // dW's operands in bf16 planes: 16-bit data with weights
  int px = 1, pdy = 1;                           // planes of dW's operands
};
static XBwd x_bwd_layout(const XShape& s, bool combine, bool x_slots, bool direct, bool need_x, bool need_w,
                         bool need_g) {
  XWork c;
  XBwd b;
  b.split = combine && s.dtype != MB_F32;
  b.px = b.split ? 2 : s.np;
  b.pdy = b.split && s.dtype == MB_F16 ? 2 : s.np;
  if (need_w) b.xs = c.take(b.px * s.rows * 2 * s.Dp);
  // dx takes dy in its own type; dW reads the same rows unless it needs planes of them
  if (need_x || need_g || b.pdy == s.np) b.dys = c.take(s.np * s.rows * 2 * s.Op);
  if (need_w) b.dyw = b.pdy == s.np ? b.dys : c.take(b.pdy * s.rows * 2 * s.Op);
  if ((need_x || need_g) && !direct) b.ws = c.take((int64_t)s.np * s.E * s.O * s.Dp * 2);
  if (need_x && !x_slots && s.k > 1) b.dxb = c.take(s.R * s.Dp * 4);
  if (need_g) b.dgp = c.take(s.R * 4 * 2 * xgemm_n_tiles(s.D, s.dtype));
  if (need_w) {
    b.kc = xgemm_kc(s.E, s.O, s.D, s.R, s.dtype);
    const int64_t parts = xgemm_parts(s.E, s.R, b.kc);
    if (parts) {
      b.parts = c.take(parts * s.O * s.D * 4);
      b.pre = c.take((s.E + 1) * 4);
    }
  }
  b.bytes = c.used;
  return b;
}

static unsigned x_grid(int64_t units) {
  const int64_t most = (int64_t)16 * sm_count();
  return (unsigned)(units < 1 ? 1 : units < most ? units : most);
}

template <typename F>
static int x_types(int dtype, const F& f) {
  if (dtype == MB_F32) return f(float());
  return dtype == MB_BF16 ? f(bf16()) : f(f16());
}

static XMove move_rows(int kind, const XShape& s, const void* src, int64_t rows, int64_t lds, int d, int dp, int64_t plane,
                       void* out) {
  const int size = dtype_size(s.dtype);
  XMove m{};
  m.kind = kind;
  m.planes = s.np;
  m.d = d; m.dp = dp; m.kdiv = 1; m.vec = aligned16(src) && lds % 8 == 0;
  m.rows = rows; m.lds = lds; m.plane = plane;
  m.src = src; m.out = out;
  m.lo = (const char*)src;
  m.hi = m.lo + ((rows - 1) * lds + d) * size;
  return m;
}
static XMove move_scatter(const XShape& s, const void* src, int64_t lds, int d, int dp, int kdiv, int planes,
                          const float* scale, void* out) {
  XMove m = move_rows(MOVE_SCATTER, s, src, s.R / kdiv, lds, d, dp, s.rows * dp, out);
  m.planes = planes;
  m.kdiv = kdiv;
  m.scale = scale;
  return m;
}
static XMove move_stage(const XShape& s, const void* w, void* out) {
  const int64_t rows = (int64_t)s.E * s.O;
  return move_rows(MOVE_STAGE, s, w, rows, s.D, s.D, s.Dp, rows * s.Dp, out);
}
static XMove move_pad(const XShape& s, int dp, int planes, void* out) {
  XMove m = move_rows(MOVE_PAD, s, nullptr, (int64_t)s.E * XP_BM, 0, 0, dp, s.rows * dp, out);
  m.planes = planes;
  return m;
}
static XMove move_zero(const XShape& s, void* out, int d) {
  XMove m{};
  m.kind = MOVE_ZERO;
  m.d = d; m.dp = 8; m.kdiv = 1;                 // one lane reads a slot: almost all have an expert
  m.rows = s.R; m.out = out;
  return m;
}

// Blocks in proportion to the vectors that each job moves
template <typename T>
static int x_moves(const XShape& s, XMoves& mv, const int32_t* plan, cudaStream_t st) {
  if (mv.n > XMOVES) {
    set_error("expert_linear: %d row jobs in one launch", mv.n);
    return MB_E_ARG;
  }
  int64_t units[XMOVES], all = 0;
  for (int q = 0; q < mv.n; ++q) {
    const bool pad = mv.m[q].kind == MOVE_PAD;   // half of the candidates on average, written only
    units[q] = (mv.m[q].rows * mv.m[q].kdiv * (mv.m[q].dp / 8) / (pad ? 4 : 1) + 255) / 256;
    all += units[q];
  }
  const int64_t most = (int64_t)16 * sm_count();
  unsigned at = 0;
  for (int q = 0; q < mv.n; ++q) {
    const int64_t b = all <= most ? units[q] : units[q] * most / all;
    mv.m[q].block0 = at;
    mv.m[q].blocks = (unsigned)(b < 1 ? 1 : b);
    at += mv.m[q].blocks;
  }
  k_rows_move<T><<<at, 256, 0, st>>>(mv, plan, s.lay);
  return check_launch("expert_linear (rows)");
}

// sums of rows (buf not null) and of partial weight gradients (dg not null) in one launch
template <typename T>
static int x_rows_sum(const float* buf, int64_t ldb, T* out, int64_t tokens, int k, int d, const int32_t* slot_row,
                      const float* dgpart, int nparts, float* dg, cudaStream_t st) {
  constexpr int V = kVec<T>;
  const bool vec = d % V == 0 && aligned16(out);
  const unsigned nb = buf ? x_grid(vec ? (tokens * (d / V) + 255) / 256 : (tokens + 7) / 8) : 0;
  const unsigned ng = dg ? x_grid((tokens * k + 255) / 256) : 0;
  if (vec)
    k_rows_sum<T, V><<<nb + ng, 256, 0, st>>>(buf, ldb, out, tokens, k, d, slot_row, nb, dgpart, nparts, dg);
  else
    k_rows_sum<T, 1><<<nb + ng, 256, 0, st>>>(buf, ldb, out, tokens, k, d, slot_row, nb, dgpart, nparts, dg);
  return check_launch("expert_linear (sum)");
}

}  // namespace mb

using namespace mb;

extern "C" int mace_b200_expert_plan_words(int64_t slots, int32_t E, int64_t* words) {
  if (slots < 0 || slots > (int64_t)1 << 29 || E < 1 || E > MB_PLAN_MAX_EXPERTS || !words) {
    set_error("expert_plan: bad sizes (slots %lld, experts %d, at most %d)", (long long)slots, E, MB_PLAN_MAX_EXPERTS);
    return MB_E_ARG;
  }
  *words = xplan(slots, E).words;
  return 0;
}

extern "C" int mace_b200_expert_plan(const int32_t* experts, int64_t slots, int32_t E, int32_t* plan, void* stream) {
  int64_t words = 0;
  if (int rc = mace_b200_expert_plan_words(slots, E, &words)) return rc;
  if (!plan || (slots > 0 && !experts)) {
    set_error("expert_plan: null pointer");
    return MB_E_ARG;
  }
  const XPlan p = xplan(slots, E);
  cudaStream_t st = (cudaStream_t)stream;
  if (slots <= 4096) return plan_one<1>(experts, p, plan, st);
  if (slots <= XP_CLUSTER_SLOTS) return plan_one<8>(experts, p, plan, st);
  k_plan_count<<<p.nblk, 256, 8 * E * 4, st>>>(experts, p, plan);
  if (int rc = check_launch("expert_plan")) return rc;
  k_plan_scan<<<1, 1024, (3 * E + 2) * 4, st>>>(p, plan);
  if (int rc = check_launch("expert_plan")) return rc;
  k_plan_place<<<p.nblk, 256, 8 * E * 4, st>>>(experts, p, plan);
  return check_launch("expert_plan");
}

extern "C" uint64_t mace_b200_capture_id(void* stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo((cudaStream_t)stream, &status, &id) != cudaSuccess) {
    cudaGetLastError();                            // the legacy stream while another one captures: not in a capture itself
    return 0;
  }
  return status == cudaStreamCaptureStatusNone ? 0 : id;
}

extern "C" int mace_b200_expert_linear_workspace(int64_t tokens, int32_t k, int32_t E, int32_t D, int32_t O,
                                                 int32_t dtype, int32_t x_per_slot, int32_t weighted, int32_t backward,
                                                 int64_t* bytes) {
  XShape s;
  if (int rc = x_shape("expert_linear_workspace", s, tokens, k, E, D, O, dtype)) return rc;
  if (!bytes) {
    set_error("expert_linear_workspace: null pointer");
    return MB_E_ARG;
  }
  *bytes = backward ? x_bwd_layout(s, weighted != 0, x_per_slot != 0, false, true, true, weighted != 0).bytes
                    : x_fwd_layout(s, weighted != 0, false).bytes;
  return 0;
}

extern "C" int mace_b200_expert_linear_few(const void* x, int64_t ldx, int32_t x_per_slot, const void* w,
                                           const int32_t* experts, const float* weights, void* out, int64_t tokens,
                                           int32_t k, int32_t E, int32_t D, int32_t O, int32_t dtype, void* stream) {
  XShape s;
  if (int rc = x_shape("expert_linear_few", s, tokens, k, E, D, O, dtype)) return rc;
  if (s.R > MB_FEW_MAX_SLOTS) {
    set_error("expert_linear_few: %lld slots (at most %d)", (long long)s.R, MB_FEW_MAX_SLOTS);
    return MB_E_ARG;
  }
  if (s.R == 0) return 0;
  if (!x || !w || !experts || !out || ldx < D) {
    set_error("expert_linear_few: null pointer or row stride %lld below the width", (long long)ldx);
    return MB_E_ARG;
  }
  cudaStream_t st = (cudaStream_t)stream;
  return x_types(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = kVec<T>;
    const bool vec = D % V == 0 && ldx % V == 0 && aligned16(x) && aligned16(w);
    const int kx = x_per_slot ? 1 : k;
    const int L = (vec ? D / V : D) <= 64 ? 8 : 32;   // narrow rows: four outputs per warp
    const dim3 grid((O + 128 / L - 1) / (128 / L), (unsigned)(weights ? tokens : s.R));
    auto go = [&](auto kern) {
      kern<<<grid, 128, 0, st>>>((const T*)x, ldx, kx, (const T*)w, experts, weights, (T*)out, k, E, D, O);
      return check_launch("expert_linear_few");
    };
    auto form = [&](auto v, auto l) {
      constexpr int VV = decltype(v)::value, LL = decltype(l)::value;
      return weights ? go(k_expert_few<T, VV, LL, false>) : go(k_expert_few<T, VV, LL, true>);
    };
    using One = std::integral_constant<int, 1>;
    using Vec = std::integral_constant<int, V>;
    using Narrow = std::integral_constant<int, 8>;
    using Wide = std::integral_constant<int, 32>;
    if (vec) return L == 8 ? form(Vec(), Narrow()) : form(Vec(), Wide());
    return L == 8 ? form(One(), Narrow()) : form(One(), Wide());
  });
}

extern "C" int mace_b200_expert_linear_fwd(const void* x, int64_t ldx, int32_t x_per_slot, const void* w,
                                           const int32_t* plan, const float* weights, void* out, void* workspace,
                                           int64_t tokens, int32_t k, int32_t E, int32_t D, int32_t O, int32_t dtype,
                                           void* stream) {
  XShape s;
  if (int rc = x_shape("expert_linear_fwd", s, tokens, k, E, D, O, dtype)) return rc;
  if (s.R == 0) return 0;
  if (!x || !w || !plan || !out || !workspace || ldx < D) {
    set_error("expert_linear_fwd: null pointer or row stride %lld below the width", (long long)ldx);
    return MB_E_ARG;
  }
  cudaStream_t st = (cudaStream_t)stream;
  const bool combine = weights != nullptr, direct = w_direct(s, w);
  const XFwd f = x_fwd_layout(s, combine, direct);
  char* base = (char*)workspace;
  return x_types(dtype, [&](auto t) {
    using T = decltype(t);
    const bool sum = f.y >= 0;
    XMoves mv{};
    mv.add(move_scatter(s, x, ldx, D, s.Dp, x_per_slot ? 1 : k, s.np, nullptr, base + f.xs));
    if (!direct) mv.add(move_stage(s, w, base + f.ws));
    if (!sum) mv.add(move_zero(s, out, O));
    if (int rc = x_moves<T>(s, mv, plan, st)) return rc;
    XGemm g{};
    g.mode = XG_FWD; g.dtype = dtype;
    g.a = base + f.xs; g.rows = s.rows; g.lda = s.Dp;
    g.b = direct ? w : base + f.ws; g.ldb = s.Dp;
    g.E = E; g.M = 0; g.N = O; g.K = D;
    g.plan = plan; g.lay = s.lay; g.scale = weights;
    g.out = sum ? (void*)(base + f.y) : out;
    g.ldo = sum ? s.Op : O;
    g.out32 = sum;
    if (int rc = xgemm_launch(g, st)) return rc;
    if (!sum) return 0;
    return x_rows_sum<T>((const float*)(base + f.y), s.Op, (T*)out, tokens, k, O, plan + s.lay.o_slot, nullptr, 0, nullptr, st);
  });
}

extern "C" int mace_b200_expert_linear_bwd(const void* dy, const void* x, int64_t ldx, int32_t x_per_slot,
                                           const void* w, const int32_t* plan, const float* weights, void* dx, void* dw,
                                           float* dweights, void* workspace, int64_t tokens, int32_t k, int32_t E,
                                           int32_t D, int32_t O, int32_t dtype, void* stream) {
  XShape s;
  if (int rc = x_shape("expert_linear_bwd", s, tokens, k, E, D, O, dtype)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (s.R == 0) {
    if (dw && cudaMemsetAsync(dw, 0, (int64_t)E * O * D * dtype_size(dtype), st) != cudaSuccess)
      return check_launch("expert_linear_bwd");
    return 0;
  }
  if (!dy || !x || !w || !plan || !workspace || ldx < D || (dweights && !weights)) {
    set_error("expert_linear_bwd: null pointer or row stride %lld below the width", (long long)ldx);
    return MB_E_ARG;
  }
  const bool combine = weights != nullptr, direct = w_direct(s, w);
  const XBwd b = x_bwd_layout(s, combine, x_per_slot != 0, direct, dx != nullptr, dw != nullptr, dweights != nullptr);
  char* base = (char*)workspace;
  const int kx = x_per_slot ? 1 : k, ky = combine ? k : 1;
  return x_types(dtype, [&](auto t) {
    using T = decltype(t);
    const bool sum = b.dxb >= 0;
    XMoves mv{};
    if (b.dys >= 0) mv.add(move_scatter(s, dy, O, O, s.Op, ky, s.np, nullptr, base + b.dys));
    // the weights scale the rows of x, not those of dy: dy stays exact for dx and dweights, and x is read only here.
    // dW sums over whole segments: their padding rows are zeros in both operands (elsewhere a padding row is never stored).
    if (dw) {
      if (b.dyw != b.dys) mv.add(move_scatter(s, dy, O, O, s.Op, ky, b.pdy, nullptr, base + b.dyw));
      mv.add(move_scatter(s, x, ldx, D, s.Dp, kx, b.px, weights, base + b.xs));
      mv.add(move_pad(s, s.Op, b.pdy, base + b.dyw));
      mv.add(move_pad(s, s.Dp, b.px, base + b.xs));
    }
    if (b.ws >= 0) mv.add(move_stage(s, w, base + b.ws));
    if (dx && !sum) mv.add(move_zero(s, dx, D));
    if (int rc = x_moves<T>(s, mv, plan, st)) return rc;
    if (dw) {
      XGemm g{};
      g.mode = XG_WGRAD; g.dtype = dtype; g.split = b.split;
      g.a = base + b.dyw; g.lda = s.Op;
      g.b = base + b.xs; g.ldb = s.Dp;
      g.rows = s.rows;
      g.E = E; g.M = O; g.N = D; g.K = 0;
      g.plan = plan; g.lay = s.lay;
      g.out = dw; g.ldo = D; g.kc = b.kc;
      if (b.parts >= 0) {
        g.parts = (float*)(base + b.parts);
        g.pre = (int32_t*)(base + b.pre);
      }
      if (int rc = xgemm_launch(g, st)) return rc;
    }
    if (!dx && !dweights) return 0;
    XGemm g{};
    g.mode = XG_DGRAD; g.dtype = dtype;
    g.a = base + b.dys; g.rows = s.rows; g.lda = s.Op;
    g.b = direct ? w : base + b.ws; g.ldb = s.Dp;
    g.E = E; g.M = 0; g.N = D; g.K = O;
    g.plan = plan; g.lay = s.lay; g.scale = weights;
    g.out = sum ? (void*)(base + b.dxb) : dx;
    g.ldo = sum ? s.Dp : D;
    g.out32 = sum;
    if (dweights) {
      g.x = x; g.ldx = ldx; g.kdiv = kx;
      g.dgpart = (float*)(base + b.dgp);
    }
    if (int rc = xgemm_launch(g, st)) return rc;
    if (!sum && !dweights) return 0;
    return x_rows_sum<T>(sum ? (const float*)(base + b.dxb) : nullptr, s.Dp, (T*)dx, tokens, k, D, plan + s.lay.o_slot,
                         dweights ? (const float*)(base + b.dgp) : nullptr, 2 * xgemm_n_tiles(D, dtype), dweights, st);
  });
}
