// Linear maps in 8-bit integers, a scale for each token and each output channel:
//   s_t = max_k |x[t][k]| / 127,  q[t][k] = nearest(x[t][k] / s_t),  y[t][n] = (sum_k q[t][k] w[n][k]) s_t s_n + b_n
// The sums are exact in int32 (k <= MB_INT8_MAX_K), y is fp32 arithmetic on them, rounded once.  q is the nearest whole number
// of the exact quotient, ties to even (a remainder by fma corrects the rounded quotient), so it does not depend on who divides.
//
// Three kernels.  k_quant_rows: a warp per row.  k_int8_few: up to 8 tokens; a CTA quantizes them into shared memory while its
// first weights are on their way, then each warp takes whole rows of w with dp4a: bound by the weights' bytes and latency.
// k_int8_gemm: tcgen05 kind::i8 from TMA tiles (SWIZZLE_128B, 128 bytes of K a stage).  Output channels are the rows of an MMA
// and tokens its columns: few tokens take a narrow tile, a lane holds one channel (its scale and bias stay in registers), and
// a warp stores 32 neighbouring channels of a token at once, whatever the alignment of y.
// Persistent CTAs, one per SM: warp 0 loads, warp 1 issues, warps 4-11 drain one of two accumulators.  CG = 2: pairs of CTAs
// (cta_group::2) on 256 channels, each with its own 128 and half of the tokens' rows.  Every wait is bounded; a tile whose
// wait expired is NaN.
#include <cuda.h>

#include <type_traits>

#include "dtypes.cuh"
#include "tc.cuh"
#include "tensor_map.cuh"

namespace mb {

// Scale of a row, its reciprocal, and the power of two that keeps both normal (a tiny row's scale is subnormal)
struct Q8 {
  float s, inv, up;
};
__device__ __forceinline__ Q8 q8_of(float scale) {
  Q8 k;
  k.up = scale < 0x1p-100f ? 0x1p60f : 1.f;
  k.s = scale * k.up;
  k.inv = 1.f / k.s;
  return k;
}
// nearest(x / scale) of the exact quotient, in [-127, 127]; 0 where the scale is 0 or not finite
__device__ __forceinline__ int q8(float x, const Q8& k) {
  const float s = k.s;
  x *= k.up;
  float q = rintf(x * k.inv);
  q = fminf(fmaxf(q, -127.f), 127.f);             // NaN goes to -127 here, and below to 0
  const float r = fmaf(-q, s, x), h = 0.5f * s;   // exact: the quotient is off by less than one
  const bool odd = (int)q & 1;
  if (r > h || (r == h && odd)) q += 1.f;
  if (r < -h || (r == -h && odd)) q -= 1.f;
  q = fminf(fmaxf(q, -127.f), 127.f);
  return s > 0.f && s < INFINITY && x == x ? (int)q : 0;
}
__device__ __forceinline__ uint32_t q8x4(const float* f, const Q8& k) {
  return (uint32_t)(q8(f[0], k) & 255) | (uint32_t)(q8(f[1], k) & 255) << 8 |
         (uint32_t)(q8(f[2], k) & 255) << 16 | (uint32_t)q8(f[3], k) << 24;
}
// max |x| that NaN passes through
__device__ __forceinline__ float top_of(float m, float v) {
  v = fabsf(v);
  return m >= v || m != m ? m : v;
}
__device__ __forceinline__ float warp_top(float m) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = top_of(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
__device__ __forceinline__ float q8_scale(float top) { return __fdiv_rn(top, 127.f); }

// V elements an access: 16 bytes, or 1 element where rows are not aligned.  Bytes up to ldq that hold no value are zero.
template <typename T, int V>
__global__ void __launch_bounds__(256) k_quant_rows(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, int64_t ldq,
                                                    float* __restrict__ scale, int64_t rows, int32_t k) {
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * 8;
  for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < rows; row += step) {
    const T* p = x + row * ldx;
    float top = 0.f;
#pragma unroll 4
    for (int j = lane * V; j < k; j += 32 * V) {
      float f[V];
      load_v<T, V>(p + j, f);
#pragma unroll
      for (int i = 0; i < V; ++i) top = top_of(top, f[i]);
    }
    top = warp_top(top);
    const float s = q8_scale(top);
    const Q8 qk = q8_of(s);
    if (lane == 0) scale[row] = s;
    int8_t* o = q + row * ldq;
    if constexpr (V == 1) {
      for (int j = lane; j < ldq; j += 32) o[j] = j < k ? (int8_t)q8(to_f(p[j]), qk) : (int8_t)0;
    } else {
#pragma unroll 4
      for (int j = lane * V; j < ldq; j += 32 * V) {   // ldq is a multiple of 16, k of V
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = 0.f;
        if (j < k) load_v<T, V>(p + j, f);
        if constexpr (V == 8)
          *reinterpret_cast<uint2*>(o + j) = make_uint2(q8x4(f, qk), q8x4(f + 4, qk));
        else
          *reinterpret_cast<uint32_t*>(o + j) = q8x4(f, qk);
      }
    }
  }
}

struct I8Args {
  const void* x;                                  // few: tokens to quantize, or null
  int64_t ldx;
  const int8_t *q, *w;
  const float *xs, *ws;
  const void* bias;
  void* y;
  int64_t ldq, ldw, t;
  int32_t n, k, b32, vec;                         // vec: rows of x are whole aligned vectors
  int32_t bn, tm;                                 // tokens of a tile, tiles along the channels
};

// ------------------------------------------------------------------------------------------------ few tokens
// TT tokens (a.t <= TT), R rows of w at a time and warp
template <typename T, int TT, int R>
__global__ void __launch_bounds__(256) k_int8_few(const I8Args a) {
  extern __shared__ __align__(16) unsigned char few_smem[];
  __shared__ float red[TT][8], sc[TT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kp = (a.k + 15) & ~15, kv = kp / 16, whole = a.k / 16;
  const int rows = a.n, first = (blockIdx.x * 8 + warp) * R;
  // the first vectors of this warp's rows, in flight while the tokens are quantized
  uint4 pre[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    pre[r] = make_uint4(0u, 0u, 0u, 0u);
    if (first + r < rows && lane < whole) pre[r] = __ldg(reinterpret_cast<const uint4*>(a.w + (first + r) * a.ldw) + lane);
  }
  uint4* qs = reinterpret_cast<uint4*>(few_smem);  // [TT][kv]
  if (a.x) {
    constexpr int XV = kVec<T>;
    float top[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      top[t] = 0.f;
      if (t < a.t) {
        const T* p = (const T*)a.x + t * a.ldx;
        if (a.vec) {
#pragma unroll 2
          for (int j = tid * XV; j < a.k; j += 256 * XV) {
            float f[XV];
            load_v<T, XV>(p + j, f);
#pragma unroll
            for (int i = 0; i < XV; ++i) top[t] = top_of(top[t], f[i]);
          }
        } else {
          for (int j = tid; j < a.k; j += 256) top[t] = top_of(top[t], to_f(p[j]));
        }
      }
      top[t] = warp_top(top[t]);
      if (lane == 0) red[t][warp] = top[t];
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      float m = red[t][lane & 7];
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) m = top_of(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float s = q8_scale(m);
      const Q8 qk = q8_of(s);
      if (tid == 0) sc[t] = s;
      if (t >= a.t) {
        for (int j = tid; j < kv; j += 256) qs[t * kv + j] = make_uint4(0u, 0u, 0u, 0u);
        continue;
      }
      const T* p = (const T*)a.x + t * a.ldx;
      int8_t* o = reinterpret_cast<int8_t*>(qs + t * kv);
      if (a.vec) {
        for (int j = tid * XV; j < kp; j += 256 * XV) {
          float f[XV];
#pragma unroll
          for (int i = 0; i < XV; ++i) f[i] = 0.f;
          if (j < a.k) load_v<T, XV>(p + j, f);
#pragma unroll
          for (int i = 0; i < XV; i += 4) *reinterpret_cast<uint32_t*>(o + j + i) = q8x4(f + i, qk);
        }
      } else {
        for (int j = tid; j < kp; j += 256) o[j] = j < a.k ? (int8_t)q8(to_f(p[j]), qk) : (int8_t)0;
      }
    }
  } else {
    int8_t* o = reinterpret_cast<int8_t*>(qs);
    for (int t = 0; t < TT; ++t)
      for (int j = tid; j < kp; j += 256) o[t * kp + j] = t < a.t && j < a.k ? a.q[t * a.ldq + j] : (int8_t)0;
    if (tid < TT) sc[tid] = tid < a.t ? a.xs[tid] : 0.f;
  }
  __syncthreads();
  for (int n0 = first; n0 < rows; n0 += (int)gridDim.x * 8 * R) {
    int acc[R][TT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[r][t] = 0;
    auto dot = [&](const uint4 (&v)[R], int j) {
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const uint4 u = qs[t * kv + j];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          acc[r][t] = __dp4a((int)v[r].x, (int)u.x, acc[r][t]);
          acc[r][t] = __dp4a((int)v[r].y, (int)u.y, acc[r][t]);
          acc[r][t] = __dp4a((int)v[r].z, (int)u.z, acc[r][t]);
          acc[r][t] = __dp4a((int)v[r].w, (int)u.w, acc[r][t]);
        }
      }
    };
    const bool ahead = n0 == first;
#pragma unroll 4
    for (int j = lane; j < whole; j += 32) {
      uint4 v[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        v[r] = make_uint4(0u, 0u, 0u, 0u);
        if (ahead && j == lane)
          v[r] = pre[r];
        else if (n0 + r < rows)
          v[r] = __ldg(reinterpret_cast<const uint4*>(a.w + (n0 + r) * a.ldw) + j);
      }
      dot(v, j);
    }
    if (whole < kv && lane < a.k - 16 * whole)     // the last bytes of odd rows, one by one
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (n0 + r < rows) {
          const int v = a.w[(n0 + r) * a.ldw + 16 * whole + lane];
#pragma unroll
          for (int t = 0; t < TT; ++t) acc[r][t] += v * reinterpret_cast<const int8_t*>(qs + t * kv + whole)[lane];
        }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[r][t] = __reduce_add_sync(0xffffffffu, acc[r][t]);
    int mine = 0;                                  // lane R t + r writes row r of token t
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int t = 0; t < TT; ++t)
        if (lane == t * R + r) mine = acc[r][t];
    const int t = lane / R, n = n0 + lane % R;
    if (t < a.t && t < TT && n < rows) {
      const float b = !a.bias ? 0.f : a.b32 ? ((const float*)a.bias)[n] : to_f(((const T*)a.bias)[n]);
      ((T*)a.y)[(int64_t)t * rows + n] = from_f<T>(fmaf((float)mine * sc[t], a.ws[n], b));
    }
  }
}

// ------------------------------------------------------------------------------------------------ many tokens
constexpr int I8_EPI0 = 4, I8_EPI = 8, I8_THREADS = 32 * (I8_EPI0 + I8_EPI), I8_BK = 128;
constexpr unsigned long long I8_WAIT = 2000000000ull;

template <int CG>
struct I8Cfg {
  static constexpr int A_BYTES = 128 * I8_BK, B_BYTES = 256 / CG * I8_BK, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 196608 / STAGE, SMEM = STAGES * STAGE + 256 + 1024;
  static_assert(STAGES <= 8 && SMEM <= 227 * 1024, "shared memory");
};
struct I8Bars {
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2];
  uint32_t tmem;
  int failed;
};

// kind::i8: D int32 (bits 4-5 = 2), A and B signed 8-bit (1 at bits 7-9 and 10-12), both K-major
__host__ __device__ constexpr uint32_t i8_idesc(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
template <int CG>
__device__ __forceinline__ void mma_i8_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate));
}

template <typename T, int CG>
__global__ void __launch_bounds__(I8_THREADS, 1)
    k_int8_gemm(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q, const I8Args g) {
  using C = I8Cfg<CG>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  I8Bars& B = *reinterpret_cast<I8Bars*>(smem + C::STAGES * C::STAGE);
  volatile int* failed = &B.failed;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = CG == 2 ? (int)cluster_ctarank() : 0, cta = blockIdx.x / CG, ctas = gridDim.x / CG;
  if (warp == 1) {
    tmem_alloc<CG>(&B.tmem, 512);
    if (lane == 0) {
      for (int s = 0; s < C::STAGES; ++s) {
        mbar_init(&B.full[s], 1);
        mbar_init(&B.empty[s], 1);
      }
      for (int a = 0; a < 2; ++a) {
        mbar_init(&B.acc_full[a], 1);
        mbar_init(&B.acc_empty[a], I8_EPI * CG);
      }
      B.failed = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();         // the peer's barriers are initialised
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = B.tmem;
  const int tiles = g.tm * (int)((g.t + g.bn - 1) / g.bn), nk = (g.k + I8_BK - 1) / I8_BK, bh = g.bn / CG;

  if (warp == 0) {
    if (lane == 0) {
      int seq = 0;
      bool ok = true;
      const uint32_t bytes = CG * (uint32_t)(C::A_BYTES + bh * I8_BK);
      for (int t = cta; ok && t < tiles; t += ctas) {
        const int n0 = t / g.tm, m0 = (t - n0 * g.tm) * (128 * CG) + rank * 128;
        for (int kb = 0; kb < nk; ++kb, ++seq) {
          const int s = seq % C::STAGES;
          if (*failed || !mbar_wait_ns(&B.empty[s], ((seq / C::STAGES) & 1) ^ 1, I8_WAIT)) {
            *failed = 1;
            ok = false;
            break;
          }
          const uint32_t bar = CG == 2 ? mapa_u32(smem_u32(&B.full[s]), 0) : smem_u32(&B.full[s]);
          if (rank == 0) mbar_arrive_tx(&B.full[s], bytes);
          const uint32_t a = smem_u32(smem + s * C::STAGE);
          tma_load_2d<CG>(a, &map_w, kb * I8_BK, m0, bar);
          tma_load_2d<CG>(a + C::A_BYTES, &map_q, kb * I8_BK, n0 * g.bn + rank * bh, bar);
        }
      }
      if (!ok && rank == 0)                      // copies in flight land before the block ends (bounded)
        for (int q = seq - C::STAGES < 0 ? 0 : seq - C::STAGES; q < seq; ++q)
          mbar_wait_ns(&B.full[q % C::STAGES], (q / C::STAGES) & 1, I8_WAIT);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = i8_idesc(128 * CG, g.bn);
      int seq = 0, tc = 0;
      bool ok = true;
      uint64_t* last_bar = nullptr;
      uint32_t last_par = 0;
      for (int t = cta; ok && t < tiles; t += ctas, ++tc) {
        const int acc = tc & 1;
        if (*failed || !mbar_wait_ns(&B.acc_empty[acc], ((tc >> 1) & 1) ^ 1, I8_WAIT)) {
          *failed = 1;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int kb = 0; kb < nk; ++kb, ++seq) {
          const int s = seq % C::STAGES;
          if (!mbar_wait_ns(&B.full[s], (seq / C::STAGES) & 1, I8_WAIT)) {
            *failed = 1;
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t a = smem_u32(smem + s * C::STAGE), b = a + C::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < I8_BK / 32; ++kk)
            mma_i8_ss<CG>(tmem + acc * 256, sw128_desc(a + kk * 32), sw128_desc(b + kk * 32), idesc, (kb | kk) ? 1u : 0u);
          mma_commit_to<CG>(&B.empty[s]);
          last_bar = &B.empty[s];
          last_par = (seq / C::STAGES) & 1;
        }
        if (!ok) break;
        mma_commit_to<CG>(&B.acc_full[acc]);
        last_bar = &B.acc_full[acc];
        last_par = (tc >> 1) & 1;
      }
      if (*failed && last_bar) mbar_wait_ns(last_bar, last_par, I8_WAIT);
    }
  } else if (warp >= I8_EPI0) {
    const int q4 = warp & 3, hf = (warp - I8_EPI0) >> 2, hw = g.bn / 2;
    int tc = 0;
    bool lost = false;                           // warp-uniform
    for (int t = cta; t < tiles; t += ctas, ++tc) {
      const int tn = t / g.tm, acc = tc & 1;
      const int n = (t - tn * g.tm) * (128 * CG) + rank * 128 + q4 * 32 + lane;
      const bool on = n < g.n;
      float ws = on ? g.ws[n] : 0.f;
      const float b = !on || !g.bias ? 0.f : g.b32 ? ((const float*)g.bias)[n] : to_f(((const T*)g.bias)[n]);
      if (!lost) {
        lost = __shfl_sync(0xffffffffu, *failed, 0) || !__all_sync(0xffffffffu, mbar_wait_ns(&B.acc_full[acc], (tc >> 1) & 1, I8_WAIT));
        if (lost) *failed = 1;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
      if (lost) ws = __int_as_float(0x7fc00000);
      for (int c = 0; c < hw; c += 32) {
        const int64_t t0 = (int64_t)tn * g.bn + hf * hw + c;
        const int w = hw - c < 32 ? hw - c : 32, left = g.t - t0 < w ? (int)(g.t - t0) : w;   // tokens here
        uint32_t u[32];
        if (!lost) {
          tmem_ld32(tmem + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * 256 + hf * hw + c), u);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) u[i] = 0;
        }
        if (c + 32 >= hw && !lost) {             // the accumulator is free
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 2)
              mbar_arrive_cluster(mapa_u32(smem_u32(&B.acc_empty[acc]), 0));
            else
              mbar_arrive(&B.acc_empty[acc]);
          }
        }
        const float xs = lane < left ? g.xs[t0 + lane] : 0.f;
        T* y = (T*)g.y + t0 * g.n + n;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float s = __shfl_sync(0xffffffffu, xs, i);
          if (i < left && on) y[(int64_t)i * g.n] = from_f<T>(fmaf((float)(int)u[i] * s, ws, b));
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();         // no CTA leaves while its peer can still signal it or read its operands
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_dealloc<CG>(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------------ host side
template <typename T>
static int quant_go(const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int32_t k, cudaStream_t st) {
  constexpr int V = kVec<T>;
  const bool vec = k % V == 0 && ldx % V == 0 && aligned16(x) && ldq % 16 == 0 && aligned16(q);
  const int64_t want = (rows + 7) / 8, most = 8 * (int64_t)sm_count();
  const unsigned grid = (unsigned)(want < most ? want : most);
  if (vec)
    k_quant_rows<T, V><<<grid, 256, 0, st>>>((const T*)x, ldx, q, ldq, scale, rows, k);
  else
    k_quant_rows<T, 1><<<grid, 256, 0, st>>>((const T*)x, ldx, q, ldq, scale, rows, k);
  return check_launch("quantize_rows");
}

constexpr int I8_FEW = 8, I8_FEW_SMEM = 128 * 1024;   // most tokens of k_int8_few, most bytes of them

template <typename T, int TT, int R>
static int few_go(const I8Args& a, cudaStream_t st) {
  static int ready_dev = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("int8_linear (device)");
  if (ready_dev != dev) {
    if (cudaFuncSetAttribute(k_int8_few<T, TT, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, I8_FEW_SMEM) != cudaSuccess) {
      set_error("int8_linear: cannot reserve shared memory");
      return MB_E_CUDA;
    }
    ready_dev = dev;
  }
  const int smem = TT * ((a.k + 15) & ~15);
  const int64_t want = ((int64_t)a.n + 8 * R - 1) / (8 * R), most = 8 * (int64_t)sm_count();
  k_int8_few<T, TT, R><<<(unsigned)(want < most ? want : most), 256, smem, st>>>(a);
  return check_launch("int8_linear");
}

template <typename T>
static int few_any(const I8Args& a, cudaStream_t st) {
  const bool wide = a.n >= 32 * sm_count();       // rows enough for several a warp
  if (a.t <= 1) return wide ? few_go<T, 1, 4>(a, st) : few_go<T, 1, 1>(a, st);
  if (a.t <= 2) return wide ? few_go<T, 2, 4>(a, st) : few_go<T, 2, 1>(a, st);
  if (a.t <= 4) return wide ? few_go<T, 4, 4>(a, st) : few_go<T, 4, 1>(a, st);
  return wide ? few_go<T, 8, 4>(a, st) : few_go<T, 8, 1>(a, st);
}

template <typename T, int CG>
static int i8_go(I8Args a, cudaStream_t st) {
  using C = I8Cfg<CG>;
  static int ready_dev = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("int8_linear (device)");
  auto kern = k_int8_gemm<T, CG>;
  if (ready_dev != dev) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) {
      set_error("int8_linear: cannot reserve %d bytes of shared memory", C::SMEM);
      return MB_E_CUDA;
    }
    ready_dev = dev;
  }
  const int units = sm_count() / CG;
  a.tm = (a.n + 128 * CG - 1) / (128 * CG);
  // the widest tile of tokens that leaves every SM one, 32 at least
  a.bn = 256;
  while (a.bn > 32 && (int64_t)a.tm * ((a.t + a.bn - 1) / a.bn) < units) a.bn /= 2;
  const int64_t tiles = (int64_t)a.tm * ((a.t + a.bn - 1) / a.bn);
  if (tiles > 0x7fffffff) {
    set_error("int8_linear: too many tiles (%lld)", (long long)tiles);
    return MB_E_ARG;
  }
  CUtensorMap mw, mq;
  if (int rc = tensor_map_2d("int8_linear", &mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.w, a.k, a.n, a.ldw, I8_BK, 128)) return rc;
  if (int rc = tensor_map_2d("int8_linear", &mq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.q, a.k, a.t, a.ldq, I8_BK, a.bn / CG)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles < units ? tiles : units) * CG);
  cfg.blockDim = dim3(I8_THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CG > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kern, mw, mq, a);
  return check_launch("int8_linear");
}

template <typename T>
static int i8_any(const I8Args& a, cudaStream_t st) {
  // pairs of CTAs where full tiles of both give every pair several
  const int64_t pairs = (int64_t)((a.n + 255) / 256) * ((a.t + 255) / 256);
  return pairs >= 2 * (sm_count() / 2) && a.k >= 512 ? i8_go<T, 2>(a, st) : i8_go<T, 1>(a, st);
}

static bool rows16(const void* p, int64_t ld) { return aligned16(p) && ld % 16 == 0; }

template <typename F>
static int i8_type(int dtype, const F& f) {
  return dtype == MB_F32 ? f(float()) : dtype == MB_BF16 ? f(bf16()) : f(f16());
}

}  // namespace mb

using namespace mb;

extern "C" int mace_b200_quantize_rows(const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int32_t k,
                                       int32_t dtype, void* stream) {
  if (rows < 0 || k < 1 || ldx < k || ldq < k || !dtype_ok(dtype)) {
    set_error("quantize_rows: bad arguments (rows %lld, width %d, row strides %lld and %lld, type %d)", (long long)rows, k,
              (long long)ldx, (long long)ldq, dtype);
    return MB_E_ARG;
  }
  if (rows == 0) return 0;
  if (!x || !q || !scale) {
    set_error("quantize_rows: null pointer");
    return MB_E_ARG;
  }
  if (sm_count() < 1) {
    set_error("quantize_rows: no CUDA device");
    return MB_E_CUDA;
  }
  return i8_type(dtype, [&](auto t) { return quant_go<decltype(t)>(x, ldx, q, ldq, scale, rows, k, (cudaStream_t)stream); });
}

extern "C" int mace_b200_int8_linear_few(int64_t tokens, int32_t k) {
  return tokens <= I8_FEW && (tokens <= 1 ? 1 : tokens <= 2 ? 2 : tokens <= 4 ? 4 : 8) * (int64_t)((k + 15) & ~15) <= I8_FEW_SMEM;
}

extern "C" int mace_b200_int8_linear(const void* x, int64_t ldx, int8_t* xq, int64_t ldq, float* xscale, const int8_t* wq,
                                     int64_t ldw, const float* wscale, const void* bias, void* y, int64_t tokens, int32_t k,
                                     int32_t n, int32_t dtype, int32_t btype, void* stream) {
  if (tokens < 0 || tokens > 0x7fffff00 || k < 1 || n < 1 || n > 0x7fffff00 || k > MB_INT8_MAX_K || ldw < k || (x && ldx < k) || !dtype_ok(dtype) ||
      (btype != dtype && btype != MB_F32)) {
    set_error("int8_linear: bad arguments (tokens %lld, in %d (at most %d), out %d, row strides %lld and %lld, types %d, %d)",
              (long long)tokens, k, MB_INT8_MAX_K, n, (long long)ldx, (long long)ldw, dtype, btype);
    return MB_E_ARG;
  }
  if (tokens == 0) return 0;
  const bool few = mace_b200_int8_linear_few(tokens, k);
  if (!wq || !wscale || !y || (!(x && few) && (!xq || !xscale || ldq < k))) {
    set_error("int8_linear: null pointer");
    return MB_E_ARG;
  }
  if (!rows16(wq, ldw) || (!few && !rows16(xq, ldq))) {
    set_error("int8_linear: rows of 8-bit values must start on 16 bytes");
    return MB_E_ARG;
  }
  if (sm_count() < 1) {
    set_error("int8_linear: no CUDA device");
    return MB_E_CUDA;
  }
  I8Args a{};
  a.x = x; a.ldx = ldx; a.q = xq; a.ldq = ldq; a.xs = xscale; a.w = wq; a.ldw = ldw; a.ws = wscale; a.bias = bias; a.y = y;
  a.t = tokens; a.n = n; a.k = k; a.b32 = btype == MB_F32;
  cudaStream_t st = (cudaStream_t)stream;
  return i8_type(dtype, [&](auto t) {
    using T = decltype(t);
    a.vec = x && k % kVec<T> == 0 && ldx % kVec<T> == 0 && aligned16(x);
    if (few) return few_any<T>(a, st);
    if (x)
      if (int rc = quant_go<T>(x, ldx, xq, ldq, xscale, tokens, k, st)) return rc;
    return i8_any<T>(a, st);
  });
}
