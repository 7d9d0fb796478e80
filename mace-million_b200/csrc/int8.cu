// Linear maps in 8-bit integers, a scale for each token and each output channel:
//   s_t = max_k |x[t][k]| / 127,  q[t][k] = nearest(x[t][k] / s_t),  y[t][n] = (sum_k q[t][k] w[n][k]) s_t s_n + b_n
// The sums are exact in int32 (k <= MB_INT8_MAX_K), y is fp32 arithmetic on them, rounded once: (sum s_n) s_t + b_n, in this order, as
// sum s_t of tokens beyond 1e33 would overflow where y does not.  q is the nearest whole number
// of the exact quotient, ties to even (a remainder by fma corrects the rounded quotient), so it does not depend on who divides.
//
// Three kernels.  k_quant_rows: a row stays in the registers of 32 to 256 threads, read once.  k_int8_few: up to 4 tokens; a CTA quantizes them into shared memory while its
// first weights are on their way, then each warp takes whole rows of w with dp4a: bound by the weights' bytes and latency.
// k_int8_gemm: tcgen05 kind::i8 from TMA tiles (SWIZZLE_128B, 128 bytes of K a stage).  Output channels are the rows of an MMA
// and tokens its columns: few tokens take a narrow tile, a lane holds one channel (its scale and bias stay in registers), and
// a warp stores 32 neighbouring channels of a token at once, whatever the alignment of y.  What drains a tile is short code on
// scales in shared memory, fetched a tile ahead; 128 x 256 results take 2.9 us an SM, 5.4 cycles a store.
// Persistent CTAs, one per SM: warp 0 loads, warp 1 issues, warps 4-11 drain one of two accumulators.  CG = 2: pairs of CTAs
// (cta_group::2) on 256 channels, each with its own 128 and half of the tokens' rows.  Every wait is bounded; a tile whose
// wait expired is NaN.
//
// Measured on a B200 (cuBLAS bf16 1.67 PFLOP/s, so 3.3 POP/s for 8 bits): 16,384 x 4096 x 4096 bf16 202 us; alone the quantization takes 42
// (4.8 TB/s) and the product of 8-bit tokens 164 (3.4 POP/s, the tensor cores 87% busy); 16,384 x 1024 x 1024 31 us (10 and 19; the drain of a tile takes as
// long as its 8 K blocks); 24,001 x 515 x 1001 fp16 42 us (13 and 28: elements of two bytes in rows of any alignment); 192 x 128 x 512
// fp32 6 us (two launches); one token 1024 x 1024 2.7 us, 4096 x 4096 5.0 us (3.4 TB/s of weights).  Few tokens by dp4a / by the
// tensor cores, 512 x 2048: 4 tokens 5.1 / 6.3 us, 5 tokens 8.4 / 6.4.
#include <cuda.h>

#include <type_traits>

#include "dtypes.cuh"
#include "tc.cuh"
#include "tensor_map.cuh"

namespace mb {

// Scale of a row, its reciprocal, and the power of two that keeps both normal (a tiny row's scale is subnormal); half: half of the
// scale where the short way of q8x4 holds, else NaN
struct Q8 {
  float scale, s, inv, up, half;
};
__device__ __forceinline__ Q8 q8_of(float scale) {
  Q8 k;
  k.scale = scale;
  k.up = scale < 0x1p-100f ? 0x1p60f : 1.f;
  k.s = scale * k.up;
  k.inv = 1.f / k.s;
  k.half = scale >= 0x1p-100f && scale < 0x1p120f ? 0.5f * scale : __int_as_float(0x7fc00000);
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
// Four of them as bytes.  Usually the rounded quotient is the one: x inv + 1.5 2^23 has it in its low bits, and the remainder shows
// that it is: |x - q s| < s / 2.  A tie (bf16 has many: 500 x 4096 3.9 us by the long way, 3.1 so) goes to the even neighbour; what
// is off by more, tiny and unusual scales take the long way.
__device__ __forceinline__ uint32_t q8x4(const float* f, const Q8& k) {
  constexpr float MAGIC = 12582912.f;
  const float2 inv = make_float2(k.inv, k.inv), big = make_float2(MAGIC, MAGIC), less = make_float2(-MAGIC, -MAGIC);
  const float2 neg = make_float2(-k.s, -k.s), a = make_float2(f[0], f[1]), b = make_float2(f[2], f[3]);
  const float2 ta = __ffma2_rn(a, inv, big), tb = __ffma2_rn(b, inv, big);
  const float2 ra = __ffma2_rn(__fadd2_rn(ta, less), neg, a), rb = __ffma2_rn(__fadd2_rn(tb, less), neg, b);
  const float m = fmaxf(fmaxf(fabsf(ra.x), fabsf(ra.y)), fmaxf(fabsf(rb.x), fabsf(rb.y)));
  uint32_t w[4] = {__float_as_uint(ta.x), __float_as_uint(ta.y), __float_as_uint(tb.x), __float_as_uint(tb.y)};
  if (!(m < k.half)) {
    if (!(m == k.half))
      return (uint32_t)(q8(f[0], k) & 255) | (uint32_t)(q8(f[1], k) & 255) << 8 | (uint32_t)(q8(f[2], k) & 255) << 16 |
             (uint32_t)q8(f[3], k) << 24;
    const float r[4] = {ra.x, ra.y, rb.x, rb.y};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (fabsf(r[i]) == k.half && (w[i] & 1)) w[i] += r[i] > 0.f ? 1u : ~0u;
  }
  return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}
// max |x| that NaN passes through
__device__ __forceinline__ float top_of(float m, float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
  return r;
}
__device__ __forceinline__ float warp_top(float m) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = top_of(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
// of a 16-byte vector: two 16-bit elements at a time
__device__ __forceinline__ float top16(const uint4& u, float) {
  return top_of(top_of(fabsf(__uint_as_float(u.x)), __uint_as_float(u.y)), top_of(fabsf(__uint_as_float(u.z)), __uint_as_float(u.w)));
}
template <typename T2>
__device__ __forceinline__ T2 top_pair(const uint4& u) {
  const T2 a = *reinterpret_cast<const T2*>(&u.x), b = *reinterpret_cast<const T2*>(&u.y), c = *reinterpret_cast<const T2*>(&u.z),
           d = *reinterpret_cast<const T2*>(&u.w);
  return __hmax2_nan(__hmax2_nan(__habs2(a), __habs2(b)), __hmax2_nan(__habs2(c), __habs2(d)));
}
__device__ __forceinline__ float top16(const uint4& u, bf16) {
  const __nv_bfloat162 m = top_pair<__nv_bfloat162>(u);
  return top_of(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float top16(const uint4& u, f16) {
  const __half2 m = top_pair<__half2>(u);
  return top_of(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float q8_scale(float top) { return __fdiv_rn(top, 127.f); }

// Largest value of the G threads of a group (a block of 256 or G threads; `red` is one buffer of two that calls alternate)
template <int G>
__device__ __forceinline__ float group_top(float m, float* red) {
  m = warp_top(m);
  if constexpr (G > 32) {
    constexpr int W = G / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) red[warp] = m;
    __syncthreads();
    m = red[warp / W * W + (lane & (W - 1))];
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) m = top_of(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  return m;
}

template <int G>
constexpr int q8_threads = G < 256 ? 256 : G;
// Rows of whole aligned vectors that G threads hold, NV vectors each: read once.  Bytes up to ldq that hold no value are zero.
template <typename T, int G, int NV>
__global__ void __launch_bounds__(q8_threads<G>) k_quant_rows(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q,
                                                              int64_t ldq, float* __restrict__ scale, int64_t rows, int32_t k) {
  constexpr int V = kVec<T>, RPB = q8_threads<G> / G;
  __shared__ float red[2][q8_threads<G> / 32];
  const int t = threadIdx.x % G, g = threadIdx.x / G;
  int buf = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB, buf ^= 1) {
    const int64_t row = r0 + g;
    const T* p = x + (row < rows ? row : r0) * ldx;
    uint4 u[NV];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * G + t) * V;
      u[i] = make_uint4(0u, 0u, 0u, 0u);
      if (j < k) u[i] = *reinterpret_cast<const uint4*>(p + j);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) top = top_of(top, top16(u[i], T()));
    top = group_top<G>(top, red[buf]);
    if (row >= rows) continue;
    const Q8 qk = q8_of(q8_scale(top));
    if (t == 0) scale[row] = qk.scale;
    int8_t* o = q + row * ldq;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * G + t) * V;
      if (j >= ldq) continue;
      float f[V];
      unpack16(u[i], f, T());
      if constexpr (V == 8)
        *reinterpret_cast<uint2*>(o + j) = make_uint2(q8x4(f, qk), q8x4(f + 4, qk));
      else
        *reinterpret_cast<uint32_t*>(o + j) = q8x4(f, qk);
    }
  }
}

// Any rows, a warp each, an element an access and four neighbours a lane.  NV > 0: up to 128 NV values stay in registers; else the
// row is read twice (the second time from L1 or L2).  words: rows of q are aligned to four bytes.
template <typename T, int NV>
__global__ void __launch_bounds__(256) k_quant_any(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, int64_t ldq,
                                                   float* __restrict__ scale, int64_t rows, int32_t k, bool words) {
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * 8;
  for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < rows; row += step) {
    const T* p = x + row * ldx;
    int8_t* o = q + row * ldq;
    float top = 0.f;
    auto put = [&](int64_t j, const float (&f)[4], const Q8& qk) {
      const uint32_t w = q8x4(f, qk);
      if (words) {
        if (j < ldq) *reinterpret_cast<uint32_t*>(o + j) = w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j + i < ldq) o[j + i] = (int8_t)(w >> (8 * i));
      }
    };
    if constexpr (NV > 0) {
      T v[NV][4];
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = 128 * n + 4 * lane + i;
          v[n][i] = from_f<T>(0.f);
          if (j < k) v[n][i] = p[j];
        }
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = top_of(top, to_f(v[n][i]));
      const Q8 qk = q8_of(q8_scale(warp_top(top)));
      if (lane == 0) scale[row] = qk.scale;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const float f[4] = {to_f(v[n][0]), to_f(v[n][1]), to_f(v[n][2]), to_f(v[n][3])};
        put(128 * n + 4 * lane, f, qk);
      }
      for (int64_t j = 128 * NV + lane; j < ldq; j += 32) o[j] = 0;
    } else {
#pragma unroll 8
      for (unsigned j = lane; j < (unsigned)k; j += 32) top = top_of(top, to_f(p[j]));   // (a step beyond widths next to 2^31 passes 31 bits)
      const Q8 qk = q8_of(q8_scale(warp_top(top)));
      if (lane == 0) scale[row] = qk.scale;
#pragma unroll 2
      for (int64_t j = 4 * lane; j < ldq; j += 128) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = j + i < k ? to_f(p[j + i]) : 0.f;
        put(j, f, qk);
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
  const unsigned rows = a.n, first = (blockIdx.x * 8 + warp) * R;   // (a grid's step beyond 2^31 - 256 rows passes 31 bits)
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
      const Q8 qk = q8_of(q8_scale(m));
      if (tid == 0) sc[t] = qk.scale;
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
  for (unsigned n0 = first; n0 < rows; n0 += gridDim.x * 8 * R) {
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
    const int t = lane / R;
    const unsigned n = n0 + lane % R;
    if (t < a.t && t < TT && n < rows) {
      const float b = !a.bias ? 0.f : a.b32 ? ((const float*)a.bias)[n] : to_f(((const T*)a.bias)[n]);
      ((T*)a.y)[(int64_t)t * rows + n] = from_f<T>(fmaf((float)mine * a.ws[n], sc[t], b));
    }
  }
}

// ------------------------------------------------------------------------------------------------ many tokens
constexpr int I8_EPI0 = 4, I8_EPI = 8, I8_THREADS = 32 * (I8_EPI0 + I8_EPI), I8_BK = 128;
constexpr unsigned long long I8_WAIT = 2000000000ull;

struct I8Bars {
  float xs[I8_EPI][128];                         // the scales of a draining warp's tokens
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2];
  uint32_t tmem;
  int failed, never;                             // never: a flag that stays 0
};
template <int CG>
struct I8Cfg {
  static constexpr int A_BYTES = 128 * I8_BK, B_BYTES = 256 / CG * I8_BK, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 196608 / STAGE, SMEM = STAGES * STAGE + sizeof(I8Bars) + 1024;
  static_assert(STAGES <= 8 && SMEM <= 227 * 1024, "shared memory");
};
// kind::i8: D int32 (bits 4-5 = 2), A and B signed 8-bit (1 at bits 7-9 and 10-12), both K-major
__host__ __device__ constexpr uint32_t i8_idesc(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
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
      B.failed = B.never = 0;
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
    const uint32_t lead = elect_lane(), smem0 = smem_u32(smem), full0 = smem_u32(B.full), empty0 = smem_u32(B.empty);
    const uint32_t target = CG == 2 ? mapa_u32(full0, 0) : full0, bytes = CG * (uint32_t)(C::A_BYTES + bh * I8_BK);
    const int tm = g.tm;
    int s = 0;
    uint32_t par = 1;
    bool ok = true, wrapped = false;
    for (int t = cta; ok && t < tiles; t += ctas) {
      const int tn = t / tm, m0 = (t - tn * tm) * (128 * CG) + rank * 128, n0 = tn * g.bn + rank * bh;
      for (int kb = 0; kb < nk; ++kb) {
        if (!mbar_wait_warp(empty0 + 8 * s, par, I8_WAIT, failed)) {
          *failed = 1;
          ok = false;
          break;
        }
        const uint32_t a = smem0 + s * C::STAGE;
        // both CTAs' bytes arrive at the first one's barrier
        mbar_arrive_tx_lead(rank == 0 ? lead : 0u, full0 + 8 * s, bytes);
        tma_load_2d_lead<CG>(lead, a, &map_w, kb * I8_BK, m0, target + 8 * s);
        tma_load_2d_lead<CG>(lead, a + C::A_BYTES, &map_q, kb * I8_BK, n0, target + 8 * s);
        if (++s == C::STAGES) s = 0, par ^= 1, wrapped = true;
      }
    }
    if (!ok && rank == 0)                        // copies in flight land before the block ends (bounded)
      for (int q = 0; q < C::STAGES; ++q) {      // places before s: this round's, the others: the round before
        if (q >= s && !wrapped) break;
        mbar_wait_ns(&B.full[q], q < s ? par ^ 1 : par, I8_WAIT);
      }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t lead = elect_lane(), smem0 = smem_u32(smem), full0 = smem_u32(B.full), empty0 = smem_u32(B.empty);
      const uint32_t acc_full0 = smem_u32(B.acc_full), acc_empty0 = smem_u32(B.acc_empty);
      const uint32_t idesc = i8_idesc(128 * CG, g.bn);
      const uint64_t a_base = sw128_desc(smem0), b_base = sw128_desc(smem0 + C::A_BYTES);
      int s = 0, acc = 0;
      uint32_t par = 0, acc_par = 1, last_bar = 0, last_par = 0;
      bool ok = true;
      for (int t = cta; ok && t < tiles; t += ctas) {
        if (!mbar_wait_warp(acc_empty0 + 8 * acc, acc_par, I8_WAIT, failed)) {
          *failed = 1;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem + acc * 256;
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait_warp(full0 + 8 * s, par, I8_WAIT, failed)) {
            *failed = 1;
            ok = false;
            break;
          }
          const uint64_t off = (uint64_t)((uint32_t)(s * C::STAGE) >> 4);
#pragma unroll
          for (int kk = 0; kk < I8_BK / 32; ++kk)
            mma_i8_ss_lead<CG>(lead, d, a_base + off + kk * 2, b_base + off + kk * 2, idesc, (kb | kk) ? 1u : 0u);
          mma_commit_lead<CG>(lead, empty0 + 8 * s);
          last_bar = empty0 + 8 * s;
          last_par = par;
          if (++s == C::STAGES) s = 0, par ^= 1;
        }
        if (!ok) break;
        mma_commit_lead<CG>(lead, acc_full0 + 8 * acc);
        last_bar = acc_full0 + 8 * acc;
        last_par = acc_par ^ 1;
        acc ^= 1;
        if (acc == 0) acc_par ^= 1;
      }
      if (*failed && last_bar) mbar_wait_warp(last_bar, last_par, I8_WAIT, &B.never);
    }
  } else if (warp >= I8_EPI0) {
    const int q4 = warp & 3, hf = (warp - I8_EPI0) >> 2, hw = g.bn / 2, tm = g.tm, n_all = g.n;
    const int64_t tokens = g.t;
    float* xs = B.xs[warp - I8_EPI0];
    int acc = 0;
    uint32_t acc_par = 0;
    bool lost = false;                           // warp-uniform
    // the next tile's: this lane's channel, and the scales of the half's tokens (lane l has those of l, 32 + l, ..)
    float next_ws = 0.f, next_b = 0.f, next_xs[4];
    auto fetch = [&](int t) {
      const int tn = t / tm, n = (t - tn * tm) * (128 * CG) + rank * 128 + q4 * 32 + lane;
      const int64_t first = (int64_t)tn * g.bn + hf * hw;
      const bool on = n < n_all;
      next_ws = on ? g.ws[n] : 0.f;
      next_b = !on || !g.bias ? 0.f : g.b32 ? ((const float*)g.bias)[n] : to_f(((const T*)g.bias)[n]);
#pragma unroll
      for (int q = 0; q < 4; ++q) next_xs[q] = 32 * q + lane < hw && first + 32 * q + lane < tokens ? g.xs[first + 32 * q + lane] : 0.f;
    };
    if (cta < tiles) fetch(cta);
    for (int t = cta; t < tiles; t += ctas) {
      const int tn = t / tm, n = (t - tn * tm) * (128 * CG) + rank * 128 + q4 * 32 + lane;
      const int64_t first = (int64_t)tn * g.bn + hf * hw;
      const bool on = n < n_all;
      float ws = next_ws;
      const float b = next_b;
#pragma unroll
      for (int q = 0; q < 4; ++q) xs[32 * q + lane] = next_xs[q];
      __syncwarp();
      if (!lost) lost = !mbar_wait_warp(smem_u32(&B.acc_full[acc]), acc_par, I8_WAIT, failed);
      if (lost) {
        *failed = 1;
        ws = __int_as_float(0x7fc00000);
      }
      if (t + ctas < tiles) fetch(t + ctas);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      T* y = (T*)g.y + first * n_all + n;
#pragma unroll 1                                // short code: unrolled, 16,384 x 512 x 512 fp16 takes 10.4 us instead of 9.8
      for (int c = 0; c < hw; c += 32) {
        const int w = hw - c < 32 ? hw - c : 32;
        const int64_t rest = tokens - first - c;
        const int left = rest < w ? (int)rest : w;             // tokens here (<= 0: none)
        uint32_t u[32];
        if (!lost) {
          tmem_ld32(tmem + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * 256 + hf * hw + c), u);
          tmem_wait_ld();
          if (c + 32 >= hw) {                    // the accumulator is free
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              if constexpr (CG == 2)
                mbar_arrive_remote(mapa_u32(smem_u32(&B.acc_empty[acc]), 0));
              else
                mbar_arrive(&B.acc_empty[acc]);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) u[i] = 0;
        }
        // the tokens' rows one after the other, 32 neighbouring channels a store
        const float4* s4 = reinterpret_cast<const float4*>(xs + c);
        auto put = [&](float sum, float s, bool here) {
          const float v = fmaf(sum * ws, s, b);
          if (here) *y = from_f<T>(v);
          y += n_all;
        };
        if (left == 32) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 f = s4[i / 4];
            put((float)(int)u[i], f.x, on);
            put((float)(int)u[i + 1], f.y, on);
            put((float)(int)u[i + 2], f.z, on);
            put((float)(int)u[i + 3], f.w, on);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 f = s4[i / 4];
            put((float)(int)u[i], f.x, i < left && on);
            put((float)(int)u[i + 1], f.y, i + 1 < left && on);
            put((float)(int)u[i + 2], f.z, i + 2 < left && on);
            put((float)(int)u[i + 3], f.w, i + 3 < left && on);
          }
        }
      }
      __syncwarp();                              // the scales are read
      acc ^= 1;
      if (acc == 0) acc_par ^= 1;
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
template <typename T, int G, int NV>
static int quant_held(const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int32_t k, cudaStream_t st) {
  constexpr int RPB = q8_threads<G> / G;
  const int64_t want = (rows + RPB - 1) / RPB, most = (2048 / q8_threads<G>) * (int64_t)sm_count();
  k_quant_rows<T, G, NV><<<(unsigned)(want < most ? want : most), q8_threads<G>, 0, st>>>((const T*)x, ldx, q, ldq, scale, rows, k);
  return check_launch("quantize_rows");
}
template <typename T>
static int quant_go(const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int32_t k, cudaStream_t st) {
  constexpr int V = kVec<T>;
  if (k % V == 0 && ldx % V == 0 && aligned16(x) && ldq % 16 == 0 && aligned16(q)) {   // (the pad of ldq < k + 16 is held, too)
    const int64_t nv = (ldq + V - 1) / V;
    // a warp a row as far as its registers go (16,384 x 768 fp32 7.3 us, 128 threads a row 14.8; 16,384 x 2048 fp16 17.7 and 25.3), then
    // small groups with full registers (16,384 x 8192 fp16: 256 threads 70 us, 512 103; 4096 wide: 128 threads 37 us, a warp 43)
    if (ldq < k + 16) {
      if (nv <= 32) return quant_held<T, 32, 1>(x, ldx, q, ldq, scale, rows, k, st);
      if (nv <= 64) return quant_held<T, 32, 2>(x, ldx, q, ldq, scale, rows, k, st);
      if (nv <= 128) return quant_held<T, 32, 4>(x, ldx, q, ldq, scale, rows, k, st);
      if (nv <= 256) return quant_held<T, 32, 8>(x, ldx, q, ldq, scale, rows, k, st);
      if (nv <= 512) return quant_held<T, 128, 4>(x, ldx, q, ldq, scale, rows, k, st);
      if (nv <= 1024) return quant_held<T, 256, 4>(x, ldx, q, ldq, scale, rows, k, st);
      if (nv <= 2048) return quant_held<T, 256, 8>(x, ldx, q, ldq, scale, rows, k, st);
    }
  }
  const int64_t want = (rows + 7) / 8, most = 8 * (int64_t)sm_count();
  const bool words = ldq % 4 == 0 && (reinterpret_cast<uintptr_t>(q) & 3) == 0;
  const unsigned grid = (unsigned)(want < most ? want : most);
  // a row of up to 1024 values stays in registers, in as many pieces of 128 as it has: each piece more costs 0.5 to 1.5 us of 16,384 rows (300
  // fp16: three 6.9 us, five 8.8; 515 fp16: five 9.5, eight 13.4, read twice 11.8; 900 fp16: eight 14.7, twice 18.0; 1200: ten and twice 12.5)
  const auto any = [&](auto nv) {
    k_quant_any<T, decltype(nv)::value><<<grid, 256, 0, st>>>((const T*)x, ldx, q, ldq, scale, rows, k, words);
    return check_launch("quantize_rows");
  };
  switch (k <= 1024 ? (k + 127) / 128 : 0) {
    case 1: return any(std::integral_constant<int, 1>());
    case 2: return any(std::integral_constant<int, 2>());
    case 3: return any(std::integral_constant<int, 3>());
    case 4: return any(std::integral_constant<int, 4>());
    case 5: return any(std::integral_constant<int, 5>());
    case 6: return any(std::integral_constant<int, 6>());
    case 7: return any(std::integral_constant<int, 7>());
    case 8: return any(std::integral_constant<int, 8>());
    default: return any(std::integral_constant<int, 0>());
  }
}

constexpr int I8_FEW = 4, I8_FEW_SMEM = 128 * 1024;   // most tokens of k_int8_few, most bytes of them

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
  // rows enough for several a warp, which then read the tokens once (4096 x 4096, two rows against one: 2 tokens 6.1 and 7.3 us, 4 tokens 9.1
  // and 11.5; 4096 x 2500 2 tokens 6.2 and 5.9)
  const bool wide = a.n >= 32 * sm_count(), some = a.n >= 24 * sm_count();
  if (a.t <= 1) return wide ? few_go<T, 1, 4>(a, st) : few_go<T, 1, 1>(a, st);
  if (a.t <= 2) return wide ? few_go<T, 2, 4>(a, st) : some ? few_go<T, 2, 2>(a, st) : few_go<T, 2, 1>(a, st);
  return wide ? few_go<T, 4, 4>(a, st) : some ? few_go<T, 4, 2>(a, st) : few_go<T, 4, 1>(a, st);
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
  // the tile of tokens whose rounds over the SMs take least: a tile's products (2 cycles a column and K block, 300 a K block at
  // least) or its drain (40 cycles a column), whichever is longer, and what a tile costs besides
  const int nk = (a.k + I8_BK - 1) / I8_BK;
  double least = 0.0;
  for (int bn = 256; bn >= 32 * CG; bn -= 32 * CG) {
    const int64_t t = (int64_t)a.tm * ((a.t + bn - 1) / bn);
    const double mma = (double)nk * (2 * bn > 300 ? 2 * bn : 300), drain = 40.0 * bn;
    const double cost = (double)((t + units - 1) / units) * ((mma > drain ? mma : drain) + 800);
    if (bn == 256 || cost <= least) least = cost, a.bn = bn;
  }
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
  return tokens <= I8_FEW && (tokens <= 1 ? 1 : tokens <= 2 ? 2 : 4) * (int64_t)((k + 15) & ~15) <= I8_FEW_SMEM;
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
