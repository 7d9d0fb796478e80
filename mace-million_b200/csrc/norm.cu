// Layer norm over the last dimension of rows that may be strided (the 0e block of the node features has rows 512 apart):
//   mu = mean(x), var = mean((x - mu)^2), r = 1 / sqrt(var + eps), xh = (x - mu) r, y = xh w + b
// and its backward pass, with a = dy w:
//   dx = r (a - mean(a) - xh mean(a xh)), dw = sum over rows of dy xh, db = sum over rows of dy.
// Statistics and sums are fp32 whatever the type of x; every output is rounded once.
//
// Bound: HBM bytes (forward x and y, backward x, dy and dx, each once).  A row stays in registers between the sums
// and the output, so nothing is read twice.  Groups of G threads own a row; an element's column belongs to the same
// thread in every row, so the backward pass accumulates dw and db in registers over the rows of a block, and a second
// small kernel adds the blocks' partial sums in a fixed order (no atomics: results do not depend on the schedule).
// V is the elements per access: 16 bytes where the width, the row strides and the addresses allow it, else 1.
// Widths that no group holds in registers take the *_wide kernels, which read the row once per sum, one element per access:
// 2,000 x 20,001 bf16 70 / 203 us (2.3 and 1.2 TB/s), 500 x 100,000 120 / 345 us, bound by the latency of those accesses.
// Measured on a B200 (forward / backward): 65,536 x 2048 bf16 100 / 151 us (5.3 TB/s each, of 6.5 measured for a copy),
// 65,536 x 1024 bf16 45 / 80 us, 32,768 x 1024 fp32 49 / 67 us, 16,384 x 128 fp32 in rows 512 apart 3.7 / 7.9 us,
// 24,001 x 515 bf16 (one element per access) 20 / 26 us, 100,000 x 64 fp16 (8 threads a row) 6.0 / 10.8 us, with a whole
// warp a row 18 / 26.  Below 5 TB/s the issue slots bound it: unpacking, the packed arithmetic and packing are about 10
// instructions an element backward.
#include "norm.cuh"

namespace mb {

struct LnArgs {
  const void *x, *dy, *w, *b;
  void *y, *dx;
  float *mean, *rstd, *partial;
  int64_t ldx, lddy, n;
  int32_t d;
  float eps;
};

// Sums of K (a power of two) values over the G threads of a group (all threads of the block call it; `red` holds
// (threads / 32) * K floats and is free to be overwritten two calls later: callers alternate two buffers).
template <int G, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float* red) {
  if constexpr (G < 32) {                         // several groups in a warp
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int W = G < 32 ? 1 : G / 32;
  float s = 0.f;
  if constexpr (K == 4) {                         // transposed: lane L ends with value L >> 3 (6 shuffles instead of 20)
#pragma unroll
    for (int h = 2, bit = 16; h >= 1; h >>= 1, bit >>= 1) {
      const bool up = lane & bit;
#pragma unroll
      for (int q = 0; q < h; ++q) {
        const float send = up ? v[q] : v[q + h];
        const float keep = up ? v[q + h] : v[q];
        v[q] = keep + __shfl_xor_sync(0xffffffffu, send, bit);
      }
    }
    s = v[0];
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  }
  if constexpr (G <= 32) {
    if constexpr (K == 4) {
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = __shfl_sync(0xffffffffu, s, 32 / K * k);
    } else {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    }
  } else {
    if constexpr (K == 4) {
      if (lane % (32 / K) == 0) red[warp * K + lane / (32 / K)] = s;
    } else {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
      if (lane == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) red[warp * K + k] = v[k];
    }
    __syncthreads();
    // the group's W x K partial sums, one or more per lane, then over the warps by shuffles
    const float* r = red + warp / W * W * K;
    float t = lane < W * K ? r[lane] : 0.f;
#pragma unroll
    for (int o = 32; o < W * K; o += 32) t += r[o + lane];
#pragma unroll
    for (int o = (W * K < 32 ? W * K : 32) / 2; o >= K; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = __shfl_sync(0xffffffffu, t, k);
  }
}

template <int G>
constexpr int ln_threads = G < 256 ? 256 : G;
// threads per SM that the registers of a thread are budgeted for, and whether the next row is fetched ahead: worth the
// registers at up to 16 values a thread (65,536 x 512 bf16 27.1 -> 23.3 us, 16,000 x 2049 fp16 82 -> 71) and from 64
// with half the threads (20,000 x 4096 bf16 88 -> 70), not at 32 (65,536 x 1024 bf16 45.3 us without, 48.2 with)
template <int G, int NV, int V>
constexpr int ln_fwd_blocks = (NV * V >= 64 ? 512 : 1024) / ln_threads<G>;
template <int NV, int V>
constexpr bool ln_fwd_pre = NV * V != 32;
template <int G, int NV, int V>
constexpr int ln_bwd_blocks = G > 256 ? 1 : NV * V > 4 ? 2 : 3;

// The row is held as loaded (16-bit rows take half the registers of fp32 values) and unpacked at each use.
template <typename T, typename P, int G, int NV, int V>
__global__ void __launch_bounds__(ln_threads<G>, ln_fwd_blocks<G, NV, V>) k_ln_fwd(const LnArgs a) {
  constexpr int RPB = ln_threads<G> / G;
  constexpr bool KEEP = NV * V <= 8;              // parameters stay in registers over the rows, else from L1 per row
  __shared__ float red[2][ln_threads<G> / 32];
  const int t = threadIdx.x % G, g = threadIdx.x / G, d = a.d;
  const P *w = (const P*)a.w, *b = (const P*)a.b;
  float pw[KEEP ? NV : 1][V], pb[KEEP ? NV : 1][V];
  auto params = [&](int i, float (&fw)[V], float (&fb)[V]) {
    const int j = (i * G + t) * V;
#pragma unroll
    for (int q = 0; q < V; ++q) fw[q] = 1.f, fb[q] = 0.f;
    if (j < d) {
      if (w) load_p<P, V>(w + j, fw);
      if (b) load_p<P, V>(b + j, fb);
    }
  };
  if constexpr (KEEP)
#pragma unroll
    for (int i = 0; i < NV; ++i) params(i, pw[i], pb[i]);
  const float inv = 1.f / (float)d;
  constexpr bool PRE = ln_fwd_pre<NV, V>;
  Raw<T, V> nx[PRE ? NV : 1];                     // the next row, in flight while this one is worked on
  auto fetch = [&](int64_t row, auto& to) {
    const T* x = (const T*)a.x + row * a.ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * G + t) * V;
      to[i].zero();
      if (j < d) to[i].load(x + j);
    }
  };
  if constexpr (PRE) {
    const int64_t row = (int64_t)blockIdx.x * RPB + g;
    if (row < a.n) fetch(row, nx);
  }
  // the trip count is the same for every group of a block (group_sum synchronises the block)
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.n; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + g;
    const bool live = row < a.n;
    using E = Elem<V>;
    constexpr int NE = kElems<V>;
    Raw<T, V> v[NV];
    float s[1], f[V];
    E e[NE], acc[NE] = {};
    if constexpr (PRE) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = nx[i];
      if (row + (int64_t)gridDim.x * RPB < a.n) fetch(row + (int64_t)gridDim.x * RPB, nx);
    } else {
      if (live) fetch(row, v);
      else
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i].zero();
    }
    auto fold = [&] {
      E p = acc[0];
#pragma unroll
      for (int q = 1; q < NE; ++q) p = e_add(p, acc[q]);
      s[0] = e_sum(p);
    };
#pragma unroll
    for (int q = 0; q < NE; ++q) acc[q] = e_splat<E>(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i].get(f);
      to_elems<V>(f, e);
#pragma unroll
      for (int q = 0; q < NE; ++q) acc[q] = e_add(acc[q], e[q]);
    }
    fold();
    group_sum<G, 1>(s, red[0]);
    const float mu = s[0] * inv;
    const E neg = e_splat<E>(-mu);
#pragma unroll
    for (int q = 0; q < NE; ++q) acc[q] = e_splat<E>(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * G + t) * V < d) {
        v[i].again();
        v[i].get(f);
        to_elems<V>(f, e);
#pragma unroll
        for (int q = 0; q < NE; ++q) {
          const E c = e_add(e[q], neg);
          acc[q] = e_fma(c, c, acc[q]);
        }
      }
    fold();
    group_sum<G, 1>(s, red[1]);
    const float r = rsqrtf(s[0] * inv + a.eps);
    if (!live) continue;
    T* y = (T*)a.y + row * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * G + t) * V;
      if (j >= d) continue;
      float fw[V], fb[V];
      E ew[NE], eb[NE];
      if constexpr (!KEEP) params(i, fw, fb);
      to_elems<V>(KEEP ? pw[KEEP ? i : 0] : fw, ew);
      to_elems<V>(KEEP ? pb[KEEP ? i : 0] : fb, eb);
      v[i].again();
      v[i].get(f);
      to_elems<V>(f, e);
#pragma unroll
      for (int q = 0; q < NE; ++q) e[q] = e_fma(e_mul(e_add(e[q], neg), e_splat<E>(r)), ew[q], eb[q]);
      from_elems<V>(e, f);
      store_v<T, V>(y + j, f);
    }
    if (t == 0 && a.mean) {
      a.mean[row] = mu;
      a.rstd[row] = r;
    }
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(1024) k_ln_fwd_wide(const LnArgs a) {
  __shared__ float red[2][32];
  const unsigned t = threadIdx.x, d = a.d;        // columns are unsigned: they step past a width of up to 2^31 - 1
  const P *w = (const P*)a.w, *b = (const P*)a.b;
  const float inv = 1.f / (float)d;
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.ldx;
    float s[1] = {0.f};
    for (unsigned j = t; j < d; j += 1024) s[0] += to_f(x[j]);
    group_sum<1024, 1>(s, red[0]);
    const float mu = s[0] * inv;
    s[0] = 0.f;
    for (unsigned j = t; j < d; j += 1024) {
      const float c = to_f(x[j]) - mu;
      s[0] += c * c;
    }
    group_sum<1024, 1>(s, red[1]);
    const float r = rsqrtf(s[0] * inv + a.eps);
    T* y = (T*)a.y + row * d;
    for (unsigned j = t; j < d; j += 1024)
      y[j] = from_f<T>(fmaf((to_f(x[j]) - mu) * r, w ? to_f(w[j]) : 1.f, b ? to_f(b[j]) : 0.f));
    if (t == 0 && a.mean) {
      a.mean[row] = mu;
      a.rstd[row] = r;
    }
  }
}

// partial[block][0 .. d) = sum of dy xh, [d .. 2 d) = sum of dy over the block's rows.  RB rows at a time with one
// synchronisation, and the next RB rows' loads in flight meanwhile.
template <typename T, typename P, int G, int NV, int V, int RB>
__global__ void __launch_bounds__(ln_threads<G>, ln_bwd_blocks<G, NV, V>) k_ln_bwd(const LnArgs a) {
  constexpr int TH = ln_threads<G>, RPB = TH / G;
  __shared__ float red[2][TH / 32 * 2 * RB];
  extern __shared__ float cols[];                 // [RPB][2][d] when RPB > 1
  const int t = threadIdx.x % G, g = threadIdx.x / G, d = a.d;
  const P* w = (const P*)a.w;
  using E = Elem<V>;
  constexpr int NE = kElems<V>;
  E pw[NV][NE], aw[NV][NE], ab[NV][NE];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (i * G + t) * V;
    float f[V];
#pragma unroll
    for (int q = 0; q < V; ++q) f[q] = 1.f;
    if (w && j < d) load_p<P, V>(w + j, f);
    to_elems<V>(f, pw[i]);
#pragma unroll
    for (int q = 0; q < NE; ++q) aw[i][q] = ab[i][q] = e_splat<E>(0.f);
  }
  const float inv = 1.f / (float)d;
  Raw<T, V> xv[RB][NV], dv[RB][NV];
  float rs[RB], mu[RB];
  auto fetch = [&](int64_t r0) {
#pragma unroll
    for (int k = 0; k < RB; ++k) {
      const int64_t row = r0 + g * RB + k;
      const bool live = row < a.n;
      const T* x = (const T*)a.x + (live ? row : 0) * a.ldx;
      const T* dy = (const T*)a.dy + (live ? row : 0) * a.lddy;
      rs[k] = live ? a.rstd[row] : 0.f;
      mu[k] = live ? a.mean[row] : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = (i * G + t) * V;
        xv[k][i].zero();
        dv[k][i].zero();
        if (live && j < d) {
          xv[k][i].load(x + j);
          dv[k][i].load(dy + j);
        }
      }
    }
  };
  int buf = 0;
  const int64_t step = (int64_t)gridDim.x * RPB * RB;
  fetch((int64_t)blockIdx.x * RPB * RB);
  for (int64_t r0 = (int64_t)blockIdx.x * RPB * RB; r0 < a.n; r0 += step, buf ^= 1) {
    // xh and up = dy w stay in registers between the sums and dx
    E xh[RB][NV][NE], up[RB][NV][NE];
    float rc[RB], s[2 * RB];
#pragma unroll
    for (int k = 0; k < RB; ++k) {
      rc[k] = rs[k];
      const E neg = e_splat<E>(-mu[k]), r = e_splat<E>(rs[k]);
      E s1[NE], s2[NE];
#pragma unroll
      for (int q = 0; q < NE; ++q) s1[q] = s2[q] = e_splat<E>(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const bool in = (i * G + t) * V < d;
        float f[V];
        E dy[NE];
        xv[k][i].get(f);
        to_elems<V>(f, xh[k][i]);
        dv[k][i].get(f);
        to_elems<V>(f, dy);
#pragma unroll
        for (int q = 0; q < NE; ++q) {
          // dy is 0 beyond the width, so nothing there reaches a sum; x - mu could be anything finite
          xh[k][i][q] = e_mul(e_add(xh[k][i][q], neg), r);
          up[k][i][q] = e_mul(dy[q], pw[i][q]);
          s1[q] = e_add(s1[q], up[k][i][q]);
          if (in) {
            s2[q] = e_fma(up[k][i][q], xh[k][i][q], s2[q]);
            aw[i][q] = e_fma(dy[q], xh[k][i][q], aw[i][q]);
          }
          ab[i][q] = e_add(ab[i][q], dy[q]);
        }
      }
      E p1 = s1[0], p2 = s2[0];
#pragma unroll
      for (int q = 1; q < NE; ++q) p1 = e_add(p1, s1[q]), p2 = e_add(p2, s2[q]);
      s[2 * k] = e_sum(p1);
      s[2 * k + 1] = e_sum(p2);
    }
    if (r0 + step < a.n) fetch(r0 + step);
    group_sum<G, 2 * RB>(s, red[buf]);
    if (a.dx) {
#pragma unroll
      for (int k = 0; k < RB; ++k) {
        const int64_t row = r0 + g * RB + k;
        if (row >= a.n) continue;
        T* dx = (T*)a.dx + row * d;
        const E m1 = e_splat<E>(-s[2 * k] * inv), m2 = e_splat<E>(-s[2 * k + 1] * inv), r = e_splat<E>(rc[k]);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int j = (i * G + t) * V;
          if (j >= d) continue;
          float f[V];
#pragma unroll
          for (int q = 0; q < NE; ++q)
            up[k][i][q] = e_mul(r, e_fma(xh[k][i][q], m2, e_add(up[k][i][q], m1)));
          from_elems<V>(up[k][i], f);
          store_v<T, V>(dx + j, f);
        }
      }
    }
  }
  if (!a.partial) return;
  float* out = a.partial + (int64_t)blockIdx.x * 2 * d;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float fw[V], fb[V];
      from_elems<V>(aw[i], fw);
      from_elems<V>(ab[i], fb);
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const int j = (i * G + t) * V + q;
        if (j < d) {
          out[j] = fw[q];
          out[d + j] = fb[q];
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float fw[V], fb[V];
      from_elems<V>(aw[i], fw);
      from_elems<V>(ab[i], fb);
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const int j = (i * G + t) * V + q;
        if (j < d) {
          cols[(2 * g) * d + j] = fw[q];
          cols[(2 * g + 1) * d + j] = fb[q];
        }
      }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < 2 * d; j += TH) {
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < RPB; ++q) s += cols[q * 2 * d + j];
      out[j] = s;
    }
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(1024) k_ln_bwd_wide(const LnArgs a) {
  __shared__ float red[2][64];
  const unsigned t = threadIdx.x, d = a.d;
  const P* w = (const P*)a.w;
  const float inv = 1.f / (float)d;
  int buf = 0;
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x, buf ^= 1) {
    const T *x = (const T*)a.x + row * a.ldx, *dy = (const T*)a.dy + row * a.lddy;
    const float mu = a.mean[row], r = a.rstd[row];
    float s[2] = {0.f, 0.f};
    for (unsigned j = t; j < d; j += 1024) {
      const float up = to_f(dy[j]) * (w ? to_f(w[j]) : 1.f);
      s[0] += up;
      s[1] += up * ((to_f(x[j]) - mu) * r);
    }
    group_sum<1024, 2>(s, red[buf]);
    T* dx = (T*)a.dx + row * d;
    for (unsigned j = t; j < d; j += 1024)
      dx[j] = from_f<T>(r * (to_f(dy[j]) * (w ? to_f(w[j]) : 1.f) - s[0] * inv - (to_f(x[j]) - mu) * r * s[1] * inv));
  }
}

// dw / db partial sums of wide rows: block (column tile of 128, row split), one column per thread
template <typename T>
__global__ void __launch_bounds__(128) k_ln_cols_wide(const LnArgs a) {
  const unsigned j = blockIdx.x * 128 + threadIdx.x, d = a.d;
  if (j >= d) return;
  float sw = 0.f, sb = 0.f;
  for (int64_t row = blockIdx.y; row < a.n; row += gridDim.y) {
    const float dy = to_f(((const T*)a.dy)[row * a.lddy + j]);
    sw += dy * (to_f(((const T*)a.x)[row * a.ldx + j]) - a.mean[row]) * a.rstd[row];
    sb += dy;
  }
  float* out = a.partial + (int64_t)blockIdx.y * 2 * d;
  out[j] = sw;
  out[(int64_t)d + j] = sb;
}

// Adds the partial sums of the blocks in a fixed order: 32 columns x 32 interleaved sets of partials per block
template <typename P>
__global__ void __launch_bounds__(1024) k_ln_reduce(const float* partial, int nb, int32_t d, P* dw, P* db) {
  __shared__ float red[32][33];
  const int c = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int64_t j = (int64_t)blockIdx.x * 32 + c;
  float s = 0.f;
  if (j < 2 * (int64_t)d) {
    const float* p = partial + j;
#pragma unroll 8
    for (int k = q; k < nb; k += 32) s += p[(int64_t)k * 2 * d];
  }
  red[q][c] = s;
  __syncthreads();
  s = warp_sum(red[c][q]);                        // warp q: column q
  const int64_t o = (int64_t)blockIdx.x * 32 + q;
  if (c == 0) {
    if (o < d) {
      if (dw) dw[o] = from_f<P>(s);
    } else if (o < 2 * (int64_t)d && db) {
      db[o - d] = from_f<P>(s);
    }
  }
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int LN_BLOCKS_PER_SM = 3;              // at most, of the backward kernel: bounds the rows of partial sums

template <typename T, typename P, int G, int NV, int V>
static int ln_fwd_launch(const LnArgs& a, cudaStream_t st) {
  constexpr int RPB = ln_threads<G> / G;
  const int64_t want = (a.n + RPB - 1) / RPB, most = (int64_t)ln_fwd_blocks<G, NV, V> * sm_count();
  k_ln_fwd<T, P, G, NV, V><<<(unsigned)(want < most ? want : most), ln_threads<G>, 0, st>>>(a);
  return check_launch("layer_norm_fwd");
}

template <typename T, typename P>
static int ln_fwd_any(const LnArgs& a, bool vec, cudaStream_t st) {
  constexpr int V = kVec<T>;
  if (vec) {                                      // up to a warp per row and 8 vectors per lane, then 4 and 16 warps
    const int nv = (a.d / V + 31) / 32;
    if (a.d / V <= 8) return ln_fwd_launch<T, P, 8, 1, V>(a, st);
    if (a.d / V <= 16) return ln_fwd_launch<T, P, 16, 1, V>(a, st);
    if (nv <= 1) return ln_fwd_launch<T, P, 32, 1, V>(a, st);
    if (nv <= 2) return ln_fwd_launch<T, P, 32, 2, V>(a, st);
    if (nv <= 4) return ln_fwd_launch<T, P, 32, 4, V>(a, st);
    if (nv <= 8) return ln_fwd_launch<T, P, 32, 8, V>(a, st);
    if (nv <= 32) return ln_fwd_launch<T, P, 128, 8, V>(a, st);
    if (nv <= 128) return ln_fwd_launch<T, P, 512, 8, V>(a, st);
  } else {
    if (a.d <= 128) return ln_fwd_launch<T, P, 32, 4, 1>(a, st);
    if (a.d <= 256) return ln_fwd_launch<T, P, 32, 8, 1>(a, st);
    if (a.d <= 640) return ln_fwd_launch<T, P, 128, 5, 1>(a, st);
    if (a.d <= 1024) return ln_fwd_launch<T, P, 128, 8, 1>(a, st);
    if (a.d <= 2048) return ln_fwd_launch<T, P, 256, 8, 1>(a, st);
    if (a.d <= 4096) return ln_fwd_launch<T, P, 512, 8, 1>(a, st);
    if (a.d <= 8192) return ln_fwd_launch<T, P, 1024, 8, 1>(a, st);
  }
  const int64_t most = (int64_t)2 * sm_count();
  k_ln_fwd_wide<T, P><<<(unsigned)(a.n < most ? a.n : most), 1024, 0, st>>>(a);
  return check_launch("layer_norm_fwd");
}

// Launches and says how many rows of partial sums there are
template <typename T, typename P, int G, int NV, int V, int RB>
static int ln_bwd_launch(const LnArgs& a, int* nb, cudaStream_t st) {
  constexpr int TH = ln_threads<G>, RPB = TH / G;
  const int64_t want = (a.n + RPB * RB - 1) / (RPB * RB), most = (int64_t)ln_bwd_blocks<G, NV, V> * sm_count();
  *nb = (int)(want < most ? want : most);
  const int smem = RPB > 1 && a.partial ? RPB * 2 * a.d * 4 : 0;
  static_assert(RPB == 1 || RPB * 2 * G * NV * V * 4 <= 40 * 1024, "column sums in shared memory");
  k_ln_bwd<T, P, G, NV, V, RB><<<*nb, TH, smem, st>>>(a);
  return check_launch("layer_norm_bwd");
}

template <typename T, typename P>
static int ln_bwd_any(const LnArgs& a, bool vec, int* nb, cudaStream_t st) {
  constexpr int V = kVec<T>;
  if (vec) {
    const int c = a.d / V;
    if (c <= 8) return ln_bwd_launch<T, P, 8, 1, V, 2>(a, nb, st);
    if (c <= 16) return ln_bwd_launch<T, P, 16, 1, V, 2>(a, nb, st);
    if (c <= 32) return ln_bwd_launch<T, P, 32, 1, V, 2>(a, nb, st);
    if (c <= 64) return ln_bwd_launch<T, P, 64, 1, V, 2>(a, nb, st);
    if (c <= 128) return ln_bwd_launch<T, P, 128, 1, V, 2>(a, nb, st);
    if (c <= 256) return ln_bwd_launch<T, P, 256, 1, V, 2>(a, nb, st);
    if (c <= 512) return ln_bwd_launch<T, P, 512, 1, V, 2>(a, nb, st);
    if (c <= 1024) return ln_bwd_launch<T, P, 512, 2, V, 1>(a, nb, st);
  } else {
    if (a.d <= 128) return ln_bwd_launch<T, P, 32, 4, 1, 2>(a, nb, st);
    if (a.d <= 256) return ln_bwd_launch<T, P, 64, 4, 1, 2>(a, nb, st);
    if (a.d <= 640) return ln_bwd_launch<T, P, 128, 5, 1, 2>(a, nb, st);
    if (a.d <= 1024) return ln_bwd_launch<T, P, 256, 4, 1, 2>(a, nb, st);
    if (a.d <= 2048) return ln_bwd_launch<T, P, 512, 4, 1, 2>(a, nb, st);
    if (a.d <= 4096) return ln_bwd_launch<T, P, 512, 8, 1, 1>(a, nb, st);
  }
  const int64_t most = (int64_t)2 * sm_count();
  *nb = (int)(a.n < 64 ? a.n : 64);
  if (a.dx) {
    k_ln_bwd_wide<T, P><<<(unsigned)(a.n < most ? a.n : most), 1024, 0, st>>>(a);
    if (int rc = check_launch("layer_norm_bwd")) return rc;
  }
  if (a.partial) {
    k_ln_cols_wide<T><<<dim3(((unsigned)a.d + 127) / 128, *nb), 128, 0, st>>>(a);
    return check_launch("layer_norm_bwd");
  }
  return 0;
}

int col_sums(const float* partial, int nb, int32_t d, void* dw, void* db, int ptype, cudaStream_t st) {
  const unsigned blocks = (unsigned)((2 * (int64_t)d + 31) / 32);
  if (ptype == MB_F32)
    k_ln_reduce<float><<<blocks, 1024, 0, st>>>(partial, nb, d, (float*)dw, (float*)db);
  else if (ptype == MB_BF16)
    k_ln_reduce<bf16><<<blocks, 1024, 0, st>>>(partial, nb, d, (bf16*)dw, (bf16*)db);
  else
    k_ln_reduce<f16><<<blocks, 1024, 0, st>>>(partial, nb, d, (f16*)dw, (f16*)db);
  return check_launch("norm parameter gradients");
}

template <typename F>
static int ln_types(int dtype, int ptype, const F& f) {
  if (dtype == MB_F32) return f(float(), float());
  if (dtype == MB_BF16) return ptype == MB_F32 ? f(bf16(), float()) : f(bf16(), bf16());
  return ptype == MB_F32 ? f(f16(), float()) : f(f16(), f16());
}

static int ln_check(const char* who, int64_t n, int32_t d, int64_t ldx, int32_t dtype, int32_t ptype) {
  if (n < 0 || d < 1 || ldx < d) {
    set_error("%s: bad sizes (rows %lld, width %d, row stride %lld)", who, (long long)n, d, (long long)ldx);
    return MB_E_ARG;
  }
  if (!dtype_ok(dtype) || (ptype != dtype && ptype != MB_F32)) {
    set_error("%s: unsupported types (x %d, parameters %d)", who, dtype, ptype);
    return MB_E_ARG;
  }
  if (sm_count() < 1) {
    set_error("%s: no CUDA device", who);
    return MB_E_CUDA;
  }
  return 0;
}

// 16-byte accesses: width and strides whole vectors, every address 16-byte aligned
static bool ln_vec(int32_t d, int64_t ldx, int64_t lddy, int dtype, const void* p0, const void* p1, const void* p2,
                   const void* p3, const void* p4) {
  const int v = 16 / dtype_size(dtype);
  return d % v == 0 && ldx % v == 0 && lddy % v == 0 && aligned16(p0) && aligned16(p1) && aligned16(p2) &&
         aligned16(p3) && aligned16(p4);
}

}  // namespace mb

using namespace mb;

extern "C" int mace_b200_layer_norm_fwd(const void* x, int64_t ldx, const void* w, const void* b, void* y, float* mean,
                                        float* rstd, int64_t n, int32_t d, double eps, int32_t dtype, int32_t ptype,
                                        void* stream) {
  if (int rc = ln_check("layer_norm_fwd", n, d, ldx, dtype, ptype)) return rc;
  if (n == 0) return 0;
  if (!x || !y || !mean != !rstd) {
    set_error("layer_norm_fwd: null pointer");
    return MB_E_ARG;
  }
  LnArgs a{};
  a.x = x; a.w = w; a.b = b; a.y = y; a.mean = mean; a.rstd = rstd;
  a.ldx = ldx; a.n = n; a.d = d; a.eps = (float)eps;
  const bool vec = ln_vec(d, ldx, 0, dtype, x, w, b, y, nullptr);
  return ln_types(dtype, ptype, [&](auto t, auto p) {
    return ln_fwd_any<decltype(t), decltype(p)>(a, vec, (cudaStream_t)stream);
  });
}

extern "C" int mace_b200_layer_norm_bwd_workspace(int64_t n, int32_t d, int64_t* floats) {
  if (n < 0 || d < 1 || !floats) {
    set_error("layer_norm_bwd_workspace: bad arguments (rows %lld, width %d)", (long long)n, d);
    return MB_E_ARG;
  }
  const int64_t most = (int64_t)LN_BLOCKS_PER_SM * (sm_count() > 0 ? sm_count() : 1);
  *floats = 2 * (int64_t)d * (n < most ? n : most);
  return 0;
}

extern "C" int mace_b200_layer_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w,
                                        const float* mean, const float* rstd, void* dx, void* dw, void* db,
                                        float* workspace, int64_t n, int32_t d, int32_t dtype, int32_t ptype,
                                        void* stream) {
  if (int rc = ln_check("layer_norm_bwd", n, d, ldx < lddy ? ldx : lddy, dtype, ptype)) return rc;
  if (n > 0 && (!dy || !x || !mean || !rstd || ((dw || db) && !workspace))) {
    set_error("layer_norm_bwd: null pointer");
    return MB_E_ARG;
  }
  LnArgs a{};
  a.x = x; a.dy = dy; a.w = w; a.dx = dx; a.mean = (float*)mean; a.rstd = (float*)rstd;
  a.partial = (dw || db) ? workspace : nullptr;
  a.ldx = ldx; a.lddy = lddy; a.n = n; a.d = d;
  const bool vec = ln_vec(d, ldx, lddy, dtype, x, dy, w, dx, nullptr);
  return ln_types(dtype, ptype, [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    int nb = 0;
    if (n > 0)
      if (int rc = ln_bwd_any<T, P>(a, vec, &nb, (cudaStream_t)stream)) return rc;
    if (!dw && !db) return 0;
    return col_sums(workspace, nb, d, dw, db, ptype, (cudaStream_t)stream);
  });
}
