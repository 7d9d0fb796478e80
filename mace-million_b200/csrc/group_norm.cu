// Group norm with an activation, channels last: a sample is a run of rows [C], its channels are `groups` runs of C / groups.
//   mu, var over the rows and channels of a group, r = 1 / sqrt(var + eps), xh = (x - mu) r, z = xh w + b, y = f(z)
// and its backward pass, with dz = dy f'(z) and a = dz w:
//   dx = r (a - mean(a) - xh mean(a xh)), dw = sum over rows of dz xh, db = sum over rows of dz.
// f: identity, silu z s(z), gelu z Phi(z) or relu.  Statistics and sums are fp32; every output is rounded once.
//
// Bound: HBM bytes (forward x and y, backward x, dy and dx, each once).  A cluster of P CTAs and a block of whole groups own a
// sample's rows of those columns: a CTA keeps its rows in shared memory between the sums and the output, exchanges sums of
// its groups with the cluster through distributed shared memory, and no row is read twice while P CTAs hold them.  Rows beyond
// that are read again, last ones first, as L2 has those.
// A thread owns V channels of one group (16 bytes, or what divides a group) and every TR-th row, and takes its sums relative to
// its own first row: of one thread's few hundred rows they lose at most that number of fp32 roundings, whatever the mean.
// Threads, CTAs and clusters are joined as (count, mean, sum of squared deviations), so nothing cancels.  No atomics: parameter
// gradients are added up over a CTA's samples in registers, then over CTAs by a second small kernel in a fixed order.
#include "dtypes.cuh"
#include "norm.cuh"
#include "tc.cuh"

namespace mb {

struct GnArgs {
  const void *x, *dy, *w, *b;
  void* out;                                      // y, or dx (null: parameter gradients only)
  float *mean, *rstd, *partial;                   // partial [cluster rows][2][C]: sums of dz xh, of dz (null: none)
  const void* off;                                // [n + 1], null: samples of `len` rows
  int64_t ldx, lddy, rows, n, len;
  int32_t c, groups, cg, gpb, act, off64, p32, cap;   // gpb: groups of a column block; cap: row steps kept in shared memory
  float eps;
};

// Rows of a sample; false: the offsets descend or leave the rows there
__device__ __forceinline__ bool gn_range(const GnArgs& a, int64_t s, int64_t& lo, int64_t& hi) {
  if (!a.off) {
    lo = s * a.len;
    hi = lo + a.len;
    return true;
  }
  auto at = [&](int64_t i) { return a.off64 ? ((const int64_t*)a.off)[i] : (int64_t)((const int32_t*)a.off)[i]; };
  const int64_t u = at(s), v = at(s + 1), before = s ? at(s - 1) : 0;
  lo = u < 0 ? 0 : u < a.rows ? u : a.rows;
  hi = v < lo ? lo : v < a.rows ? v : a.rows;
  return u >= before && v >= u && v <= a.rows;
}

// Rows outside of all samples are zero
template <typename T>
__device__ __forceinline__ void gn_clear(const GnArgs& a) {
  if (!a.off || !a.out) return;
  auto at = [&](int64_t i) {
    const int64_t v = a.off64 ? ((const int64_t*)a.off)[i] : (int64_t)((const int32_t*)a.off)[i];
    return v < 0 ? 0 : v < a.rows ? v : a.rows;
  };
  const int64_t head = a.n ? at(0) : a.rows, tail = a.n ? at(a.n) : a.rows;
  const int64_t id = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
  const int64_t step = (int64_t)gridDim.x * gridDim.y * gridDim.z * blockDim.x;
  T* out = (T*)a.out;
  for (int64_t i = id * blockDim.x + threadIdx.x; i < head * a.c; i += step) out[i] = from_f<T>(0.f);
  for (int64_t i = tail * a.c + id * blockDim.x + threadIdx.x; i < a.rows * a.c; i += step) out[i] = from_f<T>(0.f);
}

// V consecutive elements of T as one access of 16, 8 or sizeof(T) bytes
template <typename T, int V>
struct GnVec {
  using Word = std::conditional_t<V == 1, T, std::conditional_t<V * sizeof(T) == 8, uint2, uint4>>;
  Word u;
  __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const Word*>(p); }
  __device__ __forceinline__ void get(float (&f)[V]) const {
    if constexpr (V == 1) {
      f[0] = to_f(u);
    } else if constexpr (V * sizeof(T) == 16) {
      unpack16(u, f, T());
    } else if constexpr (sizeof(T) == 4) {
      f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y);
    } else {
      float g[8];
      unpack16(make_uint4(u.x, u.y, 0u, 0u), g, T());
#pragma unroll
      for (int q = 0; q < 4; ++q) f[q] = g[q];
    }
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
    if constexpr (V == 1) {
      u = from_f<T>(f[0]);
    } else if constexpr (V * sizeof(T) == 16) {
      u = pack16<T>(f);
    } else if constexpr (sizeof(T) == 4) {
      u = make_uint2(__float_as_uint(f[0]), __float_as_uint(f[1]));
    } else {
      u = make_uint2(pack2(f[0], f[1], T()), pack2(f[2], f[3], T()));
    }
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Word*>(p) = u; }
};

// f(z) and f'(z).  16-bit results take the fast exponential (2 ulp of fp32 and |z| 2^-24).
template <typename T>
__device__ __forceinline__ float gn_exp(float v) {
  if constexpr (sizeof(T) == 4) return expf(v);
  return __expf(v);
}
template <typename T>
__device__ __forceinline__ float gn_sigmoid(float z) {
  if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-z));
  return __fdividef(1.f, 1.f + __expf(-z));       // 0 where the exponential is above 2^126
}
template <typename T, int V>
__device__ __forceinline__ void gn_act(float (&z)[V], int act) {
  if (act == MB_ACT_SILU) {
#pragma unroll
    for (int q = 0; q < V; ++q) z[q] *= gn_sigmoid<T>(z[q]);
  } else if (act == MB_ACT_GELU) {
#pragma unroll
    for (int q = 0; q < V; ++q) z[q] *= normcdff(z[q]);
  } else if (act == MB_ACT_RELU) {
#pragma unroll
    for (int q = 0; q < V; ++q) z[q] = z[q] < 0.f ? 0.f : z[q];   // NaN stays
  }
}
template <typename T, int V>
__device__ __forceinline__ void gn_act_grad(const float (&z)[V], float (&d)[V], int act) {   // d *= f'(z)
  if (act == MB_ACT_SILU) {
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const float s = gn_sigmoid<T>(z[q]);
      d[q] *= s * fmaf(z[q], 1.f - s, 1.f);
    }
  } else if (act == MB_ACT_GELU) {
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const float pdf = 0.3989422804014327f * gn_exp<T>(-0.5f * z[q] * z[q]);
      d[q] *= fmaf(z[q], pdf, normcdff(z[q]));
    }
  } else if (act == MB_ACT_RELU) {
#pragma unroll
    for (int q = 0; q < V; ++q) d[q] = z[q] <= 0.f ? 0.f : d[q];
  }
}

// V parameters, fp32 or of type T
template <typename T, int V>
__device__ __forceinline__ void gn_param(const void* p, int32_t p32, int c, float other, float (&f)[V]) {
#pragma unroll
  for (int q = 0; q < V; ++q) f[q] = !p ? other : p32 ? ((const float*)p)[c + q] : to_f(((const T*)p)[c + q]);
}

// How a thread of a CTA walks over the CTA's rows and columns
struct GnWalk {
  int g0, ng, c0, nvec, tc, tr, r, col, tiles;
  bool on;
};
template <int V>
__device__ __forceinline__ GnWalk gn_walk(const GnArgs& a) {
  GnWalk k;
  k.g0 = blockIdx.y * a.gpb;
  k.ng = a.groups - k.g0 < a.gpb ? a.groups - k.g0 : a.gpb;
  k.c0 = k.g0 * a.cg;
  k.nvec = k.ng * a.cg / V;
  const int th = blockDim.x;
  k.tc = k.nvec < th ? k.nvec : th;
  k.tr = th / k.tc;
  k.r = threadIdx.x / k.tc;
  k.col = threadIdx.x - k.r * k.tc;
  k.tiles = (k.nvec + k.tc - 1) / k.tc;
  k.on = k.r < k.tr;
  return k;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) { return __int_as_float(ld_cluster_s32(addr)); }

// Sum over the 8 lanes of an octet
__device__ __forceinline__ float octet_sum(float v) {
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Shared memory: red [threads] pairs | grp [2][3][gpb] (by parity of the sample: what this CTA found) | fin [2][gpb] | kept rows
__device__ __forceinline__ size_t gn_shared_floats(int threads, int gpb) { return 2 * (size_t)threads + 8 * (size_t)gpb; }

template <typename T, int V>
__global__ void __launch_bounds__(512, 2) k_gn_fwd(const GnArgs a) {
  constexpr int U = 4;
  extern __shared__ __align__(16) float gn_smem[];
  const GnWalk k = gn_walk<V>(a);
  const int th = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = th >> 5;
  const int P = gridDim.x, rank = blockIdx.x;
  float2* red = reinterpret_cast<float2*>(gn_smem);
  float* grp0 = gn_smem + 2 * th;
  float* fin = grp0 + 6 * a.gpb;
  using Vec = GnVec<T, V>;
  Vec* kept = reinterpret_cast<Vec*>(gn_smem + ((gn_shared_floats(th, a.gpb) + 3) & ~(size_t)3)) + threadIdx.x;
  const int cgv = a.cg / V;
  gn_clear<T>(a);
  int par = 0;
  for (int64_t s = blockIdx.z; s < a.n; s += gridDim.z, par ^= 1) {
    int64_t lo, hi;
    const bool good = gn_range(a, s, lo, hi);
    const int64_t len = hi - lo, r0 = lo + len * rank / P, nr = lo + len * (rank + 1) / P - r0;
    float* grp = grp0 + par * 3 * a.gpb;
    for (int g = threadIdx.x; g < 3 * k.ng; g += th) grp[g / k.ng * a.gpb + g % k.ng] = 0.f;
    const int64_t mine = k.on && nr > k.r ? (nr - k.r + k.tr - 1) / k.tr : 0;   // rows of this thread
    // ---------------------------------------------------------------------------------------- sums
    for (int t = 0; t < k.tiles; ++t) {
      const int v0 = t * k.tc, cv = v0 + k.col;
      const bool on = cv < k.nvec;
      const T* x = (const T*)a.x + (r0 + k.r) * a.ldx + k.c0 + cv * V;
      const int64_t step = (int64_t)k.tr * a.ldx;
      float piv[V], s1[V], s2[V];
#pragma unroll
      for (int q = 0; q < V; ++q) piv[q] = s1[q] = s2[q] = 0.f;
      if (on && mine > 0) {
        Vec v;
        v.load(x);
        v.get(piv);
        auto add = [&](const Vec& u, int64_t i) {
          float f[V];
          const int64_t at = i * k.tiles + t;
          if (at < a.cap) kept[at * th] = u;
          u.get(f);
#pragma unroll
          for (int q = 0; q < V; ++q) {
            const float e = f[q] - piv[q];
            s1[q] += e;
            s2[q] = fmaf(e, e, s2[q]);
          }
        };
        int64_t i = 0;
        for (; i + U <= mine; i += U) {
          Vec u[U];
#pragma unroll
          for (int j = 0; j < U; ++j) u[j].load(x + (i + j) * step);
#pragma unroll
          for (int j = 0; j < U; ++j) add(u[j], i + j);
        }
        for (; i < mine; ++i) {
          Vec u;
          u.load(x + i * step);
          add(u, i);
        }
      }
      // V channels to (mean, squared deviations) of mine * V values
      float mu = 0.f, m2 = 0.f;
      if (on && mine > 0) {
        const float inv = 1.f / (float)mine;
        float m[V];
#pragma unroll
        for (int q = 0; q < V; ++q) {
          const float d = s1[q] * inv;
          m[q] = piv[q] + d;
          mu += m[q];
          m2 += fmaxf(fmaf(-s1[q], d, s2[q]), 0.f * s2[q]);   // not below 0, NaN stays
        }
        mu *= 1.f / (float)V;
#pragma unroll
        for (int q = 0; q < V; ++q) m2 = fmaf((m[q] - mu) * (m[q] - mu), (float)mine, m2);
      }
      __syncthreads();                            // red is free (and grp is zero)
      red[threadIdx.x] = make_float2(mu, m2);
      __syncthreads();
      for (int g = warp; g < k.ng; g += warps) {
        const int a0 = g * cgv - v0 > 0 ? g * cgv - v0 : 0, a1 = (g + 1) * cgv - v0;
        const int w = (a1 < k.nvec - v0 ? (a1 < k.tc ? a1 : k.tc) : (k.nvec - v0 < k.tc ? k.nvec - v0 : k.tc)) - a0;
        if (w <= 0) continue;
        const int entries = w * k.tr;
        const float cnt = (float)nr * (float)(w * V);
        float sum = 0.f, dev = 0.f;
        for (int e = lane; e < entries; e += 32) {
          const int r = e / w, n = nr > r ? (int)((nr - r + k.tr - 1) / k.tr) : 0;
          sum = fmaf((float)n, red[r * k.tc + a0 + (e - r * w)].x, sum);
        }
        sum = warp_sum(sum) * (float)V;
        const float mean = cnt > 0.f ? sum / cnt : 0.f;
        for (int e = lane; e < entries; e += 32) {
          const int r = e / w, n = nr > r ? (int)((nr - r + k.tr - 1) / k.tr) : 0;
          const float2 v = red[r * k.tc + a0 + (e - r * w)];
          if (n > 0) dev += fmaf((v.x - mean) * (v.x - mean), (float)(n * V), v.y);
        }
        dev = warp_sum(dev);
        if (lane == 0 && cnt > 0.f) {             // join with the tiles before
          const float c0 = grp[g], m0 = grp[a.gpb + g], n1 = c0 + cnt, d = mean - m0;
          grp[g] = n1;
          grp[a.gpb + g] = fmaf(d, cnt / n1, m0);
          grp[2 * a.gpb + g] += fmaf(d * d, c0 * (cnt / n1), dev);
        }
      }
    }
    if (P > 1)
      cluster_sync();
    else
      __syncthreads();
    // ---------------------------------------------------------------------------------------- statistics of the cluster
    for (int g = threadIdx.x >> 3; g < (k.ng + 3) / 4 * 4; g += th >> 3) {
      const int q = threadIdx.x & 7, gg = g < k.ng ? g : k.ng - 1;
      float cnt = 0.f, m = 0.f, m2 = 0.f;
      if (q < P) {
        if (P > 1) {
          const uint32_t at = mapa_u32(smem_u32(grp + gg), q);
          cnt = ld_cluster_f32(at);
          m = ld_cluster_f32(at + 4 * a.gpb);
          m2 = ld_cluster_f32(at + 8 * a.gpb);
        } else {
          cnt = grp[gg], m = grp[a.gpb + gg], m2 = grp[2 * a.gpb + gg];
        }
      }
      const float n = octet_sum(cnt), mean = n > 0.f ? octet_sum(cnt * m) / n : 0.f;
      const float d = m - mean;
      m2 = octet_sum(cnt > 0.f ? fmaf(d * d, cnt, m2) : 0.f);
      if (q == 0 && g < k.ng) {
        const float bad = good ? 0.f : __int_as_float(0x7fc00000);
        const float rs = rsqrtf((n > 0.f ? m2 / n : 0.f) + a.eps) + bad;
        fin[2 * g] = mean + bad;
        fin[2 * g + 1] = rs;
        if (a.mean && rank == 0) {
          a.mean[s * a.groups + k.g0 + g] = mean + bad;
          a.rstd[s * a.groups + k.g0 + g] = rs;
        }
      }
    }
    __syncthreads();
    // ---------------------------------------------------------------------------------------- outputs
    for (int t = 0; t < k.tiles; ++t) {
      const int cv = t * k.tc + k.col;
      if (cv >= k.nvec || mine == 0) continue;
      const int c = k.c0 + cv * V, g = cv / cgv;
      float w[V], b[V];
      gn_param<T, V>(a.w, a.p32, c, 1.f, w);
      gn_param<T, V>(a.b, a.p32, c, 0.f, b);
      const float mean = fin[2 * g], rs = fin[2 * g + 1];
#pragma unroll
      for (int q = 0; q < V; ++q) w[q] *= rs;
      const T* x = (const T*)a.x + (r0 + k.r) * a.ldx + c;
      T* y = (T*)a.out + (r0 + k.r) * (int64_t)a.c + c;
      const int64_t step = (int64_t)k.tr * a.ldx, ystep = (int64_t)k.tr * a.c;
      auto put = [&](Vec v, int64_t i) {
        float f[V];
        v.get(f);
#pragma unroll
        for (int q = 0; q < V; ++q) f[q] = fmaf(f[q] - mean, w[q], b[q]);
        gn_act<T, V>(f, a.act);
        v.set(f);
        v.store(y + i * ystep);
      };
      const int64_t have = a.cap > t ? (a.cap - t + k.tiles - 1) / k.tiles : 0;   // rows kept
      int64_t i = mine - 1;
      for (; i >= have + U - 1; i -= U) {
        Vec u[U];
#pragma unroll
        for (int j = 0; j < U; ++j) u[j].load(x + (i - j) * step);
#pragma unroll
        for (int j = 0; j < U; ++j) put(u[j], i - j);
      }
      for (; i >= have; --i) {
        Vec u;
        u.load(x + i * step);
        put(u, i);
      }
#pragma unroll 2
      for (; i >= 0; --i) put(kept[(i * k.tiles + t) * th], i);
    }
  }
  if (P > 1) cluster_sync();                      // no CTA leaves while its peers may read its sums
}

template <typename T, int V>
__global__ void __launch_bounds__(256, 2) k_gn_bwd(const GnArgs a) {
  constexpr int U = 2;
  extern __shared__ __align__(16) float gn_smem[];
  const GnWalk k = gn_walk<V>(a);
  const int th = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = th >> 5;
  const int P = gridDim.x, rank = blockIdx.x;
  float2* red = reinterpret_cast<float2*>(gn_smem);
  float* grp0 = gn_smem + 2 * th;
  float* fin = grp0 + 6 * a.gpb;
  using Vec = GnVec<T, V>;
  Vec* kept = reinterpret_cast<Vec*>(gn_smem + ((gn_shared_floats(th, a.gpb) + 3) & ~(size_t)3)) + threadIdx.x;
  const int cgv = a.cg / V;
  gn_clear<T>(a);
  float tw[V], tb[V];                             // sums of dz xh and dz over the samples (one tile of columns)
#pragma unroll
  for (int q = 0; q < V; ++q) tw[q] = tb[q] = 0.f;
  float* part = a.partial ? a.partial + ((int64_t)blockIdx.z * P + rank) * 2 * a.c : nullptr;
  int par = 0;
  bool first = true;
  for (int64_t s = blockIdx.z; s < a.n; s += gridDim.z, par ^= 1, first = false) {
    int64_t lo, hi;
    gn_range(a, s, lo, hi);
    const int64_t len = hi - lo, r0 = lo + len * rank / P, nr = lo + len * (rank + 1) / P - r0;
    float* grp = grp0 + par * 3 * a.gpb;
    for (int g = threadIdx.x; g < 2 * k.ng; g += th) grp[g / k.ng * a.gpb + g % k.ng] = 0.f;
    const int64_t mine = k.on && nr > k.r ? (nr - k.r + k.tr - 1) / k.tr : 0;
    const int64_t xstep = (int64_t)k.tr * a.ldx, dstep = (int64_t)k.tr * a.lddy, ostep = (int64_t)k.tr * a.c;
    // ---------------------------------------------------------------------------------------- sums
    for (int t = 0; t < k.tiles; ++t) {
      const int v0 = t * k.tc, cv = v0 + k.col;
      const bool on = cv < k.nvec && mine > 0;
      const int c = k.c0 + cv * V;
      float sw[V], sb[V], s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int q = 0; q < V; ++q) sw[q] = sb[q] = 0.f;
      if (on) {
        float w[V], b[V];
        gn_param<T, V>(a.w, a.p32, c, 1.f, w);
        gn_param<T, V>(a.b, a.p32, c, 0.f, b);
        const int64_t st = s * a.groups + k.g0 + cv / cgv;
        const float mean = a.mean[st], rs = a.rstd[st];
        const T* x = (const T*)a.x + (r0 + k.r) * a.ldx + c;
        const T* dy = (const T*)a.dy + (r0 + k.r) * a.lddy + c;
        auto add = [&](const Vec& u, const Vec& v, int64_t i) {
          const int64_t at = i * k.tiles + t;
          if (at < a.cap) {
            kept[2 * at * th] = u;
            kept[(2 * at + 1) * th] = v;
          }
          float f[V], d[V], z[V];
          u.get(f);
          v.get(d);
#pragma unroll
          for (int q = 0; q < V; ++q) {
            f[q] = (f[q] - mean) * rs;
            z[q] = fmaf(f[q], w[q], b[q]);
          }
          gn_act_grad<T, V>(z, d, a.act);
#pragma unroll
          for (int q = 0; q < V; ++q) {
            sw[q] = fmaf(d[q], f[q], sw[q]);
            sb[q] += d[q];
          }
        };
        int64_t i = 0;
        for (; i + U <= mine; i += U) {
          Vec u[U], v[U];
#pragma unroll
          for (int j = 0; j < U; ++j) u[j].load(x + (i + j) * xstep), v[j].load(dy + (i + j) * dstep);
#pragma unroll
          for (int j = 0; j < U; ++j) add(u[j], v[j], i + j);
        }
        for (; i < mine; ++i) {
          Vec u, v;
          u.load(x + i * xstep);
          v.load(dy + i * dstep);
          add(u, v, i);
        }
#pragma unroll
        for (int q = 0; q < V; ++q) {
          s1 = fmaf(w[q], sb[q], s1);
          s2 = fmaf(w[q], sw[q], s2);
          tw[q] += sw[q];
          tb[q] += sb[q];
        }
      }
      if (k.tiles > 1 && part && cv < k.nvec)      // one thread a column: its sums of all samples lie in memory
#pragma unroll
        for (int q = 0; q < V; ++q) {
          part[c + q] = first ? sw[q] : part[c + q] + sw[q];
          part[a.c + c + q] = first ? sb[q] : part[a.c + c + q] + sb[q];
        }
      __syncthreads();                            // red is free (and grp is zero)
      red[threadIdx.x] = make_float2(s1, s2);
      __syncthreads();
      for (int g = warp; g < k.ng; g += warps) {
        const int a0 = g * cgv - v0 > 0 ? g * cgv - v0 : 0, a1 = (g + 1) * cgv - v0;
        const int w = (a1 < k.nvec - v0 ? (a1 < k.tc ? a1 : k.tc) : (k.nvec - v0 < k.tc ? k.nvec - v0 : k.tc)) - a0;
        if (w <= 0) continue;
        float u = 0.f, v = 0.f;
        for (int e = lane; e < w * k.tr; e += 32) {
          const int r = e / w;
          const float2 p = red[r * k.tc + a0 + (e - r * w)];
          u += p.x;
          v += p.y;
        }
        u = warp_sum(u);
        v = warp_sum(v);
        if (lane == 0) {
          grp[g] += u;
          grp[a.gpb + g] += v;
        }
      }
    }
    if (!a.out) continue;
    if (P > 1)
      cluster_sync();
    else
      __syncthreads();
    const float inv = 1.f / ((float)len * (float)a.cg);
    for (int g = threadIdx.x >> 3; g < (k.ng + 3) / 4 * 4; g += th >> 3) {
      const int q = threadIdx.x & 7, gg = g < k.ng ? g : k.ng - 1;
      float u = 0.f, v = 0.f;
      if (q < P) {
        if (P > 1) {
          const uint32_t at = mapa_u32(smem_u32(grp + gg), q);
          u = ld_cluster_f32(at);
          v = ld_cluster_f32(at + 4 * a.gpb);
        } else {
          u = grp[gg], v = grp[a.gpb + gg];
        }
      }
      u = octet_sum(u);
      v = octet_sum(v);
      if (q == 0 && g < k.ng) {
        fin[2 * g] = u * inv;
        fin[2 * g + 1] = v * inv;
      }
    }
    __syncthreads();
    // ---------------------------------------------------------------------------------------- dx
    for (int t = 0; t < k.tiles; ++t) {
      const int cv = t * k.tc + k.col;
      if (cv >= k.nvec || mine == 0) continue;
      const int c = k.c0 + cv * V, g = cv / cgv;
      float w[V], b[V];
      gn_param<T, V>(a.w, a.p32, c, 1.f, w);
      gn_param<T, V>(a.b, a.p32, c, 0.f, b);
      const int64_t st = s * a.groups + k.g0 + g;
      const float mean = a.mean[st], rs = a.rstd[st], m1 = fin[2 * g], m2 = fin[2 * g + 1];
      const T* x = (const T*)a.x + (r0 + k.r) * a.ldx + c;
      const T* dy = (const T*)a.dy + (r0 + k.r) * a.lddy + c;
      T* dx = (T*)a.out + (r0 + k.r) * (int64_t)a.c + c;
      auto put = [&](Vec u, const Vec& v, int64_t i) {
        float f[V], d[V], z[V];
        u.get(f);
        v.get(d);
#pragma unroll
        for (int q = 0; q < V; ++q) {
          f[q] = (f[q] - mean) * rs;
          z[q] = fmaf(f[q], w[q], b[q]);
        }
        gn_act_grad<T, V>(z, d, a.act);
#pragma unroll
        for (int q = 0; q < V; ++q) f[q] = rs * (fmaf(d[q], w[q], -m1) - f[q] * m2);
        u.set(f);
        u.store(dx + i * ostep);
      };
      const int64_t have = a.cap > t ? (a.cap - t + k.tiles - 1) / k.tiles : 0;
      int64_t i = mine - 1;
      for (; i >= have + U - 1; i -= U) {
        Vec u[U], v[U];
#pragma unroll
        for (int j = 0; j < U; ++j) u[j].load(x + (i - j) * xstep), v[j].load(dy + (i - j) * dstep);
#pragma unroll
        for (int j = 0; j < U; ++j) put(u[j], v[j], i - j);
      }
      for (; i >= have; --i) {
        Vec u, v;
        u.load(x + i * xstep);
        v.load(dy + i * dstep);
        put(u, v, i);
      }
      for (; i >= 0; --i) {
        const int64_t at = i * k.tiles + t;
        put(kept[2 * at * th], kept[(2 * at + 1) * th], i);
      }
    }
  }
  if (part && k.tiles == 1) {                     // over the rows of threads, in their order
    float* cols = gn_smem;                        // [th] at a time
#pragma unroll
    for (int q = 0; q < 2 * V; ++q) {
      __syncthreads();
      cols[threadIdx.x] = q < V ? tw[q < V ? q : 0] : tb[q < V ? 0 : q - V];
      __syncthreads();
      if (k.on && k.r == 0) {
        float v = 0.f;
        for (int r = 0; r < k.tr; ++r) v += cols[r * k.tc + k.col];
        part[(q < V ? 0 : a.c) + k.c0 + k.col * V + (q < V ? q : q - V)] = v;
      }
    }
  }
  if (P > 1) cluster_sync();
}

// ------------------------------------------------------------------------------------------------ host side
// How a call is cut: column blocks of whole groups, CTAs of a cluster, threads, row steps in shared memory, clusters in flight
struct GnCut {
  int gpb, ncb, p, th, cap, smem;
  int64_t nz;
};

// Row segments of a column block are 64 bytes at least (two sectors).  A CTA keeps up to GN_KEEP bytes, so that two fit an SM and
// one loads while the other stores; a sample takes as many CTAs as hold it, and while the GPU is not full, more, down to 8 KB each.
constexpr int GN_KEEP = 96 * 1024;
template <int V>
static GnCut gn_cut(const GnArgs& a, int size, int slabs, int threads_max) {
  GnCut k{};
  const int64_t rows = a.off ? (a.n ? (a.rows + a.n - 1) / a.n : 0) : a.len;
  const int64_t bytes = rows * a.c * size * slabs, sms = sm_count();
  int64_t want = (bytes + GN_KEEP - 1) / GN_KEEP;
  const int64_t fill = (2 * sms + a.n - 1) / a.n, least = bytes / 8192;
  if (want < (fill < least ? fill : least)) want = fill < least ? fill : least;
  if (want < 1) want = 1;
  const int gmin = (64 + a.cg * size - 1) / (a.cg * size);      // groups of the narrowest block
  int64_t ncb = a.groups / gmin < want ? a.groups / gmin : want;
  if (ncb < 1) ncb = 1;
  k.gpb = (int)((a.groups + ncb - 1) / ncb);
  // the per-group words of a block stay below 32 KB
  if (k.gpb > 1024) k.gpb = 1024;
  k.ncb = (a.groups + k.gpb - 1) / k.gpb;
  k.p = 1;
  while (k.p < 8 && (int64_t)k.p * k.ncb < want && rows >= 2 * k.p) k.p *= 2;
  const int64_t slab = (rows + k.p - 1) / k.p * k.gpb * a.cg * size * slabs;
  const int nvec = k.gpb * a.cg / V, acc = V * size;
  k.th = slab <= 8192 ? 128 : slab <= 32768 ? 256 : threads_max;
  while (k.th < threads_max && k.th < nvec && nvec > 128) k.th *= 2;
  const int tiles = (nvec + k.th - 1) / k.th, tr = nvec < k.th ? k.th / nvec : 1;
  const int64_t steps = ((rows + k.p - 1) / k.p + tr - 1) / tr * tiles;
  const int per = k.th * acc * slabs, most = GN_KEEP / per;
  k.cap = (int)(steps < most ? steps : most);
  k.smem = (int)((((2 * (size_t)k.th + 8 * (size_t)k.gpb + 3) & ~(size_t)3) * 4) + (size_t)k.cap * per);
  return k;
}

template <auto KERN>
static int gn_launch(GnArgs& a, GnCut& k, cudaStream_t st, const char* what) {
  static int ready_dev = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return check_launch(what);
  if (ready_dev != dev) {
    if (cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != cudaSuccess) {
      set_error("%s: cannot reserve shared memory", what);
      return MB_E_CUDA;
    }
    ready_dev = dev;
  }
  a.gpb = k.gpb;
  a.cap = k.cap;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(k.p, k.ncb, (unsigned)k.nz);
  cfg.blockDim = dim3(k.th);
  cfg.dynamicSmemBytes = k.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = k.p;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = k.p > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, KERN, a);
  return check_launch(what);
}

// Clusters in flight: what threads (registers) and shared memory let be resident, and no more than there are samples
static int64_t gn_depth(const GnArgs& a, const GnCut& k, int threads_sm) {
  int per = threads_sm / k.th;
  const int by_smem = (220 * 1024) / (k.smem + 1024);
  if (by_smem < per) per = by_smem;
  if (per < 1) per = 1;
  const int64_t ctas = (int64_t)k.p * k.ncb, z = ((int64_t)per * sm_count() + ctas - 1) / ctas;
  return z < a.n ? z : a.n;
}

// Elements of an access: 16 or 8 bytes where they divide a group and everything is aligned to them, else one
static int gn_vec(const GnArgs& a, int size) {
  for (int bytes = 16; bytes >= 8; bytes /= 2) {
    const int v = bytes / size;
    const uintptr_t p = (uintptr_t)a.x | (uintptr_t)a.dy | (uintptr_t)a.out;
    if (a.cg % v == 0 && a.ldx % v == 0 && a.lddy % v == 0 && p % bytes == 0) return v;
  }
  return 1;
}

constexpr int GN_FWD_THREADS = 512, GN_FWD_SM = 1024, GN_BWD_THREADS = 256, GN_BWD_SM = 512;

template <typename T, int V>
static int gn_fwd_go(GnArgs& a, cudaStream_t st) {
  GnCut k = gn_cut<V>(a, sizeof(T), 1, GN_FWD_THREADS);
  k.nz = gn_depth(a, k, GN_FWD_SM);
  if (k.nz < 1) k.nz = 1;
  return gn_launch<k_gn_fwd<T, V>>(a, k, st, "group_norm_fwd");
}
template <typename T>
static int gn_fwd_any(GnArgs& a, cudaStream_t st) {
  const int v = gn_vec(a, sizeof(T));
  if (v == 16 / (int)sizeof(T)) return gn_fwd_go<T, 16 / sizeof(T)>(a, st);
  return v > 1 ? gn_fwd_go<T, 8 / sizeof(T)>(a, st) : gn_fwd_go<T, 1>(a, st);
}
template <typename T, int V>
static int gn_bwd_go(GnArgs& a, int64_t* parts, bool launch, cudaStream_t st) {
  GnCut k = gn_cut<V>(a, sizeof(T), 2, GN_BWD_THREADS);
  k.nz = gn_depth(a, k, GN_BWD_SM);
  if (k.nz < 1) k.nz = 1;
  *parts = k.nz * k.p;
  return launch ? gn_launch<k_gn_bwd<T, V>>(a, k, st, "group_norm_bwd") : 0;
}
template <typename T>
static int gn_bwd_any(GnArgs& a, int64_t* parts, bool launch, cudaStream_t st) {
  const int v = gn_vec(a, sizeof(T));
  if (v == 16 / (int)sizeof(T)) return gn_bwd_go<T, 16 / sizeof(T)>(a, parts, launch, st);
  return v > 1 ? gn_bwd_go<T, 8 / sizeof(T)>(a, parts, launch, st) : gn_bwd_go<T, 1>(a, parts, launch, st);
}

static int gn_check(const char* who, const GnArgs& a, int32_t dtype, int32_t ptype) {
  if (a.rows < 0 || a.n < 0 || a.c < 1 || a.groups < 1 || a.c % a.groups || a.ldx < a.c ||
      (!a.off && (a.len < 0 || (a.n && a.rows / a.n != a.len) || a.rows != a.n * a.len))) {
    set_error("%s: bad sizes (rows %lld, samples %lld of %lld, channels %d, groups %d, row stride %lld)", who, (long long)a.rows,
              (long long)a.n, (long long)a.len, a.c, a.groups, (long long)a.ldx);
    return MB_E_ARG;
  }
  if (!dtype_ok(dtype) || (ptype != dtype && ptype != MB_F32)) {
    set_error("%s: unsupported types (x %d, parameters %d)", who, dtype, ptype);
    return MB_E_ARG;
  }
  if (a.act < MB_ACT_NONE || a.act > MB_ACT_RELU) {
    set_error("%s: unknown activation %d", who, a.act);
    return MB_E_ARG;
  }
  return 0;
}

static GnArgs gn_args(const void* x, int64_t ldx, const void* w, const void* b, const void* offsets, int32_t off64, int64_t rows,
                      int64_t n, int64_t len, int32_t c, int32_t groups, int32_t act, int32_t ptype) {
  GnArgs a{};
  a.x = x; a.w = w; a.b = b; a.off = offsets; a.off64 = off64;
  a.ldx = ldx; a.rows = rows; a.n = n; a.len = len; a.c = c; a.groups = groups; a.act = act;
  a.cg = groups > 0 ? c / groups : 0;
  a.p32 = ptype == MB_F32;
  return a;
}

template <typename F>
static int gn_type(int dtype, const F& f) {
  return dtype == MB_F32 ? f(float()) : dtype == MB_BF16 ? f(bf16()) : f(f16());
}

}  // namespace mb

using namespace mb;

extern "C" int mace_b200_group_norm_fwd(const void* x, int64_t ldx, const void* w, const void* b, const void* offsets,
                                        int32_t offsets64, void* y, float* mean, float* rstd, int64_t rows, int64_t n,
                                        int64_t len, int32_t c, int32_t groups, double eps, int32_t act, int32_t dtype,
                                        int32_t ptype, void* stream) {
  GnArgs a = gn_args(x, ldx, w, b, offsets, offsets64, rows, n, len, c, groups, act, ptype);
  if (int rc = gn_check("group_norm_fwd", a, dtype, ptype)) return rc;
  if (rows > 0 && (!x || !y || !mean != !rstd)) {
    set_error("group_norm_fwd: null pointer");
    return MB_E_ARG;
  }
  if (sm_count() < 1) {
    set_error("group_norm_fwd: no CUDA device");
    return MB_E_CUDA;
  }
  a.out = y; a.mean = mean; a.rstd = rstd; a.eps = (float)eps;
  if (n == 0 && rows > 0) {                       // rows of no sample
    if (cudaMemsetAsync(y, 0, (size_t)rows * c * dtype_size(dtype), (cudaStream_t)stream) != cudaSuccess)
      return check_launch("group_norm_fwd");
    return 0;
  }
  if (n == 0) return 0;
  return gn_type(dtype, [&](auto t) { return gn_fwd_any<decltype(t)>(a, (cudaStream_t)stream); });
}

// Rows of partial sums there can be: a cluster of at most 8 CTAs for each sample, or what is resident and one cluster more
static int64_t gn_parts(int64_t n) {
  const int64_t most = (int64_t)(GN_BWD_SM / 128) * (sm_count() > 0 ? sm_count() : 1) + 8;
  return 8 * n < most ? 8 * n : most;
}

extern "C" int mace_b200_group_norm_bwd_workspace(int64_t n, int32_t c, int64_t* floats) {
  if (n < 0 || c < 1 || !floats) {
    set_error("group_norm_bwd_workspace: bad arguments (samples %lld, channels %d)", (long long)n, c);
    return MB_E_ARG;
  }
  *floats = 2 * (int64_t)c * gn_parts(n);
  return 0;
}

extern "C" int mace_b200_group_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, const void* b,
                                        const void* offsets, int32_t offsets64, const float* mean, const float* rstd, void* dx,
                                        void* dw, void* db, float* workspace, int64_t rows, int64_t n, int64_t len, int32_t c,
                                        int32_t groups, int32_t act, int32_t dtype, int32_t ptype, void* stream) {
  GnArgs a = gn_args(x, ldx < lddy ? ldx : lddy, w, b, offsets, offsets64, rows, n, len, c, groups, act, ptype);
  if (int rc = gn_check("group_norm_bwd", a, dtype, ptype)) return rc;
  if ((rows > 0 && (!dy || !x)) || (n > 0 && (!mean || !rstd)) || ((dw || db) && !workspace)) {
    set_error("group_norm_bwd: null pointer");
    return MB_E_ARG;
  }
  if (sm_count() < 1) {
    set_error("group_norm_bwd: no CUDA device");
    return MB_E_CUDA;
  }
  a.ldx = ldx; a.lddy = lddy; a.dy = dy; a.out = dx; a.mean = (float*)mean; a.rstd = (float*)rstd;
  a.partial = dw || db ? workspace : nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  int64_t parts = 0;
  if (n == 0 && rows > 0 && dx && cudaMemsetAsync(dx, 0, (size_t)rows * c * dtype_size(dtype), st) != cudaSuccess)
    return check_launch("group_norm_bwd");
  if (n > 0 && rows > 0 && (dx || a.partial)) {
    const int64_t most = gn_parts(n);
    if (int rc = gn_type(dtype, [&](auto t) { return gn_bwd_any<decltype(t)>(a, &parts, false, st); })) return rc;
    if (parts > most) {
      set_error("group_norm_bwd: %lld rows of partial sums, room for %lld", (long long)parts, (long long)most);
      return MB_E_ARG;
    }
    if (int rc = gn_type(dtype, [&](auto t) { return gn_bwd_any<decltype(t)>(a, &parts, true, st); })) return rc;
  }
  if (!a.partial) return 0;
  return col_sums(workspace, (int)parts, c, dw, db, ptype, st);
}
