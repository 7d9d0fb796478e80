// Group norm with an activation, channels last: a sample is a run of rows [C], its channels are `groups` runs of C / groups.
//   mu, var over the rows and channels of a group, r = 1 / sqrt(var + eps), xh = (x - mu) r, z = xh w + b, y = f(z)
// and its backward pass, with dz = dy f'(z) and a = dz w:
//   dx = r (a - mean(a) - xh mean(a xh)), dw = sum over rows of dz xh, db = sum over rows of dz.
// f: identity, silu z s(z), gelu z Phi(z) or relu.  Statistics and sums are fp32; every output is rounded once.
//
// Bound: HBM bytes (forward x and y, backward x, dy and dx, each once).  Two forms of the same kernels:
//  * on the chip (GN_WHOLE): a cluster of P <= 8 CTAs owns a sample's rows of a block of whole groups.  A CTA keeps its rows in shared
//    memory between the sums and the output and exchanges sums of its groups with the cluster through distributed shared memory.
//    Rows that do not fit (ragged samples far above the mean) are read again.
//  * larger ones stream: GN_SUMS (partial sums of P parts of a sample to the workspace), a small kernel that adds up the parts, and
//    GN_APPLY, which reads the rows again, last ones first: of tensors larger than L2 that one still has those (64 x 2048 x 512 bf16 75 + 130
//    us, first ones first 75.5 + 133; 24,000 x 512 fp32, which L2 holds, 46 + 60 and 43 + 60).  No barrier stands between the bytes, so
//    both run near the copy rate.  (Large samples in clusters of 8 on the chip read once, but load and store in turns: 64 x 2048 x 512
//    bf16 forward 124 us and backward 315.)
// A thread owns V channels of one group (16 bytes, or what divides a group) and every TR-th row, and takes its sums relative to
// its own first row, GN_RUN rows at a time: a sample far longer than the others, which gets no more threads than they, may have
// 10^5 rows of a thread, and that many additions of like values in a row are 0.1% off (of 137,500 times 0.1; in runs of 512 1.5e-6).
// Threads, CTAs and clusters are joined as (count, mean, sum of squared deviations), so nothing cancels.  No atomics: parameter
// gradients are added up over a CTA's samples in a thread's own places of shared memory (of columns beyond one pass of the threads: in
// the CTA's rows of the workspace), then over CTAs by a second small kernel in a fixed order.
//
// Measured on a B200 (kernels, forward / backward; a copy runs at 6.5 TB/s): 64 x 2048 x 512 bf16 in 32 groups with silu 75 / 130 us
// (3 and 5 times the tensor's bytes at 5.3 TB/s; sums 33 us, with the issue slots 80% busy, outputs 47), with gelu 92 / 163, one sample of
// 24,000 x 512 fp32 46 / 60 us (three and four launches), one of 1,029,000 x 128 fp32 272 / 495 us (5.8 and 5.3 TB/s), 384 ragged samples of
// 63 x 128 fp16 with gelu 12.2 / 25 us, 192 x 128 fp32 6.6 / 9.0 us (latency of one launch, of two), 4,000 ragged samples of 60 x 128
// bf16 57 / 131 us (what a CTA does once a sample: its offsets, sums over threads, parameters).  Samples are cut by their mean length:
// one far longer than the others gets no more CTAs than they (one of 1.1 million rows among 20,000 of 60 is 59 + 85 ms of one CTA).
#include "dtypes.cuh"
#include "norm.cuh"
#include "tc.cuh"

namespace mb {

struct GnArgs {
  const void *x, *dy, *w, *b;
  void* out;                                      // y, or dx (null: parameter gradients only)
  float *mean, *rstd, *partial;                   // partial [cluster rows][2][C]: sums of dz xh, of dz (null: none)
  float *sums, *stat;                             // [n][P][3][groups] of GN_SUMS, [n][groups][2] for GN_APPLY
  const void* off;                                // [n + 1], null: samples of `len` rows
  int* order;                                     // words of k_gn_order that say whether they ascend, null: each CTA looks for itself
  int64_t ldx, lddy, rows, n, len;
  int32_t norder;
  int32_t c, groups, cg, gpb, act, off64, p32, cap, pshift, pvec;   // gpb: groups of a column block; cap: row steps kept in shared memory
                                                  // pshift: log2 of a cluster's CTAs; pvec: parameters are aligned vectors
  float eps;
};

// Rows of a thread that are added one after the other (a multiple of GN_RING and of four); what a run gives is joined with the runs
// before it.  Those wait in the thread's place of `red`: in registers they cost the usual case, one run, up to a fifth of its time.
constexpr int GN_RUN = 512;

// CTAs of 256 threads that the registers let be resident on an SM
constexpr int GN_FWD_CTAS = 4, GN_BWD_CTAS = 2;

enum { GN_WHOLE = 0, GN_SUMS = 1, GN_APPLY = 2 };

__device__ __forceinline__ int64_t gn_off(const GnArgs& a, int64_t i) {
  return a.off64 ? ((const int64_t*)a.off)[i] : (int64_t)((const int32_t*)a.off)[i];
}
// Rows of a sample; false: the offsets leave the rows there
__device__ __forceinline__ bool gn_range(const GnArgs& a, int64_t s, int64_t& lo, int64_t& hi) {
  if (!a.off) {
    lo = s * a.len;
    hi = lo + a.len;
    return true;
  }
  const int64_t u = gn_off(a, s), v = gn_off(a, s + 1);
  lo = u < 0 ? 0 : u < a.rows ? u : a.rows;
  hi = v < lo ? lo : v < a.rows ? v : a.rows;
  return u >= 0 && v <= a.rows;
}

// Whether the offsets ascend everywhere, for a whole block.  Where they descend, samples far from there may share rows, and which
// of them wrote last would be anyone's guess: then every block writes NaN alone.  Up to GN_SCAN samples a block reads all offsets
// itself (16 a thread of 64; 900 samples of 60 x 128 bf16 17.1 -> 19.0 us), more are looked through by a launch of their own, and a
// block reads its words (4,000 samples 60 -> 62 us).  rstd then holds GN_DESCENDS, a NaN that no arithmetic gives (that is 7fffffff),
// where the backward pass finds the answer.
constexpr int GN_SCAN = 1024;
constexpr unsigned GN_DESCENDS = 0x7fc00d0du;
__device__ __forceinline__ bool gn_ascend(const GnArgs& a) {
  if (!a.off) return true;
  int bad = 0;
  if (a.order) {
    for (int i = threadIdx.x; i < a.norder; i += blockDim.x) bad |= a.order[i];
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < (int)a.n; i += blockDim.x) bad |= gn_off(a, i + 1) < gn_off(a, i);
  }
  return !__syncthreads_or(bad);
}
__global__ void __launch_bounds__(256) k_gn_order(const GnArgs a) {
  int bad = 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.n; i += (int64_t)gridDim.x * 256) bad |= gn_off(a, i + 1) < gn_off(a, i);
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) a.order[blockIdx.x] = bad;
}

// Rows outside of all samples are zero (NaN where the offsets do not ascend)
template <typename T>
__device__ __forceinline__ void gn_clear(const GnArgs& a, bool ascend) {
  if (!a.off || !a.out) return;
  auto at = [&](int64_t i) {
    const int64_t v = gn_off(a, i);
    return v < 0 ? 0 : v < a.rows ? v : a.rows;
  };
  const T none = from_f<T>(ascend ? 0.f : __int_as_float(0x7fc00000));
  const int64_t head = a.n ? at(0) : a.rows, tail = a.n ? at(a.n) : a.rows;
  const int64_t id = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
  const int64_t step = (int64_t)gridDim.x * gridDim.y * gridDim.z * blockDim.x;
  T* out = (T*)a.out;
  for (int64_t i = id * blockDim.x + threadIdx.x; i < head * a.c; i += step) out[i] = none;
  for (int64_t i = tail * a.c + id * blockDim.x + threadIdx.x; i < a.rows * a.c; i += step) out[i] = none;
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

// Rows on their way through a thread's own places in shared memory (GN_SUMS and GN_APPLY): more bytes in flight than registers hold.
// Elements of two bytes alone cannot be copied so.
constexpr int GN_RING = 8;
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// fp32 rows forward are as fast through registers (1,029,000 x 128 267 us, through the ring 295; bf16 64 x 2048 x 512 94 and 76).
template <int MODE, typename T, int V, bool BWD>
constexpr bool gn_ring = MODE != GN_WHOLE && V * sizeof(T) >= 4 && (BWD || sizeof(T) == 2);

// V elements as Elem<V> (packed pairs where V > 1) and back
template <typename T, int V>
__device__ __forceinline__ void gn_get(const GnVec<T, V>& v, Elem<V> (&e)[kElems<V>]) {
  float f[V];
  v.get(f);
  to_elems<V>(f, e);
}
template <typename T, int V>
__device__ __forceinline__ void gn_set(GnVec<T, V>& v, const Elem<V> (&e)[kElems<V>]) {
  float f[V];
  from_elems<V>(e, f);
  v.set(f);
}

// 1 / (1 + exp(-z)).  fp32 results take expf and a division; 16-bit ones 2^(-z log2 e) and a reciprocal, each approximate to
// 2^-22 (the exponent's rounding |z| 2^-24): 0 where the power is above 2^126, at z below -87.3.
__device__ __forceinline__ float pow2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
template <typename T>
__device__ __forceinline__ float gn_sigmoid(float z) {
  if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-z));
  return rcp_fast(1.f + pow2_fast(-1.4426950408889634f * z));
}
template <typename T>
__device__ __forceinline__ float2 gn_sigmoid(float2 z) {
  if constexpr (sizeof(T) == 4) return make_float2(gn_sigmoid<T>(z.x), gn_sigmoid<T>(z.y));
  const float2 t = e_mul(z, e_splat<float2>(-1.4426950408889634f));
  const float2 d = e_add(make_float2(pow2_fast(t.x), pow2_fast(t.y)), e_splat<float2>(1.f));
  return make_float2(rcp_fast(d.x), rcp_fast(d.y));
}
// Phi(z) and the normal density of z.  16-bit results: the tail Phi(-|z|) = t poly(t) exp(-z^2 / 2), t = 1 / (1 + 0.3 |z|), whose
// coefficients have the least largest relative error over |z| <= 5.5 (a linear program over a grid) with 1e-4 allowed up to 14.2: in fp32
// 3e-6 and 4e-5 of the tail itself, so far out gelu is right to the last bit of bf16 and fp16, too.  The exponential is the
// density's, too (the complementary error function took 100 instructions).
struct GnPhi {
  float cdf, pdf;
};
template <typename T>
__device__ __forceinline__ GnPhi gn_phi(float z) {
  if constexpr (sizeof(T) == 4) return {normcdff(z), 0.3989422804014327f * expf(-0.5f * z * z)};
  const float e = pow2_fast(-0.7213475204444817f * z * z), t = rcp_fast(fmaf(0.3f, fabsf(z), 1.f));
  float h = fmaf(-0.0820684f, t, 0.23104584f);
  h = fmaf(h, t, -0.034196015f);
  h = fmaf(h, t, 0.15355037f);
  h = fmaf(h, t, 0.11137169f);
  h = fmaf(h, t, 0.12029581f) * t * e;
  return {z < 0.f ? h : 1.f - h, 0.3989422804014327f * e};
}
template <typename T>
__device__ __forceinline__ float gn_gelu(float z) { return z * gn_phi<T>(z).cdf; }
template <typename T>
__device__ __forceinline__ float gn_gelu_slope(float z) {
  const GnPhi p = gn_phi<T>(z);
  return fmaf(z, p.pdf, p.cdf);
}
__device__ __forceinline__ float2 gn_each(float2 a, float (*f)(float)) { return make_float2(f(a.x), f(a.y)); }
__device__ __forceinline__ float gn_each(float a, float (*f)(float)) { return f(a); }
__device__ __forceinline__ float gn_relu(float z) { return z < 0.f ? 0.f : z; }                       // NaN stays
__device__ __forceinline__ float gn_gate(float z, float d) { return z <= 0.f ? 0.f : d; }
__device__ __forceinline__ float2 gn_gate(float2 z, float2 d) { return make_float2(gn_gate(z.x, d.x), gn_gate(z.y, d.y)); }

template <typename T, typename E, int NE>
__device__ __forceinline__ void gn_act(E (&z)[NE], int act) {
  if (act == MB_ACT_SILU) {
#pragma unroll
    for (int q = 0; q < NE; ++q) z[q] = e_mul(z[q], gn_sigmoid<T>(z[q]));
  } else if (act == MB_ACT_GELU) {
#pragma unroll
    for (int q = 0; q < NE; ++q) z[q] = gn_each(z[q], gn_gelu<T>);
  } else if (act == MB_ACT_RELU) {
#pragma unroll
    for (int q = 0; q < NE; ++q) z[q] = gn_each(z[q], gn_relu);
  }
}
template <typename T, typename E, int NE>
__device__ __forceinline__ void gn_act_grad(const E (&z)[NE], E (&d)[NE], int act) {   // d *= f'(z)
  const E one = e_splat<E>(1.f), minus = e_splat<E>(-1.f);
  if (act == MB_ACT_SILU) {
#pragma unroll
    for (int q = 0; q < NE; ++q) {
      const E s = gn_sigmoid<T>(z[q]);
      d[q] = e_mul(d[q], e_mul(s, e_fma(z[q], e_fma(s, minus, one), one)));
    }
  } else if (act == MB_ACT_GELU) {
#pragma unroll
    for (int q = 0; q < NE; ++q) d[q] = e_mul(d[q], gn_each(z[q], gn_gelu_slope<T>));
  } else if (act == MB_ACT_RELU) {
#pragma unroll
    for (int q = 0; q < NE; ++q) d[q] = gn_gate(z[q], d[q]);
  }
}

// V parameters, fp32 or of type T
template <typename T, int V>
__device__ __forceinline__ void gn_param(const void* p, const GnArgs& a, int c, float other, Elem<V> (&e)[kElems<V>]) {
  float f[V];
#pragma unroll
  for (int q = 0; q < V; ++q) f[q] = other;
  if (p && a.p32 && a.pvec && V % 4 == 0) {
#pragma unroll
    for (int q = 0; q < V; q += 4) {
      const float4 t = *reinterpret_cast<const float4*>((const float*)p + c + q);
      f[q] = t.x, f[q + 1] = t.y, f[q + 2] = t.z, f[q + 3] = t.w;
    }
  } else if (p && !a.p32 && a.pvec) {
    GnVec<T, V> t;
    t.load((const T*)p + c);
    t.get(f);
  } else if (p) {
#pragma unroll
    for (int q = 0; q < V; ++q) f[q] = a.p32 ? ((const float*)p)[c + q] : to_f(((const T*)p)[c + q]);
  }
  to_elems<V>(f, e);
}
// A CTA's (a part's) rows of a sample of len rows: the first of them, or (rank + 1) where they end
template <int MODE>
__device__ __forceinline__ int64_t gn_cut_row(const GnArgs& a, int64_t len, int rank, int P) {
  return MODE == GN_WHOLE ? (len * rank) >> a.pshift : len * rank / P;
}

// How a thread of a CTA walks over the CTA's rows and columns: TC vector columns at a time (`tiles` times), TR rows.
// slots > 0: the groups lie within warps, in runs of cgv lanes (a power of two), so that warps take sums by shuffles and the sums of
// a group come in that many places; 0: sums go through `red`, a thread each, into one place.
struct GnWalk {
  int g0, ng, c0, nvec, tc, tr, r, col, tiles, cgv, slots, grp;   // grp: of the thread's column in the first tile
  bool on, writes;                                // writes: the lane that stores a warp's sums of its group
};
template <int V>
__device__ __forceinline__ GnWalk gn_walk(const GnArgs& a) {
  GnWalk k;
  k.g0 = blockIdx.y * a.gpb;
  k.ng = a.groups - k.g0 < a.gpb ? a.groups - k.g0 : a.gpb;
  k.c0 = k.g0 * a.cg;
  k.cgv = a.cg / V;
  k.nvec = k.ng * k.cgv;
  const int th = blockDim.x;
  k.tc = k.nvec < th ? k.nvec : th;
  k.tr = th / k.tc;
  k.r = threadIdx.x / k.tc;
  k.col = threadIdx.x - k.r * k.tc;
  k.tiles = (k.nvec + k.tc - 1) / k.tc;
  k.on = k.r < k.tr;
  const bool fits = k.cgv <= 32 && (k.cgv & (k.cgv - 1)) == 0 && k.tiles == 1 && th % k.tc == 0;
  k.slots = fits && (k.tc < 32 ? (k.tc & (k.tc - 1)) == 0 : k.tc % 32 == 0) ? (k.tc < 32 ? th / 32 : k.tr) : 0;
  if (k.slots * a.gpb > (a.gpb < th ? th : a.gpb)) k.slots = 0;   // (a narrower last block has more rows than there is room for)
  k.grp = k.col / k.cgv;
  k.writes = (threadIdx.x & 31 & (k.cgv - 1)) == 0 && (k.tc >= 32 || (threadIdx.x & 31) < k.tc);
  return k;
}
// Rows of a thread among nr
__device__ __forceinline__ int gn_count(int64_t nr, const GnWalk& k) {
  const int64_t n = nr - k.r + k.tr - 1;
  return (n >> 31) ? (int)(n / k.tr) : (int)((unsigned)n / (unsigned)k.tr);
}
// (mean relative to the first row, squared deviations) of c rows of V channels in r, joined with those of n rows more
__device__ __forceinline__ void gn_join_run(float2& r, float c, float rel, float dev, float n, float v) {
  const float d = rel - r.x, f = n / (c + n);
  r.x = fmaf(d, f, r.x);
  r.y += fmaf(d * d * v, c * f, dev);
}
// The place of this thread's warp among a group's slots
__device__ __forceinline__ int gn_slot(const GnWalk& k) { return k.tc < 32 ? threadIdx.x >> 5 : k.r; }

// Sum over the lanes of a warp that hold the same group (all of them have it)
__device__ __forceinline__ float gn_warp_sum(const GnWalk& k, float v) {
  for (int o = k.cgv >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  for (int o = k.tc; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) { return __int_as_float(ld_cluster_s32(addr)); }

// Sum over the 8 lanes of an octet
__device__ __forceinline__ float octet_sum(float v) {
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Shared memory: red [threads] pairs | grp [2][slots][3][gpb] (by parity of the sample: what this CTA found) | fin [2][gpb] | rows.
// slots gpb is at most the number of threads, or slots is one.
__host__ __device__ __forceinline__ int gn_grp_floats(int threads, int gpb) { return 3 * (gpb < threads ? threads : gpb); }
__host__ __device__ __forceinline__ int gn_shared_floats(int threads, int gpb) {
  return (2 * threads + 2 * gn_grp_floats(threads, gpb) + 2 * gpb + 3) & ~3;
}

template <int MODE, typename T, int V>
__global__ void __launch_bounds__(256, GN_FWD_CTAS) k_gn_fwd(const GnArgs a) {
  constexpr int U = 4, NE = kElems<V>;
  using E = Elem<V>;
  using Vec = GnVec<T, V>;
  extern __shared__ __align__(16) float gn_smem[];
  const GnWalk k = gn_walk<V>(a);
  const int th = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = th >> 5;
  // the second launch goes through the rows backwards
  const int P = gridDim.x, rank = MODE == GN_APPLY ? P - 1 - (int)blockIdx.x : (int)blockIdx.x;
  const int cap = MODE == GN_WHOLE ? a.cap : 0, slots = k.slots ? k.slots : 1;
  float2* red = reinterpret_cast<float2*>(gn_smem);
  float* grp0 = gn_smem + 2 * th;
  float* fin = grp0 + 2 * gn_grp_floats(th, a.gpb);
  Vec* kept = reinterpret_cast<Vec*>(gn_smem + gn_shared_floats(th, a.gpb)) + threadIdx.x;
  const int64_t step = (int64_t)k.tr * a.ldx, ystep = (int64_t)k.tr * a.c;
  const bool ascend = MODE == GN_SUMS || gn_ascend(a);
  if (MODE != GN_SUMS) gn_clear<T>(a, ascend);
  int par = 0;
  for (int64_t z = blockIdx.z; z < a.n; z += gridDim.z, par ^= 1) {
    const int64_t s = MODE == GN_APPLY ? a.n - 1 - z : z;
    int64_t lo, hi;
    const bool good = gn_range(a, s, lo, hi);
    const int64_t len = hi - lo, r0 = lo + gn_cut_row<MODE>(a, len, rank, P), nr = lo + gn_cut_row<MODE>(a, len, rank + 1, P) - r0;
    float* grp = grp0 + par * gn_grp_floats(th, a.gpb);
    if (!k.slots)
      for (int g = threadIdx.x; g < 3 * k.ng; g += th) grp[g / k.ng * a.gpb + g % k.ng] = 0.f;
    // ---------------------------------------------------------------------------------------- sums
    for (int t = 0; MODE != GN_APPLY && t < k.tiles; ++t) {
      const int v0 = t * k.tc, cv = v0 + k.col;
      const bool on = cv < k.nvec && k.on && nr > k.r;
      float mu = 0.f, m2 = 0.f, mine = 0.f;       // of this thread's rows, and how many
      if (!k.slots && nr > GN_RUN * k.tr) __syncthreads();   // red is free
      if (on) {
        const T* x = (const T*)a.x + (r0 + k.r) * a.ldx + k.c0 + cv * V;
        E piv[NE], s1[NE], s2[NE];
        Vec v;
        v.load(x);
        gn_get<T, V>(v, piv);
#pragma unroll
        for (int q = 0; q < NE; ++q) piv[q] = e_mul(piv[q], e_splat<E>(-1.f)), s1[q] = s2[q] = e_splat<E>(0.f);
        int at = t;                               // place among the kept vectors
        auto add = [&](const Vec& u) {
          E f[NE];
          if (at < cap) kept[at * th] = u;
          at += k.tiles;
          gn_get<T, V>(u, f);
#pragma unroll
          for (int q = 0; q < NE; ++q) {
            const E e = e_add(f[q], piv[q]);
            s1[q] = e_add(s1[q], e);
            s2[q] = e_fma(e, e, s2[q]);
          }
        };
        int64_t left = nr - k.r;                  // rows from this thread's next one on
        int n;                                    // rows of this run
        // V channels of a run to (mean, mean relative to the first row, squared deviations) of n * V values
        auto channels = [&](float& mean, float& rel, float& dev) {
          const float rows = (float)n, inv = __fdividef(1.f, rows);
          float p[V], u1[V], u2[V];
          from_elems<V>(piv, p);
          from_elems<V>(s1, u1);
          from_elems<V>(s2, u2);
          mean = rel = dev = 0.f;
#pragma unroll
          for (int q = 0; q < V; ++q) {
            const float d = u1[q] * inv;
            p[q] = d - p[q];
            mean += p[q];
            rel += d;
            dev += fmaxf(fmaf(-u1[q], d, u2[q]), 0.f * u2[q]);   // not below 0, NaN stays
          }
          mean *= 1.f / (float)V;
          rel *= 1.f / (float)V;
#pragma unroll
          for (int q = 0; q < V; ++q) dev = fmaf((p[q] - mean) * (p[q] - mean), rows, dev);
        };
        int runs = 0;                             // before this one
        auto next_run = [&] {
          float mean, rel, dev;
          channels(mean, rel, dev);
          float2 r = make_float2(rel, dev);
          if (runs > 0) {
            r = red[threadIdx.x];
            gn_join_run(r, (float)runs * GN_RUN, rel, dev, GN_RUN, (float)V);
          }
          red[threadIdx.x] = r;
          ++runs;
          n = 0;
#pragma unroll
          for (int q = 0; q < NE; ++q) s1[q] = s2[q] = e_splat<E>(0.f);
        };
        if constexpr (gn_ring<MODE, T, V, false>) {
          const uint32_t ring = smem_u32(kept), place = (uint32_t)th * sizeof(Vec);
          int64_t todo = left;
          auto issue = [&](int d) {
            if (left > 0) {
              copy_async<sizeof(Vec)>(ring + d * place, x);
              x += step;
              left -= k.tr;
            }
            copy_commit();
          };
#pragma unroll
          for (int d = 0; d < GN_RING; ++d) issue(d);
          for (n = 0; todo > 0;) {
            if (n == GN_RUN) next_run();
#pragma unroll
            for (int d = 0; d < GN_RING; ++d) {
              if (todo <= 0) break;
              copy_wait<GN_RING - 1>();
              add(kept[d * th]);
              issue(d);
              todo -= k.tr;
              ++n;
            }
          }
        } else {
          for (n = 0; left > (U - 1) * k.tr; left -= U * k.tr, x += U * step, n += U) {
            if (n == GN_RUN) next_run();
            Vec u[U];
  #pragma unroll
            for (int j = 0; j < U; ++j) u[j].load(x + j * step);
  #pragma unroll
            for (int j = 0; j < U; ++j) add(u[j]);
          }
          for (; left > 0; left -= k.tr, x += step, ++n) {   // (fewer than U)
            Vec u;
            u.load(x);
            add(u);
          }
        }
        float rel;
        channels(mu, rel, m2);
        mine = (float)n;
        if (runs > 0) {
          float2 r = red[threadIdx.x];
          gn_join_run(r, (float)runs * GN_RUN, rel, m2, mine, (float)V);
          float p[V], sum = 0.f;
          from_elems<V>(piv, p);
#pragma unroll
          for (int q = 0; q < V; ++q) sum += p[q];
          mu = fmaf(sum, -1.f / (float)V, r.x);
          m2 = r.y;
          mine = fmaf((float)runs, GN_RUN, mine);
        }
      }
      if (k.slots) {
        const float n = mine * (float)V, cnt = gn_warp_sum(k, n), sum = gn_warp_sum(k, n * mu);
        const float mean = cnt > 0.f ? __fdividef(sum, cnt) : 0.f;
        const float dev = gn_warp_sum(k, n > 0.f ? fmaf((mu - mean) * (mu - mean), n, m2) : 0.f);
        if (k.writes) {
          float* o = grp + gn_slot(k) * 3 * a.gpb + k.grp;
          o[0] = cnt;
          o[a.gpb] = mean;
          o[2 * a.gpb] = dev;
        }
        continue;
      }
      __syncthreads();                            // red is free (and grp is zero)
      red[threadIdx.x] = make_float2(mu, m2);
      __syncthreads();
      for (int g = warp; g < k.ng; g += warps) {
        const int a0 = g * k.cgv - v0 > 0 ? g * k.cgv - v0 : 0, a1 = (g + 1) * k.cgv - v0;
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
          if (n > 0) dev += fmaf((v.x - mean) * (v.x - mean), (float)n * (float)V, v.y);
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
    if (MODE == GN_WHOLE && P > 1)
      cluster_sync();
    else if (MODE != GN_APPLY)
      __syncthreads();
    // ---------------------------------------------------------------------------------------- statistics
    // eight lanes a group take the slots of its CTAs (GN_SUMS: of this one) in turn, twice: the mean, then the deviations from it
    for (int g = threadIdx.x >> 3; MODE != GN_APPLY && g < (k.ng + 3) / 4 * 4; g += th >> 3) {
      const int gg = g < k.ng ? g : k.ng - 1, all = MODE == GN_WHOLE ? slots << a.pshift : slots;
      const uint32_t base = smem_u32(grp + gg);
      auto word = [&](int q, int which) {
        if (MODE == GN_WHOLE && P > 1)
          return ld_cluster_f32(mapa_u32(base + 4u * (uint32_t)(((q >> a.pshift) * 3 + which) * a.gpb), q & (P - 1)));
        return grp[gg + (q * 3 + which) * a.gpb];
      };
      float n = 0.f, m = 0.f, m2 = 0.f;
      for (int q = threadIdx.x & 7; q < all; q += 8) {
        const float cnt = word(q, 0);
        n += cnt;
        m = fmaf(cnt, word(q, 1), m);
      }
      n = octet_sum(n);
      m = octet_sum(m);
      const float mean = n > 0.f ? __fdividef(m, n) : 0.f;
      for (int q = threadIdx.x & 7; q < all; q += 8) {
        const float cnt = word(q, 0), d = word(q, 1) - mean;
        if (cnt > 0.f) m2 += fmaf(d * d, cnt, word(q, 2));
      }
      m2 = octet_sum(m2);
      if ((threadIdx.x & 7) != 0 || g >= k.ng) continue;
      if (MODE == GN_SUMS) {
        float* part = a.sums + (s * P + rank) * 3 * a.groups + k.g0 + g;
        part[0] = n;
        part[a.groups] = mean;
        part[2 * a.groups] = m2;
      } else {
        const float bad = good && ascend ? 0.f : __int_as_float(0x7fc00000);
        float rs = rsqrtf((n > 0.f ? __fdividef(m2, n) : 0.f) + a.eps) + bad;
        if (!ascend) rs = __uint_as_float(GN_DESCENDS);
        fin[2 * g] = mean + bad;
        fin[2 * g + 1] = rs;
        if (a.mean && rank == 0) {
          a.mean[s * a.groups + k.g0 + g] = mean + bad;
          a.rstd[s * a.groups + k.g0 + g] = rs;
        }
      }
    }
    if (MODE == GN_SUMS) continue;
    if (MODE == GN_WHOLE) __syncthreads();
    const float* st = MODE == GN_APPLY ? a.stat + (s * a.groups + k.g0) * 2 : fin;
    // ---------------------------------------------------------------------------------------- outputs
    for (int t = 0; t < k.tiles; ++t) {
      const int cv = t * k.tc + k.col;
      if (cv >= k.nvec || !k.on || nr <= k.r) continue;
      const int c = k.c0 + cv * V, g = k.tiles == 1 ? k.grp : cv / k.cgv;
      E w[NE], b[NE];
      gn_param<T, V>(a.w, a, c, 1.f, w);
      gn_param<T, V>(a.b, a, c, 0.f, b);
      const E neg = e_splat<E>(-st[2 * g]), rs = e_splat<E>(st[2 * g + 1]);
#pragma unroll
      for (int q = 0; q < NE; ++q) w[q] = e_mul(w[q], rs);
      auto put = [&](Vec v, T* y) {
        E f[NE];
        gn_get<T, V>(v, f);
#pragma unroll
        for (int q = 0; q < NE; ++q) f[q] = e_fma(e_add(f[q], neg), w[q], b[q]);
        gn_act<T>(f, a.act);
        gn_set<T, V>(v, f);
        v.store(y);
      };
      const int have = cap > t ? (cap - t + k.tiles - 1) / k.tiles : 0;   // rows kept
      int i = gn_count(nr, k);
      const T* x = (const T*)a.x + (r0 + k.r) * a.ldx + c + (int64_t)i * step;   // one row behind the next
      T* y = (T*)a.out + (r0 + k.r) * (int64_t)a.c + c + (int64_t)i * ystep;
      if constexpr (gn_ring<MODE, T, V, false>) {
        const uint32_t ring = smem_u32(kept), place = (uint32_t)th * sizeof(Vec);
        int left = i;
        auto issue = [&](int d) {
          if (left > 0) {
            x -= step;
            copy_async<sizeof(Vec)>(ring + d * place, x);
            --left;
          }
          copy_commit();
        };
#pragma unroll
        for (int d = 0; d < GN_RING; ++d) issue(d);
        while (i > 0) {
#pragma unroll
          for (int d = 0; d < GN_RING; ++d) {
            if (i <= 0) break;
            copy_wait<GN_RING - 1>();
            y -= ystep;
            put(kept[d * th], y);
            issue(d);
            --i;
          }
        }
      } else {
        for (; i - U >= have; i -= U) {
          x -= U * step;
          y -= U * ystep;
          Vec u[U];
  #pragma unroll
          for (int j = 0; j < U; ++j) u[j].load(x + j * step);
  #pragma unroll
          for (int j = 0; j < U; ++j) put(u[j], y + j * ystep);
        }
        for (; i > have; --i) {
          x -= step;
          y -= ystep;
          Vec u;
          u.load(x);
          put(u, y);
        }
      }
      const Vec* kp = kept + (i * k.tiles + t) * th;
      const int kstep = k.tiles * th;
#pragma unroll 2
      for (; i > 0; --i) {
        kp -= kstep;
        y -= ystep;
        put(*kp, y);
      }
    }
  }
  if (MODE == GN_WHOLE && P > 1) cluster_sync();  // no CTA leaves while its peers may read its sums
}

template <int MODE, typename T, int V>
__global__ void __launch_bounds__(256, GN_BWD_CTAS) k_gn_bwd(const GnArgs a) {
  constexpr int U = 4, NE = kElems<V>;
  using E = Elem<V>;
  using Vec = GnVec<T, V>;
  extern __shared__ __align__(16) float gn_smem[];
  const GnWalk k = gn_walk<V>(a);
  const int th = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = th >> 5;
  const int P = gridDim.x, rank = MODE == GN_APPLY ? P - 1 - (int)blockIdx.x : (int)blockIdx.x;
  const int cap = MODE == GN_WHOLE ? a.cap : 0, slots = k.slots ? k.slots : 1;
  float2* red = reinterpret_cast<float2*>(gn_smem);
  float* grp0 = gn_smem + 2 * th;
  float* fin = grp0 + 2 * gn_grp_floats(th, a.gpb);
  Vec* kept = reinterpret_cast<Vec*>(gn_smem + gn_shared_floats(th, a.gpb)) + threadIdx.x;
  if (MODE != GN_SUMS && a.off) gn_clear<T>(a, __float_as_uint(a.rstd[0]) != GN_DESCENDS);
  // sums of dz xh and dz over the samples (one tile of columns): a thread's own places behind the kept rows
  float* total = gn_smem + gn_shared_floats(th, a.gpb) + (size_t)2 * (gn_ring<MODE, T, V, true> ? GN_RING : cap) * th * V * sizeof(T) / 4 + threadIdx.x;
  if (MODE != GN_APPLY && k.tiles == 1)
#pragma unroll
    for (int q = 0; q < 2 * V; ++q) total[q * th] = 0.f;
  float* part = MODE != GN_APPLY && a.partial ? a.partial + ((int64_t)blockIdx.z * P + rank) * 2 * a.c : nullptr;
  const int64_t xstep = (int64_t)k.tr * a.ldx, dstep = (int64_t)k.tr * a.lddy, ostep = (int64_t)k.tr * a.c;
  int par = 0;
  bool first = true;
  for (int64_t z = blockIdx.z; z < a.n; z += gridDim.z, par ^= 1, first = false) {
    const int64_t s = MODE == GN_APPLY ? a.n - 1 - z : z;
    int64_t lo, hi;
    gn_range(a, s, lo, hi);
    const int64_t len = hi - lo, r0 = lo + gn_cut_row<MODE>(a, len, rank, P), nr = lo + gn_cut_row<MODE>(a, len, rank + 1, P) - r0;
    float* grp = grp0 + par * gn_grp_floats(th, a.gpb);
    if (!k.slots)
      for (int g = threadIdx.x; g < 2 * k.ng; g += th) grp[g / k.ng * a.gpb + g % k.ng] = 0.f;
    // what turns x and dy into xh and dz, for the columns of a tile
    E w[NE], b[NE], neg, rs;
    auto columns = [&](int c, int g) {
      gn_param<T, V>(a.w, a, c, 1.f, w);
      gn_param<T, V>(a.b, a, c, 0.f, b);
      const int64_t st = s * a.groups + k.g0 + g;
      neg = e_splat<E>(-a.mean[st]);
      rs = e_splat<E>(a.rstd[st]);
    };
    auto both = [&](const Vec& u, const Vec& v, E (&f)[NE], E (&d)[NE]) {
      E z[NE];
      gn_get<T, V>(u, f);
      gn_get<T, V>(v, d);
#pragma unroll
      for (int q = 0; q < NE; ++q) {
        f[q] = e_mul(e_add(f[q], neg), rs);
        z[q] = e_fma(f[q], w[q], b[q]);
      }
      gn_act_grad<T>(z, d, a.act);
    };
    // ---------------------------------------------------------------------------------------- sums
    for (int t = 0; MODE != GN_APPLY && t < k.tiles; ++t) {
      const int v0 = t * k.tc, cv = v0 + k.col;
      const bool on = cv < k.nvec && k.on && nr > k.r;
      const int c = k.c0 + cv * V;
      E sw[NE], sb[NE];
      float s1 = 0.f, s2 = 0.f;
      bool fresh = first;                         // nothing of these columns lies in memory
#pragma unroll
      for (int q = 0; q < NE; ++q) sw[q] = sb[q] = e_splat<E>(0.f);
      auto put_part = [&] {
        if (k.tiles == 1 || !part || cv >= k.nvec) return;   // several tiles: one thread a column, its sums of all samples lie in memory
        float fw[V], fb[V];
        from_elems<V>(sw, fw);
        from_elems<V>(sb, fb);
#pragma unroll
        for (int q = 0; q < V; ++q) {
          part[c + q] = fresh ? fw[q] : part[c + q] + fw[q];
          part[a.c + c + q] = fresh ? fb[q] : part[a.c + c + q] + fb[q];
        }
      };
      if (!k.slots && nr > GN_RUN * k.tr) __syncthreads();   // red is free
      if (on) {
        columns(c, k.tiles == 1 ? k.grp : cv / k.cgv);
        const T* x = (const T*)a.x + (r0 + k.r) * a.ldx + c;
        const T* dy = (const T*)a.dy + (r0 + k.r) * a.lddy + c;
        int at = t;
        auto add = [&](const Vec& u, const Vec& v) {
          if (at < cap) {
            kept[2 * at * th] = u;
            kept[(2 * at + 1) * th] = v;
          }
          at += k.tiles;
          E f[NE], d[NE];
          both(u, v, f, d);
#pragma unroll
          for (int q = 0; q < NE; ++q) {
            sw[q] = e_fma(d[q], f[q], sw[q]);
            sb[q] = e_add(sb[q], d[q]);
          }
        };
        auto columns_sums = [&] {                 // of a run: to s1, s2 and the parameters' sums
          E p1 = e_splat<E>(0.f), p2 = p1;
#pragma unroll
          for (int q = 0; q < NE; ++q) {
            p1 = e_fma(w[q], sb[q], p1);
            p2 = e_fma(w[q], sw[q], p2);
          }
          s1 = e_sum(p1);
          s2 = e_sum(p2);
          if (k.tiles == 1) {
            float f[V];
            from_elems<V>(sw, f);
#pragma unroll
            for (int q = 0; q < V; ++q) total[q * th] += f[q];
            from_elems<V>(sb, f);
#pragma unroll
            for (int q = 0; q < V; ++q) total[(V + q) * th] += f[q];
          }
        };
        int runs = 0, n = 0;                      // runs before this one, and rows of it
        auto next_run = [&] {
          columns_sums();
          put_part();
          fresh = false;
          if (runs > 0) s1 += red[threadIdx.x].x, s2 += red[threadIdx.x].y;
          red[threadIdx.x] = make_float2(s1, s2);
          ++runs;
          n = 0;
#pragma unroll
          for (int q = 0; q < NE; ++q) sw[q] = sb[q] = e_splat<E>(0.f);
        };
        int64_t left = nr - k.r;
        if constexpr (gn_ring<MODE, T, V, true>) {
          const uint32_t ring = smem_u32(kept), place = (uint32_t)th * sizeof(Vec);
          int64_t todo = left;
          auto issue = [&](int d) {
            if (left > 0) {
              copy_async<sizeof(Vec)>(ring + 2 * d * place, x);
              copy_async<sizeof(Vec)>(ring + (2 * d + 1) * place, dy);
              x += xstep;
              dy += dstep;
              left -= k.tr;
            }
            copy_commit();
          };
#pragma unroll
          for (int d = 0; d < GN_RING; ++d) issue(d);
          for (; todo > 0; n += GN_RING) {
            if (n == GN_RUN) next_run();
#pragma unroll
            for (int d = 0; d < GN_RING; ++d) {
              if (todo <= 0) break;
              copy_wait<GN_RING - 1>();
              add(kept[2 * d * th], kept[(2 * d + 1) * th]);
              issue(d);
              todo -= k.tr;
            }
          }
        } else {
          for (; left > (U - 1) * k.tr; left -= U * k.tr, x += U * xstep, dy += U * dstep, n += U) {
            if (n == GN_RUN) next_run();
            Vec u[U], v[U];
  #pragma unroll
            for (int j = 0; j < U; ++j) u[j].load(x + j * xstep), v[j].load(dy + j * dstep);
  #pragma unroll
            for (int j = 0; j < U; ++j) add(u[j], v[j]);
          }
          for (; left > 0; left -= k.tr, x += xstep, dy += dstep) {
            Vec u, v;
            u.load(x);
            v.load(dy);
            add(u, v);
          }
        }
        columns_sums();
        if (runs > 0) s1 += red[threadIdx.x].x, s2 += red[threadIdx.x].y;
      }
      if (k.slots) {
        s1 = gn_warp_sum(k, s1);
        s2 = gn_warp_sum(k, s2);
        if (k.writes) {
          float* o = grp + gn_slot(k) * 3 * a.gpb + k.grp;
          o[0] = s1;
          o[a.gpb] = s2;
        }
        continue;
      }
      put_part();
      __syncthreads();                            // red is free (and grp is zero)
      red[threadIdx.x] = make_float2(s1, s2);
      __syncthreads();
      for (int g = warp; g < k.ng; g += warps) {
        const int a0 = g * k.cgv - v0 > 0 ? g * k.cgv - v0 : 0, a1 = (g + 1) * k.cgv - v0;
        const int n = (a1 < k.nvec - v0 ? (a1 < k.tc ? a1 : k.tc) : (k.nvec - v0 < k.tc ? k.nvec - v0 : k.tc)) - a0;
        if (n <= 0) continue;
        float u = 0.f, v = 0.f;
        for (int e = lane; e < n * k.tr; e += 32) {
          const int r = e / n;
          const float2 p = red[r * k.tc + a0 + (e - r * n)];
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
    if (MODE == GN_WHOLE && P > 1)
      cluster_sync();
    else if (MODE != GN_APPLY)
      __syncthreads();
    const float inv = 1.f / ((float)len * (float)a.cg);
    for (int g = threadIdx.x >> 3; MODE != GN_APPLY && g < (k.ng + 3) / 4 * 4; g += th >> 3) {
      const int gg = g < k.ng ? g : k.ng - 1, all = MODE == GN_WHOLE ? slots << a.pshift : slots;
      const uint32_t base = smem_u32(grp + gg);
      float u = 0.f, v = 0.f;
      for (int q = threadIdx.x & 7; q < all; q += 8) {
        if (MODE == GN_WHOLE && P > 1) {
          const uint32_t at = mapa_u32(base + 12u * (uint32_t)((q >> a.pshift) * a.gpb), q & (P - 1));
          u += ld_cluster_f32(at);
          v += ld_cluster_f32(at + 4 * a.gpb);
        } else {
          u += grp[gg + q * 3 * a.gpb];
          v += grp[gg + (q * 3 + 1) * a.gpb];
        }
      }
      u = octet_sum(u);
      v = octet_sum(v);
      if ((threadIdx.x & 7) != 0 || g >= k.ng) continue;
      if (MODE == GN_SUMS) {
        float* gp = a.sums + (s * P + rank) * 3 * a.groups + k.g0 + g;
        gp[0] = u;
        gp[a.groups] = v;
      } else {
        fin[2 * g] = u * inv;
        fin[2 * g + 1] = v * inv;
      }
    }
    if (MODE == GN_SUMS) continue;
    if (MODE == GN_WHOLE) __syncthreads();
    const float* fs = MODE == GN_APPLY ? a.stat + (s * a.groups + k.g0) * 2 : fin;
    // ---------------------------------------------------------------------------------------- dx
    for (int t = 0; t < k.tiles; ++t) {
      const int cv = t * k.tc + k.col;
      if (cv >= k.nvec || !k.on || nr <= k.r) continue;
      const int c = k.c0 + cv * V, g = k.tiles == 1 ? k.grp : cv / k.cgv;
      if (k.tiles > 1 || MODE == GN_APPLY) columns(c, g);
      const E m1 = e_splat<E>(-fs[2 * g]), m2 = e_splat<E>(-fs[2 * g + 1]);
      auto put = [&](Vec u, const Vec& v, T* dx) {
        E f[NE], d[NE];
        both(u, v, f, d);
#pragma unroll
        for (int q = 0; q < NE; ++q) f[q] = e_mul(rs, e_fma(f[q], m2, e_fma(d[q], w[q], m1)));
        gn_set<T, V>(u, f);
        u.store(dx);
      };
      const int have = cap > t ? (cap - t + k.tiles - 1) / k.tiles : 0;
      int i = gn_count(nr, k);
      const T* x = (const T*)a.x + (r0 + k.r) * a.ldx + c + (int64_t)i * xstep;
      const T* dy = (const T*)a.dy + (r0 + k.r) * a.lddy + c + (int64_t)i * dstep;
      T* dx = (T*)a.out + (r0 + k.r) * (int64_t)a.c + c + (int64_t)i * ostep;
      if constexpr (gn_ring<MODE, T, V, true>) {
        const uint32_t ring = smem_u32(kept), place = (uint32_t)th * sizeof(Vec);
        int left = i;
        auto issue = [&](int d) {
          if (left > 0) {
            x -= xstep;
            dy -= dstep;
            copy_async<sizeof(Vec)>(ring + 2 * d * place, x);
            copy_async<sizeof(Vec)>(ring + (2 * d + 1) * place, dy);
            --left;
          }
          copy_commit();
        };
#pragma unroll
        for (int d = 0; d < GN_RING; ++d) issue(d);
        while (i > 0) {
#pragma unroll
          for (int d = 0; d < GN_RING; ++d) {
            if (i <= 0) break;
            copy_wait<GN_RING - 1>();
            dx -= ostep;
            put(kept[2 * d * th], kept[(2 * d + 1) * th], dx);
            issue(d);
            --i;
          }
        }
      } else {
        for (; i - U >= have; i -= U) {
          x -= U * xstep;
          dy -= U * dstep;
          dx -= U * ostep;
          Vec u[U], v[U];
  #pragma unroll
          for (int j = 0; j < U; ++j) u[j].load(x + j * xstep), v[j].load(dy + j * dstep);
  #pragma unroll
          for (int j = 0; j < U; ++j) put(u[j], v[j], dx + j * ostep);
        }
        for (; i > have; --i) {
          x -= xstep;
          dy -= dstep;
          dx -= ostep;
          Vec u, v;
          u.load(x);
          v.load(dy);
          put(u, v, dx);
        }
      }
      const Vec* kp = kept + 2 * (i * k.tiles + t) * th;
      const int kstep = 2 * k.tiles * th;
      for (; i > 0; --i) {
        kp -= kstep;
        dx -= ostep;
        put(kp[0], kp[th], dx);
      }
    }
  }
  if (part && k.tiles == 1) {                     // over the rows of threads, in their order
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * V * k.tc; i += th) {
      const int q = i / k.tc, col = i - q * k.tc;
      float v = 0.f;
      for (int r = 0; r < k.tr; ++r) v += total[(int)(q * th + r * k.tc + col) - (int)threadIdx.x];
      part[(q < V ? 0 : a.c) + k.c0 + col * V + (q < V ? q : q - V)] = v;
    }
  }
  if (MODE == GN_WHOLE && P > 1) cluster_sync();
}

// The parts' sums of each sample and group, a warp each: forward (count, mean, squared deviations) to mean and rstd, backward (sums
// of a and a xh) to their means
// ORDER: the offsets are looked through (forward, ragged).  Asked for at run time, or with four loads ahead instead of eight, the join of
// 592 parts takes 2 us longer.
template <bool BWD, bool ORDER>
__global__ void __launch_bounds__(256) k_gn_join(const GnArgs a, int P) {
  const int lane = threadIdx.x & 31;
  const bool ascend = !ORDER || gn_ascend(a);
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < a.n * a.groups; i += (int64_t)gridDim.x * 8) {
    const int64_t s = i / a.groups;
    const float* p = a.sums + s * P * 3 * a.groups + (i - s * a.groups);
    const int64_t step = 3 * (int64_t)a.groups;
    int64_t lo, hi;
    const bool good = gn_range(a, s, lo, hi);
    float u = 0.f, v = 0.f;
    if constexpr (BWD) {
#pragma unroll 4
      for (int q = lane; q < P; q += 32) u += p[q * step], v += p[q * step + a.groups];
      const float inv = 1.f / ((float)(hi - lo) * (float)a.cg);
      u = warp_sum(u) * inv;
      v = warp_sum(v) * inv;
    } else {
      float n = 0.f, m2 = 0.f;
#pragma unroll 8
      for (int q = lane; q < P; q += 32) {
        const float c = p[q * step];
        n += c;
        u = fmaf(c, p[q * step + a.groups], u);
      }
      n = warp_sum(n);
      u = n > 0.f ? warp_sum(u) / n : 0.f;
#pragma unroll 8
      for (int q = lane; q < P; q += 32) {
        const float c = p[q * step], d = p[q * step + a.groups] - u;
        if (c > 0.f) m2 += fmaf(d * d, c, p[q * step + 2 * a.groups]);
      }
      m2 = warp_sum(m2);
      const float bad = good && ascend ? 0.f : __int_as_float(0x7fc00000);
      u += bad;
      v = rsqrtf((n > 0.f ? m2 / n : 0.f) + a.eps) + bad;
      if (!ascend) v = __uint_as_float(GN_DESCENDS);
    }
    if (lane == 0) {
      a.stat[2 * i] = u;
      a.stat[2 * i + 1] = v;
      if (!BWD && a.mean) {
        a.mean[i] = u;
        a.rstd[i] = v;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ host side
// How a call is cut: groups of a column block, blocks, CTAs of a cluster (or parts), threads, row steps in shared memory, samples in
// the grid
struct GnCut {
  int gpb, ncb, p, pshift, th, cap, smem;
  int64_t nz;
  bool split;
};

// A CTA keeps up to this much, so that four (forward) or two (backward) fit an SM and some load while others store
constexpr int GN_KEEP_FWD = 48 * 1024, GN_KEEP_BWD = 64 * 1024, GN_WHOLE_BYTES = 4 << 20, GN_START = 16384;

// Row segments of a column block of the whole form: 64 bytes at least (two sectors)
constexpr int GN_SEGMENT = 64;

static int64_t gn_rows(const GnArgs& a) { return a.off ? (a.n ? (a.rows + a.n - 1) / a.n : 0) : a.len; }
static int gn_blocks(const GnArgs& a, int size) {   // most column blocks of the whole form
  const int per = (GN_SEGMENT + a.cg * size - 1) / (a.cg * size), n = a.groups / per;
  return n < 1 ? 1 : n;
}
// Parts of a sample in the split form; 0: the whole form.  Sizes alone decide, so that the workspace's size does not hang on
// addresses.
static int gn_split(const GnArgs& a, int size, int slabs) {
  const int64_t bytes = gn_rows(a) * a.c * size * slabs, keep = slabs == 1 ? GN_KEEP_FWD : GN_KEEP_BWD;
  if (bytes <= keep || a.n * bytes <= GN_WHOLE_BYTES) return 0;
  // the number whose rounds over the resident CTAs take least, a CTA's start and end as long as GN_START bytes of its rows: for each
  // number of rounds the most parts that need no more
  const int64_t all = (int64_t)(slabs == 1 ? GN_FWD_CTAS : GN_BWD_CTAS) * sm_count(), r0 = (a.n + all - 1) / all;
  int64_t most = bytes / 4096 < gn_rows(a) ? bytes / 4096 : gn_rows(a);   // (each part has a row of sums of every column backward)
  if (most < 1) most = 1;
  int64_t best = 1;
  double least = 0.0;
  for (int64_t r = r0; r <= r0 + 4; ++r) {
    int64_t p = r * all / a.n;
    if (p > most) p = most;
    const double t = (double)r * ((double)bytes / (double)p + GN_START);
    if (r == r0 || t < least) best = p, least = t;
  }
  return (int)best;
}

template <int V>
static GnCut gn_cut(const GnArgs& a, int size, int slabs, int threads_sm) {
  const int keep = slabs == 1 ? GN_KEEP_FWD : GN_KEEP_BWD;
  GnCut k{};
  const int64_t rows = gn_rows(a), bytes = rows * a.c * size * slabs, sms = sm_count();
  k.p = gn_split(a, size, slabs);
  k.split = k.p > 0;
  int64_t ncb;
  if (k.split) {                                  // whole rows, or as wide blocks as one pass of a CTA's threads takes
    ncb = (a.c / V + 255) / 256;
  } else {
    int64_t want = (bytes + keep - 1) / keep;
    const int64_t fill = (2 * sms + a.n - 1) / a.n, least = bytes / 8192;
    if (want < (fill < least ? fill : least)) want = fill < least ? fill : least;
    ncb = gn_blocks(a, size);
    if (ncb > want) ncb = want;
    if (ncb < 1) ncb = 1;
    k.p = 1;
    while (k.p < 8 && k.p * ncb < want && rows >= 2 * k.p) k.p *= 2;
    for (k.pshift = 0; (1 << k.pshift) < k.p; ++k.pshift) {}
  }
  if (ncb > a.groups) ncb = a.groups;
  if (ncb > 65535) ncb = 65535;                   // of a grid's second dimension
  k.gpb = (int)((a.groups + ncb - 1) / ncb);
  if (k.gpb > 1024) k.gpb = 1024;                 // words of its groups in shared memory
  k.ncb = (a.groups + k.gpb - 1) / k.gpb;
  const int64_t slab = (rows + k.p - 1) / k.p * k.gpb * a.cg * size * slabs;
  const int nvec = k.gpb * a.cg / V;
  // about 16 vectors a thread where there are CTAs enough (what a thread does once a sample is as much as 30 of them), else 4; a
  // thread for each vector column, too.  4,000 samples of 60 x 128 bf16: 256 threads 61 us, a warp a sample of 3 x 128 a third.
  const int64_t vecs = slab / (V * size * slabs), each = a.n * k.p * k.ncb >= 4 * sms ? 16 : 4;
  for (k.th = 32; k.th < 256 && (k.th * each < vecs || k.th < nvec); k.th *= 2) {}
  const int tiles = (nvec + k.th - 1) / k.th, tr = nvec < k.th ? k.th / nvec : 1;
  const int64_t steps = ((rows + k.p - 1) / k.p + tr - 1) / tr * tiles;
  const int per = k.th * V * size * slabs, most = keep / per;
  k.cap = k.split ? 0 : (int)(steps < most ? steps : most);
  k.smem = 4 * gn_shared_floats(k.th, k.gpb) + (k.split ? (V * size >= 4 && (slabs == 2 || size == 2) ? GN_RING : 0) : k.cap) * per + (slabs == 2 ? 8 * V * k.th : 0);
  // samples in the grid: all where a CTA has much to do, else what is resident (a CTA then goes over several)
  int res = threads_sm / k.th;
  const int by_smem = (220 * 1024) / (k.smem + 1024);
  if (by_smem < res) res = by_smem;
  if (res < 1) res = 1;
  k.nz = (int64_t)res * sms / ((int64_t)k.p * k.ncb);
  if (k.nz < 1) k.nz = 1;
  if (slab >= 16384 && a.n * k.p <= 1024) k.nz = a.n;
  if (k.nz > a.n) k.nz = a.n;
  return k;
}

template <auto KERN>
static int gn_launch(GnArgs& a, const GnCut& k, cudaStream_t st, const char* what) {
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
  a.pshift = k.pshift;
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
  cfg.numAttrs = !k.split && k.p > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, KERN, a);
  return check_launch(what);
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

// Words of k_gn_order (0: blocks look at the offsets themselves), and its launch
static int gn_order_words(const GnArgs& a) {
  const int64_t want = (a.n + 1023) / 1024;
  return !a.off || a.n <= GN_SCAN ? 0 : (int)(want < sm_count() ? want : sm_count());
}
static int gn_order(const GnArgs& a, cudaStream_t st) {
  if (!a.order) return 0;
  k_gn_order<<<a.norder, 256, 0, st>>>(a);
  return check_launch("group_norm (offsets)");
}

template <bool BWD>
static int gn_join(const GnArgs& a, int p, cudaStream_t st) {
  const int64_t want = (a.n * a.groups + 7) / 8, most = 8 * (int64_t)sm_count();
  const unsigned grid = (unsigned)(want < most ? want : most);
  if (!BWD && a.off)
    k_gn_join<BWD, !BWD><<<grid, 256, 0, st>>>(a, p);
  else
    k_gn_join<BWD, false><<<grid, 256, 0, st>>>(a, p);
  return check_launch("group_norm");
}

constexpr int GN_FWD_SM = 256 * GN_FWD_CTAS, GN_BWD_SM = 256 * GN_BWD_CTAS;

template <typename T, int V>
static int gn_fwd_go(GnArgs& a, cudaStream_t st) {
  const GnCut k = gn_cut<V>(a, sizeof(T), 1, GN_FWD_SM);
  if (!k.split) return gn_launch<k_gn_fwd<GN_WHOLE, T, V>>(a, k, st, "group_norm_fwd");
  if (int rc = gn_launch<k_gn_fwd<GN_SUMS, T, V>>(a, k, st, "group_norm_fwd")) return rc;
  if (int rc = gn_join<false>(a, k.p, st)) return rc;
  return gn_launch<k_gn_fwd<GN_APPLY, T, V>>(a, k, st, "group_norm_fwd");
}
template <typename T>
static int gn_fwd_any(GnArgs& a, cudaStream_t st) {
  const int v = gn_vec(a, sizeof(T));
  if (v == 16 / (int)sizeof(T)) return gn_fwd_go<T, 16 / sizeof(T)>(a, st);
  return v > 1 ? gn_fwd_go<T, 8 / sizeof(T)>(a, st) : gn_fwd_go<T, 1>(a, st);
}
template <typename T, int V>
static int gn_bwd_go(GnArgs& a, int64_t* parts, bool launch, cudaStream_t st) {
  const GnCut k = gn_cut<V>(a, sizeof(T), 2, GN_BWD_SM);
  *parts = k.nz * k.p;
  if (!launch) return 0;
  if (!k.split) return gn_launch<k_gn_bwd<GN_WHOLE, T, V>>(a, k, st, "group_norm_bwd");
  if (int rc = gn_launch<k_gn_bwd<GN_SUMS, T, V>>(a, k, st, "group_norm_bwd")) return rc;
  if (!a.out) return 0;
  if (int rc = gn_join<true>(a, k.p, st)) return rc;
  return gn_launch<k_gn_bwd<GN_APPLY, T, V>>(a, k, st, "group_norm_bwd");
}
template <typename T>
static int gn_bwd_any(GnArgs& a, int64_t* parts, bool launch, cudaStream_t st) {
  const int v = gn_vec(a, sizeof(T));
  if (v == 16 / (int)sizeof(T)) return gn_bwd_go<T, 16 / sizeof(T)>(a, parts, launch, st);
  return v > 1 ? gn_bwd_go<T, 8 / sizeof(T)>(a, parts, launch, st) : gn_bwd_go<T, 1>(a, parts, launch, st);
}

static int gn_check(const char* who, const GnArgs& a, int32_t dtype, int32_t ptype) {
  if (a.rows < 0 || a.n < 0 || a.c < 1 || a.groups < 1 || a.groups > MB_GN_MAX_GROUPS || a.c % a.groups || a.ldx < a.c ||
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
  a.pvec = aligned16(w) && aligned16(b);
  a.p32 = ptype == MB_F32;
  return a;
}

template <typename F>
static int gn_type(int dtype, const F& f) {
  return dtype == MB_F32 ? f(float()) : dtype == MB_BF16 ? f(bf16()) : f(f16());
}

}  // namespace mb

using namespace mb;

// The workspace: the split form's sums, then forward the words of k_gn_order, backward partial sums of the parameters' gradients.
// Floats of the sums, and rows there can be of the partial ones
static int64_t gn_sums(const GnArgs& a, int size, int slabs) {
  const int64_t p = a.n ? gn_split(a, size, slabs) : 0;
  return p ? a.n * (3 * p + 2) * (int64_t)a.groups : 0;
}
static int64_t gn_parts(const GnArgs& a, int size) {
  // of a launch at most what is resident or 1024 (gn_cut), and no more than its samples have parts
  const int64_t split = gn_split(a, size, 2), p = split ? split : 8;
  int64_t some = (int64_t)(GN_BWD_SM / 32) * (sm_count() > 0 ? sm_count() : 1);
  if (some < 1024) some = 1024;
  if (some < p) some = p;
  return a.n * p < some ? a.n * p : some;
}

static int64_t gn_floats(const GnArgs& a, int size, int slabs) {   // without the words of k_gn_order
  return gn_sums(a, size, slabs) + (slabs == 2 ? 2 * (int64_t)a.c * gn_parts(a, size) : 0);
}
static void gn_place(GnArgs& a, float* ws, int size, int slabs) {
  a.sums = ws;
  a.stat = !ws ? nullptr : ws + a.n * gn_split(a, size, slabs) * 3 * (int64_t)a.groups;
  a.norder = slabs == 1 ? gn_order_words(a) : 0;
  a.order = a.norder ? reinterpret_cast<int*>(ws + gn_floats(a, size, slabs)) : nullptr;
}

extern "C" int mace_b200_group_norm_workspace(int64_t rows, int64_t n, int64_t len, int32_t c, int32_t groups, int32_t ragged,
                                              int32_t dtype, int32_t backward, int64_t* floats) {
  GnArgs a = gn_args(nullptr, c, nullptr, nullptr, ragged ? "" : nullptr, 0, rows, n, len, c, groups, MB_ACT_NONE, MB_F32);
  if (int rc = gn_check("group_norm_workspace", a, dtype, MB_F32)) return rc;
  if (!floats) {
    set_error("group_norm_workspace: null pointer");
    return MB_E_ARG;
  }
  if (sm_count() < 1) {
    set_error("group_norm_workspace: no CUDA device");
    return MB_E_CUDA;
  }
  const int size = dtype_size(dtype);
  *floats = n == 0 || rows == 0 ? 0 : gn_floats(a, size, backward ? 2 : 1) + (backward ? 0 : gn_order_words(a));
  return 0;
}

extern "C" int mace_b200_group_norm_fwd(const void* x, int64_t ldx, const void* w, const void* b, const void* offsets,
                                        int32_t offsets64, void* y, float* mean, float* rstd, float* workspace, int64_t rows,
                                        int64_t n, int64_t len, int32_t c, int32_t groups, double eps, int32_t act,
                                        int32_t dtype, int32_t ptype, void* stream) {
  GnArgs a = gn_args(x, ldx, w, b, offsets, offsets64, rows, n, len, c, groups, act, ptype);
  if (int rc = gn_check("group_norm_fwd", a, dtype, ptype)) return rc;
  if (sm_count() < 1) {
    set_error("group_norm_fwd: no CUDA device");
    return MB_E_CUDA;
  }
  if (rows > 0 && (!x || !y || !mean != !rstd || (!workspace && n > 0 && gn_floats(a, dtype_size(dtype), 1) + gn_order_words(a) > 0))) {
    set_error("group_norm_fwd: null pointer");
    return MB_E_ARG;
  }
  a.out = y; a.mean = mean; a.rstd = rstd; a.eps = (float)eps;
  if (rows == 0) return 0;
  if (n == 0) {                                   // rows of no sample
    if (cudaMemsetAsync(y, 0, (size_t)rows * c * dtype_size(dtype), (cudaStream_t)stream) != cudaSuccess)
      return check_launch("group_norm_fwd");
    return 0;
  }
  gn_place(a, workspace, dtype_size(dtype), 1);
  if (int rc = gn_order(a, (cudaStream_t)stream)) return rc;
  return gn_type(dtype, [&](auto t) { return gn_fwd_any<decltype(t)>(a, (cudaStream_t)stream); });
}

extern "C" int mace_b200_group_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, const void* b,
                                        const void* offsets, int32_t offsets64, const float* mean, const float* rstd, void* dx,
                                        void* dw, void* db, float* workspace, int64_t rows, int64_t n, int64_t len, int32_t c,
                                        int32_t groups, int32_t act, int32_t dtype, int32_t ptype, void* stream) {
  GnArgs a = gn_args(x, ldx < lddy ? ldx : lddy, w, b, offsets, offsets64, rows, n, len, c, groups, act, ptype);
  if (int rc = gn_check("group_norm_bwd", a, dtype, ptype)) return rc;
  if (sm_count() < 1) {
    set_error("group_norm_bwd: no CUDA device");
    return MB_E_CUDA;
  }
  const bool work = n > 0 && rows > 0 && (dx || dw || db);
  if (work && (!dy || !x || !mean || !rstd || !workspace)) {
    set_error("group_norm_bwd: null pointer");
    return MB_E_ARG;
  }
  a.ldx = ldx; a.lddy = lddy; a.dy = dy; a.out = dx; a.mean = (float*)mean; a.rstd = (float*)rstd;
  cudaStream_t st = (cudaStream_t)stream;
  int64_t parts = 0;
  if (n == 0 && rows > 0 && dx && cudaMemsetAsync(dx, 0, (size_t)rows * c * dtype_size(dtype), st) != cudaSuccess)
    return check_launch("group_norm_bwd");
  if (work) {
    const int size = dtype_size(dtype);
    gn_place(a, workspace, size, 2);
    a.partial = dw || db ? workspace + gn_sums(a, size, 2) : nullptr;
    const int64_t most = gn_parts(a, size);
    if (int rc = gn_type(dtype, [&](auto t) { return gn_bwd_any<decltype(t)>(a, &parts, false, st); })) return rc;
    if (parts > most) {
      set_error("group_norm_bwd: %lld rows of partial sums, room for %lld", (long long)parts, (long long)most);
      return MB_E_ARG;
    }
    if (int rc = gn_type(dtype, [&](auto t) { return gn_bwd_any<decltype(t)>(a, &parts, true, st); })) return rc;
  }
  if (!dw && !db) return 0;
  return col_sums(a.partial, (int)parts, c, dw, db, ptype, st);
}
