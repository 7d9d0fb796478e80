// Routing of tokens (atoms) to experts: scores s = softmax(l) or sigmoid(l) over E logits, a choice of k experts, weights.
// The choice ranks by v = s + bias, or by the logits themselves without a bias (the same order, and no two logits that
// differ can tie after rounding); logits of -inf are closed to the token.  With groups, a group's value is the sum of its
// two best open v (of s up to the row's common factor without a bias), and only the best top_groups groups stay open.  Ties
// go to the lowest index, NaN ranks first.  Slot j gets the j-th best expert, or -1 with weight 0 when none is open.
//   renormalise: w_j = scale s_j / S, S = sum_j s_j (0 when S = 0);  else w_j = scale s_j.
// Backward (the choice is constant): with q_j = s_j / S,
//   renormalise: ds_j = scale (dw_j - sum_i dw_i q_i) / S, else ds_j = scale dw_j;
//   softmax: dl_i = s_i (ds_i - sum_j s_j ds_j), sigmoid: dl_i = ds_i s_i (1 - s_i).
//
// One warp per token, expert i in lane i % 32 (coalesced rows), all scores in registers.  The k choices are k warp-wide
// maxima of order-preserving integer keys (redux), so the comparisons are exact.  The algorithm reads each logit once.
#include "dtypes.cuh"

namespace mb {

constexpr int RT_WARPS = 8;

struct RouteArgs {
  const void* logits;
  const float *bias, *dw;
  float* w;
  int32_t* idx;
  const int32_t* cidx;
  void* dl;
  int64_t t, ldl;
  int32_t e, k, groups, top_groups, softmax, renorm;
  float scale;
};

// float -> uint32 with the same order: -0 equals +0, NaN is above +inf, and -inf is 0 (closed)
__device__ __forceinline__ unsigned order_key(float f) {
  if (f != f) return 0xFFFFFFFFu;
  if (f == -INFINITY) return 0u;
  const unsigned u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Scores of one token's experts (lane holds i = lane + 32 j): softmax numerators and their sum, or sigmoids (sum 1).
// The functions and roundings are those of exp() and division in plain fp32 arithmetic.
template <int NE>
__device__ __forceinline__ float route_scores(const float (&l)[NE], int softmax, float (&s)[NE]) {
  if (!softmax) {
#pragma unroll
    for (int j = 0; j < NE; ++j) s[j] = 1.f / (1.f + expf(-l[j]));
    return 1.f;
  }
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < NE; ++j) m = fmaxf(m, l[j]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (m == -INFINITY) m = 0.f;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    s[j] = expf(l[j] - m);
    sum += s[j];
  }
  return warp_sum(sum);
}

template <typename T, int NE>
__device__ __forceinline__ void route_load(const RouteArgs& a, int64_t row, int lane, float (&l)[NE]) {
  const T* p = (const T*)a.logits + row * a.ldl;
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    const int i = lane + 32 * j;
    l[j] = i < a.e ? to_f(p[i]) : -INFINITY;
  }
}

template <typename T, int NE>
__global__ void __launch_bounds__(32 * RT_WARPS) k_route_fwd(const RouteArgs a) {
  extern __shared__ float sm[];                   // groups > 1: [RT_WARPS][32 NE] ranking values
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t row = (int64_t)blockIdx.x * RT_WARPS + warp; row < a.t; row += (int64_t)gridDim.x * RT_WARPS) {
    float l[NE], s[NE];
    route_load<T, NE>(a, row, lane, l);
    const float sum = route_scores<NE>(l, a.softmax, s);
    unsigned key[NE];
    float rank[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      const int i = lane + 32 * j;
      rank[j] = s[j];
      if (a.bias && i < a.e) rank[j] = (a.softmax ? s[j] / sum : s[j]) + a.bias[i];
      key[j] = l[j] == -INFINITY ? 0u : order_key(a.bias ? rank[j] : l[j]);
    }
    if (a.groups > 1) {
      float* v = sm + warp * 32 * NE;
#pragma unroll
      for (int j = 0; j < NE; ++j) v[lane + 32 * j] = l[j] == -INFINITY ? -INFINITY : rank[j];
      __syncwarp();
      const int per = a.e / a.groups;
      unsigned gk = 0u;                           // lane g: key of group g's value
      if (lane < a.groups) {
        float m1 = -INFINITY, m2 = -INFINITY;
        bool nan = false;
        for (int i = 0; i < per; ++i) {
          const float f = v[lane * per + i];
          nan |= f != f;
          m2 = fmaxf(m2, fminf(m1, f));
          m1 = fmaxf(m1, f);
        }
        if (nan)
          gk = 0xFFFFFFFFu;
        else if (m1 > -INFINITY)
          gk = order_key(m2 > -INFINITY ? m1 + m2 : m1);
      }
      __syncwarp();
      unsigned open = 0u;                         // bit g: group g stays open
      for (int q = 0; q < a.top_groups; ++q) {
        const unsigned best = __reduce_max_sync(0xffffffffu, gk);
        if (best == 0u) break;
        const int g = __ffs(__ballot_sync(0xffffffffu, gk == best)) - 1;
        open |= 1u << g;
        if (lane == g) gk = 0u;
      }
#pragma unroll
      for (int j = 0; j < NE; ++j)
        if (lane + 32 * j < a.e && !((open >> ((lane + 32 * j) / per)) & 1u)) key[j] = 0u;
    }
    float mine = 0.f;                             // lane q: score and expert of slot q
    int expert = -1;
    for (int q = 0; q < a.k; ++q) {
      unsigned b = 0u;
      int at = 0;
      float sc = 0.f;
#pragma unroll
      for (int j = 0; j < NE; ++j)
        if (key[j] > b) b = key[j], at = j, sc = s[j];
      const unsigned best = __reduce_max_sync(0xffffffffu, b);
      if (best == 0u) break;
      const unsigned i = __reduce_min_sync(0xffffffffu, b == best ? (unsigned)(lane + 32 * at) : 0xFFFFFFFFu);
      sc = __shfl_sync(0xffffffffu, sc, i & 31);
      if (lane == q) mine = sc, expert = (int)i;
      if (lane == (int)(i & 31))
#pragma unroll
        for (int j = 0; j < NE; ++j)
          if (j == at) key[j] = 0u;
    }
    const float tot = a.renorm ? warp_sum(mine) : sum;
    if (lane < a.k) {
      a.w[row * a.k + lane] = tot > 0.f || tot != tot ? a.scale * (mine / tot) : 0.f;
      a.idx[row * a.k + lane] = expert;
    }
  }
}

template <typename T, int NE>
__global__ void __launch_bounds__(32 * RT_WARPS) k_route_bwd(const RouteArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t row = (int64_t)blockIdx.x * RT_WARPS + warp; row < a.t; row += (int64_t)gridDim.x * RT_WARPS) {
    float l[NE], s[NE];
    route_load<T, NE>(a, row, lane, l);
    const float sum = route_scores<NE>(l, a.softmax, s);
    const int mine = lane < a.k ? a.cidx[row * a.k + lane] : -1;
    const float dw = lane < a.k && mine >= 0 ? a.scale * a.dw[row * a.k + lane] : 0.f;
    // scores of the chosen experts, one slot per lane
    float sc = 0.f;
    for (int q = 0; q < a.k; ++q) {
      const int i = __shfl_sync(0xffffffffu, mine, q);
      if (i < 0 || i >= a.e) continue;
      float got = 0.f;
#pragma unroll
      for (int j = 0; j < NE; ++j)
        if (j == (i >> 5)) got = s[j];
      got = __shfl_sync(0xffffffffu, got, i & 31);
      if (lane == q) sc = got;
    }
    // up = s_j ds_j for the chosen slot of this lane
    float up;
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    if (a.renorm) {
      const float tot = warp_sum(sc);
      const float q = tot > 0.f || tot != tot ? sc / tot : 0.f;
      up = q * (dw - warp_sum(dw * q));
    } else {
      up = dw * (sc * inv);
    }
    if (!a.softmax) up *= 1.f - sc;
    // renormalised softmax weights do not depend on the other experts: sum_j s_j ds_j = 0
    const float all = a.softmax && !a.renorm ? warp_sum(up) * inv : 0.f;
    float out[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) out[j] = -s[j] * all;
    for (int q = 0; q < a.k; ++q) {
      const int i = __shfl_sync(0xffffffffu, mine, q);
      const float v = __shfl_sync(0xffffffffu, up, q);
#pragma unroll
      for (int j = 0; j < NE; ++j)
        if (i == lane + 32 * j) out[j] += v;
    }
    T* dl = (T*)a.dl + row * a.e;
#pragma unroll
    for (int j = 0; j < NE; ++j)
      if (lane + 32 * j < a.e) dl[lane + 32 * j] = from_f<T>(out[j]);
  }
}

template <typename T, int NE>
static int route_launch(const RouteArgs& a, bool bwd, cudaStream_t st) {
  const int64_t want = (a.t + RT_WARPS - 1) / RT_WARPS, most = (int64_t)16 * sm_count();
  const unsigned grid = (unsigned)(want < most ? want : most);
  if (bwd) {
    k_route_bwd<T, NE><<<grid, 32 * RT_WARPS, 0, st>>>(a);
    return check_launch("route_bwd");
  }
  k_route_fwd<T, NE><<<grid, 32 * RT_WARPS, a.groups > 1 ? RT_WARPS * 32 * NE * 4 : 0, st>>>(a);
  return check_launch("route_fwd");
}

template <typename T>
static int route_any(const RouteArgs& a, bool bwd, cudaStream_t st) {
  if (a.e <= 32) return route_launch<T, 1>(a, bwd, st);
  if (a.e <= 64) return route_launch<T, 2>(a, bwd, st);
  if (a.e <= 128) return route_launch<T, 4>(a, bwd, st);
  if (a.e <= 256) return route_launch<T, 8>(a, bwd, st);
  return route_launch<T, 16>(a, bwd, st);
}

static int route_check(const char* who, const RouteArgs& a, int dtype) {
  if (a.t < 0 || a.e < 1 || a.e > MB_ROUTE_MAX_EXPERTS || a.k < 1 || a.k > MB_ROUTE_MAX_K || a.k > a.e || a.ldl < a.e) {
    set_error("%s: bad sizes (tokens %lld, experts %d, k %d, row stride %lld; at most %d experts, k at most %d)", who,
              (long long)a.t, a.e, a.k, (long long)a.ldl, MB_ROUTE_MAX_EXPERTS, MB_ROUTE_MAX_K);
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
  return 0;
}

static int route_types(const RouteArgs& a, int dtype, bool bwd, cudaStream_t st) {
  if (dtype == MB_F32) return route_any<float>(a, bwd, st);
  return dtype == MB_BF16 ? route_any<bf16>(a, bwd, st) : route_any<f16>(a, bwd, st);
}

}  // namespace mb

using namespace mb;

extern "C" int mace_b200_route_fwd(const void* logits, int64_t ldl, const float* bias, float* weights, int32_t* experts,
                                   int64_t n, int32_t E, int32_t k, int32_t softmax, int32_t groups, int32_t top_groups,
                                   int32_t renormalize, float scale, int32_t dtype, void* stream) {
  RouteArgs a{};
  a.logits = logits; a.ldl = ldl; a.bias = bias; a.w = weights; a.idx = experts;
  a.t = n; a.e = E; a.k = k; a.softmax = softmax != 0; a.renorm = renormalize != 0; a.scale = scale;
  a.groups = groups; a.top_groups = top_groups;
  if (int rc = route_check("route_fwd", a, dtype)) return rc;
  if (groups < 1 || groups > 32 || E % groups || top_groups < 1 || top_groups > groups) {
    set_error("route_fwd: bad groups (%d of %d experts, %d chosen; at most 32 groups)", groups, E, top_groups);
    return MB_E_ARG;
  }
  if (n == 0) return 0;
  if (!logits || !weights || !experts) {
    set_error("route_fwd: null pointer");
    return MB_E_ARG;
  }
  return route_types(a, dtype, false, (cudaStream_t)stream);
}

extern "C" int mace_b200_route_bwd(const float* dweights, const void* logits, int64_t ldl, const int32_t* experts,
                                   void* dlogits, int64_t n, int32_t E, int32_t k, int32_t softmax,
                                   int32_t renormalize, float scale, int32_t dtype, void* stream) {
  RouteArgs a{};
  a.logits = logits; a.ldl = ldl; a.dw = dweights; a.cidx = experts; a.dl = dlogits;
  a.t = n; a.e = E; a.k = k; a.softmax = softmax != 0; a.renorm = renormalize != 0; a.scale = scale;
  if (int rc = route_check("route_bwd", a, dtype)) return rc;
  if (n == 0) return 0;
  if (!dweights || !logits || !experts || !dlogits) {
    set_error("route_bwd: null pointer");
    return MB_E_ARG;
  }
  return route_types(a, dtype, true, (cudaStream_t)stream);
}
