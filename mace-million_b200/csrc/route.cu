// Routing of tokens (atoms) to experts: scores s = softmax(l) or sigmoid(l) over E logits, a choice of k experts, weights.
// The choice ranks by v = s + bias, or by the logits themselves without a bias (the same order, and no two logits that
// differ can tie after rounding); logits of -inf are closed to the token.  With groups, a group's value is the sum of its
// two best open v (without a bias: of their s, up to the row's common factor), and only the best top_groups groups stay
// open.  Ties go to the lowest index, NaN ranks first.  Slot j gets the j-th best expert, or -1 with weight 0 when none is
// open.
//   renormalise: w_j = scale s_j / S, S = sum_j s_j (0 when S = 0);  else w_j = scale s_j.
// Backward (the choice is constant): with q_j = s_j / S,
//   renormalise: ds_j = scale (dw_j - sum_i dw_i q_i) / S, else ds_j = scale dw_j;
//   softmax: dl_i = s_i (ds_i - sum_j s_j ds_j), sigmoid: dl_i = ds_i s_i (1 - s_i).
//
// Forward: L lanes of a warp per token, lane q holding the c experts q c .. q c + c - 1 in registers as order-preserving
// integer keys, so that a warp works on 32 / L tokens.  For k > 2 each four keys of a lane are sorted, and a choice is a
// maximum over the lists' heads in the lane and over the L lanes; the winner's list moves up.  Which expert it was is found
// once all k are known, one slot per lane, by comparing with the winner's keys in shared memory (the d-th equal key for
// the d-th equal slot, so the lowest index among equals).  Where the open groups are at most half of the experts, their
// keys are first dealt out to all lanes.  k <= 2 takes its maxima from the unsorted keys: 131,072 x 256 in k = 1 40 us,
// through sorted lists 51; at k = 4 of 128 the lists are ahead (35 us of 37), at k = 8 46 us of 57.
// Bound by issued instructions, comparisons and selections at half rate above all, not by the logits' bytes: 131,072 x 128
// bf16 sigmoid, 8 groups, k = 8 takes 59 us against 5.8 us for the bytes (85 us by maxima over unsorted keys; 85 us by a
// lane per token over keys in shared memory, whose long chains leave half of the issue slots empty; 162 us by a whole warp
// per token).  Few tokens take L = 32, which has the shortest chain.
// Backward: only the chosen logits enter, except for plain softmax weights; a warp fills a tile of zeros in shared memory
// with the k values of its tokens and copies it out in whole vectors (131,072 x 128 bf16: 11.5 us, 6.5 TB/s).
#include "dtypes.cuh"

namespace mb {

constexpr int RT_WARPS = 8;
// blocks per SM that registers are budgeted for: at 131,072 x 128 (k 8) 2 took 72 us, 3 60 us, 4 58.7 us
template <int NE>
constexpr int rt_blocks = NE <= 16 ? 4 : 3;

struct RouteArgs {
  int32_t c, span, vec;                           // forward: experts per lane, lanes per group, vector loads
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

// float -> uint32 with the same order: -0 equals +0; the sum's NaN is 0x7FFFFFFF and comes out above +inf, as 0xFFFFFFFF;
// -inf (closed) is KEY_CLOSED, and so is 0
constexpr unsigned KEY_CLOSED = 0x007FFFFFu, KEY_NAN = 0xFFFFFFFFu;
__device__ __forceinline__ unsigned order_key(float f) {
  const int u = __float_as_int(f + 0.f);
  return (unsigned)u ^ ((unsigned)(u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_float(unsigned key) {
  return __uint_as_float(key ^ ((unsigned)~((int)key >> 31) | 0x80000000u));
}

// The score's parts in plain fp32 arithmetic (exp, and a correctly rounded reciprocal): the same bits as those operations
// give anywhere, so that biased scores rank alike
__device__ __forceinline__ float sigmoid_f(float l) { return __frcp_rn(1.f + expf(-l)); }

template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int L>
__device__ __forceinline__ unsigned lanes_max(unsigned v) {
  if constexpr (L == 32) {
    return __reduce_max_sync(0xffffffffu, v);
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
}
// lowest lane of the group of L lanes (counted in the group) for which p holds, 32 or more if none
template <int L>
__device__ __forceinline__ int lanes_first(bool p, int base) {
  unsigned b = __ballot_sync(0xffffffffu, p) >> base;
  if constexpr (L < 32) b &= (1u << L) - 1u;
  return b ? __ffs(b) - 1 : 32;
}

// words of shared memory between the keys of two lanes: their 16-byte accesses do not conflict
template <int NE>
constexpr int rt_pitch = NE == 12 ? 20 : NE + 4;
// words per warp: keys, then per token the k best keys, who has them, and the open groups
template <int L, int NE, int NC>
__host__ __device__ constexpr int rt_words(int k) {
  return (NC > 0 ? 32 * rt_pitch<NE> : 0) + (32 / L * (2 * k + L) + 3) / 4 * 4;
}

// NC < NE: the open groups fit in NC keys a lane, and are dealt out to all lanes before the choice; NC = 0: one or two
// experts are chosen, straight from the keys
template <typename T, int L, int NE, int NC>
__global__ void __launch_bounds__(32 * RT_WARPS, rt_blocks<NE>) k_route_fwd(const RouteArgs a) {
  constexpr int TPW = 32 / L;                     // tokens per warp
  constexpr int NL = NC > 0 ? NC / 4 : 1, P = rt_pitch<NE>;       // lists of four keys in a lane
  extern __shared__ __align__(16) unsigned sm_rt[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane & (L - 1), base = lane & ~(L - 1);
  unsigned* keys = sm_rt + warp * rt_words<L, NE, NC>(a.k);                                    // [32][P]
  unsigned* best_of = keys + (NC > 0 ? 32 * P : 0) + lane / L * (2 * a.k + L);   // [k] of this token
  int* chosen = reinterpret_cast<int*>(best_of) + a.k;                                     // [k]
  int* opened = chosen + a.k;                                                              // [L]
  // a group's `per` experts lie in a.span lanes (a power of two), a.c in each but the last ones
  const int c = a.c, span = a.span, shift = __ffs(span) - 1, per = a.e / a.groups, mine = sub >> shift;
  const int q0 = (sub - (mine << shift)) * c, i0 = mine * per + q0;
  const int n = mine >= a.groups || q0 >= per ? 0 : per - q0 < c ? per - q0 : c;
  // the four keys from `off` on in the open group number `nth` become the lane's list u; `at`: their place from the group's
  int nth[NL], off[NL], at[NL];
  if constexpr (NC > 0 && NC < NE)
#pragma unroll
    for (int u = 0; u < NL; ++u) {
      nth[u] = (sub * NC + 4 * u) / per;
      off[u] = (sub * NC + 4 * u) % per;
      at[u] = off[u] / c * P + off[u] % c;
    }
  const bool sums = a.softmax && !a.renorm, known = a.softmax && (sums || a.bias || a.groups > 1);
  const int64_t step = (int64_t)gridDim.x * RT_WARPS * TPW;
  // every lane of a warp runs the same number of passes (the collectives are warp-wide)
  for (int64_t r0 = ((int64_t)blockIdx.x * RT_WARPS + warp) * TPW; r0 < a.t; r0 += step) {
    const int64_t row = r0 + lane / L;
    const bool live = row < a.t;
    const T* p = (const T*)a.logits + (live ? row : 0) * a.ldl;
    float l[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) l[j] = -INFINITY;
    if (a.vec) {
      constexpr int V = kVec<T>;
#pragma unroll
      for (int j = 0; j + V <= NE; j += V)
        if (live && j < n) {
          float f[V];
          load_v<T, V>(p + i0 + j, f);
#pragma unroll
          for (int q = 0; q < V; ++q) l[j + q] = f[q];
        }
    } else {
#pragma unroll
      for (int j = 0; j < NE; ++j)
        if (live && j < n) l[j] = to_f(p[i0 + j]);
    }
    float m = 0.f, sum = 1.f;
    if (known) {
      m = -INFINITY;
#pragma unroll
      for (int j = 0; j < NE; ++j) m = fmaxf(m, l[j]);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (m == -INFINITY) m = 0.f;
    }
    unsigned key[NE];
    if (a.bias) {
      float s[NE];
      if (a.softmax) {
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < NE; ++j) {
          s[j] = expf(l[j] - m);
          sum += s[j];
        }
        sum = lanes_sum<L>(sum);
#pragma unroll
        for (int j = 0; j < NE; ++j) s[j] = s[j] / sum;
      } else {
#pragma unroll
        for (int j = 0; j < NE; ++j) s[j] = sigmoid_f(l[j]);
      }
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        const float v = s[j] + (j < n ? a.bias[i0 + j] : 0.f);
        key[j] = order_key(l[j] == -INFINITY ? -INFINITY : v);
      }
    } else {
      if (sums) {
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < NE; ++j) sum += expf(l[j] - m);
        sum = lanes_sum<L>(sum);
      }
#pragma unroll
      for (int j = 0; j < NE; ++j) key[j] = order_key(l[j]);
    }
    if constexpr (NC > 0)
#pragma unroll
      for (int j = 0; j < NE; j += 4)
        *reinterpret_cast<uint4*>(keys + lane * P + j) = make_uint4(key[j], key[j + 1], key[j + 2], key[j + 3]);
    unsigned open = 0u;                           // bit g: group g stays open (up to 32 groups)
    if (a.groups > 1) {
      unsigned k1 = 0u, k2 = 0u;                  // the group's two best
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        k2 = max(k2, min(k1, key[j]));
        k1 = max(k1, key[j]);
      }
      for (int o = 1; o < span; o <<= 1) {
        const unsigned o1 = __shfl_xor_sync(0xffffffffu, k1, o), o2 = __shfl_xor_sync(0xffffffffu, k2, o);
        k2 = max(min(k1, o1), max(k2, o2));
        k1 = max(k1, o1);
      }
      const float f1 = key_float(k1), f2 = key_float(k2);
      const float v1 = a.bias ? f1 : a.softmax ? expf(f1 - m) : sigmoid_f(f1);
      const float v2 = a.bias ? f2 : a.softmax ? expf(f2 - m) : sigmoid_f(f2);
      unsigned gk = k1 == KEY_NAN || k1 <= KEY_CLOSED ? k1 : order_key(k2 > KEY_CLOSED ? v1 + v2 : v1);
      for (int q = 0; q < a.top_groups; ++q) {
        const unsigned best = lanes_max<L>(gk);
        const int g = lanes_first<L>(gk == best, base) >> shift;
        if (best <= KEY_CLOSED) continue;         // nothing open is left for this token
        open |= 1u << g;
        if (g == mine) gk = 0u;
      }
      if (!((open >> (mine & 31)) & 1u))
#pragma unroll
        for (int j = 0; j < NE; ++j) key[j] = 0u;
      else if (NC > 0 && NC < NE && sub == mine << shift)
        opened[__popc(open & ((1u << mine) - 1u))] = mine;
    }
    if constexpr (NC == 0) {
      for (int q = 0; q < a.k; ++q) {
        unsigned t[NE];                           // the lane's best, as a tree
#pragma unroll
        for (int j = 0; j < NE; ++j) t[j] = key[j];
#pragma unroll
        for (int w = NE; w > 1; w = (w + 1) / 2)
#pragma unroll
          for (int j = 0; j < w / 2; ++j) t[j] = max(t[j], t[j + (w + 1) / 2]);
        const unsigned best = lanes_max<L>(t[0]);
        if (sub == lanes_first<L>(t[0] == best, base)) {
          bool left = true;
          int at = 0;
#pragma unroll
          for (int j = 0; j < NE; ++j) {          // the first of the lane's keys that has it
            const bool hit = left && key[j] == best;
            left = left && key[j] != best;
            if (hit) key[j] = 0u, at = j;
          }
          chosen[q] = best > KEY_CLOSED ? i0 + at : -1;
        }
      }
    } else {
      __syncwarp();
      unsigned h[4 * NL];
      unsigned from[NL];                            // a list's place in shared memory, and its first expert
      if constexpr (NC < NE) {
        const int count = __popc(open);
#pragma unroll
        for (int u = 0; u < NL; ++u) {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          from[u] = 0;
          if (nth[u] < count) {
            const int g = opened[nth[u]], place = (base + (g << shift)) * P + at[u];
            v = *reinterpret_cast<const uint4*>(keys + place);
            from[u] = place | (unsigned)(g * per + off[u]) << 16;
          }
          h[4 * u] = v.x, h[4 * u + 1] = v.y, h[4 * u + 2] = v.z, h[4 * u + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int u = 0; u < NL; ++u) from[u] = (lane * P + 4 * u) | (unsigned)(i0 + 4 * u) << 16;
#pragma unroll
        for (int j = 0; j < NE; ++j) h[j] = key[j];
      }
#pragma unroll
      for (int u = 0; u < NL; ++u) {                // each four in descending order
        auto order = [&](int i, int j) {
          const unsigned hi = max(h[4 * u + i], h[4 * u + j]), lo = min(h[4 * u + i], h[4 * u + j]);
          h[4 * u + i] = hi;
          h[4 * u + j] = lo;
        };
        order(0, 1), order(2, 3), order(0, 2), order(1, 3), order(1, 2);
      }
      unsigned before = 0u;                         // the lane's last best key, and how often it had the same one
      int same = 0;
      for (int q = 0; q < a.k; ++q) {
        unsigned t[NL];                             // the best of the lists' heads, as a tree
#pragma unroll
        for (int u = 0; u < NL; ++u) t[u] = h[4 * u];
#pragma unroll
        for (int w = NL; w > 1; w = (w + 1) / 2)
#pragma unroll
          for (int u = 0; u < w / 2; ++u) t[u] = max(t[u], t[u + (w + 1) / 2]);
        const unsigned best = lanes_max<L>(t[0]);
        const bool win = sub == lanes_first<L>(t[0] == best, base);
        bool left = win;
#pragma unroll
        for (int u = 0; u < NL; ++u) {              // one of the lane's lists that have it gives its head away
          const bool hit = left && h[4 * u] == best;
          left = left && h[4 * u] != best;
#pragma unroll
          for (int x = 0; x < 4; ++x) h[4 * u + x] = hit ? (x < 3 ? h[4 * u + x + 1] : 0u) : h[4 * u + x];
        }
        if (win) {
          same = best == before ? same + 1 : 0;
          before = best;
          best_of[q] = best;
          chosen[q] = lane | same << 8;
        }
      }
      __syncwarp();
      // whose key it was: the winner's keys compared once more, one slot per lane
      for (int r = 0; r < a.k; r += L) {
        const int q = r + sub;
        const unsigned best = q < a.k ? best_of[q] : 0u;
        const int who = q < a.k ? chosen[q] : lane;
        int i = -1;
        unsigned hits = 0u;
        unsigned where[NL];
#pragma unroll
        for (int u = 0; u < NL; ++u) {
          where[u] = __shfl_sync(0xffffffffu, from[u], who & 31);
          const uint4 v = *reinterpret_cast<const uint4*>(keys + (where[u] & 0xFFFF));
          hits |= (v.x == best ? 1u : 0u) << 4 * u | (v.y == best ? 2u : 0u) << 4 * u | (v.z == best ? 4u : 0u) << 4 * u |
                  (v.w == best ? 8u : 0u) << 4 * u;
        }
        for (int x = who >> 8; x > 0; --x) hits &= hits - 1u;      // equal keys: the first ones went to earlier slots
        const int bit = __ffs(hits) - 1;
#pragma unroll
        for (int u = 0; u < NL; ++u)
          if (bit >> 2 == u) i = (int)(where[u] >> 16) + (bit & 3);
        if (q < a.k) chosen[q] = best > KEY_CLOSED ? i : -1;
      }
    }
    __syncwarp();
    // weights: the chosen logits once more, L slots at a time
    // renormalised softmax weights depend on the chosen logits alone: relative to the best of them, as in the gradient (the
    // row's largest logit may be out of exp's range above all that a bias or the groups left)
    if (a.softmax && a.renorm) {
      if (!a.bias) {                              // the first choice has it
        const int i = chosen[0];
        m = live && i >= 0 ? to_f(p[i]) : 0.f;
      } else {
        m = -INFINITY;
        for (int q = sub; q < a.k; q += L) {
          const int i = chosen[q];
          if (live && i >= 0) m = fmaxf(m, to_f(p[i]));
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (m == -INFINITY) m = 0.f;
      }
    }
    float tot = 0.f;
    for (int q = sub; q < a.k; q += L) {
      const int i = chosen[q];
      if (live && i >= 0) {
        const float v = to_f(p[i]);
        tot += a.softmax ? expf(v - m) : sigmoid_f(v);
      }
    }
    tot = a.renorm ? lanes_sum<L>(tot) : sum;
    if (live)
      for (int q = sub; q < a.k; q += L) {
        const int i = chosen[q];
        float w = 0.f;
        if (i >= 0 && (tot > 0.f || tot != tot)) {
          const float v = to_f(p[i]);
          w = a.scale * ((a.softmax ? expf(v - m) : sigmoid_f(v)) / tot);
        }
        a.w[row * a.k + q] = w;
        a.idx[row * a.k + q] = i;
      }
    __syncwarp();
  }
}

// Scores of one token's experts, one warp per token (lane holds i = lane + 32 j): softmax numerators and their sum
template <int NE>
__device__ __forceinline__ float route_scores(const float (&l)[NE], float (&s)[NE]) {
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

// Gradient of weights that depend on the chosen logits alone: slots in lanes, K2 >= k lanes per token, `tpw` tokens per
// warp.  The tile of dense rows is built in shared memory.
template <typename T, int K2>
__global__ void __launch_bounds__(32 * RT_WARPS) k_route_bwd_sparse(const RouteArgs a, int tpw, int tile_bytes) {
  extern __shared__ __align__(16) unsigned char sm_raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tok = lane / K2, q = lane & (K2 - 1);
  T* tile = reinterpret_cast<T*>(sm_raw + (int64_t)warp * tile_bytes);
  const int64_t step = (int64_t)gridDim.x * RT_WARPS * tpw;
  for (int64_t r0 = ((int64_t)blockIdx.x * RT_WARPS + warp) * tpw; r0 < a.t; r0 += step) {
    const int rows = a.t - r0 < tpw ? (int)(a.t - r0) : tpw;
    const int64_t row = r0 + tok;
    int i = -1;
    float dw = 0.f, l = -INFINITY;
    if (tok < rows && q < a.k) {
      i = a.cidx[row * a.k + q];
      if (i < 0 || i >= a.e) i = -1;
      if (i >= 0) {
        dw = a.scale * a.dw[row * a.k + q];
        l = to_f(((const T*)a.logits)[row * a.ldl + i]);
      }
    }
    for (int o = lane * 16; o < tile_bytes; o += 512)
      *reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(tile) + o) = make_uint4(0u, 0u, 0u, 0u);
    float sc;
    if (a.softmax) {
      float m = l;
#pragma unroll
      for (int o = K2 / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      sc = i >= 0 ? expf(l - (m == -INFINITY ? 0.f : m)) : 0.f;
    } else {
      sc = i >= 0 ? sigmoid_f(l) : 0.f;
    }
    float up;
    if (a.renorm) {
      const float tot = lanes_sum<K2>(sc);
      const float w = tot > 0.f || tot != tot ? sc / tot : 0.f;
      up = w * (dw - lanes_sum<K2>(dw * w));
    } else {
      up = dw * sc;
    }
    if (!a.softmax) up *= 1.f - sc;
    __syncwarp();
    if (i >= 0) tile[tok * a.e + i] = from_f<T>(up);
    __syncwarp();
    T* dl = (T*)a.dl + r0 * a.e;
    const int total = rows * a.e;
    if ((reinterpret_cast<uintptr_t>(dl) & 15) == 0) {
      const int nv = total / kVec<T>;
      for (int o = lane; o < nv; o += 32) reinterpret_cast<uint4*>(dl)[o] = reinterpret_cast<const uint4*>(tile)[o];
      for (int o = nv * kVec<T> + lane; o < total; o += 32) dl[o] = tile[o];
    } else {
      for (int o = lane; o < total; o += 32) dl[o] = tile[o];
    }
    __syncwarp();
  }
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

// Gradient of plain softmax weights (not renormalised), one warp per token: dl_i = s_i (ds_i - sum_j s_j ds_j)
template <typename T, int NE>
__global__ void __launch_bounds__(32 * RT_WARPS) k_route_bwd(const RouteArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t row = (int64_t)blockIdx.x * RT_WARPS + warp; row < a.t; row += (int64_t)gridDim.x * RT_WARPS) {
    float l[NE], s[NE];
    route_load<T, NE>(a, row, lane, l);
    const float sum = route_scores<NE>(l, s);
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const int mine = lane < a.k ? a.cidx[row * a.k + lane] : -1;
    const float dw = lane < a.k && mine >= 0 ? a.scale * a.dw[row * a.k + lane] : 0.f;
    float out[NE], all = 0.f;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      s[j] *= inv;
      out[j] = 0.f;
    }
    for (int q = 0; q < a.k; ++q) {
      const int i = __shfl_sync(0xffffffffu, mine, q);
      const float v = __shfl_sync(0xffffffffu, dw, q);
#pragma unroll
      for (int j = 0; j < NE; ++j)
        if (i == lane + 32 * j) out[j] = s[j] * v, all += out[j];
    }
    all = warp_sum(all);
    T* dl = (T*)a.dl + row * a.e;
#pragma unroll
    for (int j = 0; j < NE; ++j)
      if (lane + 32 * j < a.e) dl[lane + 32 * j] = from_f<T>(out[j] - s[j] * all);
  }
}

static unsigned route_grid(int64_t tokens, int per_block, int blocks_per_sm) {
  const int64_t want = (tokens + per_block - 1) / per_block, most = (int64_t)blocks_per_sm * sm_count();
  return (unsigned)(want < most ? want : most);
}

template <typename T, int NE>
static int route_bwd_dense(const RouteArgs& a, cudaStream_t st) {
  k_route_bwd<T, NE><<<route_grid(a.t, RT_WARPS, 16), 32 * RT_WARPS, 0, st>>>(a);
  return check_launch("route_bwd");
}

template <typename T, int K2>
static int route_bwd_sparse(const RouteArgs& a, cudaStream_t st) {
  // tokens per warp: as many as there are lanes for, within 4 KB of rows
  const int row = a.e * (int)sizeof(T);
  int tpw = 32 / K2;
  while (tpw > 1 && tpw * row > 4096) tpw /= 2;
  const int tile = (tpw * row + 15) / 16 * 16;
  k_route_bwd_sparse<T, K2><<<route_grid(a.t, RT_WARPS * tpw, 8), 32 * RT_WARPS, RT_WARPS * tile, st>>>(a, tpw, tile);
  return check_launch("route_bwd");
}

template <typename T>
static int route_bwd_any(const RouteArgs& a, cudaStream_t st) {
  if (!a.softmax || a.renorm) {
    if (a.k == 1) return route_bwd_sparse<T, 1>(a, st);
    if (a.k <= 2) return route_bwd_sparse<T, 2>(a, st);
    if (a.k <= 4) return route_bwd_sparse<T, 4>(a, st);
    if (a.k <= 8) return route_bwd_sparse<T, 8>(a, st);
    if (a.k <= 16) return route_bwd_sparse<T, 16>(a, st);
    return route_bwd_sparse<T, 32>(a, st);
  }
  if (a.e <= 32) return route_bwd_dense<T, 1>(a, st);
  if (a.e <= 64) return route_bwd_dense<T, 2>(a, st);
  if (a.e <= 128) return route_bwd_dense<T, 4>(a, st);
  if (a.e <= 256) return route_bwd_dense<T, 8>(a, st);
  return route_bwd_dense<T, 16>(a, st);
}

template <typename T, int L, int NE, int NC>
static int route_fwd_go(const RouteArgs& a, cudaStream_t st) {
  const int smem = RT_WARPS * rt_words<L, NE, NC>(a.k) * 4;
  static_assert(RT_WARPS * rt_words<L, NE, NC>(MB_ROUTE_MAX_K) * 4 <= 48 * 1024, "shared memory of a block");
  k_route_fwd<T, L, NE, NC><<<route_grid(a.t, RT_WARPS * (32 / L), 8), 32 * RT_WARPS, smem, st>>>(a);
  return check_launch("route_fwd");
}

template <typename T, int L, int NE>
static int route_fwd_launch(RouteArgs a, cudaStream_t st) {
  constexpr int V = kVec<T>;
  const int per = a.e / a.groups;
  a.vec = NE % V == 0 && a.c % V == 0 && per % V == 0 && a.ldl % V == 0 && aligned16(a.logits);
  if (a.k <= 2) return route_fwd_go<T, L, NE, 0>(a, st);
  if constexpr (NE % 8 == 0 && NE <= 16)
    if (a.groups > 1 && per % 4 == 0 && a.c % 4 == 0 && a.top_groups * per <= L * NE / 2)
      return route_fwd_go<T, L, NE, NE / 2>(a, st);
  return route_fwd_go<T, L, NE, NE>(a, st);
}

template <typename T, int L>
static int route_fwd_lanes(const RouteArgs& a, cudaStream_t st) {
  if (a.c <= 4) return route_fwd_launch<T, L, 4>(a, st);
  if (a.c <= 8) return route_fwd_launch<T, L, 8>(a, st);
  if (a.c <= 12) return route_fwd_launch<T, L, 12>(a, st);
  if (a.c <= 16) return route_fwd_launch<T, L, 16>(a, st);
  return route_fwd_launch<T, 32, 32>(a, st);      // c > 16 only when 32 lanes are in use
}

// Lanes per group (a power of two) and experts per lane.  Many tokens: the fewest lanes that hold 16 experts or fewer each;
// below 8 tokens per scheduler: as many lanes as there are, for the shortest chain.
template <typename T>
static int route_fwd_any(RouteArgs a, cudaStream_t st) {
  constexpr int V = kVec<T>;
  const int per = a.e / a.groups;
  int most = 1;                                   // most lanes a group can have
  while (2 * most * a.groups <= 32) most *= 2;
  if (a.t < (int64_t)32 * sm_count()) {
    a.span = most;
  } else {
    a.span = 1;
    while (a.span < most && (per + a.span - 1) / a.span > 16) a.span *= 2;
  }
  a.c = (per + a.span - 1) / a.span;
  if (per % V == 0) a.c = (a.c + V - 1) / V * V;  // whole vectors; the group's last lanes hold fewer
  const int lanes = a.groups * a.span;
  if (lanes <= 4 && a.c <= 16) return route_fwd_lanes<T, 4>(a, st);
  if (lanes <= 8 && a.c <= 16) return route_fwd_lanes<T, 8>(a, st);
  if (lanes <= 16 && a.c <= 16) return route_fwd_lanes<T, 16>(a, st);
  return route_fwd_lanes<T, 32>(a, st);
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
  if (dtype == MB_F32) return bwd ? route_bwd_any<float>(a, st) : route_fwd_any<float>(a, st);
  if (dtype == MB_BF16) return bwd ? route_bwd_any<bf16>(a, st) : route_fwd_any<bf16>(a, st);
  return bwd ? route_bwd_any<f16>(a, st) : route_fwd_any<f16>(a, st);
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
