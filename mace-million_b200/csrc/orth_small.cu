// Orthogonalised matrices whose short side r is at most 128, all steps on the chip: one launch, a matrix per cluster of up to 8 CTAs.
// The formulas, the fp16 operands and the separate diagonals are those of orth.cu; what differs is where things lie:
//  * X is handled as [r][l] (a tall matrix is transposed while it is read and written) and cut along l over the CTAs.
//  * X stays in fp32 in TMEM next to the accumulators (LS and max(128, LS) of its columns), a lane is a row.  Its fp16 form lies in
//    shared memory in blocks of 64 columns (128-byte swizzled rows), which the Gram product reads K-major (K = l) and the update as
//    its MN-major operand (K = r) from the same bytes.
//  * A1, then b A + c A A over it, is one 128 x 128 plane in shared memory; each thread turns its own elements.
//  * With several CTAs the Gram product's partial sums are added through distributed shared memory: of two each adds the other's to
//    its own (the same sums in both), of more each adds a slice in the order of the ranks and stores it, rounded, to all.
// 256 threads: eight warps hold the rows (two halves of the columns), one thread issues the products between block barriers.
// Bound: latency.  A step is three products of 8 to 16 MMAs and three passes over TMEM, each behind a barrier (1,450 cycles for 8
// MMAs of 64, 500 to 2,000 a pass).  Measured on a B200 (5 steps, bf16): 8 of 64 x 128 20 us, 128 x 128 26, 256 x 128 33,
// 512 x 128 47 (two CTAs; a third of it the sums through distributed shared memory), 89 of 512 x 128 95 (178 CTAs on 148 SMs:
// two rounds).  The kernel over the whole GPU took 82, 82 and 187 us for the first, the second and the last.
#include <type_traits>

#include "dtypes.cuh"
#include "orth.cuh"
#include "tc.cuh"

namespace mb {

constexpr int OS_THREADS = 256, OS_BLOCK = 128 * 128;   // bytes of 128 rows of 64 fp16 columns
constexpr int OS_MAX_LS = 256, OS_MAX_P = 8;

struct OsArgs {
  const void* g;
  bf16* out;
  int64_t ldb, ldg;
  int32_t m, n, r, l, ls, tall, vec;              // ls: columns of a CTA (a multiple of 64)
  OrPoly poly;
};

struct OsShared {
  double norm[2];                                 // of the CTA, of the matrix
  double red[8];
  alignas(16) float d[128], e[128];
  uint64_t bar;
  uint32_t tmem;
  int failed;
};

__device__ __forceinline__ uint32_t os_piece(int row, int col8) {   // 16-byte piece col8 of a row in blocks of 64 columns
  return (uint32_t)((col8 >> 3) * OS_BLOCK + row * 128 + (((col8 & 7) ^ (row & 7)) << 4));
}
__device__ __forceinline__ double ld_cluster_f64(uint32_t a) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_u32x4(uint32_t a, const uint4& v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void st_cluster_f32(uint32_t a, float x) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(x) : "memory");
}

// The lane's own of its 32 values, which becomes 0 (selects: a store in a branch for each was ten times as long)
__device__ __forceinline__ float os_diagonal(float (&v)[32], int lane) {
  float d = 0.f;
#pragma unroll
  for (int x = 0; x < 32; ++x) {
    const bool on = x == lane;
    d = on ? v[x] : d;
    v[x] = on ? 0.f : v[x];
  }
  return d;
}

template <typename T>
__global__ void __launch_bounds__(OS_THREADS, 1) k_orth_small(const __grid_constant__ OsArgs g) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ OsShared S;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, P = gridDim.x, rank = blockIdx.x;
  // rp: columns of A that are worked on, 64 where that is enough (with one CTA)
  const int row = (warp & 3) * 32 + lane, half = warp >> 2, ls = g.ls, rp = g.r <= 64 && P == 1 ? 64 : 128;
  const uint32_t plane = smem_u32(smem), xs = plane + 2 * OS_BLOCK;   // A1 / B1, X, partial sums
  const uint32_t sums = xs + ls / 64 * OS_BLOCK;
  const uint32_t cols = ls == 64 ? 256u : ls == 128 ? 256u : 512u;
  if (warp == 0) {
    tmem_alloc<1>(&S.tmem, cols);
    if (lane == 0) {
      mbar_init(&S.bar, 1);
      S.failed = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  if (tid < 128) S.d[tid] = S.e[tid] = 0.f;       // (rows from rp on have none)
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tx = S.tmem, td = tx + ls, lanes = (uint32_t)((warp & 3) * 32) << 16;   // X, accumulators
  const int c0 = rank * ls, h0 = half * (ls / 2), hw = ls / 2;        // this CTA's columns, this warp's of them
  auto barrier = [&] {                            // over the matrix
    if (P > 1)
      cluster_sync();
    else
      __syncthreads();
  };

  // ---------------------------------------------------------------------------------------------- G and its norm
  const T* gp = (const T*)g.g + blockIdx.y * g.ldb;
  double sq = 0.0;
  for (int c = 0; c < hw; c += 32) {
    const int j0 = c0 + h0 + c, nc = g.l - j0;
    uint32_t u[32];
    float f[32];
#pragma unroll
    for (int x = 0; x < 32; ++x) f[x] = 0.f;
    if (row < g.r && nc > 0) {
      if (g.tall) {
        const T* p = gp + (int64_t)j0 * g.ldg + row;
        if (nc >= 32) {
          T t[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) t[x] = p[(int64_t)x * g.ldg];
#pragma unroll
          for (int x = 0; x < 32; ++x) f[x] = to_f(t[x]);
        } else {
          for (int x = 0; x < 32; ++x)
            if (x < nc) f[x] = to_f(p[(int64_t)x * g.ldg]);
        }
      } else {
        const T* p = gp + (int64_t)row * g.ldg + j0;
        constexpr int V = kVec<T>;
        if (g.vec && nc >= 32) {
#pragma unroll
          for (int q = 0; q < 32 / V; ++q) {
            float t[V];
            load_v<T, V>(p + q * V, t);
#pragma unroll
            for (int x = 0; x < V; ++x) f[q * V + x] = t[x];
          }
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x)
            if (x < nc) f[x] = to_f(p[x]);
        }
      }
    }
    __syncwarp();
    // 32 squares in fp32 where they neither overflow nor vanish, else in fp64
    float s32 = 0.f, top = 0.f;
#pragma unroll
    for (int x = 0; x < 32; ++x) {
      s32 = fmaf(f[x], f[x], s32);
      top = fmaxf(top, fabsf(f[x]));
      u[x] = __float_as_uint(f[x]);
    }
    if (top > 1e-15f && top < 1e15f)
      sq += (double)s32;
    else
#pragma unroll
      for (int x = 0; x < 32; ++x) {
        const double v = __uint_as_float(u[x]);
        sq = fma(v, v, sq);
      }
    __syncwarp();
    tmem_st32(tx + lanes + h0 + c, u);
  }
  tmem_wait_st();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
  if (lane == 0) S.red[warp] = sq;
  __syncthreads();
  if (tid == 0) {
    sq = 0.0;
    for (int q = 0; q < 8; ++q) sq += S.red[q];
    S.norm[0] = sq;
  }
  barrier();
  if (tid == 0) {
    sq = 0.0;
    for (int q = 0; q < P; ++q) sq += P > 1 ? ld_cluster_f64(mapa_u32(smem_u32(S.norm), q)) : S.norm[0];
    S.norm[1] = (double)g.poly.s / (sqrt(sq) + g.poly.eps);
  }
  __syncthreads();
  const float scale = (float)S.norm[1];

  // X's 32 columns from c on to TMEM and, rounded, to shared memory
  auto put_x = [&](int c, const float (&v)[32], bool keep) {
    if (keep) {
      uint32_t u[32];
#pragma unroll
      for (int x = 0; x < 32; ++x) u[x] = __float_as_uint(v[x]);
      tmem_st32(tx + lanes + h0 + c, u);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float f[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) f[x] = v[8 * q + x];
      sts128(xs + os_piece(row, (h0 + c) / 8 + q), pack16<f16>(f));
    }
  };
  for (int c = 0; c < hw; c += 32) {
    uint32_t u[32];
    float v[32];
    tmem_ld32(tx + lanes + h0 + c, u);
    tmem_wait_ld();
#pragma unroll
    for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(u[x]) * scale;
    put_x(c, v, true);
  }
  tmem_wait_st();

  int phase = 0;
  bool pending = false;                           // an arrival at the cluster's barrier that was not waited for
  // What the threads wrote is there for the products; `issue` runs in one thread; all wait for its products (bounded)
  auto products = [&](auto issue) {
    asm volatile("fence.proxy.async;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t lead = elect_lane();
      issue(lead);
      mma_commit_lead<1>(lead, smem_u32(&S.bar));
    }
    if (!mbar_wait_ns(&S.bar, phase & 1, OR_WAIT)) S.failed = 1;
    ++phase;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  };
  const uint32_t id_a = f16_idesc(128, rp, false, false, false), id_x = f16_idesc(128, ls, false, false, true);

  for (int step = 0; step < g.poly.steps; ++step) {
    const float ca = g.poly.a[step], cb = g.poly.b[step], cc = g.poly.c[step];
    const bool last = step == g.poly.steps - 1;
    // -------------------------------------------------------------------------------------------- A = X X^T
    products([&](uint32_t lead) {
      for (int k = 0; k < ls / 16; ++k) {
        const uint64_t a = sw128_desc(xs + (k >> 2) * OS_BLOCK + (k & 3) * 32);
        mma_f16_ss_lead<1>(lead, td, a, a, id_a, k ? 1u : 0u);
      }
    });
    // eight columns of A at a time: the diagonal apart (dia: the column among them, or outside of 0 .. 7), the rest to the plane
    const float sc = g.poly.inv_s * g.poly.inv_s * OR_SA;
    if (P == 1) {
#pragma unroll 1
      for (int c = half * (rp / 2); c < (half + 1) * (rp / 2); c += 32) {
        uint32_t u[32];
        float v[32];
        tmem_ld32(td + lanes + c, u);
        tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(u[x]) * sc;
        if (c == (warp & 3) * 32) S.d[row] = os_diagonal(v, lane) * (1.f / OR_SA);   // it runs through this piece
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float f[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) f[x] = v[8 * q + x];
          sts128(plane + os_piece(row, c / 8 + q), pack16<f16>(f));
        }
      }
      __syncthreads();
    } else {
      if (pending) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      pending = false;
#pragma unroll 1
      for (int c = half * (rp / 2); c < (half + 1) * (rp / 2); c += 32) {
        uint32_t u[32];
        tmem_ld32(td + lanes + c, u);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 8; ++q)
          sts128(sums + (uint32_t)((c / 4 + q) * 128 + row) * 16, make_uint4(u[4 * q], u[4 * q + 1], u[4 * q + 2], u[4 * q + 3]));
      }
      cluster_sync();
      if (P == 2) {                               // each CTA adds all of the other's to its own
        const uint32_t peer = mapa_u32(sums, rank ^ 1);
#pragma unroll 1
        for (int c = half * 64; c < half * 64 + 64; c += 32) {
          uint32_t u[32];
          float v[32];
          float4 t[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) t[q] = ld_cluster_f32x4(peer + (uint32_t)((c / 4 + q) * 128 + row) * 16);
          tmem_ld32(td + lanes + c, u);
          tmem_wait_ld();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            v[4 * q] = (__uint_as_float(u[4 * q]) + t[q].x) * sc, v[4 * q + 1] = (__uint_as_float(u[4 * q + 1]) + t[q].y) * sc;
            v[4 * q + 2] = (__uint_as_float(u[4 * q + 2]) + t[q].z) * sc, v[4 * q + 3] = (__uint_as_float(u[4 * q + 3]) + t[q].w) * sc;
          }
          if (c == (warp & 3) * 32) S.d[row] = os_diagonal(v, lane) * (1.f / OR_SA);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float f[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] = v[8 * q + x];
            sts128(plane + os_piece(row, c / 8 + q), pack16<f16>(f));
          }
        }
        // this CTA has read its peer's sums; it waits for its peer before it writes its own again
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        pending = true;
      }
      // else 2048 / P pieces of eight columns of a row for this CTA: 8 / P for a thread
      auto slice = [&](auto np) {
        constexpr int PP = decltype(np)::value, PER = 8 / PP;
        float f[PER][8];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int p = rank * (2048 / PP) + k * OS_THREADS + tid;
          const uint32_t at = sums + (uint32_t)((p / 128 * 2) * 128 + (p & 127)) * 16;
          float4 t[PP][2];
#pragma unroll
          for (int q = 0; q < PP; ++q) {
            const uint32_t from = mapa_u32(at, q);
            t[q][0] = ld_cluster_f32x4(from);
            t[q][1] = ld_cluster_f32x4(from + 2048);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float4 v = t[0][h];
#pragma unroll
            for (int q = 1; q < PP; ++q) v.x += t[q][h].x, v.y += t[q][h].y, v.z += t[q][h].z, v.w += t[q][h].w;
            f[k][4 * h] = v.x * sc, f[k][4 * h + 1] = v.y * sc, f[k][4 * h + 2] = v.z * sc, f[k][4 * h + 3] = v.w * sc;
          }
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int p = rank * (2048 / PP) + k * OS_THREADS + tid, i = p & 127, c8 = p / 128, dia = i - 8 * c8;
          float dv = 0.f;
#pragma unroll
          for (int x = 0; x < 8; ++x)
            if (x == dia) dv = f[k][x] * (1.f / OR_SA), f[k][x] = 0.f;
          const uint4 w = pack16<f16>(f[k]);
          const uint32_t at = plane + os_piece(i, c8), da = smem_u32(&S.d[i]);
#pragma unroll
          for (int q = 0; q < PP; ++q) {
            st_cluster_u32x4(mapa_u32(at, q), w);
            if (dia >= 0 && dia < 8) st_cluster_f32(mapa_u32(da, q), dv);
          }
        }
      };
      if (P == 4)
        slice(std::integral_constant<int, 4>());
      else if (P == 8)
        slice(std::integral_constant<int, 8>());
      if (P > 2)
        cluster_sync();
      else
        __syncthreads();
    }
    // -------------------------------------------------------------------------------------------- b A + c A A
    products([&](uint32_t lead) {
      for (int k = 0; k < rp / 16; ++k) {
        const uint64_t a = sw128_desc(plane + (k >> 2) * OS_BLOCK + (k & 3) * 32);
        mma_f16_ss_lead<1>(lead, td, a, a, id_a, k ? 1u : 0u);
      }
    });
    {
      // b a1 + c (a1 (d_i + d_j) + sq), all times SB: a1's plane is SA a1, the accumulator SA^2 sq
      const float di = S.d[row], k2 = cc * (OR_SB / OR_SA), k1 = fmaf(k2, di, cb * (OR_SB / OR_SA)), k3 = cc * (OR_SB / (OR_SA * OR_SA));
#pragma unroll 1
      for (int c = half * (rp / 2); c < (half + 1) * (rp / 2); c += 32) {
        uint32_t u[32];
        float v[32];
        tmem_ld32(td + lanes + c, u);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float f[8];
          unpack16(lds128(plane + os_piece(row, c / 8 + q)), f, f16());
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 dj = *reinterpret_cast<const float4*>(&S.d[c + 8 * q + 4 * h]);
            const float t[4] = {dj.x, dj.y, dj.z, dj.w};
#pragma unroll
            for (int x = 0; x < 4; ++x)
              v[8 * q + 4 * h + x] = fmaf(f[4 * h + x], fmaf(k2, t[x], k1), __uint_as_float(u[8 * q + 4 * h + x]) * k3);
          }
        }
        if (c == (warp & 3) * 32) S.e[row] = fmaf(cb, di, fmaf(cc * di, di, os_diagonal(v, lane) * (1.f / OR_SB)));
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float f[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) f[x] = v[8 * q + x];
          sts128(plane + os_piece(row, c / 8 + q), pack16<f16>(f));
        }
      }
      __syncthreads();
    }
    // -------------------------------------------------------------------------------------------- X <- a X + (b A + c A A) X
    products([&](uint32_t lead) {
      for (int k = 0; k < rp / 16; ++k)
        mma_f16_ss_lead<1>(lead, td, sw128_desc(plane + (k >> 2) * OS_BLOCK + (k & 3) * 32), sw128_desc_mn(xs + k * 2048, OS_BLOCK), id_x,
                           k ? 1u : 0u);
    });
    const float el = S.e[row];
    const bool grow = g.poly.grow >> step & 1;
    if (last && pending) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (last) barrier();                          // every CTA's S.failed is final
    float bad = 0.f;
    if (last) {
      for (int q = 0; q < P; ++q)
        if (P > 1 ? ld_cluster_s32(mapa_u32(smem_u32(&S.failed), q)) : *(volatile int*)&S.failed) bad = __int_as_float(0x7fc00000);
    }
#pragma unroll 1
    for (int c = 0; c < hw; c += 32) {
      uint32_t u[32], w[32];
      float v[32];
      tmem_ld32(tx + lanes + h0 + c, u);
      tmem_ld32(td + lanes + h0 + c, w);
      tmem_wait_ld();
      if (grow) {
#pragma unroll
        for (int x = 0; x < 32; ++x) v[x] = or_update<true>(ca, el, __uint_as_float(u[x]), __uint_as_float(w[x]) * (1.f / OR_SB));
      } else {
#pragma unroll
        for (int x = 0; x < 32; ++x) v[x] = or_update<false>(ca, el, __uint_as_float(u[x]), __uint_as_float(w[x]) * (1.f / OR_SB));
      }
      if (!last) {
        put_x(c, v, true);
        continue;
      }
      const int j0 = c0 + h0 + c, nc = g.l - j0;
      if (row < g.r && nc > 0) {
        bf16* o = g.out + (int64_t)blockIdx.y * g.m * g.n;
#pragma unroll
        for (int x = 0; x < 32; ++x) v[x] = fmaf(v[x], g.poly.inv_s, bad);
        if (g.tall) {
          o += (int64_t)j0 * g.n + row;
          if (nc >= 32) {
#pragma unroll
            for (int x = 0; x < 32; ++x) o[(int64_t)x * g.n] = from_f<bf16>(v[x]);
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (x < nc) o[(int64_t)x * g.n] = from_f<bf16>(v[x]);
          }
        } else {
          o += (int64_t)row * g.n + j0;
          if (nc >= 32 && g.n % 8 == 0 && (reinterpret_cast<uintptr_t>(g.out) & 15) == 0) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float f[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) f[x] = v[8 * q + x];
              *(reinterpret_cast<uint4*>(o) + q) = pack16<bf16>(f);
            }
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (x < nc) o[x] = from_f<bf16>(v[x]);
          }
        }
      }
      __syncwarp();
    }
    if (!last) tmem_wait_st();
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  barrier();                                      // no CTA leaves while its peers may read its shared memory
  if (warp == 0) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_dealloc<1>(tx, cols);
  }
}

// ------------------------------------------------------------------------------------------------ host side
static int os_ctas(int32_t l) {
  int p = 1;
  while (p * OS_MAX_LS < l) p *= 2;
  return p;
}

bool orth_small(int64_t batch, int32_t m, int32_t n) {
  const int32_t r = m < n ? m : n, l = m < n ? n : m;
  return r <= 128 && l <= OS_MAX_P * OS_MAX_LS && batch <= 65535;
}

template <typename T>
static int os_go(OsArgs& a, int p, int64_t batch, cudaStream_t st) {
  static int ready_dev = -1;
  int dev = 0;
  constexpr int MOST = 1024 + (2 + OS_MAX_LS / 64) * OS_BLOCK + 65536;
  if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("orthogonalize (device)");
  if (ready_dev != dev) {
    if (cudaFuncSetAttribute(k_orth_small<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST) != cudaSuccess) {
      set_error("orthogonalize: cannot reserve %d bytes of shared memory", MOST);
      return MB_E_CUDA;
    }
    ready_dev = dev;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p, (unsigned)batch);
  cfg.blockDim = dim3(OS_THREADS);
  cfg.dynamicSmemBytes = 1024 + (2 + a.ls / 64) * OS_BLOCK + (p > 1 ? 65536 : 0);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = p;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, k_orth_small<T>, a);
  return check_launch("orthogonalize");
}

int orth_small_launch(const void* gp, int64_t ldb, int64_t ldg, void* out, int64_t batch, int32_t m, int32_t n, const OrPoly& poly,
                      int32_t dtype, cudaStream_t st) {
  OsArgs a{};
  a.g = gp; a.out = (bf16*)out; a.ldb = ldb; a.ldg = ldg; a.m = m; a.n = n; a.poly = poly;
  a.tall = m > n;
  a.r = a.tall ? n : m;
  a.l = a.tall ? m : n;
  const int p = os_ctas(a.l), v = 16 / dtype_size(dtype);
  a.ls = ((a.l + p - 1) / p + 63) / 64 * 64;
  a.vec = ldg % v == 0 && (batch == 1 || ldb % v == 0) && aligned16(gp);
  return dtype == MB_F32    ? os_go<float>(a, p, batch, st)
         : dtype == MB_BF16 ? os_go<bf16>(a, p, batch, st)
                            : os_go<f16>(a, p, batch, st);
}

}  // namespace mb
