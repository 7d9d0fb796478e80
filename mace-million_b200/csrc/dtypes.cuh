// Element types of the operators that take fp32, bf16 or fp16 tensors (MB_F32 / MB_BF16 / MB_F16): conversions to and
// from fp32, one element or one 16-byte vector at a time.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace mb {

using bf16 = __nv_bfloat16;
using f16 = __half;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(f16 v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ f16 from_f<f16>(float v) { return __float2half_rn(v); }

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);   // elements of one 16-byte vector

// 16 bytes <-> kVec<T> floats
__device__ __forceinline__ void unpack16(const uint4& u, float (&f)[4], float) {
  f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack16(const uint4& u, float (&f)[8], bf16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void unpack16(const uint4& u, float (&f)[8], f16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
// two floats to one 32-bit word of two 16-bit elements (round to nearest even), the first in the low half
__device__ __forceinline__ uint32_t pack2(float a, float b, bf16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, f16) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&f)[8]) {
  return make_uint4(pack2(f[0], f[1], T()), pack2(f[2], f[3], T()), pack2(f[4], f[5], T()), pack2(f[6], f[7], T()));
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&f)[4]) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

// V consecutive elements as floats / from floats: V = kVec<T> is one 16-byte access (16-byte aligned), V = 1 one element
template <typename T, int V>
__device__ __forceinline__ void load_v(const T* p, float (&f)[V]) {
  if constexpr (V == 1)
    f[0] = to_f(*p);
  else
    unpack16(*reinterpret_cast<const uint4*>(p), f, T());
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float (&f)[V]) {
  if constexpr (V == 1)
    *p = from_f<T>(f[0]);
  else
    *reinterpret_cast<uint4*>(p) = pack16<T>(f);
}
// Arithmetic on one element or on a packed pair (one instruction for both); roundings are explicit, nothing is contracted
template <int V>
using Elem = std::conditional_t<V == 1, float, float2>;
template <int V>
constexpr int kElems = V == 1 ? 1 : V / 2;
__device__ __forceinline__ float e_add(float a, float b) { return __fadd_rn(a, b); }
__device__ __forceinline__ float e_mul(float a, float b) { return __fmul_rn(a, b); }
__device__ __forceinline__ float e_fma(float a, float b, float c) { return __fmaf_rn(a, b, c); }
__device__ __forceinline__ float2 e_add(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 e_mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 e_fma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
template <typename E>
__device__ __forceinline__ E e_splat(float v);
template <>
__device__ __forceinline__ float e_splat<float>(float v) { return v; }
template <>
__device__ __forceinline__ float2 e_splat<float2>(float v) { return make_float2(v, v); }
__device__ __forceinline__ float e_sum(float a) { return a; }
__device__ __forceinline__ float e_sum(float2 a) { return a.x + a.y; }
// V floats as elements and back
template <int V>
__device__ __forceinline__ void to_elems(const float (&f)[V], Elem<V> (&e)[kElems<V>]) {
  if constexpr (V == 1) {
    e[0] = f[0];
  } else {
#pragma unroll
    for (int q = 0; q < V / 2; ++q) e[q] = make_float2(f[2 * q], f[2 * q + 1]);
  }
}
template <int V>
__device__ __forceinline__ void from_elems(const Elem<V> (&e)[kElems<V>], float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = e[0];
  } else {
#pragma unroll
    for (int q = 0; q < V / 2; ++q) f[2 * q] = e[q].x, f[2 * q + 1] = e[q].y;
  }
}

// The same, kept as loaded until used: V elements of T in the fewest registers
template <typename T, int V>
struct Raw {
  uint4 u;
  __device__ __forceinline__ void zero() { u = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&f)[V]) const { unpack16(u, f, T()); }
  // unpack again at the next use instead of keeping the floats
  __device__ __forceinline__ void again() { asm volatile("" : "+r"(u.x), "+r"(u.y), "+r"(u.z), "+r"(u.w)); }
};
template <typename T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void zero() { v = from_f<T>(0.f); }
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_f(v); }
  __device__ __forceinline__ void again() {}
};
// V parameters of type P (as many bytes as V elements of a possibly narrower type need)
template <typename P, int V>
__device__ __forceinline__ void load_p(const P* p, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = to_f(*p);
  } else if constexpr (V == kVec<P>) {
    unpack16(*reinterpret_cast<const uint4*>(p), f, P());
  } else {                                        // fp32 parameters of 16-bit rows: two vectors
    static_assert(V == 8 && sizeof(P) == 4, "parameter vector");
    float a[4], b[4];
    unpack16(reinterpret_cast<const uint4*>(p)[0], a, float());
    unpack16(reinterpret_cast<const uint4*>(p)[1], b, float());
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = a[i];
      f[4 + i] = b[i];
    }
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline int dtype_size(int dt) { return dt == MB_F32 ? 4 : 2; }
inline bool dtype_ok(int dt) { return dt == MB_F32 || dt == MB_BF16 || dt == MB_F16; }
int sm_count();                                  // SMs of the current device (cached per device), <= 0 on failure

}  // namespace mb
