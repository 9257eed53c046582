// Shared helpers of the row operators (layer_norm.hip, logprobs.hip,
// act8.hip): element types, 8-element vectors at any alignment, wave
// reductions without LDS.
//
// Element types are a template argument DT with the codes of the C ABI:
// 0 = fp32, 1 = bf16, 2 = fp16.  Arithmetic is in fp32 everywhere; a value is
// rounded to DT once, when it is stored (round to nearest, ties to even).
#pragma once

#include "../common.h"

namespace {

template <int DT>
struct Elem;
template <>
struct Elem<0> {
  typedef float raw;
  static __device__ __forceinline__ float up(raw v) { return v; }
  static __device__ __forceinline__ raw down(float f) { return f; }
};
template <>
struct Elem<1> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float up(raw v) { return zk::bf16_to_f32(v); }
  static __device__ __forceinline__ raw down(float f) { return zk::f32_to_bf16(f); }
};
template <>
struct Elem<2> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float up(raw v) {
    return (float)__builtin_bit_cast(_Float16, v);
  }
  static __device__ __forceinline__ raw down(float f) {
    return __builtin_bit_cast(uint16_t, (_Float16)f);
  }
};

// 16 / 8 bytes at the element's own alignment: one global_load / store
// (unaligned vector accesses are legal for global memory on gfx950; an odd row
// length only costs the cache lines that a vector straddles).
typedef uint32_t Bytes16 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t Bytes8 __attribute__((ext_vector_type(2), aligned(1)));

// 8 elements as loaded (a row in flight takes half the registers in 16 bits).
template <int DT>
struct Raw8 {
  uint32_t v[DT == 0 ? 8 : 4];
};

// the first n (<= 8; may be negative) elements, zeros behind them
template <int DT>
__device__ __forceinline__ Raw8<DT> raw8(const typename Elem<DT>::raw* p, int n) {
  Raw8<DT> r;
  if (n >= 8) {
    const Bytes16 a = *reinterpret_cast<const Bytes16*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = a[i];
    if constexpr (DT == 0) {
      const Bytes16 b = *reinterpret_cast<const Bytes16*>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) r.v[4 + i] = b[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < (DT == 0 ? 8 : 4); ++i) {
      if constexpr (DT == 0) {
        r.v[i] = i < n ? __float_as_uint(p[i]) : 0u;
      } else {
        r.v[i] = (2 * i < n ? (uint32_t)p[2 * i] : 0u) |
                 (2 * i + 1 < n ? (uint32_t)p[2 * i + 1] << 16 : 0u);
      }
    }
  }
  return r;
}

template <int DT>
__device__ __forceinline__ float raw_at(const Raw8<DT>& r, int i) {
  if constexpr (DT == 0) {
    return __uint_as_float(r.v[i]);
  } else {
    return Elem<DT>::up((uint16_t)(r.v[i >> 1] >> (16 * (i & 1))));
  }
}

template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::raw* p, float (&f)[8]) {
  if constexpr (DT == 0) {
    const Bytes16 a = *reinterpret_cast<const Bytes16*>(p);
    const Bytes16 b = *reinterpret_cast<const Bytes16*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = __uint_as_float(a[i]);
      f[4 + i] = __uint_as_float(b[i]);
    }
  } else {
    const Bytes16 a = *reinterpret_cast<const Bytes16*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = Elem<DT>::up((uint16_t)(a[i] & 0xffffu));
      f[2 * i + 1] = Elem<DT>::up((uint16_t)(a[i] >> 16));
    }
  }
}

// the first n (0..8) elements; the rest are `fill`
template <int DT>
__device__ __forceinline__ void load8_n(const typename Elem<DT>::raw* p, int n, float fill,
                                        float (&f)[8]) {
  if (n >= 8) {
    load8<DT>(p, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? Elem<DT>::up(p[i]) : fill;
  }
}

// Two values to bf16 in one v_cvt_pk_bf16_f32 (two separate conversions take four
// instructions).
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, b16x2));
}

template <int DT>
__device__ __forceinline__ uint32_t pair16(float lo, float hi) {
  if constexpr (DT == 1) {
    return bf16_pair(lo, hi);
  } else {
    return (uint32_t)Elem<DT>::down(lo) | ((uint32_t)Elem<DT>::down(hi) << 16);
  }
}

template <int DT>
__device__ __forceinline__ void store8(typename Elem<DT>::raw* p, const float (&f)[8]) {
  if constexpr (DT == 0) {
    Bytes16 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = __float_as_uint(f[i]);
      b[i] = __float_as_uint(f[4 + i]);
    }
    *reinterpret_cast<Bytes16*>(p) = a;
    *reinterpret_cast<Bytes16*>(p + 4) = b;
  } else {
    Bytes16 a;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = pair16<DT>(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<Bytes16*>(p) = a;
  }
}

template <int DT>
__device__ __forceinline__ void store8_n(typename Elem<DT>::raw* p, int n, const float (&f)[8]) {
  if (n >= 8) {
    store8<DT>(p, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = Elem<DT>::down(f[i]);
  }
}

// Sum over aligned groups of G lanes (a power of two up to 64); every lane of
// the group ends with the total.  Fixed order.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

}  // namespace
