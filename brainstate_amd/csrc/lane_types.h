// Element types and matrix-core helpers of the sequence-layer operators (delta_*.hip, norm.hip,
// int8.hip).
#pragma once

#include "common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

using bs_f32x4 = __attribute__((__vector_size__(4 * sizeof(float)))) float;
using bs_bf16x8 = __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16;
using bs_u16x8 = __attribute__((__vector_size__(8 * sizeof(uint16_t)))) uint16_t;

// Storage of one element; bf16 and fp16 are held by their bits.
struct bs_bf16 { uint16_t u; };
struct bs_f16 { uint16_t u; };

__device__ __forceinline__ float bs_to_f32(float x) { return x; }
__device__ __forceinline__ float bs_to_f32(bs_bf16 x) {
  return __uint_as_float((uint32_t)x.u << 16);
}
__device__ __forceinline__ float bs_to_f32(bs_f16 x) {
  return (float)__builtin_bit_cast(_Float16, x.u);
}

template <typename T>
__device__ __forceinline__ T bs_from_f32(float x);
template <>
__device__ __forceinline__ float bs_from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ bs_bf16 bs_from_f32<bs_bf16>(float x) {  // to nearest, ties to even
  return bs_bf16{__builtin_bit_cast(uint16_t, (__bf16)x)};
}
template <>
__device__ __forceinline__ bs_f16 bs_from_f32<bs_f16>(float x) {
  return bs_f16{__builtin_bit_cast(uint16_t, (_Float16)x)};
}

// Four neighbouring values in one store; p is aligned to all four.
template <typename T>
__device__ __forceinline__ void bs_store4(T* p, const bs_f32x4& x) {
  if constexpr (sizeof(T) == 4) {
    *(bs_f32x4*)p = x;
  } else {
    uint2 v;
    v.x = bs_from_f32<T>(x[0]).u | (uint32_t)bs_from_f32<T>(x[1]).u << 16;
    v.y = bs_from_f32<T>(x[2]).u | (uint32_t)bs_from_f32<T>(x[3]).u << 16;
    *(uint2*)p = v;
  }
}

// Element i of an array whose type is known at run time (gates, norm weights).
__device__ __forceinline__ float bs_load_any(const void* p, int dtype, int64_t i) {
  if (dtype == BS_F32) return ((const float*)p)[i];
  if (dtype == BS_BF16) return bs_to_f32(((const bs_bf16*)p)[i]);
  return bs_to_f32(((const bs_f16*)p)[i]);
}
__device__ __forceinline__ void bs_store_any(void* p, int dtype, int64_t i, float x) {
  if (dtype == BS_F32) ((float*)p)[i] = x;
  else if (dtype == BS_BF16) ((bs_bf16*)p)[i] = bs_from_f32<bs_bf16>(x);
  else ((bs_f16*)p)[i] = bs_from_f32<bs_f16>(x);
}

static inline int bs_dtype_ok(int d) { return d == BS_F32 || d == BS_BF16 || d == BS_F16; }
static inline int bs_dtype_size(int d) { return d == BS_F32 ? 4 : 2; }

// ---------------------------------------------------------------- products in 32 bits
// The matrix cores multiply bf16.  A 32-bit value is the exact sum of three bf16 values (its
// significand's 24 bits in pieces of 8, each cut off, not rounded), an fp16 value of two, so a
// product of 32-bit accuracy is the sum of those part products that reach 2^-24: part p has
// weight 2^-8p, and pairs with p + q > 2 are left out.  A pair costs one instruction, so a
// 32-bit operand against a bf16 one costs 3 and two of them 6, where the fp32 matrix
// instruction costs 16.
template <int P>
struct bs_parts { bs_bf16x8 p[P]; };

__device__ __forceinline__ uint32_t bs_pack_hi(float lo, float hi) {
  // upper 16 bits of `lo` into the lower half, of `hi` into the upper
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float bs_cut(float x) {
  return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
}

// Parts of four values, as two words of two bf16 each.
template <int P>
__device__ __forceinline__ void bs_split4(const float* x, uint2* out) {
  float r[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
  for (int p = 0; p < P; ++p) {
    out[p] = make_uint2(bs_pack_hi(r[0], r[1]), bs_pack_hi(r[2], r[3]));
    if (p + 1 < P) {
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] -= bs_cut(r[i]);
    }
  }
}

template <int P>
__device__ __forceinline__ bs_parts<P> bs_split8(const float* x) {
  uint2 a[P], b[P];
  bs_split4<P>(x, a);
  bs_split4<P>(x + 4, b);
  bs_parts<P> o;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint4 w = make_uint4(a[p].x, a[p].y, b[p].x, b[p].y);
    o.p[p] = __builtin_bit_cast(bs_bf16x8, w);
  }
  return o;
}

// acc += a b over 32 products a lane group: parts p, q with p + q <= S.
template <int S, int PA, int PB>
__device__ __forceinline__ bs_f32x4 bs_mma(const bs_parts<PA>& a, const bs_parts<PB>& b,
                                           bs_f32x4 acc) {
#pragma unroll
  for (int s = S; s >= 0; --s)
#pragma unroll
    for (int p = 0; p <= s; ++p)
      if (p < PA && s - p < PB)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[p], b.p[s - p], acc, 0, 0, 0);
  return acc;
}
