// Operands of the gated delta rule shared by its kernels (delta_step.hip, delta_chunk.hip,
// delta_grad.hip).
#pragma once

#include "lane_types.h"

// log decays below this are taken as this: exp of it is 0, and sums of 64 of them keep the
// differences of the others exact to 1e-9 in 64 bits, so g = -inf resets the state.
#define BS_DELTA_G_MIN (-1e4f)

#define BS_DELTA_MAX_DIM 128

int bs_delta_check(const bs_delta_in* in, const char* who);

// Offset in elements of (batch, token, head) with strides s.
__device__ __forceinline__ int64_t bs_delta_at(const int64_t* s, int64_t b, int64_t t, int h) {
  return b * s[0] + t * s[1] + (int64_t)h * s[2];
}

__device__ __forceinline__ float bs_delta_g(const bs_delta_in& in, int64_t b, int64_t t, int h) {
  const float g = bs_load_any(in.g, in.g_dtype, bs_delta_at(in.g_stride, b, t, h));
  return g < BS_DELTA_G_MIN ? BS_DELTA_G_MIN : g;   // NaN stays
}
__device__ __forceinline__ float bs_delta_beta(const bs_delta_in& in, int64_t b, int64_t t,
                                               int h) {
  return bs_load_any(in.beta, in.beta_dtype, bs_delta_at(in.beta_stride, b, t, h));
}
