// Rows of values in the lanes of a wave or workgroup, shared by the norms (norm.hip, layer_norm.hip).
#pragma once

#include "lane_types.h"

#include <type_traits>

namespace {

template <int V>
using Int = std::integral_constant<int, V>;

constexpr int kVec = 8;

// How a lane's 8 columns lie: rows of whole runs; rows whose last lane takes the row's last 8
// columns, some of them a second time (it stores the same values there and leaves them out of
// sums); rows of fewer than 8 columns.  Either way a row's loads have no branch and are in flight
// together; they and the stores are of 16 bytes and any alignment.
enum Mode { kWhole, kTail, kSmall };

template <int MODE>
struct Cols {
  int c, at;              // the first column, and where its 8 are loaded
  bool in;
  float m[MODE == kTail ? kVec : 1];
  __device__ __forceinline__ Cols() {}
  __device__ __forceinline__ Cols(int first, int dim) {
    c = first, in = c < dim;
    at = MODE == kSmall ? c : min(c, dim - kVec);
    if (MODE == kTail)
#pragma unroll
      for (int j = 0; j < kVec; ++j) m[j] = in && at + j >= c ? 1.f : 0.f;
  }
  __device__ __forceinline__ float once(int j, float x) const {    // x, where column j counts
    return MODE == kTail ? m[j] * x : x;
  }
};

template <typename T, int MODE>
struct Vec8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* row, const Cols<MODE>& k, int dim) {
    if (MODE != kSmall) {
      __builtin_memcpy(w, row + k.at, sizeof(w));
    } else {
      T t[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) t[j] = k.at + j < dim ? row[k.at + j] : T{};
      __builtin_memcpy(w, t, sizeof(w));
    }
  }
  // as numbers; 0 for a lane past the row
  __device__ __forceinline__ void values(bool in, float* x) const {
    T t[kVec];
    __builtin_memcpy(t, w, sizeof(w));
#pragma unroll
    for (int j = 0; j < kVec; ++j) x[j] = in ? bs_to_f32(t[j]) : 0.f;
  }
  static __device__ __forceinline__ void store(T* row, const Cols<MODE>& k, int dim,
                                               const float* x) {
    if (!k.in) return;
    if (MODE != kSmall) {
      uint4 o[sizeof(T) / 2];
      if constexpr (sizeof(T) == 4) {
        o[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                          __float_as_uint(x[3]));
        o[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]),
                          __float_as_uint(x[7]));
      } else {
        uint32_t* u = (uint32_t*)o;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          u[j] = bs_from_f32<T>(x[2 * j]).u | (uint32_t)bs_from_f32<T>(x[2 * j + 1]).u << 16;
      }
      __builtin_memcpy(row + k.at, o, sizeof(o));
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (k.at + j < dim) row[k.at + j] = bs_from_f32<T>(x[j]);
    }
  }
};

template <typename W, int NV, int MODE>
__device__ __forceinline__ void load_typed(const W* p, const Cols<MODE>* k, int dim,
                                           float (*w)[kVec]) {
  Vec8<W, MODE> v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i].load(p, k[i], dim);
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i].values(k[i].in, w[i]);
}

template <int NV, int MODE>
__device__ __forceinline__ void load_weight(const void* p, int dtype, const Cols<MODE>* k, int dim,
                                            float fill, float (*w)[kVec]) {
  if (!p) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < kVec; ++j) w[v][j] = fill;
  } else if (dtype == BS_F32) {
    load_typed<float, NV>((const float*)p, k, dim, w);
  } else if (dtype == BS_BF16) {
    load_typed<bs_bf16, NV>((const bs_bf16*)p, k, dim, w);
  } else {
    load_typed<bs_f16, NV>((const bs_f16*)p, k, dim, w);
  }
}

// Sums over the lanes of a row: TPR of a wave, or (TPR = 0) the whole workgroup, where `turn`
// alternates so that one barrier a sum is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float* x, float (*sh)[16][N], int& turn) {
#pragma unroll
  for (int d = 1; d < (TPR ? TPR : 64); d <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += __shfl_xor(x[i], d);
  if (TPR == 0) {
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) sh[turn][wave][i] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.f;
    for (int k = 0; k < waves; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] += sh[turn][k][i];
    turn ^= 1;
  }
}

}  // namespace
