// The Philox 4x32-10 generator (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011)
// and the elements that dropout keeps.
#pragma once

#include "common.h"

struct U4 {
  uint32_t x, y, z, w;
};

__device__ __forceinline__ U4 philox(U4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c.x;
    const uint64_t p1 = (uint64_t)0xCD9E8D57u * c.z;
    c = U4{(uint32_t)(p1 >> 32) ^ c.y ^ k0, (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c.w ^ k1,
           (uint32_t)p0};
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}

// Element (row, column) is kept where word column % 4 of counter (column / 4, site, row) is not
// below `drop`.
struct Dropout {
  uint32_t k0, k1, site, drop;
  __device__ __forceinline__ Dropout(uint64_t seed, const int64_t* at, uint32_t s, uint32_t d) {
    if (at) seed = (uint64_t)*at;
    k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32), site = s, drop = d;
  }
  __device__ __forceinline__ uint32_t four(int64_t row, int quad) const {
    const U4 r = philox(U4{(uint32_t)quad, site, (uint32_t)row, (uint32_t)(row >> 32)}, k0, k1);
    return (r.x >= drop) | (r.y >= drop) << 1 | (r.z >= drop) << 2 | (r.w >= drop) << 3;
  }
  // bit j: element (row, column + j) is kept, for 8 of them
  __device__ __forceinline__ uint32_t eight(int64_t row, int column) const {
    const int quad = column >> 2, off = column & 3;
    uint32_t bits = four(row, quad) | four(row, quad + 1) << 4;
    if (off) bits = (bits | four(row, quad + 2) << 8) >> off;
    return bits;
  }
};
