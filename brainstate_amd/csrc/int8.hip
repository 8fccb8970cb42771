// Products of 8-bit integers with a scale for each token and each output channel:
//
//   a_m = max_k |x_mk| / 127,  x8 = round(127 x / max_k |x_mk|),  y_mn = a_m w_scale_n sum_k x8_mk w8_nk + bias_n
//
// Sums are exact (32-bit integers on the matrix cores), so no order of them changes a bit.
// quant_kernel writes the tokens' integers in rows padded with zeros to whole 128-byte steps: the
// products then need no test of k on that side, and what the weights' side reads past a row's end
// is multiplied by 0.
//
// Few tokens (skinny_kernel): bound by the weights' bytes, and below a few MB by the latency of
// one pass over k.  Each workgroup has 16 channels and its waves share k; weights go straight from
// memory to the matrix instruction, whose operand is 16 rows x 64 bytes.  One token x 4,096 x
// 4,096: 6.0 us (2.8 TB/s; 16.9 MB fetched for 16.8), with 3.7 before it for the token's integers.
// Many tokens (tile_kernel): bound by the matrix cores; tiles of both operands are staged in LDS
// by direct loads, two deep, 16-byte pieces in an order that keeps the reads off each other's
// banks (no conflicts counted).  8,192 x 4,096 x 4,096: in a run of calls 162 us with the 24 of
// quant_kernel, so 138 (2.0 POP/s; a large library product of this type 2.1), under the tracer 157
// (1.75 POP/s); the matrix cores are busy in 49 % of the cycles.
#include "lane_types.h"

#include <type_traits>

namespace {

using i32x4 = __attribute__((__vector_size__(4 * sizeof(int)))) int;
using i32x16 = __attribute__((__vector_size__(16 * sizeof(int)))) int;

constexpr int kStep = 128;    // bytes of k in one step of the kernels

// ------------------------------------------------------------------ tokens to 8 bits
// Bound by bytes: 8,192 x 4,096 bfloat16 24 us (4.2 TB/s).
// A row to a workgroup; V vectors of 8 values of it to a lane's registers (the rest, if any, is
// read again for the second pass).  V is 1 for rows of up to 2,048 values and 4 above: us by 1 / 4
// at 8,192 rows of 2,048 12.7 / 18.5, of 4,096 22.2 / 24.0, of 8,192 42.5 / 36.5.
template <typename T, int V>
__global__ __launch_bounds__(256) void quant_kernel(const T* x, int64_t stride, int k, int ld,
                                                    int8_t* x8, float* scale) {
  __shared__ uint32_t sh[4];
  const int64_t row = blockIdx.x;
  const T* p = x + row * stride;
  T held[V][8];
  auto load = [&](int c, T* t) {
    if (c + 8 <= k) {
      __builtin_memcpy(t, p + c, 8 * sizeof(T));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = c + j < k ? p[c + j] : T{};
    }
  };
  uint32_t top = 0;     // of |x| as bits: ordered like the values, NaN above infinity
  auto raise = [&](const T* t) {
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(bs_to_f32(t[j])) & 0x7FFFFFFFu);
  };
#pragma unroll
  for (int v = 0; v < V; ++v) load(threadIdx.x * 8 + 2048 * v, held[v]);
#pragma unroll
  for (int v = 0; v < V; ++v) raise(held[v]);
  for (int c = threadIdx.x * 8 + 2048 * V; c < k; c += 2048) {
    T t[8];
    load(c, t);
    raise(t);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = top;
  __syncthreads();
  top = max(max(sh[0], sh[1]), max(sh[2], sh[3]));
  const float most = __uint_as_float(top), a = most / 127.f;
  if (threadIdx.x == 0) scale[row] = a;
  // 127 x is exact for 16-bit values, so quotients of exactly a half round to even there; both
  // sides of the quotient are divided by 256 where 127 x could overflow
  const float up = most > 1e36f ? 127.f / 256.f : 127.f;
  const float den = most > 1e36f ? most / 256.f : most;
  const bool ok = a > 0.f && a < INFINITY;    // a row of 0, or with NaN or infinity, is 0: its
                                              // scale makes the result 0 or NaN
  int8_t* q = x8 + row * ld;
  auto store = [&](int c, const T* t) {
    uint32_t r[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int n = ok ? (int)rintf(up * bs_to_f32(t[j]) / den) : 0;
      r[j >> 2] |= (uint32_t)(n & 255) << 8 * (j & 3);
    }
    if (c + 8 <= ld) {
      __builtin_memcpy(q + c, r, 8);
    } else {
      for (int j = 0; c + j < ld; ++j) q[c + j] = (int8_t)(r[j >> 2] >> 8 * (j & 3));
    }
  };
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = threadIdx.x * 8 + 2048 * v;
    if (c < ld) store(c, held[v]);
  }
  for (int c = threadIdx.x * 8 + 2048 * V; c < ld; c += 2048) {
    T t[8];
    load(c, t);
    store(c, t);
  }
}

__global__ __launch_bounds__(256) void pad_kernel(const int8_t* x, int k, int ld, int8_t* x8) {
  const int64_t row = blockIdx.x;
  for (int c = threadIdx.x; c < ld; c += 256) x8[row * ld + c] = c < k ? x[row * k + c] : 0;
}

struct Out {
  void* y;
  const float *a, *w;       // scales
  const void* bias;
  int y_dtype, bias_dtype, m, n;
  bool wide;                // rows of y start on 4 values
};

__device__ __forceinline__ void put(const Out& o, int m, int n, int acc, float w, float b) {
  bs_store_any(o.y, o.y_dtype, (int64_t)m * o.n + n, fmaf((float)acc, o.a[m] * w, b));
}

// 16 bytes of a row of weights at k, which may start anywhere; 0 past the row's end.
__device__ __forceinline__ i32x4 load_w(const int8_t* row, int k, int k_len) {
  i32x4 r = {0, 0, 0, 0};
  if (k + 16 <= k_len) {
    __builtin_memcpy(&r, row + k, 16);
  } else {
    int8_t t[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) t[j] = k + j < k_len ? row[k + j] : (int8_t)0;
    __builtin_memcpy(&r, t, 16);
  }
  return r;
}

// ------------------------------------------------------------------ few tokens
// MT tiles of 16 tokens.  A lane group g takes bytes 32g..32g+31 of a step for two products, so
// the four groups read a row's 128 bytes side by side; tokens are taken in the same order.
template <int MT>
__global__ __launch_bounds__(256) void skinny_kernel(const int8_t* x8, int ld, const int8_t* w8,
                                                     int k_len, Out o) {
  __shared__ i32x4 sh[4][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const int8_t* wr = w8 + (int64_t)min(n0 + r, o.n - 1) * k_len;
  const int8_t* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xr[t] = x8 + (int64_t)min(m0 + 16 * t + r, o.m - 1) * ld + 32 * g;
  i32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = i32x4{0, 0, 0, 0};
  for (int k = wave * kStep; k < ld; k += 4 * kStep) {
    const i32x4 b0 = load_w(wr, k + 32 * g, k_len), b1 = load_w(wr, k + 32 * g + 16, k_len);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(xr[t] + k), b0, acc[t], 0, 0,
                                                     0);
      acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(xr[t] + k + 16), b1, acc[t],
                                                     0, 0, 0);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) sh[wave][t][lane] = acc[t];
  __syncthreads();
  for (int t = wave; t < MT; t += 4) {
    i32x4 s = sh[0][t][lane];
#pragma unroll
    for (int v = 1; v < 4; ++v) s += sh[v][t][lane];
    const int n = n0 + r;
    if (n >= o.n) continue;
    const float w = o.w[n], b = o.bias ? bs_load_any(o.bias, o.bias_dtype, n) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = m0 + 16 * t + 4 * g + i;
      if (m < o.m) put(o, m, n, s[i], w, b);
    }
  }
}

// ------------------------------------------------------------------ many tokens
typedef const __attribute__((address_space(1))) void* GlobalPtr;
typedef __attribute__((address_space(3))) void* LdsPtr;

// Tile of BM tokens x BN channels, WM x WN waves, products of 32 x 32 x 32.
template <int BM, int BN, int WM, int WN, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(const int8_t* x8, int ld,
                                                            const int8_t* w8, int k_len, Out o,
                                                            int tiles_m, int tiles_n) {
  constexpr int W = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
  constexpr int LA = BM * kStep / 1024 / W, LB = BN * kStep / 1024 / W;   // 1 KB loads a wave
  // two steps of both operands, as arrays of their own: a read of one then does not wait for the
  // loads into the other
  __shared__ __attribute__((aligned(16))) int8_t sa0[BM * kStep];
  __shared__ __attribute__((aligned(16))) int8_t sb0[BN * kStep];
  __shared__ __attribute__((aligned(16))) int8_t sa1[BM * kStep];
  __shared__ __attribute__((aligned(16))) int8_t sb1[BN * kStep];
  __shared__ float scales[BM];
  // workgroups go round the 8 XCDs: each gets a run of tiles, 8 rows of tiles deep, so that the 32
  // tiles it works on at a time share 8 + 4 runs of rows in its L2
  const int tiles = tiles_m * tiles_n, per = (tiles + 7) / 8;
  const int tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || tile >= tiles) return;
  const int band = tile / (8 * tiles_n), in_band = tile % (8 * tiles_n);
  const int deep = min(8, tiles_m - 8 * band);
  const int m0 = (8 * band + in_band % deep) * BM, n0 = in_band / deep * BN;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / WN, wn = wave % WN, r = lane & 31, g = lane >> 5;

  // Load i of a wave fills rows 8 (wave LA + i) .. + 7; lane: row lane / 8, place lane % 8, which
  // holds piece (place ^ (row / 2) % 8): 16 rows' pieces then lie on different banks.
  auto key = [](int row) { return row >> 1 & 7; };
  auto piece = [&](int i) { return (lane & 7) ^ key(8 * i + (lane >> 3)); };
  const int8_t* ga[LA];
  const int8_t* gb[LB];
#pragma unroll
  for (int i = 0; i < LA; ++i)
    ga[i] = x8 + (int64_t)min(m0 + 8 * (wave * LA + i) + (lane >> 3), o.m - 1) * ld +
            16 * piece(wave * LA + i);
#pragma unroll
  for (int i = 0; i < LB; ++i)
    gb[i] = w8 + (int64_t)min(n0 + 8 * (wave * LB + i) + (lane >> 3), o.n - 1) * k_len;
  const int last = max(k_len - 16, 0);     // DIRECT: the last whole piece of a row

  auto stage = [&](int k, int8_t* sa, int8_t* sb) {
#pragma unroll
    for (int i = 0; i < LA; ++i)
      __builtin_amdgcn_global_load_lds((GlobalPtr)(ga[i] + k),
                                       (LdsPtr)(sa + (wave * LA + i) * 1024), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      if constexpr (DIRECT) {
        __builtin_amdgcn_global_load_lds((GlobalPtr)(gb[i] + min(k + 16 * piece(wave * LB + i), last)),
                                         (LdsPtr)(sb + (wave * LB + i) * 1024), 16, 0, 0);
      } else {
        *(i32x4*)(sb + (wave * LB + i) * 1024 + lane * 16) =
            load_w(gb[i], k + 16 * piece(wave * LB + i), k_len);
      }
    }
  };
  i32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  // a step's four products, the operands of each read while the one before runs
  auto multiply = [&](const int8_t* sa, const int8_t* sb) {
    i32x4 a[2][TM], b[2][TN];
    auto read = [&](int s) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int row = (wm * TM + i) * 32 + r;
        a[s & 1][i] = *(const i32x4*)(sa + row * kStep + 16 * ((2 * s + g) ^ key(row)));
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int row = (wn * TN + j) * 32 + r;
        b[s & 1][j] = *(const i32x4*)(sb + row * kStep + 16 * ((2 * s + g) ^ key(row)));
      }
    };
    read(0);
#pragma unroll
    for (int s = 0; s < kStep / 32; ++s) {
      if (s + 1 < kStep / 32) read(s + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] =
              __builtin_amdgcn_mfma_i32_32x32x32_i8(a[s & 1][i], b[s & 1][j], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // every wave's direct loads have to be in LDS before any wave passes the barrier
  auto arrive = [&]() {
    __builtin_amdgcn_s_waitcnt(0x0F70);     // vmcnt 0
    __syncthreads();
  };
  for (int i = threadIdx.x; i < BM; i += 64 * W) scales[i] = o.a[min(m0 + i, o.m - 1)];
  stage(0, sa0, sb0);
  for (int k = 0; k < ld; k += 2 * kStep) {
    arrive();
    if (k + kStep < ld) stage(k + kStep, sa1, sb1);
    multiply(sa0, sb0);
    if (k + kStep < ld) {
      arrive();
      if (k + 2 * kStep < ld) stage(k + 2 * kStep, sa0, sb0);
      multiply(sa1, sb1);
    }
  }
  // 16 rows at a time through a wave's own part of sa0, so that a lane stores 4 neighbouring
  // channels and 8 or 16 lanes a whole run of a row; groups of 4 in an order (group ^ row) that
  // spreads the banks
  constexpr int C = TN * 32, L = C / 4;
  __syncthreads();
  int* turn = (int*)(sa0 + wave * 16 * C * 4);
  const int cg = lane % L, n = n0 + wn * C + 4 * cg;
  float w[4], bias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = n + i < o.n ? o.w[n + i] : 0.f;
    bias[i] = o.bias && n + i < o.n ? bs_load_any(o.bias, o.bias_dtype, n + i) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int row = 8 * (e >> 2) + 4 * g + (e & 3), col = 32 * j + r;
          turn[row * C + ((((col >> 2) ^ row) & (L - 1)) << 2) + (col & 3)] = acc[i][j][8 * h + e];
        }
      __builtin_amdgcn_wave_barrier();     // one wave's LDS accesses are done in order
#pragma unroll
      for (int q = 0; q < 16 * L / 64; ++q) {
        const int row = q * (64 / L) + lane / L;
        const int mi = (wm * TM + i) * 32 + 16 * h + row, m = m0 + mi;
        const i32x4 v = *(const i32x4*)(turn + row * C + (((cg ^ row) & (L - 1)) << 2));
        if (m >= o.m) continue;
        const float am = scales[mi];
        bs_f32x4 y;
#pragma unroll
        for (int x = 0; x < 4; ++x) y[x] = fmaf((float)v[x], am * w[x], bias[x]);
        const int64_t at = (int64_t)m * o.n + n;
        if (o.wide && n < o.n) {
          if (o.y_dtype == BS_F32) bs_store4((float*)o.y + at, y);
          else if (o.y_dtype == BS_BF16) bs_store4((bs_bf16*)o.y + at, y);
          else bs_store4((bs_f16*)o.y + at, y);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (n + x < o.n) bs_store_any(o.y, o.y_dtype, at + x, y[x]);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
}

template <int BM, int BN, int WM, int WN>
void launch_tile(const int8_t* x8, int ld, const int8_t* w8, int k, const Out& o,
                 hipStream_t st) {
  const int tm = (o.m + BM - 1) / BM, tn = (o.n + BN - 1) / BN;
  const int grid = (tm * tn + 7) / 8 * 8;
  if (k % 16 == 0 && (uintptr_t)w8 % 16 == 0)
    tile_kernel<BM, BN, WM, WN, true><<<grid, 64 * WM * WN, 0, st>>>(x8, ld, w8, k, o, tm, tn);
  else
    tile_kernel<BM, BN, WM, WN, false><<<grid, 64 * WM * WN, 0, st>>>(x8, ld, w8, k, o, tm, tn);
}

// Skinny while one round of workgroups (one a CU) holds the call, with as few tokens each as that
// allows: a workgroup's time is its share of k, which more tokens a workgroup only lengthen.  Past
// that the weights are read again for every 64 tokens and the tiles' LDS pays, but up to 32 tokens
// a tile of 64 is mostly empty.  us at tokens x k x channels, skinny by 16 / 32 / 64 tokens, tile:
//   64 x 1,000 x 300    7.4 /  8.0 / 10.0, 12.9      512 x 1,000 x 300   - / - / 10.8, 13.8
//   32 x 4,096 x 4,096 13.8 / 13.2 / 15.3, 20.2      128 x 4,096 x 4,096 - / - / 25.0, 21.0
//   64 x 4,096 x 4,096 21.0 / 17.6 / 18.9, 20.5       64 x 2,048 x 8,192 19.3 / 15.8 / 14.1, 12.7
// Tiles are as large as still give every CU one.  us by 64 / 128 / 256 at 4,096 x 4,096:
//   512 tokens 26.0 / 33.7 / -, 1,024 37.5 / 36.6 / 65.4, 2,048 68.0 / 57.4 / 70.3,
//   4,096 123.6 / 100.6 / 83.8, 8,192 236.8 / 192.5 / 159.4
void product(const int8_t* x8, int ld, const int8_t* w8, int k, const Out& o, hipStream_t st) {
  const int64_t tn = (o.n + 15) / 16, tm = (o.m + 15) / 16, cus = bs_num_cus();
  const auto grid = [&](int mt) { return dim3((unsigned)tn, (unsigned)((tm + mt - 1) / mt)); };
  if (tm == 1 || tn * tm <= cus)
    skinny_kernel<1><<<grid(1), 256, 0, st>>>(x8, ld, w8, k, o);
  else if (tm == 2 || tn * ((tm + 1) / 2) <= cus)
    skinny_kernel<2><<<grid(2), 256, 0, st>>>(x8, ld, w8, k, o);
  else if (tn * ((tm + 3) / 4) <= cus)
    skinny_kernel<4><<<grid(4), 256, 0, st>>>(x8, ld, w8, k, o);
  else if ((int64_t)((o.m + 255) / 256) * ((o.n + 255) / 256) >= cus)
    launch_tile<256, 256, 2, 4>(x8, ld, w8, k, o, st);
  else if ((int64_t)((o.m + 127) / 128) * ((o.n + 127) / 128) >= cus)
    launch_tile<128, 128, 2, 2>(x8, ld, w8, k, o, st);
  else
    launch_tile<64, 64, 2, 2>(x8, ld, w8, k, o, st);
}

int padded(int k) { return (k + kStep - 1) / kStep * kStep; }

int check(int64_t m, int32_t k, int32_t n, const char* who) {
  BS_CHECK_ARG(m >= 0 && m <= 0x7FFFF000 && k >= 1 && k <= 65536 && n >= 0 && n <= 0x0FFFFF00,
               "%s: %lld tokens of %d values (1..65536), %d channels", who, (long long)m, k, n);
  // the largest tiles' and the skinny form's workgroups, rounded up, stay below 2^32 threads
  const int64_t tiles = ((m + 255) / 256) * (((int64_t)n + 255) / 256);
  BS_CHECK_ARG(tiles < (1 << 23) - 8, "%s: %lld tokens x %d channels exceed one launch", who,
               (long long)m, n);
  return BS_OK;
}

// A launch has fewer than 2^32 threads (past that the count wraps without an error), so rows that
// take a workgroup each go in pieces of this many: f(first row, rows).
constexpr int64_t kRowsAtOnce = 1 << 23;
template <typename F>
void row_pieces(int64_t m, F&& f) {
  for (int64_t r = 0; r < m; r += kRowsAtOnce)
    f(r, (unsigned)(m - r < kRowsAtOnce ? m - r : kRowsAtOnce));
}

int quantize(const void* x, int dtype, int64_t m, int k, int64_t stride, int ld, int8_t* x8,
             float* scale, hipStream_t st) {
  auto run = [&](auto* p) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    row_pieces(m, [&](int64_t r, unsigned rows) {
      if (ld <= 2048)
        quant_kernel<T, 1><<<rows, 256, 0, st>>>(p + r * stride, stride, k, ld, x8 + r * ld,
                                                 scale + r);
      else
        quant_kernel<T, 4><<<rows, 256, 0, st>>>(p + r * stride, stride, k, ld, x8 + r * ld,
                                                 scale + r);
    });
  };
  if (dtype == BS_F32) run((const float*)x);
  else if (dtype == BS_BF16) run((const bs_bf16*)x);
  else run((const bs_f16*)x);
  BS_CHECK_LAUNCH();
  return BS_OK;
}

}  // namespace

extern "C" int bs_int8_quantize(const void* x, int32_t dtype, int64_t m, int32_t k,
                                int64_t stride, int8_t* x8, float* scale, bs_stream_t stream) {
  if (int rc = check(m, k, 0, "bs_int8_quantize")) return rc;
  BS_CHECK_ARG(bs_dtype_ok(dtype), "bs_int8_quantize: dtype %d unknown", dtype);
  if (m == 0) return BS_OK;
  BS_CHECK_ARG(x && x8 && scale, "bs_int8_quantize: NULL pointer");
  return quantize(x, dtype, m, k, stride, k, x8, scale, bs_stream(stream));
}

extern "C" size_t bs_int8_workspace_size(int64_t m, int32_t k) {
  if (m < 0 || k < 1 || k > 65536) return 0;
  return (size_t)m * padded(k) + (size_t)m * sizeof(float);
}

extern "C" int bs_int8_linear(const void* x, int32_t x_dtype, int64_t stride, const float* x_scale,
                              int64_t m, int32_t k, int32_t n, const int8_t* w8,
                              const float* w_scale, const void* bias, int32_t bias_dtype, void* y,
                              int32_t y_dtype, void* workspace, size_t workspace_bytes,
                              bs_stream_t stream) {
  if (int rc = check(m, k, n, "bs_int8_linear")) return rc;
  BS_CHECK_ARG((x_scale || bs_dtype_ok(x_dtype)) && bs_dtype_ok(bias_dtype) &&
                   bs_dtype_ok(y_dtype), "bs_int8_linear: dtype unknown");
  if (m == 0 || n == 0) return BS_OK;
  BS_CHECK_ARG(x && w8 && w_scale && y, "bs_int8_linear: NULL pointer");
  const size_t need = bs_int8_workspace_size(m, k);
  BS_CHECK_ARG(workspace && workspace_bytes >= need,
               "bs_int8_linear: workspace of %zu bytes needed", need);
  hipStream_t st = bs_stream(stream);
  const int ld = padded(k);
  int8_t* x8 = (int8_t*)workspace;
  float* a = (float*)(x8 + (size_t)m * ld);
  if (x_scale) {
    row_pieces(m, [&](int64_t r, unsigned rows) {
      pad_kernel<<<rows, 256, 0, st>>>((const int8_t*)x + r * k, k, ld, x8 + r * ld);
    });
    BS_CHECK_LAUNCH();
  } else if (int rc = quantize(x, x_dtype, m, k, stride, ld, x8, a, st)) {
    return rc;
  }
  const Out o = {y, x_scale ? x_scale : a, w_scale, bias, y_dtype, bias_dtype, (int)m, n,
                 n % 4 == 0 && (uintptr_t)y % 16 == 0};
  product(x8, ld, w8, k, o, st);
  BS_CHECK_LAUNCH();
  return BS_OK;
}
