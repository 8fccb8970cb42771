// Products with 4-bit weights u in 0..15, two to a byte, and a scale for each channel and group of
// G input values:
//
//   y_mn = sum_groups scale_n,group (sum_k in group x_mk (u_nk - 8)) + bias_n
//
// Tokens are taken as they are: 16-bit ones by the matrix instruction of their type, 32-bit ones as
// three exact bf16 parts (lane_types.h).  u - 8 has 4 bits and is exact in either type, so the
// products are exact and the sums 32-bit; a group's sum is multiplied by its scale in 32 bits, when
// it is whole, so no weight is ever rounded.  u - 8 goes through the instruction that makes a float
// of a 4-bit integer, which gives sixteenths: sums are taken 16 times at the end.
//
// Few tokens (few_kernel): bound by the weights' bytes, and below a few MB by the latency of one
// pass over k: 4,096 x 4,096 with groups of 128 for one token in bf16 5.5 us, 8,192 x 8,192 13 us (2.7
// TB/s).  Many tokens (tile_kernel): bound by the matrix cores, and by unpacking and LDS, which the
// products of one tile wait for: 8,192 tokens x 4,096 x 4,096 in bf16 296 to 314 us, 875 to 930 TFLOP/s
// beside a library product's 1,480 to 1,620 of weights that are whole; in 32 bits 810 to 840 us (library 1,820).
#include "lane_types.h"

#include <type_traits>

namespace {

using bs_f32x16 = __attribute__((__vector_size__(16 * sizeof(float)))) float;
using bs_f16x8 = __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16;

constexpr int kStep = 128;    // values of k in one step of the kernels, of one group or several

// How tokens of a type meet the matrix cores: parts of 16 bits.
template <typename T>
struct Form {                 // bfloat16, and 32 bits by parts of it
  static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
  static __device__ __forceinline__ uint32_t pair(float a, float b) {  // exact in either type
    return bs_pack_hi(a, b);
  }
  static __device__ __forceinline__ bs_f32x4 mma16(const uint4& a, const uint4& b, bs_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bs_bf16x8, a),
                                                   __builtin_bit_cast(bs_bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ bs_f32x16 mma32(const uint4& a, const uint4& b, bs_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bs_bf16x8, a),
                                                   __builtin_bit_cast(bs_bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Form<bs_f16> {
  static constexpr int kParts = 1;
  static __device__ __forceinline__ uint32_t pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
  }
  static __device__ __forceinline__ bs_f32x4 mma16(const uint4& a, const uint4& b, bs_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(bs_f16x8, a),
                                                  __builtin_bit_cast(bs_f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ bs_f32x16 mma32(const uint4& a, const uint4& b, bs_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(bs_f16x8, a),
                                                  __builtin_bit_cast(bs_f16x8, b), c, 0, 0, 0);
  }
};

// 8 weights as (u - 8) / 16 in the matrix cores' type.
template <typename T>
__device__ __forceinline__ uint4 weights(uint32_t u) {
  u ^= 0x88888888u;           // two's complement
  uint32_t v = u >> 4;
  asm("" : "+v"(v));          // else the bytes below are cut out of u, an instruction each
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {        // the instruction takes a byte of a register by itself
    f[2 * i] = __builtin_amdgcn_cvt_off_f32_i4((int)(u >> 8 * i & 255));
    f[2 * i + 1] = __builtin_amdgcn_cvt_off_f32_i4((int)(v >> 8 * i & 255));
  }
  return make_uint4(Form<T>::pair(f[0], f[1]), Form<T>::pair(f[2], f[3]),
                    Form<T>::pair(f[4], f[5]), Form<T>::pair(f[6], f[7]));
}

struct Out {
  void* y;
  const void* bias;
  int y_dtype, bias_dtype, m, n;
};

// Parts of 8 neighbouring tokens' values, 0 from `left` on.
template <typename T>
__device__ __forceinline__ void token_parts(const T* p, int left, uint4* out) {
  T t[8];
  if (left >= 8) {
    __builtin_memcpy(t, p, sizeof(t));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = j < left ? p[j] : T{};
  }
  if constexpr (sizeof(T) == 4) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = t[j];
    const bs_parts<3> s = bs_split8<3>(f);
#pragma unroll
    for (int i = 0; i < 3; ++i) out[i] = __builtin_bit_cast(uint4, s.p[i]);
  } else {
    __builtin_memcpy(out, t, 16);
  }
}

// Words of a row of weights from byte `at`, 0 past the row's end.
template <int WORDS>
__device__ __forceinline__ void load_words(const uint8_t* row, int at, int bytes, bool whole,
                                           uint32_t* w) {
  if (whole || at + 4 * WORDS <= bytes) {
    __builtin_memcpy(w, row + at, 4 * WORDS);
  } else {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      uint32_t r = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (at + 4 * i + j < bytes) r |= (uint32_t)row[at + 4 * i + j] << 8 * j;
      w[i] = r;
    }
  }
}

// ------------------------------------------------------------------ few tokens
// A workgroup has 16 channels and MT tiles of 16 tokens; its 8 waves share k, a step each in turn.
// Of a group a lane group g takes the values G / 4 g .. of its channel and tokens.
constexpr int kFewWaves = 8;

template <typename T, int MT, int G>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(const T* x, int64_t stride,
                                                             const uint8_t* w4, const float* scale,
                                                             int k_len, Out o) {
  constexpr int PI = Form<T>::kParts, H = kStep / G, W = G / 32;    // groups, words of a group
  __shared__ bs_f32x4 sh[kFewWaves][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT, n = min(n0 + r, o.n - 1);
  const int bytes = (k_len + 1) / 2, groups = (k_len + G - 1) / G;
  const uint8_t* wr = w4 + (int64_t)n * bytes;
  const float* sr = scale + (int64_t)n * groups;
  const T* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xr[t] = x + (int64_t)min(m0 + 16 * t + r, o.m - 1) * stride;
  bs_f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = bs_f32x4{0.f, 0.f, 0.f, 0.f};
  auto load = [&](int k, bool whole, uint32_t (*w)[W], float* s) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      load_words<W>(wr, (k + G * h + G / 4 * g) / 2, bytes, whole, w[h]);
      const int at = k / G + h;
      s[h] = whole || at < groups ? sr[at] : 0.f;
    }
  };
  auto multiply = [&](int k, bool whole, uint32_t (*w)[W], const float* s) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      bs_f32x4 c[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) c[t] = bs_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const uint4 b = weights<T>(w[h][i]);
        const int at = k + G * h + G / 4 * g + 8 * i;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          uint4 a[PI];
          token_parts(xr[t] + at, whole ? 8 : k_len - at, a);
#pragma unroll
          for (int p = PI - 1; p >= 0; --p) c[t] = Form<T>::mma16(a[p], b, c[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(s[h], c[t][e], acc[t][e]);
    }
  };
  const int whole = k_len / kStep;             // steps without an end
  constexpr int kBatch = 4;                    // steps whose weights are in flight together
  int step = wave;
  for (; step + (kBatch - 1) * kFewWaves < whole; step += kBatch * kFewWaves) {
    uint32_t w[kBatch][H][W];
    float s[kBatch][H];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) load(kStep * (step + i * kFewWaves), true, w[i], s[i]);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) multiply(kStep * (step + i * kFewWaves), true, w[i], s[i]);
  }
  for (; kStep * step < k_len; step += kFewWaves) {
    uint32_t w[H][W];
    float s[H];
    const bool in = step < whole;
    load(kStep * step, in, w, s);
    multiply(kStep * step, in, w, s);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) sh[wave][t][lane] = acc[t];
  __syncthreads();
  // a lane one token and channel
  for (int i = threadIdx.x; i < MT * 256; i += 64 * kFewWaves) {
    const int t = i >> 8, e = i >> 4 & 15, c = i & 15;       // token 16 t + e, channel c
    const float* p = (const float*)&sh[0][t][16 * (e >> 2) + c] + (e & 3);
    float y = 0.f;
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) y += p[v * MT * 256];
    y *= 16.f;
    const int m = m0 + 16 * t + e;
    if (m >= o.m || n0 + c >= o.n) continue;
    if (o.bias) y += bs_load_any(o.bias, o.bias_dtype, n0 + c);
    bs_store_any(o.y, o.y_dtype, (int64_t)m * o.n + n0 + c, y);
  }
}

// ------------------------------------------------------------------ many tokens
typedef const __attribute__((address_space(1))) void* GlobalPtr;
typedef __attribute__((address_space(3))) void* LdsPtr;

// Tokens as parts in rows padded with zeros to whole steps.
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(const T* x, int64_t stride, int k, int ld,
                                                  int64_t plane, uint16_t* to) {
  const int64_t row = blockIdx.x;
  for (int c = threadIdx.x * 8; c < ld; c += 2048) {
    uint4 p[Form<T>::kParts];
    token_parts(x + row * stride + c, k - c, p);
#pragma unroll
    for (int i = 0; i < Form<T>::kParts; ++i) *(uint4*)(to + i * plane + row * ld + c) = p[i];
  }
}

// Tiles of 32 TM WM tokens x 32 TN WN channels, WM x WN waves, products of 32 x 32 x 16.  Tokens are
// staged in LDS by direct loads, two steps deep, 16-byte pieces in an order that keeps the reads off
// each other's banks; a wave's weights go straight to its registers.  Of a group lane group g takes
// the values G / 2 g ..
template <typename T, int TM, int TN, int WM, int WN, int G>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(const uint16_t* x, int64_t ld,
                                                            int64_t plane, const uint8_t* w4,
                                                            const float* scale, int k_len, Out o,
                                                            int tiles_m, int tiles_n) {
  constexpr int PI = Form<T>::kParts, W = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN;
  constexpr int LA = BM * 256 / 1024 / W, H = kStep / G, S = G / 16;   // products of a group
  __shared__ __attribute__((aligned(16))) uint16_t sa0[PI][BM * kStep];
  __shared__ __attribute__((aligned(16))) uint16_t sa1[PI][BM * kStep];
  // workgroups go round the 8 XCDs: each gets a run of tiles, 8 rows of tiles deep, so that the
  // tiles it works on at a time share their rows in its L2
  const int tiles = tiles_m * tiles_n, per = (tiles + 7) / 8;
  const int tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || tile >= tiles) return;
  const int band = tile / (8 * tiles_n), in_band = tile % (8 * tiles_n);
  const int deep = min(8, tiles_m - 8 * band);
  const int m0 = (8 * band + in_band % deep) * BM, n0 = in_band / deep * BN;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / WN, wn = wave % WN, r = lane & 31, g = lane >> 5;
  const int bytes = (k_len + 1) / 2, groups = (k_len + G - 1) / G;

  // places as a base of all lanes, which moves along k, and a lane's own 32 bits
  const char* xb = (const char*)(x + (int64_t)m0 * ld);
  uint32_t ga[LA];
#pragma unroll
  for (int i = 0; i < LA; ++i) {
    const int row = 4 * (wave * LA + i) + (lane >> 4);
    ga[i] = (uint32_t)min(row, o.m - 1 - m0) * (uint32_t)(2 * ld) + 16 * ((lane & 15) ^ (row & 15));
  }
  const uint8_t* wb = w4 + (int64_t)n0 * bytes;
  const float* sb = scale + (int64_t)n0 * groups;
  uint32_t gb[TN], gs[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = min((wn * TN + j) * 32 + r, o.n - 1 - n0);
    gb[j] = (uint32_t)n * bytes, gs[j] = (uint32_t)n * groups;
  }
  auto stage = [&](int k, uint16_t (*sa)[BM * kStep]) {
#pragma unroll
    for (int p = 0; p < PI; ++p) {
      const char* at = xb + (p * plane + k) * 2;
#pragma unroll
      for (int i = 0; i < LA; ++i)
        __builtin_amdgcn_global_load_lds((GlobalPtr)(at + ga[i]),
                                         (LdsPtr)(sa[p] + (wave * LA + i) * 512), 16, 0, 0);
    }
  };
  struct Weights { uint32_t w[TN][H][S]; float s[TN][H]; } b;
  auto load = [&](int k) {
    // of a whole step no lane has a test of its own: at a branch of the lanes every load in flight,
    // the next tokens' too, would be waited for
    if (k + kStep <= k_len) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          __builtin_memcpy(b.w[j][h], wb + (k + G * h) / 2 + (gb[j] + G / 4 * g), 4 * S);
          b.s[j][h] = sb[k / G + h + gs[j]];
        }
    } else {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          load_words<S>(wb + gb[j], (k + G * h + G / 2 * g) / 2, bytes, false, b.w[j][h]);
          b.s[j][h] = k / G + h < groups ? sb[gs[j] + k / G + h] : 0.f;
        }
    }
  };
  bs_f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  // A step is 8 products deep, of 16 values each, in two halves: a half's weights are unpacked, and
  // the next 32 tokens read, beside the products before them.
  auto multiply = [&](const uint16_t (*sa)[BM * kStep], int next) {
    Weights now = b;
    if (next < k_len) load(next);
    bs_f32x16 c[TM][TN];
    uint4 wf[TN][4], wn[TN][4], a[4][PI], an[4][PI];
    auto unpack = [&](int half, uint4 (*to)[4]) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          to[j][u] = weights<T>(now.w[j][(4 * half + u) / S][(4 * half + u) % S]);
    };
    auto tokens = [&](int t, uint4 (*to)[PI]) {       // of half t / TM, rows t % TM
      const int row = (wm * TM + t % TM) * 32 + r;
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int p = 0; p < PI; ++p) {
          const int at = 4 * (t / TM) + u, piece = G / 8 * (at / S) + G / 16 * g + at % S;
          to[u][p] = *(const uint4*)(sa[p] + row * kStep + 8 * (piece ^ (row & 15)));
        }
    };
    unpack(0, wf);
    tokens(0, a);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < 2 * TM; ++t) {
      const int i = t % TM, half = t / TM;
      if (t + 1 < 2 * TM) tokens(t + 1, an);
      if (t == 0) unpack(1, wn);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int h = (4 * half + u) / S, at = (4 * half + u) % S;
          if (at == 0)
#pragma unroll
            for (int e = 0; e < 16; ++e) c[i][j][e] = 0.f;
#pragma unroll
          for (int p = PI - 1; p >= 0; --p) c[i][j] = Form<T>::mma32(a[u][p], wf[j][u], c[i][j]);
          if (at == S - 1)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              acc[i][j][e] = fmaf(now.s[j][h], c[i][j][e], acc[i][j][e]);
        }
      __builtin_amdgcn_sched_group_barrier(0x100, 4 * PI, 0);      // the next tokens first,
#pragma unroll
      for (int q = 0; q < 4 * TN * PI; ++q) {                      // then products with 16 others
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, 16, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int p = 0; p < PI; ++p) a[u][p] = an[u][p];
        if (t == TM - 1)
#pragma unroll
          for (int j = 0; j < TN; ++j) wf[j][u] = wn[j][u];
      }
    }
  };
  // every wave's direct loads have to be in LDS before any wave passes the barrier
  auto arrive = [&]() {
    __builtin_amdgcn_s_waitcnt(0x0F70);     // vmcnt 0
    __syncthreads();
  };
  stage(0, sa0);
  load(0);
  for (int k = 0; k < k_len; k += 2 * kStep) {
    arrive();
    if (k + kStep < k_len) stage(k + kStep, sa1);
    multiply(sa0, k + kStep);
    if (k + kStep < k_len) {
      arrive();
      if (k + 2 * kStep < k_len) stage(k + 2 * kStep, sa0);
      multiply(sa1, k + 2 * kStep);
    }
  }
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + (wn * TN + j) * 32 + r;
    if (n >= o.n) continue;
    const float bias = o.bias ? bs_load_any(o.bias, o.bias_dtype, n) : 0.f;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int m = m0 + (wm * TM + i) * 32 + 8 * (e >> 2) + 4 * g + (e & 3);
        if (m < o.m) bs_store_any(o.y, o.y_dtype, (int64_t)m * o.n + n, fmaf(16.f, acc[i][j][e], bias));
      }
  }
}

// ------------------------------------------------------------------ weights to 4 bits
// A run of 8 values a lane, G / 8 lanes a group.
template <typename T, int G>
__global__ __launch_bounds__(256) void quantize_kernel(const T* w, int64_t stride, int k, int64_t n,
                                                       uint8_t* w4, float* scale) {
  constexpr int L = G / 8;
  const int groups = (k + G - 1) / G, bytes = (k + 1) / 2;
  const int64_t u = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  const int64_t row = u / groups;
  if (row >= n) return;                        // whole groups of lanes leave together
  const int group = (int)(u % groups), c = group * G + threadIdx.x % L * 8;
  float f[8];
  uint32_t top = 0;           // of |w| as bits: ordered like the values, NaN above infinity
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f[j] = c + j < k ? bs_to_f32(w[row * stride + c + j]) : 0.f;
    top = max(top, __float_as_uint(f[j]) & 0x7FFFFFFFu);
  }
#pragma unroll
  for (int d = 1; d < L; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  const float most = __uint_as_float(top), a = most / 7.f;
  if (threadIdx.x % L == 0) scale[row * groups + group] = a;
  // 7 w is exact for 16-bit values, so quotients of exactly a half round to even there; both sides of
  // the quotient are divided by 16 where 7 w could overflow.  In 32 bits it is off by 3 roundings, so one
  // beside a half is formed again in 64: 7 w is exact there, and a quotient of 27 bits by 24 that is no
  // half is 2^-28 away from one.  8,192 x 8,192: 124 us in 32 bits (123 without), 90 in bf16.
  const float up = most > 1e37f ? 7.f / 16.f : 7.f, den = most > 1e37f ? most / 16.f : most;
  const bool ok = most > 0.f && most < INFINITY;   // a group of 0, or with NaN or infinity, is 0: its
                                                   // scale makes the result 0 or NaN
  auto nearest = [&](float x) {
    const float q = up * x / den;
    float r = rintf(q);
    if constexpr (sizeof(T) == 4)
      if (fabsf(fabsf(q - r) - 0.5f) < 1e-5f) r = (float)rint(7.0 * (double)x / (double)most);
    return (int)r + 8;
  };
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    if (c + j >= k) continue;
    const int lo = ok ? nearest(f[j]) : 8, hi = ok ? nearest(f[j + 1]) : 8;
    w4[row * bytes + (c + j) / 2] = (uint8_t)(lo | hi << 4);
  }
}

template <typename F>
void by_group(int group, F&& f) {
  if (group == 32) f(std::integral_constant<int, 32>());
  else if (group == 64) f(std::integral_constant<int, 64>());
  else f(std::integral_constant<int, 128>());
}
template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == BS_F32) f(float());
  else if (dtype == BS_BF16) f(bs_bf16());
  else f(bs_f16());
}

int padded(int k) { return (k + kStep - 1) / kStep * kStep; }

int check(int64_t m, int32_t k, int64_t n, int32_t group, const char* who) {
  BS_CHECK_ARG(group == 32 || group == 64 || group == 128, "%s: groups of %d (32, 64, 128)", who,
               group);
  // few_kernel's workgroups of 512 threads for 16 channels stay below 2^32 threads
  BS_CHECK_ARG(m >= 0 && m <= 0x7FFFF000 && k >= 1 && k <= 65536 && n >= 0 && n < 0x07FFFF00,
               "%s: %lld tokens of %d values (1..65536), %lld channels", who, (long long)m, k,
               (long long)n);
  // the smallest tiles' workgroups, rounded up, stay below 2^32 threads
  const int64_t tiles = ((m + 63) / 64) * ((n + 63) / 64);
  BS_CHECK_ARG(tiles < (1 << 23) - 8, "%s: %lld tokens x %lld channels exceed one launch", who,
               (long long)m, (long long)n);
  return BS_OK;
}

// Whether few_kernel takes the call: it unpacks each weight once, but a workgroup reads all tokens for
// its 16 channels.  Against the best tiles, of 4,096 x 4,096 weights in groups of 128, tokens in bf16: 16
// tokens 7.7 us (24), 32 tokens 12 (25), 64 tokens 22 (25), in 32 bits 43 (47).  Of 8,192 x 8,192, which
// are two rounds of its workgroups: 32 tokens 40 us (52), 64 tokens 71 (52), in 32 bits 16 tokens 52 (84),
// 32 tokens 104 (86).
bool few(int dtype, int64_t m, int64_t n) {
  return m <= (dtype == BS_F32 ? 16 : 32) || (m <= 64 && (n + 15) / 16 <= bs_num_cus());
}

// Whether tile_kernel reads the tokens where they are.
bool in_place(const void* x, int dtype, int k, int64_t stride) {
  return dtype != BS_F32 && k % kStep == 0 && stride % 8 == 0 && (uintptr_t)x % 16 == 0 &&
         stride >= 0 && stride < 1 << 22;      // a tile's rows are addressed in 32 bits
}

template <typename T, int TM, int TN, int WM, int WN, int G>
void launch_tile(const uint16_t* x, int64_t ld, int64_t plane, const uint8_t* w4,
                 const float* scale, int k, const Out& o, hipStream_t st) {
  const int tm = (o.m + 32 * TM * WM - 1) / (32 * TM * WM);
  const int tn = (o.n + 32 * TN * WN - 1) / (32 * TN * WN);
  tile_kernel<T, TM, TN, WM, WN, G><<<(tm * tn + 7) / 8 * 8, 64 * WM * WN, 0, st>>>(
      x, ld, plane, w4, scale, k, o, tm, tn);
}

template <typename T, int G>
void many(const uint16_t* x, int64_t ld, int64_t plane, const uint8_t* w4, const float* scale,
          int k, const Out& o, hipStream_t st) {
  // A launch takes its rounds of a workgroup a CU, and a round of tiles of 128 x 256, 64 x 256, 64 x 128
  // and 64 x 64 about 75, 46, 34 and 25 us at 4,096 values in groups of 128 in bf16.  Whole rounds, in
  // which every CU has one: 85, 51, 37 and 30; in fp16 82, 49, 36, 30; groups of 64 -, 58, 41, 34; of 32
  // -, 82, 58, 47; 32-bit tokens in groups of 128 -, 108, 75, 55; of 64 -, 112, 79, 58; of 32 -, -, 96,
  // 69: in that proportion within an eighth.  Of 48 calls of 100 to 8,192 tokens x 4,096 channels the
  // choice was the fastest tile but in three (1,500 and 2,500 tokens in groups of 64, 106 us for 88 and
  // 158 for 139; 2,500 in groups of 128, 131 for 120).  The largest tiles: 8,192 tokens x 4,096 channels
  // 304 us (365, 379, 517 with the others).  1,500 tokens: 72 (88, 79, 100); 700 tokens: 46 with the
  // second (70, 48, 52); 512 tokens: 35 with the third (69, 45, 36); 256 tokens: 26 with the last (67, 44,
  // 34).  With the other groups' or 32-bit sums beside them the larger ones do not fit the registers.
  auto rounds = [&](int bm, int bn) {
    const int64_t tiles = (int64_t)((o.m + bm - 1) / bm) * ((o.n + bn - 1) / bn);
    return (tiles + bs_num_cus() - 1) / bs_num_cus();
  };
  constexpr bool kLarge = sizeof(T) == 2 && G == kStep, kWide = sizeof(T) == 2 || G > 32;
  const int64_t large = 75 * rounds(128, 256), wide = 46 * rounds(64, 256),
                mid = 34 * rounds(64, 128), small = 25 * rounds(64, 64);
  const int64_t least = mid < small ? mid : small, wider = kWide && wide < least ? wide : least;
  if (kLarge && large <= wider)
    launch_tile<T, kLarge ? 4 : 2, 1, 1, kLarge ? 8 : 4, G>(x, ld, plane, w4, scale, k, o, st);
  else if (kWide && wide <= least)
    launch_tile<T, 2, 1, 1, kWide ? 8 : 4, G>(x, ld, plane, w4, scale, k, o, st);
  else if (mid <= small)
    launch_tile<T, 2, 1, 1, 4, G>(x, ld, plane, w4, scale, k, o, st);
  else
    launch_tile<T, 1, 1, 2, 2, G>(x, ld, plane, w4, scale, k, o, st);
}

template <typename T, int G>
void run(const T* x, int64_t stride, int64_t m, const uint8_t* w4, const float* scale, int k,
         const Out& o, void* workspace, hipStream_t st) {
  if (few(o.y_dtype, m, o.n)) {
    const unsigned tn = (unsigned)((o.n + 15) / 16);
    if (m <= 16)
      few_kernel<T, 1, G><<<dim3(tn, 1), 64 * kFewWaves, 0, st>>>(x, stride, w4, scale, k, o);
    else if (m <= 32)
      few_kernel<T, 2, G><<<dim3(tn, 1), 64 * kFewWaves, 0, st>>>(x, stride, w4, scale, k, o);
    else
      few_kernel<T, 4, G><<<dim3(tn, 1), 64 * kFewWaves, 0, st>>>(x, stride, w4, scale, k, o);
    return;
  }
  const uint16_t* from = (const uint16_t*)x;
  int64_t ld = stride, plane = 0;
  if (workspace) {
    ld = padded(k), plane = m * ld, from = (const uint16_t*)workspace;
    constexpr int64_t kAtOnce = 1 << 23;       // a launch has fewer than 2^32 threads
    for (int64_t r = 0; r < m; r += kAtOnce)
      pad_kernel<T><<<(unsigned)(m - r < kAtOnce ? m - r : kAtOnce), 256, 0, st>>>(
          x + r * stride, stride, k, (int)ld, plane, (uint16_t*)workspace + r * ld);
  }
  many<T, G>(from, ld, plane, w4, scale, k, o, st);
}

}  // namespace

extern "C" int bs_int4_quantize(const void* w, int32_t dtype, int64_t n, int32_t k, int64_t stride,
                                int32_t group, uint8_t* w4, float* scale, bs_stream_t stream) {
  if (int rc = check(0, k, n, group, "bs_int4_quantize")) return rc;
  BS_CHECK_ARG(bs_dtype_ok(dtype), "bs_int4_quantize: dtype %d unknown", dtype);
  if (n == 0) return BS_OK;
  BS_CHECK_ARG(w && w4 && scale, "bs_int4_quantize: NULL pointer");
  const int64_t groups = (k + group - 1) / group, per = 256 / (group / 8);
  // a launch has fewer than 2^32 threads: rows in pieces
  const int64_t most = (1ll << 23) * per / groups;
  hipStream_t st = bs_stream(stream);
  for (int64_t r = 0; r < n; r += most) {
    const int64_t rows = n - r < most ? n - r : most;
    const unsigned grid = (unsigned)((rows * groups + per - 1) / per);
    by_type(dtype, [&](auto t) {
      using T = decltype(t);
      by_group(group, [&](auto g) {
        quantize_kernel<T, g.value><<<grid, 256, 0, st>>>((const T*)w + r * stride, stride, k, rows,
                                                          w4 + r * ((k + 1) / 2),
                                                          scale + r * groups);
      });
    });
    BS_CHECK_LAUNCH();
  }
  return BS_OK;
}

extern "C" size_t bs_int4_workspace_size(const void* x, int32_t dtype, int64_t stride, int64_t m,
                                         int32_t k, int32_t n) {
  if (m < 0 || k < 1 || k > 65536 || !bs_dtype_ok(dtype)) return 0;
  if (few(dtype, m, n) || in_place(x, dtype, k, stride)) return 0;
  return (size_t)m * padded(k) * 2 * (dtype == BS_F32 ? 3 : 1);
}

extern "C" int bs_int4_linear(const void* x, int32_t dtype, int64_t stride, int64_t m, int32_t k,
                              int32_t n, int32_t group, const uint8_t* w4, const float* w_scale,
                              const void* bias, int32_t bias_dtype, void* y, void* workspace,
                              size_t workspace_bytes, bs_stream_t stream) {
  if (int rc = check(m, k, n, group, "bs_int4_linear")) return rc;
  BS_CHECK_ARG(bs_dtype_ok(dtype) && bs_dtype_ok(bias_dtype), "bs_int4_linear: dtype unknown");
  if (m == 0 || n == 0) return BS_OK;
  BS_CHECK_ARG(x && w4 && w_scale && y, "bs_int4_linear: NULL pointer");
  const size_t need = bs_int4_workspace_size(x, dtype, stride, m, k, n);
  BS_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
               "bs_int4_linear: workspace of %zu bytes needed", need);
  const Out o = {y, bias, dtype, bias_dtype, (int)m, n};
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    by_group(group, [&](auto g) {
      run<T, g.value>((const T*)x, stride, m, w4, w_scale, k, o, need ? workspace : nullptr,
                      bs_stream(stream));
    });
  });
  BS_CHECK_LAUNCH();
  return BS_OK;
}
