// Decay attention over chunks of 64 tokens: the walk over a sequence's chunks, forward and for the
// gradients (decay.h has its formulas), and the carry of states from segment to segment.
//
// A chunk costs two products with the state and two within the chunk.  A workgroup walks the
// chunks of one segment and head; each of its 4 waves has 32 value columns of the state in
// registers, so the state never leaves them inside a segment:
//
//   att^T = K Q^T          rows j, columns i: a lane has 16 neighbouring j of one i
//   O^T   = S^T Q^T + V^T att^T     rows are value columns, a lane has 16 neighbouring of one token
//   S     = K^T V          a lane has one value column and runs of 8 rows, which is what the next
//                          S^T Q^T takes from it
//
// Rows of a tile are dealt so that a product leaves in a lane what the next one takes from it; the
// transposed operands (K^T, V^T) are read from LDS by its transposing reads.
//
// 8,192 tokens of 32 heads of 128 x 128 in bf16 (268 MB, 53 us at a large copy's 5.1 TB/s): sum_kernel
// 46 us, scan_kernel 20, walk_kernel 112.  The walk is bound by what a wave issues: a chunk takes it
// about 1,100 vector instructions, most of them splits of the state and its scaled values into parts,
// 120 products and 110 reads of LDS, and with two waves a SIMD the vector units are busy 40 %, the matrix
// cores 30 % and LDS 20 % of the time.  8 waves of 16 columns, four a SIMD, take the same 111 us, since
// each reads Q, K and att again for half the columns; the three gradients' walks of 4 x 2,048 tokens, 16
// heads, take 252 us this way and 303 that way.
//
// Numbers: the state and all sums are 32-bit; products take 32-bit operands as three exact bf16
// parts (lane_types.h).  Sums of log decays are 64-bit, since their differences are exponents.  An
// infinity or NaN reaches the outputs and states from its token on, as by the formula.
#include "decay.h"
#include "decay_slots.h"

namespace {

constexpr int kThreads = 256;
constexpr int kPitch = 128;      // values of a row of V in LDS

template <typename T> constexpr int kParts = sizeof(T) == 4 ? 3 : 2;
template <> constexpr int kParts<bs_bf16> = 1;

typedef __attribute__((__vector_size__(4 * sizeof(short)))) short i16x4;
typedef __attribute__((address_space(3))) i16x4* LdsTile;
using bs_u32x4 = __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t;

// 4 rows x 16 columns of 16-bit values for 16 lanes, transposed: lane l gives the place of the 4
// columns 4 (l % 4) .. of row l / 4 % 4 and receives the 4 rows of column l % 16.
__device__ __forceinline__ uint2 turn4(const void* tile, int bytes) {
  return __builtin_bit_cast(
      uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTile)((const char*)tile + bytes)));
}

// acc += a b over 16 products: parts p, q with p + q <= 2.
template <int PA, int PB>
__device__ __forceinline__ bs_f32x16 mma(const bs_parts<PA>& a, const bs_parts<PB>& b,
                                         bs_f32x16 acc) {
#pragma unroll
  for (int s = 2; s >= 0; --s)
#pragma unroll
    for (int p = 0; p <= s; ++p)
      if (p < PA && s - p < PB)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[p], b.p[s - p], acc, 0, 0, 0);
  return acc;
}

__device__ __forceinline__ bs_f32x16 zero16() {
  bs_f32x16 r;
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = 0.f;
  return r;
}

// Where piece `piece` (8 values) of row `row` lies in a tile of rows of D values, in bytes.  Pieces are
// in an order that spreads over the banks both the same piece of 16 rows and, for the transposing
// reads, 4 neighbouring pieces of 4 rows.  Piece c ^ piece lies at place ^ (16 c), and rows 16 (of 128
// values) or 32 apart have one order.
template <int D>
__device__ __forceinline__ int place(int row, int piece) {
  const int key = D == 128 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2 | (row >> 2 & 3);
  return row * (2 * D) + ((piece ^ key) << 4);
}
__device__ __forceinline__ bs_bf16x8 piece_at(const uint16_t* tile, int bytes) {
  return *(const bs_bf16x8*)((const char*)tile + bytes);
}

// Three bf16 parts of 8 floats (lane_types.h), what a part leaves by the exact sum x - part.
struct Splitter {
  uint32_t low, high;           // -1 in either half, in scalar registers
  __device__ __forceinline__ Splitter() : low(0x0000BF80u), high(0xBF800000u) {
    asm volatile("" : "+s"(low), "+s"(high));
  }
  template <int P>
  __device__ __forceinline__ bs_parts<P> split(const float* x) const {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    uint32_t w[P][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
      for (int p = 0; p < P; ++p) {
        w[p][i] = bs_pack_hi(a, b);
        if (p + 1 < P) {
          const bf16x2 v = __builtin_bit_cast(bf16x2, w[p][i]);
          a = __builtin_amdgcn_fdot2_f32_bf16(v, __builtin_bit_cast(bf16x2, low), a, false);
          b = __builtin_amdgcn_fdot2_f32_bf16(v, __builtin_bit_cast(bf16x2, high), b, false);
        }
      }
    }
    bs_parts<P> o;
#pragma unroll
    for (int p = 0; p < P; ++p)
      o.p[p] = __builtin_bit_cast(bs_bf16x8, make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]));
    return o;
  }
};

// The same parts with a value's rest from that value alone.  Splitter's dot product takes its neighbour
// times 0, which an infinity makes NaN: no matter where a product sums over both, but the values of a
// key are rows of the state.
struct Cutter {
  template <int P>
  __device__ __forceinline__ bs_parts<P> split(const float* x) const { return bs_split8<P>(x); }
};

// An operand's rows of one head; strides in bytes.
struct HeadRows {
  const char* p;
  int64_t batch, token;
  template <typename T>
  static __device__ __forceinline__ HeadRows of(const DecayOperand& x, int h) {
    constexpr int64_t n = sizeof(T);
    return {(const char*)x.p + (h / x.rep) * x.stride[2] * n, x.stride[0] * n, x.stride[1] * n};
  }
};

// The rows of a chunk in processing order, 8 neighbouring values at a time, 0 past the last row and
// the row's end: buffer loads, whose bounds the hardware checks.
template <typename T, bool VEC>     // VEC: rows start on 16 bytes and end on 8 values
struct ChunkRows {
  __amdgpu_buffer_rsrc_t rs;
  uint32_t step;
  int dim, rows, back;
  __device__ __forceinline__ ChunkRows(const HeadRows& x, const DecayChunk& c, int d, int b) {
    step = (uint32_t)x.token;
    const uint64_t p = (uint64_t)(x.p + c.batch * x.batch + c.token * x.token);
    const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32 |
                          (uint32_t)__builtin_amdgcn_readfirstlane((int)p);
    rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0,
                                           (uint32_t)(c.rows - 1) * step + d * (int)sizeof(T),
                                           0x00027000);
    dim = d, rows = c.rows, back = b;
  }
  __device__ __forceinline__ void raw(int row, int d, uint4* x) const {
    constexpr int W = sizeof(T) / 2;
    const int have = row < rows ? dim : 0;
    const uint32_t at = (uint32_t)(back ? rows - 1 - row : row) * step;
    if constexpr (VEC) {
      const uint32_t o = d < have ? at + d * (uint32_t)sizeof(T) : 0xFFFFFF00u;
#pragma unroll
      for (int i = 0; i < W; ++i)
        x[i] = __builtin_bit_cast(uint4,
                                  __builtin_amdgcn_raw_buffer_load_b128(rs, o + 16 * i, 0, 0));
    } else {
      uint32_t e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t o = d + j < have ? at + (d + j) * (uint32_t)sizeof(T) : 0xFFFFFFF0u;
        if constexpr (W == 1) e[j] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rs, o, 0, 0);
        else e[j] = __builtin_amdgcn_raw_buffer_load_b32(rs, o, 0, 0);
      }
      if constexpr (W == 1) {
        x[0] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16,
                          e[6] | e[7] << 16);
      } else {
        x[0] = make_uint4(e[0], e[1], e[2], e[3]);
        x[1] = make_uint4(e[4], e[5], e[6], e[7]);
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ void floats(const uint4* x, float* f) {
  T t[8];
  __builtin_memcpy(t, x, sizeof(t));
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = bs_to_f32(t[j]);
}

template <typename T, typename S>
__device__ __forceinline__ bs_parts<kParts<T>> parts_of(const S& sp, const uint4* x) {
  if constexpr (kParts<T> == 1) {
    bs_parts<1> o;
    o.p[0] = __builtin_bit_cast(bs_bf16x8, x[0]);
    return o;
  } else {
    float f[8];
    floats<T>(x, f);
    return sp.template split<kParts<T>>(f);
  }
}

// A chunk's rows of D padded values on their way into LDS.
template <typename T, int D>
struct Staged {
  static constexpr int kPer = D / 8, kRows = kThreads / kPer, kN = 64 / kRows, W = sizeof(T) / 2;
  uint4 x[kN][W];
  template <bool VEC>
  __device__ __forceinline__ void load(const ChunkRows<T, VEC>& r) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      r.raw(threadIdx.x / kPer + i * kRows, threadIdx.x % kPer * 8, x[i]);
  }
  // as bf16 parts, [part][64][D]
  template <typename S>
  __device__ __forceinline__ void put(uint16_t* to, const S& sp) const {
    const int at = place<D>(threadIdx.x / kPer, threadIdx.x % kPer);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const bs_parts<kParts<T>> p = parts_of<T>(sp, x[i]);
#pragma unroll
      for (int k = 0; k < kParts<T>; ++k)
        *(bs_bf16x8*)((char*)to + (k * 64 + i * kRows) * 2 * D + at) = p.p[k];
    }
  }
  // as they are, [64][D]: 16-bit values in the order of place(), 32-bit ones in a row's order
  __device__ __forceinline__ void put_raw(void* to) const {
    const int at = place<D>(threadIdx.x / kPer, threadIdx.x % kPer);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int row = threadIdx.x / kPer + i * kRows, d = threadIdx.x % kPer * 8;
      if constexpr (W == 1) {
        *(uint4*)((char*)to + i * kRows * 2 * D + at) = x[i][0];
      } else {
        *(uint4*)((float*)to + row * D + d) = x[i][0];
        *(uint4*)((float*)to + row * D + d + 4) = x[i][W - 1];
      }
    }
  }
};

// Coefficients of a chunk, by processing order.
struct Coef {
  float grow[64], left[64];      // exp(run_i), exp(total - run_i)
  float high[64], low[64];       // run_i log2 e = high + low
  float total;                   // exp(total)
};

constexpr double kLog2e = 1.4426950408889634;

__device__ __forceinline__ float exp_of(double x) { return __builtin_amdgcn_exp2f((float)x); }

// The log decay of the lane's row.
__device__ __forceinline__ float decay_of(const DecayPlan& p, const DecayChunk& c, int back, int h) {
  const int lane = threadIdx.x & 63;
  // from the last token to the first, a decay belongs to the row after its token
  const int at = back ? c.rows - lane : lane;
  if (lane < c.rows && (!back || lane > 0 || c.next_g))
    return bs_load_any(p.g, p.g_dtype, bs_delta_at(p.g_stride, c.batch, c.token + at, h));
  return 0.f;
}

// By one wave, lane = row, from decay_of.  Returns total (times log2 e).
__device__ __forceinline__ double coefficients(float g, Coef& o) {
  const int lane = threadIdx.x & 63;
  g = g < BS_DELTA_G_MIN ? BS_DELTA_G_MIN : g;
  double x = (double)g * kLog2e;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  const double total = __shfl(x, 63);
  o.high[lane] = (float)x;
  o.low[lane] = (float)(x - (double)(float)x);
  o.grow[lane] = exp_of(x);
  o.left[lane] = exp_of(total - x);
  if (lane == 0) o.total = exp_of(total);
  return total;
}

struct Place {                   // a lane's place in the products of 32 x 32
  int m, g;
  // fresh: formed anew where it stands, so that what follows from it is not kept in registers over
  // a loop (places in LDS, which would spill)
  __device__ __forceinline__ explicit Place(bool fresh) {
    int lane = threadIdx.x & 63;
    if (fresh) asm volatile("" : "+v"(lane));
    m = lane & 31, g = lane >> 5;
  }
  // Where this lane reads 4 rows 16 ks + 8 g + 4 second .. (and 32 D ks further on) x 4 columns of a
  // 16-bit tile for the transposing read: `piece` and the upper or lower half of it, by what column
  // of 4 (lane % 4) it gives for the 16 lanes it reads with.
  template <int D>
  __device__ __forceinline__ int turn(int piece, int upper, int second) const {
    return place<D>(8 * g + 4 * second + (m >> 2 & 3), piece) + 8 * upper;
  }
};

// Row m of a tile of value columns (and of att^T): lane group g then has 16 neighbouring ones.
__device__ __forceinline__ int value_row(int m) {
  return 16 * (m >> 2 & 1) + 4 * (m >> 3) + (m & 3);
}

// V^T of 32 value columns from `col`: fragments of 16 tokens each, 8 values a lane.
template <typename T>
__device__ __forceinline__ void turned_v(const void* v, int col, const Place& l,
                                         uint4 (*r)[sizeof(T) / 2]) {
  if constexpr (sizeof(T) == 2) {
    const int x = l.m & 3, half = l.m >> 4, piece = col / 8 + 2 * (x & 1) + half;
    const int a = l.turn<kPitch>(piece, x >> 1, 0), b = l.turn<kPitch>(piece, x >> 1, 1);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const uint2 p = turn4(v, a + ks * 32 * kPitch), q = turn4(v, b + ks * 32 * kPitch);
      r[ks][0] = make_uint4(p.x, p.y, q.x, q.y);
    }
  } else {
    const uint32_t* p = (const uint32_t*)v + 8 * l.g * kPitch + col + value_row(l.m);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks, p += 16 * kPitch) {
      r[ks][0] = make_uint4(p[0], p[kPitch], p[2 * kPitch], p[3 * kPitch]);
      r[ks][1] = make_uint4(p[4 * kPitch], p[5 * kPitch], p[6 * kPitch], p[7 * kPitch]);
    }
  }
}

// The wave's 32 columns of a state: element e of tile rt is row 32 rt + 16 (e / 8) + 8 g + e % 8.
template <int RT>
struct Columns {
  bs_f32x16 s[RT];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < RT; ++i) s[i] = zero16();
  }
  // f(tile, element, its offset in bytes): a buffer's bounds leave out what the lane does not have,
  // so the offset is whole in the one register that they are checked against
  template <typename F>
  static __device__ __forceinline__ void each(const DecayRun& r, const DecayState& st, int col,
                                              const Place& l, F&& f) {
    const int c = col + value_row(l.m), have = c < r.dv ? r.dc - 8 * l.g : 0;
    const uint32_t at = 4u * (c * st.col + 8 * l.g * st.row), row = 4u * st.row;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int d = 32 * i + 16 * (e >> 3) + (e & 7);
        f(i, e, d < have ? at + d * row : 0x80000000u);
      }
  }
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t place_of(const DecayRun& r,
                                                                   const DecayState& st,
                                                                   int64_t at) {
    const uint64_t p = (uint64_t)(st.p + at * r.dc * r.dv);
    const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32 |
                          (uint32_t)__builtin_amdgcn_readfirstlane((int)p);
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 4 * r.dc * r.dv, 0x00027000);
  }
  __device__ __forceinline__ void load(const DecayRun& r, const DecayState& st, int64_t at, int col,
                                       const Place& l) {
    clear();
    if (!st.p) return;
    const __amdgpu_buffer_rsrc_t rs = place_of(r, st, at);
    each(r, st, col, l, [&](int i, int e, uint32_t at) {
      s[i][e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, 0));
    });
  }
  __device__ __forceinline__ void store(const DecayRun& r, const DecayState& st, int64_t at,
                                        float scale, int col, const Place& l) const {
    const __amdgpu_buffer_rsrc_t rs = place_of(r, st, at);
    each(r, st, col, l, [&](int i, int e, uint32_t at) {
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(scale * s[i][e]), rs, at, 0, 0);
    });
  }
  // as saved states lie: tile by tile, 4 values of a lane side by side
  static __device__ __forceinline__ int64_t saved_at(const DecayRun& r, int64_t slot_head, int wave) {
    return slot_head * decay_saved(r.dc, r.dv) + wave * ((r.dc + 31) / 32 * 1024) +
           (threadIdx.x & 63) * 4;
  }
  __device__ __forceinline__ void save(const DecayRun& r, int64_t slot_head, int wave) const {
    float* p = r.save + saved_at(r, slot_head, wave);
#pragma unroll
    for (int i = 0; i < RT; ++i)
      if (32 * i < r.dc) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *(float4*)(p + (4 * i + e) * 256) = make_float4(s[i][4 * e], s[i][4 * e + 1],
                                                          s[i][4 * e + 2], s[i][4 * e + 3]);
      }
  }
  // this lane's part of the product with a saved state
  __device__ __forceinline__ float product(const DecayRun& r, int64_t slot_head, int wave) const {
    const float* p = r.saved + saved_at(r, slot_head, wave);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < RT; ++i)
      if (32 * i < r.dc) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 x = *(const float4*)(p + (4 * i + e) * 256);
          sum = fmaf(x.x, s[i][4 * e], sum), sum = fmaf(x.y, s[i][4 * e + 1], sum);
          sum = fmaf(x.z, s[i][4 * e + 2], sum), sum = fmaf(x.w, s[i][4 * e + 3], sum);
        }
      }
    return sum;
  }
  // s = decay s + K^T (left V) with V's turned fragments of 16 tokens each
  template <typename T, int DC>
  __device__ __forceinline__ void add(const uint16_t* k, const uint4 (*v)[sizeof(T) / 2],
                                      const Coef& co, float scale, const Place& l,
                                      const Splitter& sp) {
    constexpr int PI = kParts<T>;
    const float total = co.total;
#pragma unroll
    for (int i = 0; i < RT; ++i) s[i] *= total;
    const int x = l.m & 3, piece = 2 * (l.m >> 4) + (x & 1);
    const int first = l.turn<DC>(piece, x >> 1, 0), second = l.turn<DC>(piece, x >> 1, 1);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      float f[8];
      floats<T>(v[ks], f);
      const float* lf = co.left + 16 * ks + 8 * l.g;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= scale * lf[j];
      const bs_parts<3> vp = sp.split<3>(f);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        bs_parts<PI> kp;
#pragma unroll
        for (int p = 0; p < PI; ++p) {
          const int at = (p * 64 + 16 * ks) * 2 * DC;
          const uint2 a = turn4(k, (first ^ 64 * i) + at), b = turn4(k, (second ^ 64 * i) + at);
          kp.p[p] = __builtin_bit_cast(bs_bf16x8, make_uint4(a.x, a.y, b.x, b.y));
        }
        s[i] = mma(kp, vp, s[i]);
      }
    }
  }
};

struct Carry {
  float* factor;               // [segs][hv]: decay of a state over the slots a segment takes
  DecayLink* link;             // [segs]
};

// What the slots of a segment that the next one goes on with add to the state, from zero.
template <typename T, int RT, bool VEC>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void sum_kernel(DecayRun run,
                                                                             DecayPlan plan,
                                                                             Carry carry) {
  constexpr int DC = 32 * RT, PI = kParts<T>;
  __shared__ __attribute__((aligned(16))) uint16_t lk[PI * 64 * DC];
  __shared__ __attribute__((aligned(16))) T lv[64 * kPitch];
  __shared__ Coef coef[2];
  const int seg = blockIdx.x, h = blockIdx.y;
  int from = seg * plan.per, to = min(from + plan.per, plan.seq.slots);
  const DecayLink link = link_of(plan.seq, run.back, from, to);
  if (h == 0 && threadIdx.x == 0) carry.link[seg] = link;
  if (link.seq < 0) return;
  const Place l(false);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = 32 * wave;
  const bool live = col < run.dv;
  Chunks chunks(plan.seq, from, to, run.back);
  DecayChunk c;
  auto none = [](int) {};
  const Splitter sp;
  const HeadRows kh = HeadRows::of<T>(run.k, h), vh = HeadRows::of<T>(run.v, h);
  Staged<T, DC> k;
  Staged<T, kPitch> v;
  auto load = [&](const DecayChunk& at) {
    k.load(ChunkRows<T, VEC>(kh, at, run.dc, run.back));
    v.load(ChunkRows<T, VEC>(vh, at, run.dv, run.back));
  };
  double decay = 0.0;
  float g = 0.f;                  // of the chunk that is loaded next, a chunk ahead of its use
  bool more = chunks.next(plan.seq, c, none);
  if (more) {
    load(c);
    if (wave == 3) decay += coefficients(decay_of(plan, c, run.back, h), coef[0]);
  }
  bool ahead = more && chunks.next(plan.seq, c, none);
  if (ahead && wave == 3) g = decay_of(plan, c, run.back, h);
  Columns<RT> s;
  s.clear();
  for (int at = 0; more; at ^= 1) {
    const Place l(true);
    __syncthreads();
    k.put(lk, Cutter());
    v.put_raw(lv);
    __syncthreads();
    more = ahead;
    if (more) {
      load(c);
      if (wave == 3) decay += coefficients(g, coef[at ^ 1]);
      ahead = chunks.next(plan.seq, c, none);
      if (ahead && wave == 3) g = decay_of(plan, c, run.back, h);
    }
    if (live) {
      const Place l(true);
      uint4 vf[4][sizeof(T) / 2];
      turned_v<T>(lv, col, l, vf);
      s.template add<T, DC>(lk, vf, coef[at], run.add_scale, l, sp);
    }
  }
  if (live) s.store(run, run.start, (int64_t)seg * plan.hv + h, 1.f, col, l);
  if (threadIdx.x == 192) carry.factor[seg * plan.hv + h] = exp_of(decay);
}

// The states before the segments, in place of the segments' sums: a lane has one element of a
// head's state.
__global__ __launch_bounds__(256) void scan_kernel(DecayRun run, DecayPlan plan, Carry carry) {
  const int n = run.dc * run.dv, e = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
  if (e >= n) return;
  const int r = e / run.dv, c = e % run.dv;
  float* p = run.start.p + (int64_t)h * n + e;
  const int64_t step = (int64_t)plan.hv * n;
  float state = 0.f;
  constexpr int kAhead = 8;      // segments whose loads are in flight together
  for (int i0 = 0; i0 < plan.segs; i0 += kAhead) {
    float x[kAhead], factor[kAhead];
    DecayLink link[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = min(i0 + i, plan.segs - 1), seg = run.back ? plan.segs - 1 - at : at;
      x[i] = p[seg * step];
      link[i] = carry.link[seg], factor[i] = carry.factor[seg * plan.hv + h];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i0 + i >= plan.segs) break;
      p[(run.back ? plan.segs - 1 - i0 - i : i0 + i) * step] = state;
      if (link[i].seq < 0) continue;
      if (link[i].first)
        state = run.first.p ? run.first.p[((int64_t)link[i].seq * plan.hv + h) * n +
                                          r * run.first.row + c * run.first.col]
                            : 0.f;
      state = fmaf(factor[i], state, x[i]);
    }
  }
}

struct Runs { DecayRun r[3]; };

template <typename T>
__device__ void zero_rows(const DecayPlan& plan, T* o, int dv, int h) {
  zero_outside(plan.seq, o, plan.hv, dv, h, 0, kPitch);
}

// sum_j P_ij for row i and sum_i P_ij for column j of a 32 x 32 tile, of which a lane has 16 j of
// one i: the first in lane i of either group, the second of j = 16 g + m / 2.
__device__ __forceinline__ void pair_sums(const float* p, const Place& l, double& row,
                                          double& col) {
  double v[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = p[e];
  row = 0.0;
#pragma unroll
  for (int e = 0; e < 16; ++e) row += v[e];
  row += __shfl_xor(row, 32);
#pragma unroll
  for (int w = 8; w >= 1; w >>= 1) {     // lanes 2 w apart share out their values
    const bool up = l.m & 2 * w;
#pragma unroll
    for (int k = 0; k < w; ++k) {
      const double mine = up ? v[k + w] : v[k], other = up ? v[k] : v[k + w];
      v[k] = mine + __shfl_xor(other, 2 * w);
    }
  }
  col = v[0] + __shfl_xor(v[0], 1);
}

// 8 values of a row of V as it lies in LDS; `at`: where the row's piece g lies (16-bit), or value 8 g.
template <typename T>
__device__ __forceinline__ void straight_v(const T* v, int at, int step, uint4* x) {
  if constexpr (sizeof(T) == 2) {
    x[0] = *(const uint4*)((const char*)v + (at ^ 32 * step));
  } else {
    x[0] = *(const uint4*)(v + at + 16 * step);
    x[1] = *(const uint4*)(v + at + 16 * step + 4);
  }
}

// Sets infinities and NaN among the values of a word to 0; whether there were any.
template <typename T>
__device__ __forceinline__ bool drop_values(uint32_t& w) {
  constexpr uint32_t kExp = std::is_same<T, bs_f16>::value ? 0x7C00u : 0x7F80u;   // bits of an exponent
  const bool high = (w & kExp << 16) == kExp << 16, low = (w & kExp) == kExp;
  if constexpr (sizeof(T) == 4) {
    w = high ? 0u : w;
    return high;
  } else {
    w = high ? w & 0xFFFFu : w;
    w = low ? w & 0xFFFF0000u : w;
    return high | low;
  }
}

// Value `col` of row j of V.
template <typename T>
__device__ __forceinline__ float value_at(const T* v, int j, int col) {
  if constexpr (sizeof(T) == 4) return v[j * kPitch + col];
  else return bs_to_f32(*(const T*)((const char*)v + place<kPitch>(j, col >> 3) + 2 * (col & 7)));
}

template <typename T, int RT, bool VEC, bool GRAD>
__global__ __launch_bounds__(kThreads, kParts<T> == 1 ? 2 : 1) void walk_kernel(Runs runs,
                                                                              DecayPlan plan) {
  constexpr int DC = 32 * RT, PI = kParts<T>, W = sizeof(T) / 2;
  __shared__ __attribute__((aligned(16))) uint16_t lq[PI * 64 * DC];
  __shared__ __attribute__((aligned(16))) uint16_t lk[PI * 64 * DC];
  __shared__ __attribute__((aligned(16))) T lv[64 * kPitch];
  __shared__ __attribute__((aligned(16))) uint16_t la[3 * 64 * 64];     // att, [part][i][j]
  __shared__ Coef coef[2];
  __shared__ float dots[GRAD ? 4 : 1][64];
  __shared__ float edge[4];
  __shared__ double sums[GRAD ? 3 : 1][2][32];       // of P's tiles
  const DecayRun& run = runs.r[blockIdx.z];
  const int seg = blockIdx.x, h = blockIdx.y;
  if (seg >= plan.segs) {
    if (run.o_f32) zero_rows(plan, (float*)run.o, run.dv, h);
    else zero_rows(plan, (T*)run.o, run.dv, h);
    return;
  }
  const int from = seg * plan.per, to = min(from + plan.per, plan.seq.slots);
  const Place l(false);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = 32 * wave;
  const bool live = col < run.dv;
  Chunks chunks(plan.seq, from, to, run.back);
  const int n = run.dc * run.dv;
  auto empty = [&](int seq) {                 // a sequence without tokens keeps its state
    if (!run.last.p) return;
    const int64_t at = ((int64_t)seq * plan.hv + h) * n;
    for (int e = threadIdx.x; e < n; e += kThreads) {
      const int r = e / run.dv, c = e % run.dv;
      run.last.p[at + r * run.last.row + c * run.last.col] =
          run.first.p ? run.first.p[at + r * run.first.row + c * run.first.col] : 0.f;
    }
  };
  const Splitter sp;
  const HeadRows qh = HeadRows::of<T>(run.q, h), kh = HeadRows::of<T>(run.k, h),
                 vh = HeadRows::of<T>(run.v, h), dh = HeadRows::of<T>(run.dot, h);
  Staged<T, DC> q, k;
  Staged<T, kPitch> v;
  auto load = [&](const DecayChunk& at) {
    q.load(ChunkRows<T, VEC>(qh, at, run.dc, run.back));
    k.load(ChunkRows<T, VEC>(kh, at, run.dc, run.back));
    v.load(ChunkRows<T, VEC>(vh, at, run.dv, run.back));
  };
  auto put = [&]() {
    q.put(lq, sp);
    k.put(lk, Cutter());
    v.put_raw(lv);
  };
  DecayChunk c, next;
  float g = 0.f;                  // of the next chunk, loaded an iteration ahead of its use
  if (!chunks.next(plan.seq, c, empty)) return;
  load(c);
  if (wave == 3) coefficients(decay_of(plan, c, run.back, h), coef[0]);
  bool more = chunks.next(plan.seq, next, empty);
  if (more && wave == 3) g = decay_of(plan, next, run.back, h);
  Columns<RT> s;
  if (live && !c.first) s.load(run, run.start, (int64_t)seg * plan.hv + h, col, l);
  put();
  __syncthreads();
  for (int at = 0;; at ^= 1) {
    const Place l(true);
    if (more) load(next);
    const Coef& co = coef[at];
    if (live && c.first) s.load(run, run.first, (int64_t)c.seq * plan.hv + h, col, l);
    if (wave < 3) {                           // att^T: the tiles (0, 0), (0, 1), (1, 1)
      const int jt = wave >> 1, it = (wave + 1) >> 1, i = 32 * it + l.m;
      bs_f32x16 a = zero16();
      const int j = 32 * jt + value_row(l.m);
      constexpr int kPairs = GRAD ? kPitch / 32 : 1;     // fragments loaded together
      uint4 px[kPairs][W];
      auto load_pairs = [&](int half) {
        const ChunkRows<T, VEC> rows(dh, c, run.dv, run.back);
#pragma unroll
        for (int s = 0; s < kPairs; ++s)
          rows.raw(i, 16 * (kPairs * half + s) + 8 * l.g, px[s]);
      };
      if (GRAD && run.pairs) load_pairs(0);
      const int ka = place<DC>(j, l.g), qa = place<DC>(i, l.g);
#pragma unroll
      for (int s = 0; s < DC / 16; ++s) {
        bs_parts<PI> kp, qp;
#pragma unroll
        for (int p = 0; p < PI; ++p) {
          kp.p[p] = piece_at(lk, (ka ^ 32 * s) + p * 128 * DC);
          qp.p[p] = piece_at(lq, (qa ^ 32 * s) + p * 128 * DC);
        }
        a = mma(kp, qp, a);
      }
      const float high = co.high[i], low = co.low[i];
      const int j0 = 32 * jt + 16 * l.g;
      float w[16];
#pragma unroll
      for (int e = 0; e < 16; ++e)
        w[e] = j0 + e <= i ? run.att_scale * a[e] *
                                 __builtin_amdgcn_exp2f((high - co.high[j0 + e]) +
                                                        (low - co.low[j0 + e]))
                           : 0.f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const bs_parts<3> p = sp.split<3>(w + 8 * half);
#pragma unroll
        for (int x = 0; x < 3; ++x)
          *(bs_bf16x8*)((char*)la + (place<64>(i, j0 / 8) ^ 16 * half) + x * 128 * 64) = p.p[x];
      }
      if (GRAD && run.pairs) {
        a = zero16();
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int s = 0; s < kPairs; ++s) {
            uint4 y[W];
            straight_v(lv, W == 1 ? place<kPitch>(j, l.g) : j * kPitch + 8 * l.g,
                       kPairs * half + s, y);
            a = mma(parts_of<T>(sp, y), parts_of<T>(sp, px[s]), a);
          }
          if (half == 0) load_pairs(1);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] *= a[e];
        double row, column;
        pair_sums(w, l, row, column);
        if (l.g == 0) sums[wave][0][l.m] = row;
        if (!(l.m & 1)) sums[wave][1][16 * l.g + l.m / 2] = column;
      }
    } else if (more) {
      coefficients(g, coef[at ^ 1]);
    }
    __builtin_amdgcn_sched_barrier(0);        // phase by phase: registers for one at a time
    bs_f32x16 o[2] = {zero16(), zero16()};
    if (!GRAD && live && run.save && !c.first) s.save(run, (int64_t)c.slot * plan.hv + h, wave);
    if (GRAD && live && run.saved && !c.first) {
      float sum = s.product(run, (int64_t)(c.slot + 1) * plan.hv + h, wave);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
      if ((threadIdx.x & 63) == 0) edge[wave] = sum;
    }
    if (live) {
      uint4 dx[2][2][W];
      if (GRAD && run.dot.p) {
        const ChunkRows<T, VEC> rows(dh, c, run.dv, run.back);
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            rows.raw(32 * it + l.m, col + 16 * l.g + 8 * half, dx[it][half]);
      }
      const int qa = place<DC>(l.m, l.g);
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = s.s[i][8 * half + e];
          const bs_parts<3> st = sp.split<3>(f);
#pragma unroll
          for (int it = 0; it < 2; ++it) {
            bs_parts<PI> qp;
#pragma unroll
            for (int p = 0; p < PI; ++p)
              qp.p[p] = piece_at(lq, (qa ^ 16 * (4 * i + 2 * half)) + (p * 64 + 32 * it) * 2 * DC);
            o[it] = mma(st, qp, o[it]);
          }
        }
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        const int i = 32 * it + l.m;
        o[it] *= run.grow_scale * co.grow[i];
        if (GRAD && run.dot.p) {
          float sum = 0.f;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float f[8];
            floats<T>(dx[it][half], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(f[e], o[it][8 * half + e], sum);
          }
          sum += __shfl_xor(sum, 32);
          if (l.g == 0) dots[wave][i] = sum;
        }
      }
    }
    __syncthreads();                          // att
    if (live) {
      uint4 vf[4][W];
      turned_v<T>(lv, col, l, vf);
      // A token takes nothing from a later one, but its 0 in att times an infinity or NaN is NaN.  One in
      // a value column leaves every row of that column of the state so: a look at one row tells.  Such
      // values are left out of the product here and taken one by one below.
      const bool was = isfinite(s.s[0][0]);
      s.template add<T, DC>(lk, vf, co, run.add_scale, l, sp);
      uint32_t apart = 0;                      // bit m: column value_row(m) has such values
      if (__ballot(was && !isfinite(s.s[0][0]))) {
        bool any = false;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
          for (int w = 0; w < W; ++w) {
            any |= drop_values<T>(vf[ks][w].x) | drop_values<T>(vf[ks][w].y) |
                   drop_values<T>(vf[ks][w].z) | drop_values<T>(vf[ks][w].w);
            __builtin_amdgcn_sched_barrier(0);
          }
        const uint64_t hit = __ballot(any);
        apart = (uint32_t)hit | (uint32_t)(hit >> 32);
      }
      const int aa = place<64>(l.m, l.g);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const bs_parts<PI> vp = parts_of<T>(sp, vf[ks]);
#pragma unroll
        for (int it = ks >> 1; it < 2; ++it) {
          bs_parts<3> ap;
#pragma unroll
          for (int p = 0; p < 3; ++p)
            ap.p[p] = piece_at(la, (aa ^ 32 * ks) + (p * 64 + 32 * it) * 128);
          o[it] = mma(vp, ap, o[it]);
        }
      }
      const int oc = col + 16 * l.g;
      if (apart) {
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll 1
          for (int j = 0; j <= 32 * it + l.m; ++j) {
            const char* p = (const char*)la + place<64>(32 * it + l.m, j >> 3) + 2 * (j & 7);
            float a = 0.f;
#pragma unroll
            for (int x = 2; x >= 0; --x) a += bs_to_f32(*(const bs_bf16*)(p + x * 128 * 64));
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (apart >> (8 * (e >> 2) + 4 * l.g + (e & 3)) & 1) {
                const float x = value_at(lv, j, oc + e);
                if (!isfinite(x)) o[it][e] = fmaf(a, x, o[it][e]);
              }
          }
      }
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        const int i = 32 * it + l.m;
        // rows past the chunk's end lie past the buffer's
        const int row = run.back ? c.rows - 1 - i : i;
        auto put_out = [&](auto* out) {
          using O = typename std::remove_pointer<decltype(out)>::type;
          const int step = plan.hv * run.dv * (int)sizeof(O);
          const uint64_t p = (uint64_t)(out + ((c.batch * plan.seq.tokens + c.token) * plan.hv + h) *
                                                  run.dv);
          const uint64_t base =
              (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32 |
              (uint32_t)__builtin_amdgcn_readfirstlane((int)p);
          const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
              (void*)base, 0, (c.rows - 1) * step + run.dv * (int)sizeof(O), 0x00027000);
          auto at = [&](int e) {
            return row >= 0 && row < c.rows && oc + e < run.dv
                       ? (uint32_t)(row * step) + (oc + e) * (uint32_t)sizeof(O)
                       : 0xFFFFFF00u;
          };
          if (run.vec_o) {
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
              bs_u32x4 x[sizeof(O) / 2];
              O t[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) t[j] = bs_from_f32<O>(o[it][e + j]);
              __builtin_memcpy(x, t, sizeof(t));
              const uint32_t to = at(e);
#pragma unroll
              for (int j = 0; j < (int)sizeof(O) / 2; ++j)
                __builtin_amdgcn_raw_buffer_store_b128(x[j], rs, to + 16 * j, 0, 0);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const O x = bs_from_f32<O>(o[it][e]);
              if constexpr (sizeof(O) == 4)
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x), rs, at(e), 0, 0);
              else
                __builtin_amdgcn_raw_buffer_store_b16(x.u, rs, at(e), 0, 0);
            }
          }
        };
        if (run.o_f32) put_out((float*)run.o);
        else put_out((T*)run.o);
      }
      if (c.last && run.last.p) {
        float scale = 1.f;
        if (run.back) {
          const float g = bs_load_any(plan.g, plan.g_dtype,
                                      bs_delta_at(plan.g_stride, c.batch, c.token, h));
          scale = exp_of((g < BS_DELTA_G_MIN ? BS_DELTA_G_MIN : g) * kLog2e);
        }
        s.store(run, run.last, (int64_t)c.seq * plan.hv + h, scale, col, l);
      }
    }
    __syncthreads();                          // the chunk's last readers are through
    if (GRAD && run.dot.p && threadIdx.x < c.rows) {
      const int i = threadIdx.x, m = i & 31;
      double sum = dots[0][i];
      for (int w = 1; 32 * w < run.dv; ++w) sum += dots[w][i];
      if (run.pairs)
        sum += i < 32 ? sums[0][0][m] - sums[0][1][m] - sums[1][1][m]
                      : sums[1][0][m] + sums[2][0][m] - sums[2][1][m];
      const int64_t row = c.batch * plan.seq.tokens + c.token + (run.back ? c.rows - 1 - i : i);
      run.dots[(int64_t)h * run.rows + row] = sum;
    }
    if (GRAD && run.saved && !c.first && threadIdx.x == 0) {
      float sum = edge[0];
      for (int w = 1; 32 * w < run.dv; ++w) sum += edge[w];
      // the decay of the next chunk's first token stands between
      run.edge[(int64_t)c.slot * plan.hv + h] = co.grow[0] * sum;
    }
    if (!more) return;
    put();
    c = next;
    more = chunks.next(plan.seq, next, empty);
    if (more && wave == 3) g = decay_of(plan, next, run.back, h);
    __syncthreads();
  }
}

// Sequences without tokens keep their states.
__global__ __launch_bounds__(256) void keep_kernel(const float* from, float* to, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    to[i] = from ? from[i] : 0.f;
}

// f(element, tiles of 32 rows of a state, whether operands' rows start on 16 bytes and end on 8
// values)
template <typename F>
void by_type(int dtype, int wide, int vec, F&& f) {
  using Two = std::integral_constant<int, 2>;
  using Four = std::integral_constant<int, 4>;
  auto sized = [&](auto t) {
    auto placed = [&](auto rt) {
      if (vec) f(t, rt, std::true_type());
      else f(t, rt, std::false_type());
    };
    if (wide) placed(Four());
    else placed(Two());
  };
  if (dtype == BS_F32) sized(float());
  else if (dtype == BS_BF16) sized(bs_bf16());
  else sized(bs_f16());
}

int vectors(const DecayOperand& x, int dim, int dtype) {
  const int per = 16 / bs_dtype_size(dtype);
  int ok = dim % 8 == 0 && (uintptr_t)x.p % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && x.stride[i] % per == 0;
  return ok;
}

int64_t align16(int64_t n) { return (n + 15) / 16 * 16; }

}  // namespace

DecayPlan decay_plan(const bs_delta_in& in, int seqs, int tokens, const int32_t* offsets) {
  DecayPlan p;
  p.seq = delta_plan(seqs, tokens, offsets);
  p.hv = in.hv, p.g = in.g, p.g_dtype = in.g_dtype;
  for (int i = 0; i < 3; ++i) p.g_stride[i] = in.g_stride[i];
  // As many segments as the card takes workgroups at a time: 8,192 tokens of 32 heads in bf16 take 165
  // us with two workgroups a CU, 195 with one, 193 with three.  Of 2 chunks at least, since a state a
  // segment is what the carry reads and writes: 16,384 tokens of one head of 128 in bf16 take 65 us so, 85
  // with 1, 68 with 4; 2,048 tokens of 4 heads 39, 36 and 56; 700 tokens of 3 heads of 48 in 32 bits, where
  // the latency of a chunk is most of it, 33, 24 and 54.
  const int64_t units = (int64_t)p.seq.slots * in.hv;
  const int64_t at_once = (in.dtype == BS_BF16 ? 2 : 1) * bs_num_cus();
  int64_t per = (units + at_once - 1) / at_once;
  per = per < 2 ? 2 : per;
  p.carry = 1;
  const int whole = (tokens + kChunk - 1) / kChunk;       // chunks of a sequence
  if (!offsets && whole && per >= whole) {
    per = per / whole * whole;
    p.carry = 0;
  }
  if (per >= p.seq.slots) {
    per = p.seq.slots;
    p.carry = 0;
  }
  p.per = (int)per;
  p.segs = p.seq.slots ? (int)((p.seq.slots + per - 1) / per) : 0;
  return p;
}

int decay_check(const bs_delta_in* in, int seqs, int tokens, const int32_t* offsets,
                const char* who) {
  if (int rc = delta_check_chunked(in, seqs, tokens, offsets, who)) return rc;
  BS_CHECK_ARG(in->hv <= 65535, "%s: %d heads exceed one launch", who, in->hv);
  const int64_t slots = offsets ? (int64_t)tokens / kChunk + seqs
                                : (int64_t)seqs * ((tokens + kChunk - 1) / kChunk);
  BS_CHECK_ARG((slots + 1) * in->hv < 1 << 22 && (int64_t)seqs * in->hv < 1 << 22,
               "%s: %d sequences of %d tokens, %d heads exceed one launch", who, seqs, tokens,
               in->hv);
  return BS_OK;
}

DecayRun decay_run(const bs_delta_in& in, const DecayOperand& q, const DecayOperand& k,
                   const DecayOperand& v, const DecayOperand& dot, int dc, int dv) {
  DecayRun r = {};
  r.q = q, r.k = k, r.v = v, r.dot = dot, r.dc = dc, r.dv = dv;
  r.first = r.last = r.start = DecayState{nullptr, dv, 1};
  r.vec = vectors(q, dc, in.dtype) && vectors(k, dc, in.dtype) && vectors(v, dv, in.dtype) &&
          (!dot.p || vectors(dot, dv, in.dtype));
  r.att_scale = r.grow_scale = in.scale, r.add_scale = 1.f;
  return r;
}

int64_t decay_carry_bytes(const bs_delta_in& in, const DecayPlan& plan) {
  if (!plan.carry) return 0;
  return align16((int64_t)plan.segs * in.hv * 4) + align16((int64_t)plan.segs * sizeof(DecayLink));
}

void decay_carry(const DecayRun& run, const DecayPlan& plan, int dtype, void* scratch,
                 hipStream_t st) {
  Carry c;
  c.factor = (float*)scratch;
  c.link = (DecayLink*)((char*)scratch + align16((int64_t)plan.segs * plan.hv * 4));
  by_type(dtype, run.dc > 64, run.vec, [&](auto t, auto rt, auto vec) {
    sum_kernel<decltype(t), rt.value, vec.value><<<dim3(plan.segs, plan.hv), kThreads, 0, st>>>(run, plan, c);
  });
  scan_kernel<<<dim3((run.dc * run.dv + 255) / 256, plan.hv), 256, 0, st>>>(run, plan, c);
}

void decay_walk(const DecayRun* runs, int n, const DecayPlan& plan, int dtype, hipStream_t st) {
  const bool grad = n > 1;     // the gradients' walks, else the forward one
  Runs r = {};
  int wide = 0, aligned = 1;
  for (int i = 0; i < n; ++i) {
    r.r[i] = runs[i];
    wide |= runs[i].dc > 64;
    aligned &= runs[i].vec;
  }
  const dim3 grid(plan.segs + (plan.seq.offsets ? 1 : 0), plan.hv, n);
  if (grid.x == 0) return;
  by_type(dtype, wide, aligned, [&](auto t, auto rt, auto vec) {
    if (grad)
      walk_kernel<decltype(t), rt.value, vec.value, true><<<grid, kThreads, 0, st>>>(r, plan);
    else walk_kernel<decltype(t), rt.value, vec.value, false><<<grid, kThreads, 0, st>>>(r, plan);
  });
}

void decay_keep(const float* from, float* to, int64_t n, hipStream_t st) {
  const int64_t blocks = (n + 255) / 256;
  keep_kernel<<<(unsigned)(blocks < 65536 ? blocks : 65536), 256, 0, st>>>(from, to, n);
}

int64_t decay_kept_bytes(const bs_delta_in& in, const DecayPlan& plan, int keep) {
  if (!keep) return 0;
  const int64_t start = plan.carry ? (int64_t)plan.segs * in.hv * in.dk * in.dv * 4 : 0;
  return align16(start) +
         (keep > 1 ? (int64_t)plan.seq.slots * in.hv * decay_saved(in.dk, in.dv) * 4 : 0);
}

float* decay_kept_saved(const bs_delta_in& in, const DecayPlan& plan, void* kept) {
  return (float*)((char*)kept + decay_kept_bytes(in, plan, 1));
}

extern "C" size_t bs_decay_attention_kept_size(const bs_delta_in* in, int32_t seqs, int32_t tokens,
                                               int32_t packed, int32_t keep) {
  static const int32_t dummy[1] = {0};
  const int32_t* off = packed ? dummy : nullptr;
  if (decay_check(in, seqs, tokens, off, "bs_decay_attention_kept_size")) return 0;
  return (size_t)decay_kept_bytes(*in, decay_plan(*in, seqs, tokens, off), keep);
}

extern "C" size_t bs_decay_attention_workspace_size(const bs_delta_in* in, int32_t seqs,
                                                    int32_t tokens, int32_t packed, int32_t keep) {
  static const int32_t dummy[1] = {0};
  const int32_t* off = packed ? dummy : nullptr;
  if (decay_check(in, seqs, tokens, off, "bs_decay_attention_workspace_size")) return 0;
  const DecayPlan p = decay_plan(*in, seqs, tokens, off);
  return (size_t)(decay_carry_bytes(*in, p) + (keep ? 0 : decay_kept_bytes(*in, p, 1)));
}

extern "C" int bs_decay_attention(const bs_delta_in* in, int32_t seqs, int32_t tokens,
                                  const int32_t* seq_offsets, const float* initial_state,
                                  float* final_state, void* o, void* kept, int32_t keep,
                                  void* workspace, size_t workspace_bytes, bs_stream_t stream) {
  static const char* who = "bs_decay_attention";
  if (int rc = decay_check(in, seqs, tokens, seq_offsets, who)) return rc;
  if (seqs == 0 && !seq_offsets) return BS_OK;
  const DecayPlan plan = decay_plan(*in, seqs, tokens, seq_offsets);
  const size_t need =
      bs_decay_attention_workspace_size(in, seqs, tokens, seq_offsets != nullptr, keep);
  BS_CHECK_ARG(tokens == 0 || (in->q && in->k && in->v && in->g && o), "%s: NULL pointer", who);
  BS_CHECK_ARG(keep >= 0 && keep <= 2 && (kept || !decay_kept_bytes(*in, plan, keep)),
               "%s: keep %d, kept is NULL", who, keep);
  BS_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
               "%s: workspace of %zu bytes needed, %zu given", who, need,
               workspace ? workspace_bytes : (size_t)0);
  hipStream_t st = bs_stream(stream);
  const int64_t states = (int64_t)seqs * in->hv * in->dk * in->dv;
  if (plan.seq.slots == 0) {
    if (final_state && states) {
      decay_keep(initial_state, final_state, states, st);
      BS_CHECK_LAUNCH();
    }
    if (!seq_offsets || tokens == 0) return BS_OK;
  }
  const int group = in->hv / in->hk;
  auto op = [](const void* p, const int64_t* s, int rep) {
    return DecayOperand{p, {s[0], s[1], s[2]}, rep};
  };
  DecayRun run = decay_run(*in, op(in->q, in->q_stride, group), op(in->k, in->k_stride, group),
                           op(in->v, in->v_stride, 1), op(nullptr, in->v_stride, 1), in->dk,
                           in->dv);
  run.o = o;
  run.vec_o = in->dv % 8 == 0 && (uintptr_t)o % 16 == 0;
  run.first.p = const_cast<float*>(initial_state);
  run.last.p = final_state;
  if (plan.carry) {
    run.start.p = (float*)(keep ? kept : (char*)workspace + decay_carry_bytes(*in, plan));
    decay_carry(run, plan, in->dtype, workspace, st);
    BS_CHECK_LAUNCH();
  }
  if (keep > 1) run.save = decay_kept_saved(*in, plan, kept);
  decay_walk(&run, 1, plan, in->dtype, st);
  BS_CHECK_LAUNCH();
  return BS_OK;
}
