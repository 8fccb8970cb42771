// Plan and workspace of the chunked gated delta rule (delta_chunk.hip, delta_grad.hip).
#pragma once

#include "delta.h"

#include <type_traits>

constexpr int kChunk = 64;   // tokens of a chunk
constexpr int kCoef = 6 * kChunk;

// A sequence's chunks lie side by side in the workspace.  Where sequences are packed end to end
// their lengths are known on the device only; sequence n then starts at slot offsets[n] / 64 + n,
// which leaves room for every chunk of the sequences before it.
struct DeltaPlan {
  int seqs, tokens;           // tokens of each sequence, or of all of them when packed
  const int32_t* offsets;     // [seqs + 1] or NULL
  int slots;
};

struct DeltaSpan { int seq, chunks, slot; int64_t batch, first; int len; };

__device__ __forceinline__ int delta_offset(const DeltaPlan& p, int n) {
  return min(max(p.offsets[n], 0), p.tokens);
}

// Sequence n (the same in every lane): its first slot, batch row, first token and length.
__device__ __forceinline__ DeltaSpan delta_span(const DeltaPlan& p, int n) {
  n = __builtin_amdgcn_readfirstlane(n);
  DeltaSpan s;
  s.seq = n;
  if (p.offsets) {
    const int a = __builtin_amdgcn_readfirstlane(delta_offset(p, n));
    const int b = __builtin_amdgcn_readfirstlane(delta_offset(p, n + 1));
    s.batch = 0, s.first = a, s.len = max(b - a, 0);
    s.slot = a / kChunk + n;
    s.chunks = (s.len + kChunk - 1) / kChunk;
  } else {
    s.batch = n, s.first = 0, s.len = p.tokens;
    s.chunks = (s.len + kChunk - 1) / kChunk;
    s.slot = n * s.chunks;
  }
  return s;
}

// The sequence that owns a slot: the last one whose first slot is not past it, or the first one
// where every first slot is (no sequence's chunk lies there then).
__device__ __forceinline__ int delta_owner(const DeltaPlan& p, int slot) {
  if (!p.offsets) return slot / ((p.tokens + kChunk - 1) / kChunk);
  int lo = 0, hi = p.seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (delta_offset(p, mid) / kChunk + mid <= slot) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// The products are of 16 x 16 tiles over 32 values.  A product leaves rows 4g..4g+3 of a tile in
// lane group g and takes 8 values of the contracted index from it, so rows are dealt to tiles
// such that tiles 2s and 2s+1 hold rows 32s..32s+31 with 8 rows in a group, 4 in each tile: what
// one product leaves in a lane is what the next one takes from it.  delta_row is the token (or
// row of the state) of row m of tile t.
__device__ __forceinline__ int delta_row(int t, int m) {
  return 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3);
}

// Device arrays of a call, per slot and head, of fragments: the 8 values of each of 64 lanes as a
// product takes them, 1 KB side by side.  Fragment (t, s) of a matrix holds rows delta_row(t, .)
// and columns 32s + 8g .. + 7.
struct DeltaWork {
  uint16_t *kp, *qp;          // [slot][hk][parts][4][dkp / 32]: k and q, 0 past the end
  uint16_t *kt, *qt;          // [slot][hk][parts][dkp / 16][2]: their transposes
  uint16_t *inv;              // [slot][hv][3][6]: (1 + L)^-1 without its 32 x 32 block of zeros
  uint16_t *att;              // [slot][hv][3][6]: the masked q k^T; in the backward pass the
                              // transposes of both
  float *coef;                // [slot][hv][kCoef], see delta_coef
  float *ds, *dr;             // backward: [slot][hv][dkp][dvp], the gradient of the state after
                              // the chunk, and [slot][hv][64][dvp], that of R
};

// Rows of coef, 64 values each (the last in 64 bits).
enum delta_coef { kGrow = 0, kLeft = 1, kBeta = 2, kTotal = 3, kRun = 4 };
constexpr int kFrag = 512;                 // values of a fragment
constexpr int kSquare = 6 * kFrag;

// Fragment (t, s) of a lower triangular square, s <= t / 2; of an upper one, s >= t / 2.
__device__ __forceinline__ int delta_lower(int t, int s) { return t < 2 ? t : 2 * t - 2 + s; }
__device__ __forceinline__ int delta_upper(int t, int s) { return t < 2 ? 2 * t + s : t + 2; }

struct DeltaSizes {
  int64_t keys, square, coef, state, rows, bytes;
  int parts, dkp, dvp, ks;
};

static inline DeltaSizes delta_sizes(const bs_delta_in& in, int slots, int backward) {
  DeltaSizes s;
  s.parts = in.dtype == BS_BF16 ? 1 : in.dtype == BS_F16 ? 2 : 3;
  s.ks = in.dk <= 64 ? 2 : 4;
  s.dkp = 32 * s.ks;
  s.dvp = (in.dv + 31) / 32 * 32;
  s.keys = (int64_t)slots * in.hk * s.parts * kChunk * s.dkp;
  s.square = (int64_t)slots * in.hv * kSquare;
  s.coef = (int64_t)slots * in.hv * kCoef;
  s.state = backward ? (int64_t)slots * in.hv * s.dkp * s.dvp : 0;
  s.rows = backward ? (int64_t)slots * in.hv * kChunk * s.dvp : 0;
  s.bytes = s.keys * 2 * (backward ? 4 : 3) + s.square * 2 * 6 +
            (s.coef + s.state + s.rows) * 4;
  return s;
}

static inline DeltaWork delta_work(void* ws, const DeltaSizes& s, int backward) {
  DeltaWork w;
  char* p = (char*)ws;
  auto take = [&](int64_t bytes) {
    char* r = p;
    p += bytes;
    return r;
  };
  w.inv = (uint16_t*)take(s.square * 6);
  w.att = (uint16_t*)take(s.square * 6);
  w.coef = (float*)take(s.coef * 4);
  w.kp = (uint16_t*)take(s.keys * 2);
  w.qp = (uint16_t*)take(s.keys * 2);
  w.kt = (uint16_t*)take(s.keys * 2);
  w.qt = backward ? (uint16_t*)take(s.keys * 2) : nullptr;
  w.ds = backward ? (float*)take(s.state * 4) : nullptr;
  w.dr = backward ? (float*)take(s.rows * 4) : nullptr;
  return w;
}

static inline DeltaPlan delta_plan(int seqs, int tokens, const int32_t* offsets) {
  DeltaPlan p;
  p.seqs = seqs, p.tokens = tokens, p.offsets = offsets;
  p.slots = !seqs ? 0 : offsets ? tokens / kChunk + seqs
                                : seqs * ((tokens + kChunk - 1) / kChunk);
  return p;
}

int delta_check_chunked(const bs_delta_in* in, int seqs, int tokens, const int32_t* offsets,
                        const char* who);
int delta_prepare(const bs_delta_in& in, const DeltaPlan& plan, const DeltaWork& w,
                  const DeltaSizes& z, int backward, hipStream_t st);

// Four rows of NT columns (16 apart) of a chunk, 0 past the last row and column: buffer loads,
// whose bounds the hardware checks, so that the loads of a chunk stay free of branches (at a
// branch every load in flight is waited for).
template <typename T, int NT>
struct DeltaRows {
  using Raw = typename std::conditional<sizeof(T) == 4, float, uint16_t>::type;
  uint64_t base;           // the first chunk's first row
  int64_t step;            // bytes of a chunk's rows
  int bytes, row;          // of a row's columns; from row to row
  uint32_t at[NT][4];
  __device__ __forceinline__ DeltaRows(const T* first, int64_t stride, int out0, int col, int dv) {
    const uint64_t p = (uint64_t)first;      // the same in every lane
    base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32 |
           (uint32_t)__builtin_amdgcn_readfirstlane((int)p);
    row = (int)(stride * sizeof(T));
    step = (int64_t)kChunk * stride * sizeof(T);
    bytes = dv * (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < NT; ++i, col += 16)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        at[i][r] = col < dv ? (uint32_t)(out0 + r) * (uint32_t)row + col * (uint32_t)sizeof(T)
                            : 0xFFFFFFF0u;
  }
  // of chunk c of a sequence of `len`
  __device__ __forceinline__ void load(int c, int len, Raw (*x)[4]) const {
    const int rows = min(len - c * kChunk, kChunk);
    const uint32_t n = (uint32_t)(rows - 1) * (uint32_t)row + (uint32_t)bytes;
    __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)(base + c * step), 0, n, 0x00027000);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (sizeof(T) == 4)
          x[i][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, at[i][r], 0, 0));
        else
          x[i][r] = __builtin_amdgcn_raw_buffer_load_b16(rs, at[i][r], 0, 0);
      }
  }
  // what load gave, as numbers
  static __device__ __forceinline__ float value(Raw x) {
    if constexpr (sizeof(T) == 4) return x;
    else return bs_to_f32(T{x});
  }
};

// Kept matrices (states, U, dR: rows x dvp) are laid out as the backward pass's products over the
// value columns take them: fragment (t, s) has rows delta_row(t, .) and columns 32s + 8g .. + 7,
// in two halves of 4 columns, 1 KB each.  delta_kept is the place of the 4 columns 4g .. 4g + 3 of
// a slice of 16, row delta_row(t, m).
__device__ __forceinline__ int delta_kept(int t, int slice, int lane, int dvp) {
  const int m = lane & 15, g = lane >> 4;
  return (((t * (dvp >> 5) + (slice >> 1)) * 2 + (g & 1)) * 64 + 16 * (2 * (slice & 1) + (g >> 1)) +
          m) * 4;
}
// The 8 values of lane's fragment (t, s).
__device__ __forceinline__ const float* delta_kept_frag(const float* p, int t, int s, int lane,
                                                        int dvp) {
  return p + ((t * (dvp >> 5) + s) * 2 * 64 + lane) * 4;
}

// Waits for every load so far.  Ahead of a loop that keeps loads in flight: where the loop is
// entered with loads of its own in flight, the compiler has to wait in it as if it always were.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }

__device__ __forceinline__ bs_f32x4 zero4() { return bs_f32x4{0.f, 0.f, 0.f, 0.f}; }

// Parts of 8 floats in two vectors.
__device__ __forceinline__ bs_parts<3> row_parts(const float4& a, const float4& b) {
  const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  return bs_split8<3>(x);
}
__device__ __forceinline__ bs_parts<3> row_parts(const float* p) {
  return row_parts(*(const float4*)p, *(const float4*)(p + 4));
}

// Rows of a chunk, a lane one row: 8 neighbouring values of it, 0 past the row's end and past the
// last row.  Buffer loads, whose bounds the hardware checks: no branches, so nothing waits.
template <typename T>
struct DeltaRow {
  __amdgpu_buffer_rsrc_t rs;
  uint32_t at;
  int dim;              // 0 for a lane without a row
  bool vec;             // rows start on 16 bytes and end on 8 values
  __device__ __forceinline__ DeltaRow(const T* first, int64_t stride, int row, int rows, int d,
                                      bool v) {
    const uint32_t step = (uint32_t)(stride * sizeof(T));
    const uint64_t p = (uint64_t)first;
    const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32 |
                          (uint32_t)__builtin_amdgcn_readfirstlane((int)p);
    rs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)base, 0, (uint32_t)(rows - 1) * step + (uint32_t)(d * sizeof(T)), 0x00027000);
    at = (uint32_t)row * step, dim = row < rows ? d : 0, vec = v;
  }
  // values d .. d + 7
  __device__ __forceinline__ void raw(int d, uint4* x) const {
    constexpr int W = sizeof(T) / 2;           // vectors of 16 bytes
    if (vec) {
#pragma unroll
      for (int i = 0; i < W; ++i)
        x[i] = __builtin_bit_cast(
            uint4, __builtin_amdgcn_raw_buffer_load_b128(
                       rs, d < dim ? at + d * (uint32_t)sizeof(T) + 16 * i : 0xFFFFFFF0u, 0, 0));
    } else {
      uint32_t e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t o = d + j < dim ? at + (d + j) * (uint32_t)sizeof(T) : 0xFFFFFFF0u;
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
  static __device__ __forceinline__ void values(const uint4* x, float* f) {
    const T* t = (const T*)x;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = bs_to_f32(t[j]);
  }
  template <int PI>
  static __device__ __forceinline__ bs_parts<PI> parts(const uint4* x) {
    if constexpr (PI == 1) {
      bs_parts<1> o;
      o.p[0] = __builtin_bit_cast(bs_bf16x8, x[0]);
      return o;
    } else {
      float f[8];
      values(x, f);
      return bs_split8<PI>(f);
    }
  }
};

// Workgroup of a grid of units x slices: the slices of a unit (one sequence and head) read the
// same chunks, so they are given to one of the 8 XCDs, whose L2 then reads each chunk once.
struct DeltaPlace { int unit, slice; };
__device__ __forceinline__ DeltaPlace delta_place(int units, int slices) {
  const int k = blockIdx.x >> 3;
  return {(int)(blockIdx.x & 7) * ((units + 7) >> 3) + k / slices, k % slices};
}
static inline unsigned delta_grid(int64_t units, int slices) {
  return (unsigned)((units + 7) / 8 * 8 * slices);
}

// The 16 columns' rows of tile 2s + odd of an operand over 32 rows, transposed: its product with
// 1, exact.  A lane receives 4 columns of row delta_row(.., m).
template <int P>
__device__ __forceinline__ bs_f32x4 delta_turn(const bs_parts<P>& x, int odd, int lane) {
  const int m = lane & 15, g = lane >> 4;
  bs_u16x8 one;
#pragma unroll
  for (int e = 0; e < 8; ++e) one[e] = g == m >> 2 && e == 4 * odd + (m & 3) ? 0x3F80 : 0;
  const bs_bf16x8 b = __builtin_bit_cast(bs_bf16x8, one);
  bs_f32x4 r = zero4();
#pragma unroll
  for (int p = P - 1; p >= 0; --p)
    r = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.p[p], b, r, 0, 0, 0);
  return r;
}

// Whether a workgroup of the recurrences takes 32 value columns instead of 16: where 16 would not
// leave every workgroup a CU of its own.  A chunk's latency grows less than the columns do, and
// half the workgroups then take turns on a CU.  Whole forward call in us with 16 / 32 columns,
// heads of 128 x 128: 8,192 tokens x 32 heads (256 workgroups of 16) 434 / 506, x 40 heads 735 /
// 542, 2 x 4,096 x 16 186 / 231, 4 x 2,048 x 16 194 / 156.
static inline bool delta_wide(int64_t units, int dvp) {
  return units * (dvp / 16) > bs_num_cus();
}

// Rows of a packed batch before the first sequence and after the last one are no sequence's:
// their values (row t of `o`, `heads` of `d` elements a row) are 0.
template <typename T>
__device__ void zero_outside(const DeltaPlan& plan, T* o, int heads, int d, int h, int c0,
                             int cols) {
  const int a = delta_offset(plan, 0), b = max(delta_offset(plan, plan.seqs), a);
  const int c = c0 + threadIdx.x % cols, step = blockDim.x / cols;
  if (c >= d) return;
  for (int t = threadIdx.x / cols; t < plan.tokens; t += step) {
    if (t >= a && t < b) {
      t += (b - t - 1) / step * step;
      continue;
    }
    o[((int64_t)t * heads + h) * d + c] = bs_from_f32<T>(0.f);
  }
}

__device__ __forceinline__ bs_bf16x8 delta_frag(const uint16_t* p) { return *(const bs_bf16x8*)p; }

// Parts of the 8 values at `p` + step * part.
template <int PI>
__device__ __forceinline__ bs_parts<PI> delta_frags(const uint16_t* p, int64_t step) {
  bs_parts<PI> r;
#pragma unroll
  for (int i = 0; i < PI; ++i) r.p[i] = delta_frag(p + i * step);
  return r;
}

// Parts of 8 values of one lane's place in LDS, [part][..][64 lanes][2] words of 4 values.
template <int P>
__device__ __forceinline__ bs_parts<P> delta_lds(const uint2* p, int step) {
  bs_parts<P> r;
#pragma unroll
  for (int i = 0; i < P; ++i) r.p[i] = __builtin_bit_cast(bs_bf16x8, *(const uint4*)(p + i * step));
  return r;
}

template <int P>
__device__ __forceinline__ void delta_put(uint2* p, int step, const bs_f32x4& x) {
  const float v[4] = {x[0], x[1], x[2], x[3]};
  uint2 o[P];
  bs_split4<P>(v, o);
#pragma unroll
  for (int i = 0; i < P; ++i) p[i * step] = o[i];
}
