// Decay attention token by token: the form that answers, on states kept between calls.
//
//   S = exp(g) S + k v^T,  o = scale S^T q
//
// The state is the only large operand (dk dv floats read and written for 5 dk dv operations: bound
// by HBM) and is read once and written once whatever the number of tokens.  A workgroup keeps a
// slice of 32 columns of one head's state in registers: 8 lanes x 4 columns side by side make
// 128-byte pieces of a row, 32 rows a pass.  The slices of a state run on one XCD, so that pieces
// which share a line of 128 bytes find it in one L2: 256 states of 16 heads of 100 x 100 take 90 us, 4
// tokens of 64 states of 32 heads of 128 x 128 78 (107 and 99 before launch_step chose how columns are
// read, 134 and 111 then with slices dealt out one by one).
//
// 256 states of 32 heads of 128 x 128, one token: 195 to 202 us, 5.4 TB/s of states beside a large copy's 5.1;
// one state: 4.8 us, the latency of a read, a sum over rows and a write.
#include "delta.h"

namespace {

constexpr int kCols = 32;      // columns of the state a workgroup holds
constexpr int kRows = 32;      // rows a pass covers

// How a row's columns are read and written: one by one, 4 at a time, or these past the caches.
enum Columns { kSingle = 0, kFour = 1, kPast = 2 };
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float4 load_cols(const float* p, int n, int cols) {
  if (cols == kPast) {
    const f32x4 x = __builtin_nontemporal_load((const f32x4*)p);
    return make_float4(x[0], x[1], x[2], x[3]);
  }
  if (cols == kFour) return *(const float4*)p;
  return make_float4(n > 0 ? p[0] : 0.f, n > 1 ? p[1] : 0.f, n > 2 ? p[2] : 0.f,
                     n > 3 ? p[3] : 0.f);
}

__device__ __forceinline__ void store_cols(float* p, int n, int cols, const float4& r) {
  if (cols == kPast) {
    __builtin_nontemporal_store(f32x4{r.x, r.y, r.z, r.w}, (f32x4*)p);
    return;
  }
  if (cols == kFour) {
    *(float4*)p = r;
    return;
  }
  if (n > 0) p[0] = r.x;
  if (n > 1) p[1] = r.y;
  if (n > 2) p[2] = r.z;
  if (n > 3) p[3] = r.w;
}

// Sum over the 8 lane groups of a wave that hold the same columns (lanes l, l + 8, ..).
__device__ __forceinline__ float sum_rows(float x) {
  x += __shfl_xor(x, 8);
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

template <typename T, int NR>   // NR passes of 32 rows: dk <= 32 NR
__global__ __launch_bounds__(256) void decay_step_kernel(bs_delta_in in, int tokens, float* state,
                                                         int64_t n_states, const int32_t* slots,
                                                         T* o, int slices, int cols_of,
                                                         uint32_t heads) {
  __shared__ float4 part[2][4][8];
  // workgroups go round the 8 XCDs in turn; the slices of one state to the same one
  const int slice = blockIdx.x / 8 % slices;
  const uint32_t unit = blockIdx.x / 8 / slices * 8 + blockIdx.x % 8;
  if (unit >= heads) return;
  const int h = unit % in.hv;
  const int64_t b = unit / in.hv;
  const int hk = h / (in.hv / in.hk);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = slice * kCols + (tid & 7) * 4, n = in.dv - c, row0 = tid >> 3;
  const int64_t at = slots ? (int64_t)slots[b] : b;
  T* ob = o + (b * tokens * in.hv + h) * in.dv;
  if (at < 0 || at >= n_states) {           // an idle row of the batch
    for (int t = 0; t < tokens; ++t)
      for (int i = slice * kCols + tid; i < min((slice + 1) * kCols, in.dv); i += 256)
        ob[(int64_t)t * in.hv * in.dv + i] = bs_from_f32<T>(0.f);
    return;
  }
  float* sp = state + (at * in.hv + h) * (int64_t)in.dk * in.dv + c;
  const int cols = n >= 4 ? cols_of : kSingle;
  float4 s[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = row0 + i * kRows;
    s[i] = r < in.dk && n > 0 ? load_cols(sp + (int64_t)r * in.dv, n, cols)
                              : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int t = 0; t < tokens; ++t) {
    const T* qp = (const T*)in.q + bs_delta_at(in.q_stride, b, t, hk);
    const T* kp = (const T*)in.k + bs_delta_at(in.k_stride, b, t, hk);
    const T* vp = (const T*)in.v + bs_delta_at(in.v_stride, b, t, h) + c;
    const float decay = expf(bs_delta_g(in, b, t, h));
    float v[4], k[NR], q[NR];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < n ? bs_to_f32(vp[j]) : 0.f;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = row0 + i * kRows;
      q[i] = r < in.dk ? bs_to_f32(qp[r]) : 0.f;
      k[i] = r < in.dk ? bs_to_f32(kp[r]) : 0.f;
    }
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      s[i].x = fmaf(k[i], v[0], s[i].x * decay), s[i].y = fmaf(k[i], v[1], s[i].y * decay);
      s[i].z = fmaf(k[i], v[2], s[i].z * decay), s[i].w = fmaf(k[i], v[3], s[i].w * decay);
      y.x = fmaf(s[i].x, q[i], y.x), y.y = fmaf(s[i].y, q[i], y.y);
      y.z = fmaf(s[i].z, q[i], y.z), y.w = fmaf(s[i].w, q[i], y.w);
    }
    y.x = sum_rows(y.x), y.y = sum_rows(y.y), y.z = sum_rows(y.z), y.w = sum_rows(y.w);
    const int p = t & 1;        // two sets, so one barrier a token is enough
    if (lane < 8) part[p][wave][lane] = y;
    __syncthreads();
    if (tid < kCols && slice * kCols + tid < in.dv) {
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) a += ((const float*)part[p][w])[tid];
      ob[(int64_t)t * in.hv * in.dv + slice * kCols + tid] = bs_from_f32<T>(in.scale * a);
    }
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = row0 + i * kRows;
    if (r < in.dk && n > 0) store_cols(sp + (int64_t)r * in.dv, n, cols, s[i]);
  }
}

template <typename T>
void launch_step(const bs_delta_in& in, int batch, int tokens, float* state, int64_t n_states,
                 const int32_t* slots, void* o, hipStream_t st) {
  const int slices = (in.dv + kCols - 1) / kCols;
  const uint32_t heads = (uint32_t)batch * in.hv;
  const unsigned grid = (heads + 7) / 8 * 8 * slices;
  // A state is read and written once a call, and many of them exceed the caches by far: past them 256
  // states of 32 heads of 128 x 128 take 195 us (233 through them), of 16 heads of 112 x 112 94 (103).
  // Rows that do not end on 64 bytes share pieces of that size, which the caches put together: 100 x 100
  // takes 89 us (120 past them).
  const int cols = in.dv % 4 || (uintptr_t)state % 16 ? kSingle : in.dv % 16 ? kFour : kPast;
  if (in.dk <= 64)
    decay_step_kernel<T, 2><<<grid, 256, 0, st>>>(in, tokens, state, n_states, slots, (T*)o,
                                                  slices, cols, heads);
  else
    decay_step_kernel<T, 4><<<grid, 256, 0, st>>>(in, tokens, state, n_states, slots, (T*)o,
                                                  slices, cols, heads);
}

}  // namespace

extern "C" int bs_decay_attention_step(const bs_delta_in* in, int32_t batch, int32_t tokens,
                                       float* state, int64_t n_states, const int32_t* slots,
                                       void* o, bs_stream_t stream) {
  if (int rc = bs_delta_check(in, "bs_decay_attention_step")) return rc;
  BS_CHECK_ARG(batch >= 0 && tokens >= 0 && n_states >= 0,
               "bs_decay_attention_step: batch %d, tokens %d, states %lld", batch, tokens,
               (long long)n_states);
  // a launch has fewer than 2^32 threads; past that the count wraps without an error
  BS_CHECK_ARG(((int64_t)batch * in->hv + 7) * ((in->dv + kCols - 1) / kCols) < 1 << 24,
               "bs_decay_attention_step: batch %d x %d heads exceeds one launch", batch, in->hv);
  if (batch == 0 || tokens == 0) return BS_OK;
  BS_CHECK_ARG(in->q && in->k && in->v && in->g && state && o,
               "bs_decay_attention_step: NULL pointer");
  hipStream_t st = bs_stream(stream);
  if (in->dtype == BS_F32)
    launch_step<float>(*in, batch, tokens, state, n_states, slots, o, st);
  else if (in->dtype == BS_BF16)
    launch_step<bs_bf16>(*in, batch, tokens, state, n_states, slots, o, st);
  else
    launch_step<bs_f16>(*in, batch, tokens, state, n_states, slots, o, st);
  BS_CHECK_LAUNCH();
  return BS_OK;
}
