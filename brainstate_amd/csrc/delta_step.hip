// The gated delta rule token by token: the form that answers, on states kept between calls.
//
//   S' = exp(g) S,  u = beta (v - S'^T k),  S = S' + k u^T,  o = scale S^T q
//
// Both products with the state are taken from S' in one pass (S^T q = S'^T q + (k.q) u), so a
// token costs one reduction, and the state, the only large operand (dk dv floats read and
// written for 8 dk dv operations: bound by HBM), is read once and written once whatever the
// number of tokens.  A workgroup keeps a slice of 32 columns of one head's state in registers:
// 8 lanes x 4 columns side by side make 128-byte pieces of a row, 32 rows a pass.  One token of
// one sequence with 32 heads of 128 x 128 then has 128 workgroups: 5.8 us, most of it the latency
// of one read, one sum over the rows and one write.  224 live rows of 256 with such heads: 222 us,
// 4.3 TB/s beside a large copy's 5.1.
#include "delta.h"

namespace {

constexpr int kCols = 32;      // columns of the state a workgroup holds
constexpr int kRows = 32;      // rows a pass covers

__device__ __forceinline__ float4 load_cols(const float* p, int c, int dv, bool whole) {
  if (whole) return *(const float4*)(p + c);
  float4 r;
  r.x = c < dv ? p[c] : 0.f;
  r.y = c + 1 < dv ? p[c + 1] : 0.f;
  r.z = c + 2 < dv ? p[c + 2] : 0.f;
  r.w = c + 3 < dv ? p[c + 3] : 0.f;
  return r;
}

__device__ __forceinline__ void store_cols(float* p, int c, int dv, bool whole, float4 r) {
  if (whole) {
    *(float4*)(p + c) = r;
    return;
  }
  if (c < dv) p[c] = r.x;
  if (c + 1 < dv) p[c + 1] = r.y;
  if (c + 2 < dv) p[c + 2] = r.z;
  if (c + 3 < dv) p[c + 3] = r.w;
}

// Sum over the 8 lanes groups of a wave that hold the same columns (lanes l, l+8, ..).
__device__ __forceinline__ float sum_rows(float x) {
  x += __shfl_xor(x, 8);
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

template <typename T, int NR>   // NR passes of 32 rows: dk <= 32 NR
__global__ __launch_bounds__(256) void step_kernel(bs_delta_in in, int tokens, float* state,
                                                   int64_t n_states, const int32_t* slots, T* o,
                                                   int slices, int vec) {
  const int slice = blockIdx.x % slices;
  const int h = blockIdx.x / slices % in.hv;
  const int64_t b = blockIdx.x / slices / in.hv;
  const int hk = h / (in.hv / in.hk);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = slice * kCols + (tid & 7) * 4, row0 = tid >> 3;
  const int64_t at = slots ? (int64_t)slots[b] : b;
  T* ob = o + (b * tokens * in.hv + h) * in.dv;
  if (at < 0 || at >= n_states) {           // an idle row of the batch
    for (int t = 0; t < tokens; ++t)
      for (int i = tid; i < kCols && slice * kCols + i < in.dv; i += 256)
        ob[(int64_t)t * in.hv * in.dv + slice * kCols + i] = bs_from_f32<T>(0.f);
    return;
  }
  __shared__ float4 part[2][4][8][2];
  __shared__ float kq_part[2][4];
  float* sp = state + (at * in.hv + h) * (int64_t)in.dk * in.dv;
  const bool whole = vec && c + 4 <= in.dv;
  float4 s[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = row0 + i * kRows;
    s[i] = r < in.dk && c < in.dv ? load_cols(sp + (int64_t)r * in.dv, c, in.dv, whole)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int t = 0; t < tokens; ++t) {
    const T* qp = (const T*)in.q + bs_delta_at(in.q_stride, b, t, hk);
    const T* kp = (const T*)in.k + bs_delta_at(in.k_stride, b, t, hk);
    const T* vp = (const T*)in.v + bs_delta_at(in.v_stride, b, t, h);
    const float decay = expf(bs_delta_g(in, b, t, h)), beta = bs_delta_beta(in, b, t, h);
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = c + j < in.dv ? bs_to_f32(vp[c + j]) : 0.f;
    float kr[NR], kq = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), y = a;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = row0 + i * kRows;
      const float qr = r < in.dk ? bs_to_f32(qp[r]) : 0.f;
      kr[i] = r < in.dk ? bs_to_f32(kp[r]) : 0.f;
      s[i].x *= decay, s[i].y *= decay, s[i].z *= decay, s[i].w *= decay;
      a.x = fmaf(s[i].x, kr[i], a.x), a.y = fmaf(s[i].y, kr[i], a.y);
      a.z = fmaf(s[i].z, kr[i], a.z), a.w = fmaf(s[i].w, kr[i], a.w);
      y.x = fmaf(s[i].x, qr, y.x), y.y = fmaf(s[i].y, qr, y.y);
      y.z = fmaf(s[i].z, qr, y.z), y.w = fmaf(s[i].w, qr, y.w);
      kq = fmaf(kr[i], qr, kq);
    }
    a.x = sum_rows(a.x), a.y = sum_rows(a.y), a.z = sum_rows(a.z), a.w = sum_rows(a.w);
    y.x = sum_rows(y.x), y.y = sum_rows(y.y), y.z = sum_rows(y.z), y.w = sum_rows(y.w);
    kq = sum_rows(kq);
    const int p = t & 1;        // two sets, so one barrier a token is enough
    if (lane < 8) {
      part[p][wave][lane][0] = a;
      part[p][wave][lane][1] = y;
      if (lane == 0) kq_part[p][wave] = kq;
    }
    __syncthreads();
    a = part[p][0][tid & 7][0], y = part[p][0][tid & 7][1], kq = kq_part[p][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 aw = part[p][w][tid & 7][0], yw = part[p][w][tid & 7][1];
      a.x += aw.x, a.y += aw.y, a.z += aw.z, a.w += aw.w;
      y.x += yw.x, y.y += yw.y, y.z += yw.z, y.w += yw.w;
      kq += kq_part[p][w];
    }
    const float u[4] = {beta * (v[0] - a.x), beta * (v[1] - a.y), beta * (v[2] - a.z),
                        beta * (v[3] - a.w)};
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      s[i].x = fmaf(kr[i], u[0], s[i].x), s[i].y = fmaf(kr[i], u[1], s[i].y);
      s[i].z = fmaf(kr[i], u[2], s[i].z), s[i].w = fmaf(kr[i], u[3], s[i].w);
    }
    if (tid < 8) {
      const float r[4] = {fmaf(kq, u[0], y.x), fmaf(kq, u[1], y.y), fmaf(kq, u[2], y.z),
                          fmaf(kq, u[3], y.w)};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < in.dv)
          ob[(int64_t)t * in.hv * in.dv + c + j] = bs_from_f32<T>(in.scale * r[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = row0 + i * kRows;
    if (r < in.dk && c < in.dv) store_cols(sp + (int64_t)r * in.dv, c, in.dv, whole, s[i]);
  }
}

template <typename T>
void launch_step(const bs_delta_in& in, int batch, int tokens, float* state, int64_t n_states,
                 const int32_t* slots, void* o, hipStream_t st) {
  const int slices = (in.dv + kCols - 1) / kCols;
  const unsigned grid = (unsigned)((int64_t)batch * in.hv * slices);
  const int vec = in.dv % 4 == 0 && (uintptr_t)state % 16 == 0;
  if (in.dk <= 64)
    step_kernel<T, 2><<<grid, 256, 0, st>>>(in, tokens, state, n_states, slots, (T*)o, slices,
                                            vec);
  else
    step_kernel<T, 4><<<grid, 256, 0, st>>>(in, tokens, state, n_states, slots, (T*)o, slices,
                                            vec);
}

}  // namespace

int bs_delta_check(const bs_delta_in* in, const char* who) {
  BS_CHECK_ARG(in != nullptr, "%s: operands are NULL", who);
  BS_CHECK_ARG(bs_dtype_ok(in->dtype) && bs_dtype_ok(in->g_dtype) && bs_dtype_ok(in->beta_dtype),
               "%s: dtype %d / %d / %d unknown", who, in->dtype, in->g_dtype, in->beta_dtype);
  BS_CHECK_ARG(in->hk >= 1 && in->hv >= 1 && in->hv % in->hk == 0,
               "%s: %d value heads for %d key heads", who, in->hv, in->hk);
  BS_CHECK_ARG(in->dk >= 1 && in->dk <= BS_DELTA_MAX_DIM && in->dv >= 1 &&
                   in->dv <= BS_DELTA_MAX_DIM,
               "%s: head sizes %d, %d outside 1..%d", who, in->dk, in->dv, BS_DELTA_MAX_DIM);
  return BS_OK;
}

extern "C" int bs_gated_delta_step(const bs_delta_in* in, int32_t batch, int32_t tokens,
                                   float* state, int64_t n_states, const int32_t* slots, void* o,
                                   bs_stream_t stream) {
  if (int rc = bs_delta_check(in, "bs_gated_delta_step")) return rc;
  BS_CHECK_ARG(batch >= 0 && tokens >= 0 && n_states >= 0,
               "bs_gated_delta_step: batch %d, tokens %d, states %lld", batch, tokens,
               (long long)n_states);
  // a launch has fewer than 2^32 threads; past that the count wraps without an error
  BS_CHECK_ARG((int64_t)batch * in->hv * ((in->dv + kCols - 1) / kCols) < 1 << 24,
               "bs_gated_delta_step: batch %d x %d heads exceeds one launch", batch, in->hv);
  if (batch == 0 || tokens == 0) return BS_OK;
  BS_CHECK_ARG(in->q && in->k && in->v && in->g && in->beta && state && o,
               "bs_gated_delta_step: NULL pointer");
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
