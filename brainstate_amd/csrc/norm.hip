// The norms before and after a block, its gate, residual scale and residual, in one pass, and
// their gradients.  With r(x) = (mean x^2 + eps)^-1/2 over a row:
//
//   p = y r(y) post,  t = scale silu(gate) p,  s = residual + t,  normed = s r(s) pre
//
// (a part that is not given is left out).  Bound by bytes: a row is read once into registers,
// where both norms' sums are taken in 32 bits, and its results are written once; s is rounded
// only when it is stored.  A row belongs to TPR lanes with 8 NV values each, so a norm over a
// head of 128 values shares a wave with three others and one of 16,384 takes 1,024 threads.
// Workgroups stay for many rows: a lane's columns are the same in each, so the weights are read
// once and the weights' gradients are summed in registers, then over the workgroups in their
// order (grad_sum_kernel): the same bits every time.
#include "lane_types.h"

namespace {

constexpr int kVec = 8;

// Rows start at any element: 16-byte loads of any alignment, single ones at a row's end.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int left, float* x) {
  if (left >= kVec) {
    T t[kVec];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int j = 0; j < kVec; ++j) x[j] = bs_to_f32(t[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j) x[j] = j < left ? bs_to_f32(p[j]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int left, const float* x) {
  if (left >= kVec) {
    T t[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) t[j] = bs_from_f32<T>(x[j]);
    __builtin_memcpy(p, t, sizeof(t));
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (j < left) p[j] = bs_from_f32<T>(x[j]);
  }
}

template <int NV>
__device__ __forceinline__ void load_weight(const void* p, int dtype, int c0, int step, int dim,
                                            float fill, float (*w)[kVec]) {
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int c = c0 + v * step + j;
      w[v][j] = p && c < dim ? bs_load_any(p, dtype, c) : fill;
    }
}

// Sums over the TPR lanes of a row; `turn` alternates so that one barrier a sum is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float* x, float (*sh)[16][N], int& turn) {
#pragma unroll
  for (int d = 1; d < (TPR < 64 ? TPR : 64); d <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += __shfl_xor(x[i], d);
  if (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) sh[turn][wave][i] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = 0.f;
#pragma unroll
      for (int k = 0; k < TPR / 64; ++k) x[i] += sh[turn][k][i];
    }
    turn ^= 1;
  }
}

__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + expf(-z)); }

template <typename T, int TPR, int NV>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_kernel(bs_norm_in in, T* stream,
                                                                     T* normed) {
  constexpr int RPB = TPR >= 256 ? 1 : 256 / TPR;
  __shared__ float sh[2][16][1];
  const int t = threadIdx.x % TPR, c0 = t * kVec, step = TPR * kVec, dim = in.dim;
  int turn = 0;
  float post[NV][kVec], scale[NV][kVec], pre[NV][kVec];
  load_weight<NV>(in.post, in.post_dtype, c0, step, dim, 1.f, post);
  load_weight<NV>(in.scale, in.scale_dtype, c0, step, dim, in.scale_value, scale);
  load_weight<NV>(in.pre, in.pre_dtype, c0, step, dim, 1.f, pre);
  const float inv = 1.f / (float)dim;
  const int64_t first = (int64_t)blockIdx.x * RPB, stride = (int64_t)gridDim.x * RPB;
  for (int64_t base = first; base < in.rows; base += stride) {
    const int64_t row = base + threadIdx.x / TPR;
    const bool live = row < in.rows;
    float x[NV][kVec], z[NV][kVec], s[NV][kVec];
    float sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = c0 + v * step, left = live ? dim - c : 0;
      load8((const T*)in.y + row * in.y_stride + c, left, x[v]);
      if (in.gate) load8((const T*)in.gate + row * in.gate_stride + c, left, z[v]);
      if (in.residual) load8((const T*)in.residual + row * in.residual_stride + c, left, s[v]);
#pragma unroll
      for (int j = 0; j < kVec; ++j) sum[0] = fmaf(x[v][j], x[v][j], sum[0]);
    }
    float r1 = 1.f;
    if (in.post) {
      row_sum<TPR, 1>(sum, sh, turn);
      r1 = rsqrtf(sum[0] * inv + in.eps);
    }
    sum[0] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        float a = x[v][j] * r1 * post[v][j] * scale[v][j];
        if (in.gate) a *= z[v][j] * sigmoid(z[v][j]);
        if (in.residual) a += s[v][j];
        s[v][j] = a;
        sum[0] = fmaf(a, a, sum[0]);
      }
      const int c = c0 + v * step;
      if (live) store8(stream + row * dim + c, dim - c, s[v]);
    }
    if (in.pre) {
      row_sum<TPR, 1>(sum, sh, turn);
      const float r2 = rsqrtf(sum[0] * inv + in.eps);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) s[v][j] *= r2 * pre[v][j];
        const int c = c0 + v * step;
        if (live) store8(normed + row * dim + c, dim - c, s[v]);
      }
    }
  }
}

struct NormGrad {
  const void *gs, *gn;              // gradients of stream and normed (NULL: none)
  void *dy, *dgate, *dresidual;     // NULL: not wanted
  float* part;                      // [workgroups][3][dim]: of post, scale, pre
};

// With n = s r2, dn = grad normed . pre:  ds = grad stream + r2 (dn - n mean(dn n)), and the like
// for y; sums of a row: y^2, then s^2 and dn s, then what reaches y.
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_grad_kernel(bs_norm_in in,
                                                                          NormGrad o) {
  constexpr int BLOCK = TPR > 256 ? TPR : 256, RPB = BLOCK / TPR;
  __shared__ float sh[2][16][1];
  __shared__ float sh2[2][16][2];
  __shared__ float acc[BLOCK * kVec];
  const int t = threadIdx.x % TPR, c0 = t * kVec, step = TPR * kVec, dim = in.dim;
  int turn = 0, turn2 = 0;
  float post[NV][kVec], scale[NV][kVec], pre[NV][kVec];
  float dw[3][NV][kVec];
  load_weight<NV>(in.post, in.post_dtype, c0, step, dim, 1.f, post);
  load_weight<NV>(in.scale, in.scale_dtype, c0, step, dim, in.scale_value, scale);
  load_weight<NV>(in.pre, in.pre_dtype, c0, step, dim, 1.f, pre);
#pragma unroll
  for (int i = 0; i < 3; ++i)
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < kVec; ++j) dw[i][v][j] = 0.f;
  const float inv = 1.f / (float)dim;
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < in.rows;
       base += (int64_t)gridDim.x * RPB) {
    const int64_t row = base + threadIdx.x / TPR;
    const bool live = row < in.rows;
    float x[NV][kVec], z[NV][kVec], s[NV][kVec], d[NV][kVec], dn[NV][kVec];
    float sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = c0 + v * step, left = live ? dim - c : 0;
      load8((const T*)in.y + row * in.y_stride + c, left, x[v]);
      if (in.gate) load8((const T*)in.gate + row * in.gate_stride + c, left, z[v]);
      if (in.residual) load8((const T*)in.residual + row * in.residual_stride + c, left, s[v]);
      if (o.gs) load8((const T*)o.gs + row * dim + c, left, d[v]);
      if (o.gn) load8((const T*)o.gn + row * dim + c, left, dn[v]);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        sum[0] = fmaf(x[v][j], x[v][j], sum[0]);
        if (!o.gs) d[v][j] = 0.f;
      }
    }
    float r1 = 1.f;
    if (in.post) {
      row_sum<TPR, 1>(sum, sh, turn);
      r1 = rsqrtf(sum[0] * inv + in.eps);
    }
    float two[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        x[v][j] *= r1;                                   // normalised y
        float a = x[v][j] * post[v][j] * scale[v][j];
        if (in.gate) a *= z[v][j] * sigmoid(z[v][j]);
        if (in.residual) a += s[v][j];
        s[v][j] = a;
        if (o.gn) {
          two[0] = fmaf(a, a, two[0]);
          two[1] = fmaf(dn[v][j] * pre[v][j], a, two[1]);
        }
      }
    if (o.gn) {
      row_sum<TPR, 2>(two, sh2, turn2);
      const float r2 = rsqrtf(two[0] * inv + in.eps), k = two[1] * r2 * r2 * inv;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          dw[2][v][j] = fmaf(dn[v][j], s[v][j] * r2, dw[2][v][j]);
          d[v][j] += r2 * (dn[v][j] * pre[v][j] - s[v][j] * k);
        }
    }
    sum[0] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = c0 + v * step;
      if (live && o.dresidual) store8((T*)o.dresidual + row * dim + c, dim - c, d[v]);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const float p = x[v][j] * post[v][j];
        float act = 1.f, slope = 0.f;
        if (in.gate) {
          const float sg = sigmoid(z[v][j]);
          act = z[v][j] * sg;
          slope = sg * (1.f + z[v][j] * (1.f - sg));
        }
        z[v][j] = d[v][j] * scale[v][j] * p * slope;
        dw[1][v][j] = fmaf(d[v][j] * act, p, dw[1][v][j]);
        const float dp = d[v][j] * scale[v][j] * act;
        dw[0][v][j] = fmaf(dp, x[v][j], dw[0][v][j]);
        d[v][j] = dp * post[v][j];
        sum[0] = fmaf(d[v][j], x[v][j], sum[0]);
      }
      if (live && o.dgate) store8((T*)o.dgate + row * dim + c, dim - c, z[v]);
    }
    if (in.post) row_sum<TPR, 1>(sum, sh, turn);
    const float k = in.post ? sum[0] * inv : 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) d[v][j] = r1 * (d[v][j] - x[v][j] * k);
      const int c = c0 + v * step;
      if (live && o.dy) store8((T*)o.dy + row * dim + c, dim - c, d[v]);
    }
  }
  if (!o.part) return;
#pragma unroll
  for (int i = 0; i < 3; ++i)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kVec; ++j) acc[threadIdx.x * kVec + j] = dw[i][v][j];
      __syncthreads();
      for (int e = threadIdx.x; e < TPR * kVec; e += BLOCK) {   // the rows side by side
        float a = 0.f;
        for (int k = 0; k < RPB; ++k) a += acc[k * TPR * kVec + e];
        const int c = v * step + e;
        if (c < dim) o.part[((int64_t)blockIdx.x * 3 + i) * dim + c] = a;
      }
    }
}

// Column sums of the workgroups' parts: 64 columns a workgroup, 16 waves over the parts.
__global__ __launch_bounds__(1024) void grad_sum_kernel(const float* part, int parts, int dim,
                                                        bs_norm_in in, void* dpost, void* dscale,
                                                        void* dpre) {
  __shared__ float sh[16][64];
  const int which = blockIdx.y, c = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  void* out = which == 0 ? dpost : which == 1 ? dscale : dpre;
  if (!out) return;
  float a = 0.f;
  if (c < dim)
    for (int k = w; k < parts; k += 16) a += part[((int64_t)k * 3 + which) * dim + c];
  sh[w][threadIdx.x & 63] = a;
  __syncthreads();
  if (w == 0 && c < dim) {
    for (int k = 1; k < 16; ++k) a += sh[k][threadIdx.x & 63];
    bs_store_any(out, which == 0 ? in.post_dtype : which == 1 ? in.scale_dtype : in.pre_dtype, c,
                 a);
  }
}

int check(const bs_norm_in* in, const char* who) {
  BS_CHECK_ARG(in != nullptr, "%s: operands are NULL", who);
  BS_CHECK_ARG(bs_dtype_ok(in->dtype) && bs_dtype_ok(in->post_dtype) &&
                   bs_dtype_ok(in->scale_dtype) && bs_dtype_ok(in->pre_dtype),
               "%s: dtype unknown", who);
  BS_CHECK_ARG(in->rows >= 0 && in->dim >= 1 && in->dim <= 16384,
               "%s: %lld rows of %d values (1..16384)", who, (long long)in->rows, in->dim);
  BS_CHECK_ARG(in->rows == 0 || in->y, "%s: y is NULL", who);
  return BS_OK;
}

struct Shape { int tpr, nv; };
Shape shape_of(int dim) {
  static const Shape s[] = {{16, 1}, {16, 2}, {64, 1}, {64, 2}, {256, 1}, {256, 2}, {1024, 1},
                            {1024, 2}};
  for (const Shape& x : s)
    if (dim <= x.tpr * x.nv * kVec) return x;
  return s[7];
}

int grid_of(const bs_norm_in& in, const Shape& s, int per_cu) {
  const int rpb = s.tpr >= 256 ? 1 : 256 / s.tpr;
  const int64_t need = (in.rows + rpb - 1) / rpb, most = (int64_t)per_cu * bs_num_cus();
  return (int)(need < most ? need : most);
}

constexpr int kGradPerCu = 2;

template <typename T, typename F>
void by_shape(const Shape& s, F&& f) {
  switch (s.tpr * s.nv) {
    case 16: f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>()); break;
    case 32: f(std::integral_constant<int, 16>(), std::integral_constant<int, 2>()); break;
    case 64: f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>()); break;
    case 128: f(std::integral_constant<int, 64>(), std::integral_constant<int, 2>()); break;
    case 256: f(std::integral_constant<int, 256>(), std::integral_constant<int, 1>()); break;
    case 512: f(std::integral_constant<int, 256>(), std::integral_constant<int, 2>()); break;
    case 1024: f(std::integral_constant<int, 1024>(), std::integral_constant<int, 1>()); break;
    default: f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
  }
}

template <typename T>
void launch(const bs_norm_in& in, void* stream, void* normed, hipStream_t st) {
  const Shape s = shape_of(in.dim);
  const int grid = grid_of(in, s, 8);
  by_shape<T>(s, [&](auto tpr, auto nv) {
    norm_kernel<T, tpr.value, nv.value><<<grid, tpr.value > 256 ? tpr.value : 256, 0, st>>>(
        in, (T*)stream, (T*)normed);
  });
}

template <typename T>
void launch_grad(const bs_norm_in& in, const NormGrad& o, hipStream_t st) {
  const Shape s = shape_of(in.dim);
  const int grid = grid_of(in, s, kGradPerCu);
  if (grid == 0) return;
  by_shape<T>(s, [&](auto tpr, auto nv) {
    norm_grad_kernel<T, tpr.value, nv.value><<<grid, tpr.value > 256 ? tpr.value : 256, 0, st>>>(
        in, o);
  });
}

}  // namespace

extern "C" int bs_norm_gate_residual(const bs_norm_in* in, void* stream_out, void* normed_out,
                                     bs_stream_t stream) {
  if (int rc = check(in, "bs_norm_gate_residual")) return rc;
  if (in->rows == 0) return BS_OK;
  BS_CHECK_ARG(stream_out && (!in->pre || normed_out), "bs_norm_gate_residual: output is NULL");
  hipStream_t st = bs_stream(stream);
  if (in->dtype == BS_F32) launch<float>(*in, stream_out, normed_out, st);
  else if (in->dtype == BS_BF16) launch<bs_bf16>(*in, stream_out, normed_out, st);
  else launch<bs_f16>(*in, stream_out, normed_out, st);
  BS_CHECK_LAUNCH();
  return BS_OK;
}

extern "C" size_t bs_norm_grad_workspace_size(int64_t rows, int32_t dim) {
  bs_norm_in in = {};
  in.rows = rows, in.dim = dim;
  if (rows < 1 || dim < 1 || dim > 16384) return 0;
  return (size_t)grid_of(in, shape_of(dim), kGradPerCu) * 3 * dim * sizeof(float);
}

extern "C" int bs_norm_gate_residual_grad(const bs_norm_in* in, const void* grad_stream,
                                          const void* grad_normed, void* dy, void* dpost,
                                          void* dgate, void* dscale, void* dresidual, void* dpre,
                                          void* workspace, size_t workspace_bytes,
                                          bs_stream_t stream) {
  if (int rc = check(in, "bs_norm_gate_residual_grad")) return rc;
  BS_CHECK_ARG(!grad_normed || in->pre, "bs_norm_gate_residual_grad: a gradient of normed without "
                                        "its weight");
  BS_CHECK_ARG((!dpost || in->post) && (!dgate || in->gate) && (!dscale || in->scale) &&
                   (!dresidual || in->residual) && (!dpre || in->pre),
               "bs_norm_gate_residual_grad: a gradient of an operand that is not given");
  const bool weights = dpost || dscale || dpre;
  const size_t need = weights ? bs_norm_grad_workspace_size(in->rows, in->dim) : 0;
  BS_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
               "bs_norm_gate_residual_grad: workspace of %zu bytes needed", need);
  const NormGrad o = {grad_stream, grad_normed, dy, dgate, dresidual,
                      weights ? (float*)workspace : nullptr};
  hipStream_t st = bs_stream(stream);
  if (in->dtype == BS_F32) launch_grad<float>(*in, o, st);
  else if (in->dtype == BS_BF16) launch_grad<bs_bf16>(*in, o, st);
  else launch_grad<bs_f16>(*in, o, st);
  BS_CHECK_LAUNCH();
  if (weights) {
    const int parts = grid_of(*in, shape_of(in->dim), kGradPerCu);
    grad_sum_kernel<<<dim3((in->dim + 63) / 64, 3), 1024, 0, st>>>(
        (const float*)workspace, parts, in->dim, *in, dpost, dscale, dpre);
    BS_CHECK_LAUNCH();
  }
  return BS_OK;
}
