// Layer norm of a residual stream and a dropped-out branch, its gradients, and dropout alone.  Over
// a row of n values:
//
//   stream = residual + (kept ? x / (1 - p) : 0),  h = (stream - mean) r,  normed = h weight + bias
//   with r = (mean of (stream - mean)^2 + eps)^-1/2
//   d = grad stream + r (dh - mean(dh) - h mean(dh h))  with dh = grad normed . weight
//
// d is the residual's gradient and, where x was kept, times 1 / (1 - p), that of x.  Which elements
// are kept is computed again from the seed wherever it is needed (philox.h): no mask is stored.
// Bound by bytes: a row is read once into registers, where its sums are taken in 32 bits (the
// squares about the mean, after it), and its results are written once; stream is rounded only when
// it is stored.  Workgroups stay for many rows: a lane's columns are the same in each, so the
// weights are read once and their gradients are summed in registers, then over the workgroups in
// their order (weight_sum_kernel): the same bits every time.
//
// 8,192 rows of 4,096 in bf16 with dropout of a tenth: forward 59 to 70 us (268 MB, 3.9 to 4.5 TB/s beside
// a large copy's 5.1), gradients 91 (403 MB and the mask's words again, 4.4), weights' sums 4.1; dropout
// alone 26 to 29 (134 MB, 4.6 to 5.1).  The larger figures are the tracer's, the smaller a run of calls'.
#include "philox.h"
#include "rows.h"

namespace {

// TPR lanes to a row and 256 / TPR rows to a workgroup, or (TPR = 0) a row to a workgroup.
template <typename T, int TPR, int NV, int BLOCK, int MODE, bool DROP>
__global__ __launch_bounds__(BLOCK) void layer_norm_kernel(bs_layer_norm_in in, T* stream,
                                                           T* normed, float* stats) {
  constexpr int RPB = TPR ? 256 / TPR : 1;
  __shared__ float sh[2][16][1];
  const int lanes = TPR ? TPR : blockDim.x, t = threadIdx.x % lanes;
  const int step = lanes * kVec, dim = in.dim;
  Cols<MODE> k[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) k[v] = Cols<MODE>(t * kVec + v * step, dim);
  int turn = 0;
  float weight[NV][kVec], bias[NV][kVec];
  load_weight<NV>(in.weight, in.weight_dtype, k, dim, 1.f, weight);
  load_weight<NV>(in.bias, in.bias_dtype, k, dim, 0.f, bias);
  const Dropout drop(in.seed, DROP ? in.seed_at : nullptr, in.site, in.drop);
  const float inv = 1.f / (float)dim;
  const int64_t stride = (int64_t)gridDim.x * RPB, last = in.rows - 1;
  int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / lanes;
  const int64_t turns = (in.rows - (int64_t)blockIdx.x * RPB + stride - 1) / stride;
  Vec8<T, MODE> xv[NV], rv[NV];
  // the next row's operands are loaded while this one's sums are taken
  auto load = [&](int64_t r) {
    r = r < last ? r : last;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      xv[v].load((const T*)in.x + r * in.x_stride, k[v], dim);
      if (in.residual) rv[v].load((const T*)in.residual + r * in.residual_stride, k[v], dim);
    }
  };
  load(row);
  for (int64_t turn_of = 0; turn_of < turns; ++turn_of, row += stride) {
    const bool live = row < in.rows;
    float s[NV][kVec], sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float x[kVec];
      xv[v].values(k[v].in, x);
      if (in.residual) rv[v].values(k[v].in, s[v]);
      if (DROP) {
        const uint32_t kept = drop.eight(row, k[v].at);
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[j] = kept >> j & 1 ? x[j] * in.keep_scale : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        s[v][j] = in.residual ? s[v][j] + x[j] : x[j];
        sum[0] += k[v].once(j, s[v][j]);
      }
    }
    load(row + stride);
    row_sum<TPR, 1>(sum, sh, turn);
    const float mean = sum[0] * inv;
    sum[0] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (stream && live) xv[v].store(stream + row * dim, k[v], dim, s[v]);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        s[v][j] = k[v].in && (MODE != kSmall || k[v].at + j < dim) ? s[v][j] - mean : 0.f;
        sum[0] = fmaf(k[v].once(j, s[v][j]), s[v][j], sum[0]);
      }
    }
    row_sum<TPR, 1>(sum, sh, turn);
    const float r = rsqrtf(sum[0] * inv + in.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) s[v][j] = fmaf(s[v][j] * r, weight[v][j], bias[v][j]);
      if (live) xv[v].store(normed + row * dim, k[v], dim, s[v]);
    }
    if (stats && live && t == 0) {
      stats[2 * row] = mean;
      stats[2 * row + 1] = r;
    }
  }
}

struct LayerNormGrad {
  const void *gs, *gn;              // gradients of stream and normed (NULL: none)
  const float* stats;               // [rows][2]: mean and r
  void *dx, *dresidual;             // NULL: not wanted
  float* part;                      // [workgroups][2][dim]: of weight and bias
};

template <typename T, int TPR, int NV, int BLOCK, int MODE, bool DROP>
__global__ __launch_bounds__(BLOCK) void layer_norm_grad_kernel(bs_layer_norm_in in,
                                                                LayerNormGrad o) {
  constexpr int RPB = TPR ? 256 / TPR : 1;
  __shared__ float sh[2][16][2];
  __shared__ float acc[BLOCK * kVec];
  const int lanes = TPR ? TPR : blockDim.x, t = threadIdx.x % lanes;
  const int step = lanes * kVec, dim = in.dim;
  Cols<MODE> k[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) k[v] = Cols<MODE>(t * kVec + v * step, dim);
  int turn = 0;
  float weight[NV][kVec], dw[2][NV][kVec];
  load_weight<NV>(in.weight, in.weight_dtype, k, dim, 1.f, weight);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < kVec; ++j) dw[i][v][j] = 0.f;
  const Dropout drop(in.seed, DROP ? in.seed_at : nullptr, in.site, in.drop);
  const float inv = 1.f / (float)dim;
  const int64_t stride = (int64_t)gridDim.x * RPB, last = in.rows - 1;
  int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / lanes;
  const int64_t turns = (in.rows - (int64_t)blockIdx.x * RPB + stride - 1) / stride;
  Vec8<T, MODE> xv[NV], rv[NV], gsv[NV], gnv[NV];
  float mean_of, r_of;
  auto load = [&](int64_t r) {
    r = r < last ? r : last;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      xv[v].load((const T*)in.x + r * in.x_stride, k[v], dim);
      if (in.residual) rv[v].load((const T*)in.residual + r * in.residual_stride, k[v], dim);
      if (o.gs) gsv[v].load((const T*)o.gs + r * dim, k[v], dim);
      if (o.gn) gnv[v].load((const T*)o.gn + r * dim, k[v], dim);
    }
    mean_of = o.stats[2 * r], r_of = o.stats[2 * r + 1];
  };
  load(row);
  for (int64_t turn_of = 0; turn_of < turns; ++turn_of, row += stride) {
    const bool live = row < in.rows;
    const float mean = mean_of, r = r_of;
    uint32_t kept[NV];
    float h[NV][kVec], d[NV][kVec], dn[NV][kVec];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float x[kVec];
      xv[v].values(k[v].in, x);
      if (in.residual) rv[v].values(k[v].in, h[v]);
      gsv[v].values(o.gs && k[v].in && live, d[v]);       // a row that is not there gives nothing
      gnv[v].values(o.gn && k[v].in && live, dn[v]);
      if (DROP) {
        kept[v] = drop.eight(live ? row : last, k[v].at);   // of the row that was loaded
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[j] = kept[v] >> j & 1 ? x[j] * in.keep_scale : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        h[v][j] = ((in.residual ? h[v][j] + x[j] : x[j]) - mean) * r;
        dw[0][v][j] = fmaf(dn[v][j], h[v][j], dw[0][v][j]);
        dw[1][v][j] += dn[v][j];
        dn[v][j] *= weight[v][j];
        sum[0] += k[v].once(j, dn[v][j]);
        sum[1] = fmaf(k[v].once(j, dn[v][j]), h[v][j], sum[1]);
      }
    }
    load(row + stride);
    if (o.gn) row_sum<TPR, 2>(sum, sh, turn);
    const float off = sum[0] * inv, slope = sum[1] * inv;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) d[v][j] += r * (dn[v][j] - off - h[v][j] * slope);
      if (live && o.dresidual) xv[v].store((T*)o.dresidual + row * dim, k[v], dim, d[v]);
      if (DROP) {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          d[v][j] = kept[v] >> j & 1 ? d[v][j] * in.keep_scale : 0.f;
      }
      if (live && o.dx) xv[v].store((T*)o.dx + row * dim, k[v], dim, d[v]);
    }
  }
  if (!o.part) return;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const int e = k[v].at + j - v * step;
        if (MODE != kTail || k[v].m[j] != 0.f)
          if (k[v].in) acc[threadIdx.x / lanes * step + e] = dw[i][v][j];
      }
      __syncthreads();
      for (int e = threadIdx.x; e < step; e += blockDim.x) {   // the rows side by side
        const int c = v * step + e;
        if (c >= dim) continue;
        float a = 0.f;
        for (int x = 0; x < RPB; ++x) a += acc[x * step + e];
        o.part[((int64_t)blockIdx.x * 2 + i) * dim + c] = a;
      }
    }
}

// Column sums of the workgroups' parts: 32 columns a workgroup, 32 half waves over the parts.
__global__ __launch_bounds__(1024) void weight_sum_kernel(const float* part, int parts, int dim,
                                                          bs_layer_norm_in in, void* dweight,
                                                          void* dbias) {
  __shared__ float sh[32][33];
  const int which = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  void* out = which ? dbias : dweight;
  if (!out) return;
  float a = 0.f;
  if (c < dim)
    for (int k = w; k < parts; k += 32) a += part[((int64_t)k * 2 + which) * dim + c];
  sh[w][threadIdx.x & 31] = a;
  __syncthreads();
  if (w == 0 && c < dim) {
    for (int k = 1; k < 32; ++k) a += sh[k][threadIdx.x];
    bs_store_any(out, which ? in.bias_dtype : in.weight_dtype, c, a);
  }
}

struct DropoutIn {
  const void* x;
  void* y;
  int64_t stride, row0;
  uint64_t seed;
  const int64_t* seed_at;
  uint32_t units, per;              // runs of 8 columns, and of a row
  int dim;
  uint32_t site, drop;
  float scale;
};

// A run of 8 columns a lane.
template <typename T, int MODE>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutIn in) {
  const uint32_t u = blockIdx.x * 256 + threadIdx.x;
  if (u >= in.units) return;
  const uint32_t r = u / in.per;
  const int64_t row = in.row0 + r;
  const Cols<MODE> k((u - r * in.per) * kVec, in.dim);
  Vec8<T, MODE> v;
  v.load((const T*)in.x + row * in.stride, k, in.dim);
  const Dropout drop(in.seed, in.seed_at, in.site, in.drop);
  const uint32_t kept = drop.eight(row, k.at);
  float x[kVec];
  v.values(true, x);
#pragma unroll
  for (int j = 0; j < kVec; ++j) x[j] = kept >> j & 1 ? x[j] * in.scale : 0.f;
  v.store((T*)in.y + row * in.dim, k, in.dim, x);
}

int check(const bs_layer_norm_in* in, const char* who) {
  BS_CHECK_ARG(in != nullptr, "%s: operands are NULL", who);
  BS_CHECK_ARG(bs_dtype_ok(in->dtype) && bs_dtype_ok(in->weight_dtype) &&
                   bs_dtype_ok(in->bias_dtype),
               "%s: dtype unknown", who);
  BS_CHECK_ARG(in->rows >= 0 && in->dim >= 1 && in->dim <= 16384,
               "%s: %lld rows of %d values (1..16384)", who, (long long)in->rows, in->dim);
  BS_CHECK_ARG(in->rows == 0 || in->x, "%s: x is NULL", who);
  return BS_OK;
}

// Lanes to a row: 16 or a wave for short rows, else as many whole waves as it has runs of 8
// values, up to 16; two runs a lane past 8,192 values.
struct Shape { int lanes, nv; };
Shape shape_of(int dim) {
  const int runs = (dim + kVec - 1) / kVec;
  if (runs <= 16) return {16, 1};
  if (runs <= 64) return {64, 1};
  const int nv = runs > 1024 ? 2 : 1;
  return {(runs + 64 * nv - 1) / (64 * nv) * 64, nv};
}

int block_of(const Shape& s) { return s.lanes <= 64 ? 256 : s.lanes; }

int grid_of(int64_t rows, const Shape& s, int threads) {   // threads: wanted on a CU
  const int block = block_of(s), rpb = s.lanes <= 64 ? 256 / s.lanes : 1;
  const int64_t need = (rows + rpb - 1) / rpb;
  const int64_t most = (int64_t)(threads / block > 1 ? threads / block : 1) * bs_num_cus();
  return (int)(need < most ? need : most);
}

// Threads on a CU.  Forward and backward of 8,192 rows of 4,096 in bf16 take 153 us at 2,048 forward
// ones (172 at 512, 157 at 1,024, 152 at 4,096, which takes 2,048 rows of 16,384 from 48 us to 55); the
// gradients, whose workgroups each leave a row of sums, 226 us for 2,048 rows of 16,384 at 512 and
// 1,024, 257 at 2,048.
constexpr int kThreads = 2048, kGradThreads = 512;

// f(lanes of a row or 0, runs a lane, largest workgroup, mode)
template <typename F>
void by_shape(const Shape& s, int dim, F&& f) {
  auto moded = [&](auto... a) {
    if (dim % kVec == 0) f(a..., Int<kWhole>());
    else f(a..., Int<kTail>());
  };
  if (dim < kVec) f(Int<16>(), Int<1>(), Int<256>(), Int<kSmall>());
  else if (s.lanes == 16) moded(Int<16>(), Int<1>(), Int<256>());
  else if (s.lanes == 64) moded(Int<64>(), Int<1>(), Int<256>());
  else if (s.nv == 2) moded(Int<0>(), Int<2>(), Int<1024>());
  else if (s.lanes <= 512) moded(Int<0>(), Int<1>(), Int<512>());
  else moded(Int<0>(), Int<1>(), Int<1024>());
}

template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == BS_F32) f(float());
  else if (dtype == BS_BF16) f(bs_bf16());
  else f(bs_f16());
}

}  // namespace

extern "C" int bs_layer_norm(const bs_layer_norm_in* in, void* stream_out, void* normed_out,
                             float* stats, bs_stream_t stream) {
  if (int rc = check(in, "bs_layer_norm")) return rc;
  if (in->rows == 0) return BS_OK;
  BS_CHECK_ARG(normed_out, "bs_layer_norm: output is NULL");
  hipStream_t st = bs_stream(stream);
  const Shape s = shape_of(in->dim);
  const int grid = grid_of(in->rows, s, kThreads);
  by_type(in->dtype, [&](auto t) {
    using T = decltype(t);
    by_shape(s, in->dim, [&](auto tpr, auto nv, auto block, auto mode) {
      if (in->drop)
        layer_norm_kernel<T, tpr.value, nv.value, block.value, mode.value, true>
            <<<grid, block_of(s), 0, st>>>(*in, (T*)stream_out, (T*)normed_out, stats);
      else
        layer_norm_kernel<T, tpr.value, nv.value, block.value, mode.value, false>
            <<<grid, block_of(s), 0, st>>>(*in, (T*)stream_out, (T*)normed_out, stats);
    });
  });
  BS_CHECK_LAUNCH();
  return BS_OK;
}

extern "C" size_t bs_layer_norm_grad_workspace_size(int64_t rows, int32_t dim) {
  if (rows < 1 || dim < 1 || dim > 16384) return 0;
  return (size_t)grid_of(rows, shape_of(dim), kGradThreads) * 2 * dim * sizeof(float);
}

extern "C" int bs_layer_norm_grad(const bs_layer_norm_in* in, const void* grad_stream,
                                  const void* grad_normed, const float* stats, void* dx,
                                  void* dresidual, void* dweight, void* dbias, void* workspace,
                                  size_t workspace_bytes, bs_stream_t stream) {
  if (int rc = check(in, "bs_layer_norm_grad")) return rc;
  BS_CHECK_ARG((!dresidual || in->residual) && (!dweight || in->weight) && (!dbias || in->bias),
               "bs_layer_norm_grad: a gradient of an operand that is not given");
  BS_CHECK_ARG(in->rows == 0 || stats, "bs_layer_norm_grad: stats is NULL");
  const bool weights = dweight || dbias;
  const size_t need = weights ? bs_layer_norm_grad_workspace_size(in->rows, in->dim) : 0;
  BS_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
               "bs_layer_norm_grad: workspace of %zu bytes needed", need);
  const LayerNormGrad o = {grad_stream, grad_normed, stats, dx, dresidual,
                           weights ? (float*)workspace : nullptr};
  hipStream_t st = bs_stream(stream);
  const Shape s = shape_of(in->dim);
  const int grid = grid_of(in->rows, s, kGradThreads);
  if (grid)
    by_type(in->dtype, [&](auto t) {
      using T = decltype(t);
      by_shape(s, in->dim, [&](auto tpr, auto nv, auto block, auto mode) {
        if (in->drop)
          layer_norm_grad_kernel<T, tpr.value, nv.value, block.value, mode.value, true>
              <<<grid, block_of(s), 0, st>>>(*in, o);
        else
          layer_norm_grad_kernel<T, tpr.value, nv.value, block.value, mode.value, false>
              <<<grid, block_of(s), 0, st>>>(*in, o);
      });
    });
  if (weights)
    weight_sum_kernel<<<dim3((in->dim + 31) / 32, 2), 1024, 0, st>>>(
        (const float*)workspace, grid, in->dim, *in, dweight, dbias);
  BS_CHECK_LAUNCH();
  return BS_OK;
}

extern "C" int bs_dropout(const void* x, int32_t dtype, int64_t rows, int64_t dim, int64_t stride,
                          uint64_t seed, const int64_t* seed_at, uint32_t site, uint32_t drop,
                          float scale, void* y, bs_stream_t stream) {
  BS_CHECK_ARG(bs_dtype_ok(dtype), "bs_dropout: dtype unknown");
  BS_CHECK_ARG(rows >= 0 && dim >= 1 && dim <= INT32_MAX,
               "bs_dropout: %lld rows of %lld values (1..2^31 - 1)", (long long)rows,
               (long long)dim);
  if (rows == 0) return BS_OK;
  BS_CHECK_ARG(x && y, "bs_dropout: NULL pointer");
  hipStream_t st = bs_stream(stream);
  const int64_t per = (dim + kVec - 1) / kVec, most = (1ll << 31) / per;
  DropoutIn in = {x, y, stride, 0, seed, seed_at, 0, (uint32_t)per, (int)dim, site, drop, scale};
  // a launch has fewer than 2^32 threads: rows in pieces
  for (; in.row0 < rows; in.row0 += most) {
    const int64_t n = rows - in.row0 < most ? rows - in.row0 : most;
    in.units = (uint32_t)(n * per);
    const unsigned grid = (in.units + 255u) / 256;
    by_type(dtype, [&](auto t) {
      using T = decltype(t);
      if (dim < kVec) dropout_kernel<T, kSmall><<<grid, 256, 0, st>>>(in);
      else if (dim % kVec) dropout_kernel<T, kTail><<<grid, 256, 0, st>>>(in);
      else dropout_kernel<T, kWhole><<<grid, 256, 0, st>>>(in);
    });
    BS_CHECK_LAUNCH();
  }
  return BS_OK;
}
