// The norms before and after a block, its gate, residual scale and residual, in one pass, and
// their gradients.  With r(x) = (mean x^2 + eps)^-1/2 over a row:
//
//   p = y r(y) post,  t = scale silu(gate) p,  s = residual + t,  normed = s r(s) pre
//
// (a part that is not given is left out).  Bound by bytes: a row is read once into registers,
// where both norms' sums are taken in 32 bits, and its results are written once; s is rounded
// only when it is stored.  A row belongs to as many lanes as it has
// runs of 8 values, so a norm over a head of 128 values shares a wave with three others and one of
// 2,050 takes 5 waves.
// Workgroups stay for many rows: a lane's columns are the same in each, so the weights are read
// once and the weights' gradients are summed in registers, then over the workgroups in their
// order (grad_sum_kernel): the same bits every time.
// bfloat16 with every part, beside a large copy's 5.1 TB/s: 8,192 x 4,096 forward 68 us (4.9 TB/s),
// gradients 136 us with the weights' sums (3.9 TB/s; the kernel alone 129, 201 with a row's loads
// only after the row before); 4,099 x 2,050 29 and 76 us.
// Two runs a lane (past 4,096 values) do not fit the gradients' registers, which spill 340 to 436
// bytes a lane, 856 to 892 in workgroups of 1,024 (past 8,192), where the forward kernel spills 92
// to 256 as well: 4,096 x 5,120 forward 70 us (3.0 TB/s: 5 waves lie unevenly on 4 SIMDs),
// gradients 444 (0.8); 8,192 x 8,192 143 (4.7) and 1,026 (1.0); 4,096 x 16,384 245 (2.7) and 2,046
// (0.5).
#include "rows.h"

namespace {

// 1 / (1 + exp(-z)): the hardware's exponential and reciprocal, each within 1 ulp; the exponent's
// rounding adds |z| 2^-24 where exp(-z) counts beside 1.
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * z));
}

// TPR lanes to a row and 256 / TPR rows to a workgroup, or (TPR = 0) a row to a workgroup.
template <typename T, int TPR, int NV, int BLOCK, int MODE>
__global__ __launch_bounds__(BLOCK) void norm_kernel(bs_norm_in in, T* stream, T* normed) {
  constexpr int RPB = TPR ? 256 / TPR : 1;
  __shared__ float sh[2][16][1];
  const int lanes = TPR ? TPR : blockDim.x, t = threadIdx.x % lanes;
  const int step = lanes * kVec, dim = in.dim;
  Cols<MODE> k[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) k[v] = Cols<MODE>(t * kVec + v * step, dim);
  int turn = 0;
  float post[NV][kVec], scale[NV][kVec], pre[NV][kVec];
  load_weight<NV>(in.post, in.post_dtype, k, dim, 1.f, post);
  load_weight<NV>(in.scale, in.scale_dtype, k, dim, in.scale_value, scale);
  load_weight<NV>(in.pre, in.pre_dtype, k, dim, 1.f, pre);
  const float inv = 1.f / (float)dim;
  const int64_t stride = (int64_t)gridDim.x * RPB, last = in.rows - 1;
  int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / lanes;
  const int64_t turns = (in.rows - (int64_t)blockIdx.x * RPB + stride - 1) / stride;
  Vec8<T, MODE> yv[NV], zv[NV], sv[NV];
  // the next row's operands are loaded while this one's sums are taken
  auto load = [&](int64_t r) {
    r = r < last ? r : last;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      yv[v].load((const T*)in.y + r * in.y_stride, k[v], dim);
      if (in.gate) zv[v].load((const T*)in.gate + r * in.gate_stride, k[v], dim);
      if (in.residual) sv[v].load((const T*)in.residual + r * in.residual_stride, k[v], dim);
    }
  };
  load(row);
  for (int64_t turn_of = 0; turn_of < turns; ++turn_of, row += stride) {
    const bool live = row < in.rows;
    float x[NV][kVec], z[NV][kVec], s[NV][kVec];
    float sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const bool inside = k[v].in;
      yv[v].values(inside, x[v]);
      if (in.gate) zv[v].values(inside, z[v]);
      if (in.residual) sv[v].values(inside, s[v]);
#pragma unroll
      for (int j = 0; j < kVec; ++j) sum[0] = fmaf(k[v].once(j, x[v][j]), x[v][j], sum[0]);
    }
    load(row + stride);
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
        sum[0] = fmaf(k[v].once(j, a), a, sum[0]);
      }
      if (live) yv[v].store(stream + row * dim, k[v], dim, s[v]);
    }
    if (in.pre) {
      row_sum<TPR, 1>(sum, sh, turn);
      const float r2 = rsqrtf(sum[0] * inv + in.eps);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) s[v][j] *= r2 * pre[v][j];
        if (live) yv[v].store(normed + row * dim, k[v], dim, s[v]);
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
template <typename T, int TPR, int NV, int BLOCK, int MODE>
__global__ __launch_bounds__(BLOCK) void norm_grad_kernel(bs_norm_in in, NormGrad o) {
  constexpr int RPB = TPR ? 256 / TPR : 1;
  __shared__ float sh[2][16][1];
  __shared__ float sh2[2][16][2];
  __shared__ float acc[BLOCK * kVec];
  const int lanes = TPR ? TPR : blockDim.x, t = threadIdx.x % lanes;
  const int step = lanes * kVec, dim = in.dim;
  Cols<MODE> k[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) k[v] = Cols<MODE>(t * kVec + v * step, dim);
  int turn = 0, turn2 = 0;
  float post[NV][kVec], scale[NV][kVec], pre[NV][kVec];
  float dw[3][NV][kVec];
  load_weight<NV>(in.post, in.post_dtype, k, dim, 1.f, post);
  load_weight<NV>(in.scale, in.scale_dtype, k, dim, in.scale_value, scale);
  load_weight<NV>(in.pre, in.pre_dtype, k, dim, 1.f, pre);
#pragma unroll
  for (int i = 0; i < 3; ++i)
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < kVec; ++j) dw[i][v][j] = 0.f;
  const float inv = 1.f / (float)dim;
  const int64_t stride = (int64_t)gridDim.x * RPB, last = in.rows - 1;
  int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / lanes;
  const int64_t turns = (in.rows - (int64_t)blockIdx.x * RPB + stride - 1) / stride;
  Vec8<T, MODE> yv[NV], zv[NV], sv[NV], gsv[NV], gnv[NV];
  auto load = [&](int64_t r) {
    r = r < last ? r : last;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      yv[v].load((const T*)in.y + r * in.y_stride, k[v], dim);
      if (in.gate) zv[v].load((const T*)in.gate + r * in.gate_stride, k[v], dim);
      if (in.residual) sv[v].load((const T*)in.residual + r * in.residual_stride, k[v], dim);
      if (o.gs) gsv[v].load((const T*)o.gs + r * dim, k[v], dim);
      if (o.gn) gnv[v].load((const T*)o.gn + r * dim, k[v], dim);
    }
  };
  // the next row is loaded while this one's sums are formed, where registers are left for it
  constexpr bool kAhead = NV == 1;
  if (kAhead) load(row);
  for (int64_t turn_of = 0; turn_of < turns; ++turn_of, row += stride) {
    const bool live = row < in.rows;
    if (!kAhead) load(row);
    float x[NV][kVec], z[NV][kVec], s[NV][kVec], d[NV][kVec], dn[NV][kVec];
    float sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const bool inside = k[v].in;
      yv[v].values(inside, x[v]);
      if (in.gate) zv[v].values(inside, z[v]);
      if (in.residual) sv[v].values(inside, s[v]);
      gsv[v].values(o.gs && inside && live, d[v]);       // a row that is not there gives nothing
      gnv[v].values(o.gn && inside && live, dn[v]);
#pragma unroll
      for (int j = 0; j < kVec; ++j) sum[0] = fmaf(k[v].once(j, x[v][j]), x[v][j], sum[0]);
    }
    if (kAhead) load(row + stride);
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
          two[0] = fmaf(k[v].once(j, a), a, two[0]);
          two[1] = fmaf(k[v].once(j, dn[v][j]) * pre[v][j], a, two[1]);
        }
      }
    if (o.gn) {
      row_sum<TPR, 2>(two, sh2, turn2);
      const float r2 = rsqrtf(two[0] * inv + in.eps), off = two[1] * r2 * r2 * inv;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          dw[2][v][j] = fmaf(dn[v][j], s[v][j] * r2, dw[2][v][j]);
          d[v][j] += r2 * (dn[v][j] * pre[v][j] - s[v][j] * off);
        }
    }
    sum[0] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (live && o.dresidual) yv[v].store((T*)o.dresidual + row * dim, k[v], dim, d[v]);
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
        sum[0] = fmaf(k[v].once(j, d[v][j]), x[v][j], sum[0]);
      }
      if (live && o.dgate) yv[v].store((T*)o.dgate + row * dim, k[v], dim, z[v]);
    }
    if (in.post) row_sum<TPR, 1>(sum, sh, turn);
    const float off = in.post ? sum[0] * inv : 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) d[v][j] = r1 * (d[v][j] - x[v][j] * off);
      if (live && o.dy) yv[v].store((T*)o.dy + row * dim, k[v], dim, d[v]);
    }
  }
  if (!o.part) return;
#pragma unroll
  for (int i = 0; i < 3; ++i)
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
        float a = 0.f;
        if (c < dim)
          for (int x = 0; x < RPB; ++x) a += acc[x * step + e];
        if (c < dim) o.part[((int64_t)blockIdx.x * 3 + i) * dim + c] = a;
      }
    }
}

// Column sums of the workgroups' parts: 32 columns a workgroup, 32 half waves over the parts.
__global__ __launch_bounds__(1024) void grad_sum_kernel(const float* part, int parts, int dim,
                                                        bs_norm_in in, void* dpost, void* dscale,
                                                        void* dpre) {
  __shared__ float sh[32][33];
  const int which = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  void* out = which == 0 ? dpost : which == 1 ? dscale : dpre;
  if (!out) return;
  float a = 0.f;
  if (c < dim)
    for (int k = w; k < parts; k += 32) a += part[((int64_t)k * 3 + which) * dim + c];
  sh[w][threadIdx.x & 31] = a;
  __syncthreads();
  if (w == 0 && c < dim) {
    for (int k = 1; k < 32; ++k) a += sh[k][threadIdx.x];
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

// Lanes to a row: as many as it has runs of 8 values, a power of two up to a wave, whole waves
// above; two runs a lane past 4,096 values.  us at 262,144 x 128 by 16 / 64 lanes 62 / 144, at
// 131,072 x 250 by 32 / 64 63 / 90.
struct Shape { int lanes, nv; };
Shape shape_of(int dim) {
  const int runs = (dim + kVec - 1) / kVec;
  if (runs <= 16) return {16, 1};
  if (runs <= 32) return {32, 1};
  const int nv = runs > 512 ? 2 : 1;
  return {(runs + 64 * nv - 1) / (64 * nv) * 64, nv};
}
// Forward only: two runs a lane also where one would take 5 or 6 waves, which lie unevenly on a
// CU's 4 SIMDs (bfloat16, us with one / two: 8,192 x 2,560 48.5 / 44.5, x 3,000 58.8 / 48.0, 4,099 x
// 2,050 34.0 / 25.5; 4 waves, x 2,048, 32.7 / 35.3; 7 waves, x 3,584, 63.7 / 63.7).  The gradients
// would leave the registers (4,099 x 2,050 90 / 280).
Shape forward_shape_of(int dim) {
  const int runs = (dim + kVec - 1) / kVec;
  return runs > 256 && runs <= 384 ? Shape{192, 2} : shape_of(dim);
}
int block_of(const Shape& s) { return s.lanes <= 64 ? 256 : s.lanes; }

int grid_of(const bs_norm_in& in, const Shape& s, int threads) {   // threads: wanted on a CU
  const int block = block_of(s), rpb = s.lanes <= 64 ? 256 / s.lanes : 1;
  const int64_t need = (in.rows + rpb - 1) / rpb;
  const int64_t most = (int64_t)(threads / block > 1 ? threads / block : 1) * bs_num_cus();
  return (int)(need < most ? need : most);
}

// Threads a CU: a full one forward (512 / 1,024 / 2,048 / 4,096 at 8,192 x 4,096: 69.7 / 67.0 / 65.8 /
// 68.2 us); fewer for gradients, whose workgroups each leave three rows of sums (512 / 1,024 / 2,048
// at 8,192 x 2,048, loads not yet ahead: 96 / 113 / 134 us).
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
  else if (s.lanes == 32) moded(Int<32>(), Int<1>(), Int<256>());
  else if (s.lanes == 64) moded(Int<64>(), Int<1>(), Int<256>());
  else if (s.nv == 1) moded(Int<0>(), Int<1>(), Int<512>());
  else if (s.lanes <= 512) moded(Int<0>(), Int<2>(), Int<512>());
  else moded(Int<0>(), Int<2>(), Int<1024>());
}

template <typename T>
void launch(const bs_norm_in& in, void* stream, void* normed, hipStream_t st) {
  const Shape s = forward_shape_of(in.dim);
  const int grid = grid_of(in, s, kThreads);
  by_shape(s, in.dim, [&](auto tpr, auto nv, auto block, auto mode) {
    norm_kernel<T, tpr.value, nv.value, block.value, mode.value>
        <<<grid, block_of(s), 0, st>>>(in, (T*)stream, (T*)normed);
  });
}

template <typename T>
void launch_grad(const bs_norm_in& in, const NormGrad& o, hipStream_t st) {
  const Shape s = shape_of(in.dim);
  const int grid = grid_of(in, s, kGradThreads);
  if (grid == 0) return;
  by_shape(s, in.dim, [&](auto tpr, auto nv, auto block, auto mode) {
    norm_grad_kernel<T, tpr.value, nv.value, block.value, mode.value>
        <<<grid, block_of(s), 0, st>>>(in, o);
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
  return (size_t)grid_of(in, shape_of(dim), kGradThreads) * 3 * dim * sizeof(float);
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
    const int parts = grid_of(*in, shape_of(in->dim), kGradThreads);
    grad_sum_kernel<<<dim3((in->dim + 31) / 32, 3), 1024, 0, st>>>(
        (const float*)workspace, parts, in->dim, *in, dpost, dscale, dpre);
    BS_CHECK_LAUNCH();
  }
  return BS_OK;
}
