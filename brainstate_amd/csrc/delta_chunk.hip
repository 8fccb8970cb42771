// The gated delta rule over chunks of 64 tokens, forward, and the backward pass's recurrence.
//
// With run_i the sum of the log decays of a chunk up to token i, S0 the state before it and
// e_ij = exp(run_i - run_j):
//
//   (1 + L) U = R,   R_i = beta_i (v_i - exp(run_i) S0^T k_i),   L_ij = beta_i e_ij k_i.k_j (j < i)
//   S = exp(run_63) S0 + sum_j exp(run_63 - run_j) k_j u_j^T
//   o_i = scale (exp(run_i) S0^T q_i + sum_{j <= i} e_ij (q_i.k_j) u_j)
//
// so a chunk costs four products with the state and within the chunk, and one dependent step
// for 64 tokens.  prepare_kernel forms, for all chunks at once, what does not depend on the
// state: (1 + L)^-1, the masked q k^T, and q and k as bf16 parts in the order the products take
// them.  chain_kernel then walks the chunks of one sequence, head and slice of value columns.
//
// Numbers: the state, U, R, (1 + L)^-1 and all sums are 32-bit; products take them as three
// exact bf16 parts (lane_types.h).  Sums of log decays are 64-bit, since their differences are
// exponents.
#include "delta_chunk.h"

namespace {

// One chunk and value head: 4 waves, wave w has rows 16w..16w+15.
// The inverse is formed by blocks of 16: the four on the diagonal by substitution, one column a
// lane, the ones below by X_ij = -X_ii sum_k L_ik X_kj in 32-bit matrix instructions.
template <typename T, int PI, int KS, bool BWD>
__global__ __launch_bounds__(256) void prepare_kernel(bs_delta_in in, DeltaPlan plan, DeltaWork w,
                                                      int vec) {
  constexpr int DK = KS * 32, LD = DK + 8;
  __shared__ __attribute__((aligned(16))) uint16_t kl[PI][kChunk][LD];
  __shared__ float lm[kChunk][kChunk + 4];
  __shared__ float xm[kChunk][kChunk + 4];
  __shared__ double run[kChunk];
  __shared__ float bt[kChunk];
  const int slot = blockIdx.x, h = blockIdx.y;
  const int group = in.hv / in.hk, hk = h / group;
  const DeltaSpan sp = delta_span(plan, delta_owner(plan, slot));
  const int c = slot - sp.slot;
  if (c >= sp.chunks) return;
  const int64_t t0 = sp.first + (int64_t)c * kChunk;
  const int len = min(sp.len - c * kChunk, kChunk);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, g = lane >> 4;
  const bool first = h % group == 0;

  if (wave == 0) {      // lane = token
    double x = lane < len ? (double)bs_delta_g(in, sp.batch, t0 + lane, h) : 0.0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double y = __shfl_up(x, d);
      if (lane >= d) x += y;
    }
    const float b = lane < len ? bs_delta_beta(in, sp.batch, t0 + lane, h) : 0.f;
    run[lane] = x, bt[lane] = b;
    const double total = __shfl(x, 63);
    float* co = w.coef + ((int64_t)slot * in.hv + h) * kCoef;
    co[lane] = expf((float)x);
    co[kChunk + lane] = expf((float)(total - x));
    co[2 * kChunk + lane] = b;
    co[3 * kChunk + lane] = expf((float)total);
    ((double*)(co + 4 * kChunk))[lane] = x;
  }
  const int row = 16 * wave + m;
  bs_parts<PI> qf[KS], kf[KS];
  {
    const bool live = row < len;
    const int64_t t = live ? t0 + row : t0;
    const T* kp = (const T*)in.k + bs_delta_at(in.k_stride, sp.batch, t, hk);
    const T* qp = (const T*)in.q + bs_delta_at(in.q_stride, sp.batch, t, hk);
    const int64_t base = ((int64_t)slot * in.hk + hk) * PI * kChunk * DK;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 32 * s + 8 * g, left = live ? in.dk - d : 0;
      kf[s] = load_parts<PI>(kp + d, left, vec);
      qf[s] = load_parts<PI>(qp + d, left, vec);
#pragma unroll
      for (int p = 0; p < PI; ++p) {
        *(bs_bf16x8*)&kl[p][row][d] = kf[s].p[p];
        if (first) {
          *(bs_bf16x8*)(w.kp + base + ((int64_t)p * kChunk + row) * DK + d) = kf[s].p[p];
          *(bs_bf16x8*)(w.qp + base + ((int64_t)p * kChunk + row) * DK + d) = qf[s].p[p];
        }
      }
    }
  }
  __syncthreads();
  float* att = w.att + ((int64_t)slot * in.hv + h) * kChunk * kChunk;
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) {
    if (jt > (wave | 1)) {       // past the 32-token block of the diagonal: never read
      if (BWD) continue;
      break;
    }
    const int j = 16 * jt + m;
    bs_f32x4 kk = {0.f, 0.f, 0.f, 0.f}, qk = kk;
    if (jt <= wave) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        bs_parts<PI> b;
#pragma unroll
        for (int p = 0; p < PI; ++p) b.p[p] = *(const bs_bf16x8*)&kl[p][j][32 * s + 8 * g];
        kk = bs_mma<2>(kf[s], b, kk);
        qk = bs_mma<2>(qf[s], b, qk);
      }
    }
    float4 row4;
    float* r4 = (float*)&row4;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * wave + 4 * g + r;
      const float e = j <= i ? expf((float)(run[i] - run[j])) : 0.f;
      if (jt <= wave) lm[i][j] = j < i ? bt[i] * e * kk[r] : 0.f;
      else xm[i][j] = 0.f;
      const float a = j <= i ? in.scale * e * qk[r] : 0.f;
      r4[r] = a;
      if (!BWD) att[i * kChunk + j] = a;
    }
    if (BWD) *(float4*)(att + j * kChunk + 16 * wave + 4 * g) = row4;
  }
  if (first) {                    // the transposed copies: 8 lanes write a row of 64 tokens
    const int64_t base = ((int64_t)slot * in.hk + hk) * PI * kChunk * DK;
    for (int p = 0; p < PI; ++p)
      for (int d = tid >> 3; d < DK; d += 32) {
        bs_u16x8 r;
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = kl[p][8 * (tid & 7) + j][d];
        *(bs_u16x8*)(w.kt + base + ((int64_t)p * DK + d) * kChunk + 8 * (tid & 7)) = r;
      }
  }
  __syncthreads();
  {
    float x[16];
    const int o = 16 * wave;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float a = r == m ? 1.f : 0.f;
#pragma unroll
      for (int s = 0; s < r; ++s) a = fmaf(-lm[o + r][o + s], x[s], a);
      x[r] = a;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if ((r >> 2) == g) xm[o + r][o + m] = x[r];
  }
  if (BWD && first) {             // q's transposed copy, through the same LDS
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int p = 0; p < PI; ++p) *(bs_bf16x8*)&kl[p][row][32 * s + 8 * g] = qf[s].p[p];
  }
  __syncthreads();
  if (BWD && first) {
    const int64_t base = ((int64_t)slot * in.hk + hk) * PI * kChunk * DK;
    for (int p = 0; p < PI; ++p)
      for (int d = tid >> 3; d < DK; d += 32) {
        bs_u16x8 r;
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = kl[p][8 * (tid & 7) + j][d];
        *(bs_u16x8*)(w.qt + base + ((int64_t)p * DK + d) * kChunk + 8 * (tid & 7)) = r;
      }
  }
  for (int d = 1; d < 4; ++d) {
    const int j = wave, i = wave + d;
    if (i < 4) {
      bs_f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
      for (int k = j; k < i; ++k)
#pragma unroll
        for (int s = 0; s < 4; ++s)
          a = __builtin_amdgcn_mfma_f32_16x16x4f32(lm[16 * i + m][16 * k + 4 * s + g],
                                                   xm[16 * k + 4 * s + g][16 * j + m], a, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r)     // contracted rows 4g + r, as the first product left them
        b = __builtin_amdgcn_mfma_f32_16x16x4f32(xm[16 * i + m][16 * i + 4 * g + r], a[r], b, 0,
                                                 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) xm[16 * i + 4 * g + r][16 * j + m] = -b[r];
    }
    __syncthreads();
  }
  float* inv = w.inv + ((int64_t)slot * in.hv + h) * kChunk * kChunk;
  for (int e = tid; e < kChunk * 16; e += 256) {
    const int i = e >> 4, j = (e & 15) * 4;
    if (BWD) {
      if ((j | 31) < i) continue;     // row i of the transpose starts at its 32-token block
      *(float4*)(inv + i * kChunk + j) =
          make_float4(j < i ? 0.f : xm[j][i], j + 1 < i ? 0.f : xm[j + 1][i],
                      j + 2 < i ? 0.f : xm[j + 2][i], j + 3 < i ? 0.f : xm[j + 3][i]);
    } else {
      if (j > (i | 31)) continue;
      *(float4*)(inv + i * kChunk + j) = *(const float4*)&xm[i][j];
    }
  }
}

// Forward over the chunks of one sequence (z), value head (y) and slice of 16 NT value columns
// (x).  Each of 4 waves has 16 tokens of a chunk and a quarter of the state's rows; what the
// others need goes through LDS, as parts and in the lane that takes it.
template <typename T, int PI, int KS, int NT>
__global__ __launch_bounds__(256) void chain_kernel(bs_delta_in in, DeltaPlan plan, DeltaWork w,
                                                    const float* state0, float* state1, T* o,
                                                    float* keep_s, float* keep_u, int dvp) {
  constexpr int DK = KS * 32, TW = KS / 2, PO = PI == 3 ? 3 : 2;
  constexpr int kS = KS * NT * 128, kR = 2 * NT * 128;       // words of a part
  __shared__ __attribute__((aligned(16))) uint2 ls[3 * kS];
  __shared__ __attribute__((aligned(16))) uint2 lr[3 * kR];
  __shared__ __attribute__((aligned(16))) uint2 lu[3 * kR];
  __shared__ __attribute__((aligned(16))) uint2 lv[PO * kR];
  const int h = blockIdx.y, n = blockIdx.z, hk = h / (in.hv / in.hk);
  if (n >= plan.seqs) {
    zero_outside(plan, o, in.hv, in.dv, h, blockIdx.x * 16 * NT, 16 * NT);
    return;
  }
  const DeltaSpan sp = delta_span(plan, n);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, g = lane >> 4;
  const int col0 = blockIdx.x * 16 * NT + m;
  const int tok = delta_row(wave, m);                 // the row this lane feeds
  const int out0 = 32 * (wave >> 1) + 8 * g + 4 * (wave & 1);   // the 4 rows it receives
  const int blk = wave >> 1;

  bs_f32x4 s[TW][NT];
#pragma unroll
  for (int i = 0; i < TW; ++i) {
    const int t = TW * wave + i, d0 = 32 * (t >> 1) + 8 * g + 4 * (t & 1);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int c = col0 + 16 * nt;
        s[i][nt][r] = state0 && d0 + r < in.dk && c < in.dv
            ? state0[(((int64_t)n * in.hv + h) * in.dk + d0 + r) * in.dv + c] : 0.f;
      }
      delta_put<3>(ls + (((t >> 1) * NT + nt) * 64 + lane) * 2 + (t & 1), kS, s[i][nt]);
    }
  }
  __syncthreads();
  for (int c = 0; c < sp.chunks; ++c) {
    const int slot = sp.slot + c;
    const int64_t sh = (int64_t)slot * in.hv + h;
    const int64_t kb = ((int64_t)slot * in.hk + hk) * PI * kChunk * DK;
    const float* co = w.coef + sh * kCoef;
    const float4 grow = *(const float4*)(co + out0), left = *(const float4*)(co + kChunk + out0),
                 beta = *(const float4*)(co + 2 * kChunk + out0);
    const float total = co[3 * kChunk];
    const float* gr = (const float*)&grow;
    const float* lf = (const float*)&left;
    const float* be = (const float*)&beta;
    if (keep_s) {
#pragma unroll
      for (int i = 0; i < TW; ++i) {
        const int t = TW * wave + i, d0 = 32 * (t >> 1) + 8 * g + 4 * (t & 1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            keep_s[(sh * DK + d0 + r) * dvp + col0 + 16 * nt] = s[i][nt][r];
      }
    }
    bs_f32x4 ks[NT], qs[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) ks[nt] = qs[nt] = zero4();
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      const bs_parts<PI> kf = delta_frags<PI>(w.kp + kb + tok * DK + 32 * st + 8 * g, kChunk * DK);
      const bs_parts<PI> qf = delta_frags<PI>(w.qp + kb + tok * DK + 32 * st + 8 * g, kChunk * DK);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const bs_parts<3> b = delta_lds<3>(ls + ((st * NT + nt) * 64 + lane) * 2, kS);
        ks[nt] = bs_mma<2>(kf, b, ks[nt]);
        qs[nt] = bs_mma<PO - 1>(qf, b, qs[nt]);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int cc = col0 + 16 * nt;
      bs_f32x4 x;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = c * kChunk + out0 + r;
        const float v = t < sp.len && cc < in.dv
            ? bs_to_f32(((const T*)in.v)[bs_delta_at(in.v_stride, sp.batch, sp.first + t, h) + cc])
            : 0.f;
        x[r] = be[r] * (v - gr[r] * ks[nt][r]);
      }
      delta_put<3>(lr + ((blk * NT + nt) * 64 + lane) * 2 + (wave & 1), kR, x);
    }
    __syncthreads();
    bs_f32x4 u[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) u[nt] = zero4();
    const float* ip = w.inv + sh * kChunk * kChunk + tok * kChunk + 8 * g;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      if (st > blk) break;
      const bs_parts<3> a = row_parts(ip + 32 * st);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        u[nt] = bs_mma<2>(a, delta_lds<3>(lr + ((st * NT + nt) * 64 + lane) * 2, kR), u[nt]);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int at = ((blk * NT + nt) * 64 + lane) * 2 + (wave & 1);
      delta_put<PO>(lv + at, kR, u[nt]);
      bs_f32x4 x;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = lf[r] * u[nt][r];
        if (keep_u) keep_u[(sh * kChunk + out0 + r) * dvp + col0 + 16 * nt] = u[nt][r];
      }
      delta_put<3>(lu + at, kR, x);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TW; ++i) {
      const int t = TW * wave + i;
      const uint16_t* kt = w.kt + kb + delta_row(t, m) * kChunk + 8 * g;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[i][nt] *= total;
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const bs_parts<PI> a = delta_frags<PI>(kt + 32 * st, DK * kChunk);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          s[i][nt] = bs_mma<2>(a, delta_lds<3>(lu + ((st * NT + nt) * 64 + lane) * 2, kR),
                               s[i][nt]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        delta_put<3>(ls + (((t >> 1) * NT + nt) * 64 + lane) * 2 + (t & 1), kS, s[i][nt]);
    }
    const float* ap = w.att + sh * kChunk * kChunk + tok * kChunk + 8 * g;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 4; ++r) qs[nt][r] *= in.scale * gr[r];
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      if (st > blk) break;
      const bs_parts<3> a = row_parts(ap + 32 * st);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        qs[nt] = bs_mma<PO - 1>(a, delta_lds<PO>(lv + ((st * NT + nt) * 64 + lane) * 2, kR),
                                qs[nt]);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int cc = col0 + 16 * nt;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = c * kChunk + out0 + r;
        if (t < sp.len && cc < in.dv)
          o[((sp.batch * plan.tokens + sp.first + t) * in.hv + h) * in.dv + cc] =
              bs_from_f32<T>(qs[nt][r]);
      }
    }
    __syncthreads();
  }
  if (state1) {
#pragma unroll
    for (int i = 0; i < TW; ++i) {
      const int t = TW * wave + i, d0 = 32 * (t >> 1) + 8 * g + 4 * (t & 1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int cc = col0 + 16 * nt;
          if (d0 + r < in.dk && cc < in.dv)
            state1[(((int64_t)n * in.hv + h) * in.dk + d0 + r) * in.dv + cc] = s[i][nt][r];
        }
    }
  }
}

template <typename T, int PI, int KS>
void launch_prepare(const bs_delta_in& in, const DeltaPlan& plan, const DeltaWork& w,
                    int backward, hipStream_t st) {
  const dim3 grid(plan.slots, in.hv);
  int vec = (uintptr_t)in.q % 16 == 0 && (uintptr_t)in.k % 16 == 0;
  for (int i = 0; i < 3; ++i) vec = vec && in.q_stride[i] % 8 == 0 && in.k_stride[i] % 8 == 0;
  if (backward) prepare_kernel<T, PI, KS, true><<<grid, 256, 0, st>>>(in, plan, w, vec);
  else prepare_kernel<T, PI, KS, false><<<grid, 256, 0, st>>>(in, plan, w, vec);
}

template <typename T, int PI, int KS>
void launch_chain(const bs_delta_in& in, const DeltaPlan& plan, const DeltaWork& w,
                  const DeltaSizes& z, const float* s0, float* s1, void* o, float* keep_s,
                  float* keep_u, hipStream_t st) {
  const unsigned rows = plan.seqs + (plan.offsets ? 1 : 0);
  // 16 columns a workgroup
  chain_kernel<T, PI, KS, 1><<<dim3(z.dvp / 16, in.hv, rows), 256, 0, st>>>(
      in, plan, w, s0, s1, (T*)o, keep_s, keep_u, z.dvp);
}

template <typename T, int PI>
void forward(const bs_delta_in& in, const DeltaPlan& plan, const DeltaWork& w,
             const DeltaSizes& z, const float* s0, float* s1, void* o, float* keep_s,
             float* keep_u, hipStream_t st) {
  if (z.ks == 2) launch_chain<T, PI, 2>(in, plan, w, z, s0, s1, o, keep_s, keep_u, st);
  else launch_chain<T, PI, 4>(in, plan, w, z, s0, s1, o, keep_s, keep_u, st);
}

}  // namespace

int delta_prepare(const bs_delta_in& in, const DeltaPlan& plan, const DeltaWork& w,
                  const DeltaSizes& z, int backward, hipStream_t st) {
  if (plan.slots == 0 || plan.seqs == 0) return BS_OK;
  if (in.dtype == BS_BF16) {
    if (z.ks == 2) launch_prepare<bs_bf16, 1, 2>(in, plan, w, backward, st);
    else launch_prepare<bs_bf16, 1, 4>(in, plan, w, backward, st);
  } else if (in.dtype == BS_F16) {
    if (z.ks == 2) launch_prepare<bs_f16, 2, 2>(in, plan, w, backward, st);
    else launch_prepare<bs_f16, 2, 4>(in, plan, w, backward, st);
  } else {
    if (z.ks == 2) launch_prepare<float, 3, 2>(in, plan, w, backward, st);
    else launch_prepare<float, 3, 4>(in, plan, w, backward, st);
  }
  BS_CHECK_LAUNCH();
  return BS_OK;
}

int delta_check_chunked(const bs_delta_in* in, int seqs, int tokens, const int32_t* offsets,
                        const char* who) {
  if (int rc = bs_delta_check(in, who)) return rc;
  BS_CHECK_ARG(seqs >= 0 && tokens >= 0, "%s: %d sequences, %d tokens", who, seqs, tokens);
  const int64_t slots = offsets ? (int64_t)tokens / kChunk + seqs
                                : (int64_t)seqs * ((tokens + kChunk - 1) / kChunk);
  BS_CHECK_ARG(slots <= 0x7FFFFFFF / kChunk && seqs < 65535 && in->hv <= 65535,
               "%s: %d sequences of %d tokens, %d heads exceed one launch", who, seqs, tokens,
               in->hv);
  return BS_OK;
}

extern "C" size_t bs_gated_delta_workspace_size(const bs_delta_in* in, int32_t seqs,
                                                int32_t tokens, int32_t packed) {
  static const int32_t dummy[1] = {0};
  const int32_t* off = packed ? dummy : nullptr;
  if (delta_check_chunked(in, seqs, tokens, off, "bs_gated_delta_workspace_size")) return 0;
  return (size_t)delta_sizes(*in, delta_plan(seqs, tokens, off).slots, 0).bytes;
}

extern "C" int bs_gated_delta_rule(const bs_delta_in* in, int32_t seqs, int32_t tokens,
                                   const int32_t* seq_offsets, const float* initial_state,
                                   float* final_state, void* o, float* kept_states, float* kept_u,
                                   void* workspace, size_t workspace_bytes, bs_stream_t stream) {
  if (int rc = delta_check_chunked(in, seqs, tokens, seq_offsets, "bs_gated_delta_rule"))
    return rc;
  if (seqs == 0 && !seq_offsets) return BS_OK;
  const DeltaPlan plan = delta_plan(seqs, tokens, seq_offsets);
  const DeltaSizes z = delta_sizes(*in, plan.slots, 0);
  BS_CHECK_ARG(tokens == 0 || (in->q && in->k && in->v && in->g && in->beta && o),
               "bs_gated_delta_rule: NULL pointer");
  BS_CHECK_ARG(z.bytes == 0 || (workspace && workspace_bytes >= (size_t)z.bytes),
               "bs_gated_delta_rule: workspace of %lld bytes needed, %lld given",
               (long long)z.bytes, (long long)(workspace ? workspace_bytes : 0));
  hipStream_t st = bs_stream(stream);
  const DeltaWork w = delta_work(workspace, z, 0);
  if (int rc = delta_prepare(*in, plan, w, z, 0, st)) return rc;
  if (in->dtype == BS_BF16)
    forward<bs_bf16, 1>(*in, plan, w, z, initial_state, final_state, o, kept_states, kept_u, st);
  else if (in->dtype == BS_F16)
    forward<bs_f16, 2>(*in, plan, w, z, initial_state, final_state, o, kept_states, kept_u, st);
  else
    forward<float, 3>(*in, plan, w, z, initial_state, final_state, o, kept_states, kept_u, st);
  BS_CHECK_LAUNCH();
  return BS_OK;
}
