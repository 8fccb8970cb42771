// Gradients of the chunked gated delta rule (its forward: delta_chunk.hip).
//
// With dO of a chunk, dS of the state after it, the masked A_ij = scale e_ij q_i.k_j and
// K~_j = exp(total - run_j) k_j, G_i = exp(run_i):
//
//   dU = A^T dO + K~ dS
//   dR = (1 + L)^-T dU                          dv_i = beta_i dR_i
//   dS0 = exp(total) dS + scale (G q)^T dO - (beta G k)^T dR
//
// is a recurrence from the last chunk to the first, the forward one's mirror (grad_chain_kernel).
// The rest of a chunk follows from dS, dR and what the forward pass kept (S0, U), for all chunks
// at once (grad_chunk_kernel):
//
//   dL = -dR U^T (strictly below the diagonal),  dA = dO U^T (on and below it)
//   dqk = scale e dA,  dkk = beta_i e dL
//   dq = scale G dO S0^T + dqk k
//   dk = K-part of dS: exp(total - run) U dS^T,  of R: -beta G dR S0^T,  + dqk^T q + (dkk + dkk^T) k
//   dbeta_i = dR_i.v_i - G_i k_i.(S0 dR_i) + sum_j dL_ij e_ij k_i.k_j
//   drun from every exponent;  dg_t = sum of drun_i over i >= t
//
// since dL = -(1 + L)^-T (dU R^T) (1 + L)^-T = -dR U^T needs no product with the inverse beyond dR.
// dg is a difference of large sums, so everything that reaches it is in 32 bits.
#include "delta_chunk.h"

namespace {

template <typename T, int PI, int KS>
__global__ __launch_bounds__(256) void grad_chain_kernel(bs_delta_in in, DeltaPlan plan,
                                                         DeltaWork w, const T* go,
                                                         const float* gstate, T* dv,
                                                         float* dstate, int dvp) {
  constexpr int DK = KS * 32, TW = KS / 2;
  constexpr int kS = KS * 128, kR = 2 * 128;       // words of a part
  __shared__ __attribute__((aligned(16))) uint2 ls[3 * kS];
  __shared__ __attribute__((aligned(16))) uint2 lo[PI * kR];
  __shared__ __attribute__((aligned(16))) uint2 lg[2][3 * kR];
  __shared__ __attribute__((aligned(16))) uint2 lu[3 * kR];
  __shared__ __attribute__((aligned(16))) uint2 lr[3 * kR];
  const int h = blockIdx.y, n = blockIdx.z, hk = h / (in.hv / in.hk);
  if (n >= plan.seqs) {
    zero_outside(plan, dv, in.hv, in.dv, h, blockIdx.x * 16, 16);
    return;
  }
  const DeltaSpan sp = delta_span(plan, n);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, g = lane >> 4;
  const int col = blockIdx.x * 16 + m;
  const int tok = delta_row(wave, m);
  const int out0 = 32 * (wave >> 1) + 8 * g + 4 * (wave & 1);
  const int blk = wave >> 1, own = (blk * 64 + lane) * 2 + (wave & 1);

  // dO of a chunk and scale G dO, into LDS
  auto stage = [&](int c) {
    const float* co = w.coef + ((int64_t)(sp.slot + c) * in.hv + h) * kCoef;
    const float4 grow = *(const float4*)(co + out0);
    const float* gr = (const float*)&grow;
    bs_f32x4 x, y;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = c * kChunk + out0 + r;
      x[r] = t < sp.len && col < in.dv
          ? bs_to_f32(go[((sp.batch * plan.tokens + sp.first + t) * in.hv + h) * in.dv + col])
          : 0.f;
      y[r] = in.scale * gr[r] * x[r];
    }
    delta_put<PI>(lo + own, kR, x);
    delta_put<3>(lg[c & 1] + own, kR, y);
  };

  bs_f32x4 s[TW];
#pragma unroll
  for (int i = 0; i < TW; ++i) {
    const int t = TW * wave + i, d0 = 32 * (t >> 1) + 8 * g + 4 * (t & 1);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      s[i][r] = gstate && d0 + r < in.dk && col < in.dv
          ? gstate[(((int64_t)n * in.hv + h) * in.dk + d0 + r) * in.dv + col] : 0.f;
    delta_put<3>(ls + ((t >> 1) * 64 + lane) * 2 + (t & 1), kS, s[i]);
  }
  if (sp.chunks) stage(sp.chunks - 1);
  __syncthreads();
  for (int c = sp.chunks - 1; c >= 0; --c) {
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
    bs_f32x4 du = zero4();
#pragma unroll
    for (int st = 0; st < KS; ++st)
      du = bs_mma<2>(delta_frags<PI>(w.kp + kb + tok * DK + 32 * st + 8 * g, kChunk * DK),
                     delta_lds<3>(ls + (st * 64 + lane) * 2, kS), du);
#pragma unroll
    for (int r = 0; r < 4; ++r) du[r] *= lf[r];
    const float* ap = w.att + sh * kChunk * kChunk + tok * kChunk + 8 * g;
#pragma unroll
    for (int st = 0; st < 2; ++st)
      if (st >= blk)
        du = bs_mma<2>(row_parts(ap + 32 * st), delta_lds<PI>(lo + (st * 64 + lane) * 2, kR), du);
    delta_put<3>(lu + own, kR, du);
    __syncthreads();
    bs_f32x4 dr = zero4();
    const float* ip = w.inv + sh * kChunk * kChunk + tok * kChunk + 8 * g;
#pragma unroll
    for (int st = 0; st < 2; ++st)
      if (st >= blk)
        dr = bs_mma<2>(row_parts(ip + 32 * st), delta_lds<3>(lu + (st * 64 + lane) * 2, kR), dr);
    bs_f32x4 x;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = c * kChunk + out0 + r;
      const float b = be[r] * dr[r];
      x[r] = -gr[r] * b;
      w.dr[(sh * kChunk + out0 + r) * dvp + col] = dr[r];
      if (t < sp.len && col < in.dv)
        dv[((sp.batch * plan.tokens + sp.first + t) * in.hv + h) * in.dv + col] =
            bs_from_f32<T>(b);
    }
    delta_put<3>(lr + own, kR, x);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TW; ++i) {
      const int t = TW * wave + i, d0 = 32 * (t >> 1) + 8 * g + 4 * (t & 1);
#pragma unroll
      for (int r = 0; r < 4; ++r) w.ds[(sh * DK + d0 + r) * dvp + col] = s[i][r];
      s[i] *= total;
      const int64_t at = kb + delta_row(t, m) * kChunk + 8 * g;
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        s[i] = bs_mma<2>(delta_frags<PI>(w.qt + at + 32 * st, DK * kChunk),
                         delta_lds<3>(lg[c & 1] + (st * 64 + lane) * 2, kR), s[i]);
        s[i] = bs_mma<2>(delta_frags<PI>(w.kt + at + 32 * st, DK * kChunk),
                         delta_lds<3>(lr + (st * 64 + lane) * 2, kR), s[i]);
      }
      delta_put<3>(ls + ((t >> 1) * 64 + lane) * 2 + (t & 1), kS, s[i]);
    }
    if (c) stage(c - 1);
    __syncthreads();
  }
  if (dstate) {
#pragma unroll
    for (int i = 0; i < TW; ++i) {
      const int t = TW * wave + i, d0 = 32 * (t >> 1) + 8 * g + 4 * (t & 1);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (d0 + r < in.dk && col < in.dv)
          dstate[(((int64_t)n * in.hv + h) * in.dk + d0 + r) * in.dv + col] = s[i][r];
    }
  }
}

__device__ __forceinline__ float sum16(float x) {     // over the 16 lanes of a group
  x += __shfl_xor(x, 1);
  x += __shfl_xor(x, 2);
  x += __shfl_xor(x, 4);
  return x + __shfl_xor(x, 8);
}
__device__ __forceinline__ float sum4(float x) {      // over the 4 lane groups
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Four tokens (4g..4g+3 of 16 at t0) of column d of a transposed copy, parts added up.
template <int PI>
__device__ __forceinline__ bs_f32x4 column4(const uint16_t* p, int64_t step) {
  bs_f32x4 r = zero4();
#pragma unroll
  for (int i = 0; i < PI; ++i) {
    const uint2 x = *(const uint2*)(p + i * step);
    r[0] += __uint_as_float(x.x << 16), r[1] += __uint_as_float(x.x & 0xFFFF0000u);
    r[2] += __uint_as_float(x.y << 16), r[3] += __uint_as_float(x.y & 0xFFFF0000u);
  }
  return r;
}

// One chunk (x) and key head (y): 4 waves, wave w has tokens 16w..16w+15; the value heads that
// share the key head are taken in turn, their dq and dk summed in registers.
template <typename T, int PI, int KS>
__global__ __launch_bounds__(256) void grad_chunk_kernel(bs_delta_in in, DeltaPlan plan,
                                                         DeltaWork w, const T* go,
                                                         const float* keep_s, const float* keep_u,
                                                         T* dq, T* dk, void* dg, void* dbeta,
                                                         int dvp, int vec) {
  constexpr int DK = KS * 32, CT = KS * 2;
  __shared__ float lp[kChunk][kChunk + 4];
  __shared__ float lm[kChunk][kChunk + 4];
  __shared__ float cols[4][kChunk], rows[kChunk], tot[4], bsum[kChunk];
  __shared__ double run[kChunk];
  const int slot = blockIdx.x, hk = blockIdx.y, group = in.hv / in.hk;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, g = lane >> 4;
  if (slot == plan.slots) {       // packed only: rows outside all sequences
    zero_outside(plan, dq, in.hk, in.dk, hk, 0, 128);
    zero_outside(plan, dk, in.hk, in.dk, hk, 0, 128);
    const int a = delta_offset(plan, 0), b = max(delta_offset(plan, plan.seqs), a);
    for (int t = tid; t < plan.tokens; t += 256)
      if (t < a || t >= b)
        for (int h = hk * group; h < (hk + 1) * group; ++h) {
          bs_store_any(dg, in.g_dtype, (int64_t)t * in.hv + h, 0.f);
          bs_store_any(dbeta, in.beta_dtype, (int64_t)t * in.hv + h, 0.f);
        }
    return;
  }
  const DeltaSpan sp = delta_span(plan, delta_owner(plan, slot));
  const int c = slot - sp.slot;
  if (c >= sp.chunks) return;
  const int64_t t0 = sp.first + (int64_t)c * kChunk;
  const int len = min(sp.len - c * kChunk, kChunk);
  const int64_t kb = ((int64_t)slot * in.hk + hk) * PI * kChunk * DK;
  const int row = 16 * wave + m, out0 = 16 * wave + 4 * g, blk = wave >> 1;
  const bool live = row < len;

  bs_f32x4 qk[4], kk[4], aq[CT], ak[CT];
#pragma unroll
  for (int j = 0; j < 4; ++j) qk[j] = kk[j] = zero4();
#pragma unroll
  for (int i = 0; i < CT; ++i) aq[i] = ak[i] = zero4();
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const bs_parts<PI> qf = delta_frags<PI>(w.qp + kb + row * DK + 32 * s + 8 * g, kChunk * DK);
    const bs_parts<PI> kf = delta_frags<PI>(w.kp + kb + row * DK + 32 * s + 8 * g, kChunk * DK);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j <= wave) {
        const bs_parts<PI> b =
            delta_frags<PI>(w.kp + kb + (16 * j + m) * DK + 32 * s + 8 * g, kChunk * DK);
        qk[j] = bs_mma<2>(qf, b, qk[j]);
        kk[j] = bs_mma<2>(kf, b, kk[j]);
      }
  }
  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    const int64_t sh = (int64_t)slot * in.hv + h;
    const float* co = w.coef + sh * kCoef;
    const float* us = keep_u + sh * kChunk * dvp;
    const float* dr = w.dr + sh * kChunk * dvp;
    const float* s0 = keep_s + sh * DK * dvp;
    const float* ds = w.ds + sh * DK * dvp;
    const T* gp = go + ((sp.batch * plan.tokens + t0 + (live ? row : 0)) * in.hv + h) * in.dv;
    const T* vp = (const T*)in.v + bs_delta_at(in.v_stride, sp.batch, t0 + (live ? row : 0), h);
    if (tid < kChunk) run[tid] = ((const double*)(co + 4 * kChunk))[tid];
    bs_f32x4 xq[CT], xs[CT], xr[CT], da[4], dl[4];
    float dot_s = 0.f, dot_v = 0.f;
#pragma unroll
    for (int i = 0; i < CT; ++i) xq[i] = xs[i] = xr[i] = zero4();
#pragma unroll
    for (int j = 0; j < 4; ++j) da[j] = dl[j] = zero4();
    for (int e = 0; e < dvp; e += 32) {
      const int d = e + 8 * g, left = live ? in.dv - d : 0;
      const bs_parts<PI> of = load_parts<PI>(gp + d, left, vec);
      const float4 r0 = *(const float4*)(dr + row * dvp + d),
                   r1 = *(const float4*)(dr + row * dvp + d + 4);
      const bs_parts<3> rf = row_parts(r0, r1);
      const bs_parts<3> uf = row_parts(us + row * dvp + d);
      const float rr[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) dot_v = fmaf(rr[j], bs_to_f32(vp[d + j]), dot_v);
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        const int64_t at = (int64_t)(16 * i + m) * dvp + d;
        const float4 a0 = *(const float4*)(s0 + at), a1 = *(const float4*)(s0 + at + 4);
        const float4 b0 = *(const float4*)(ds + at), b1 = *(const float4*)(ds + at + 4);
        if ((i & 3) == wave) {
          float x = a0.x * b0.x;
          x = fmaf(a0.y, b0.y, x), x = fmaf(a0.z, b0.z, x), x = fmaf(a0.w, b0.w, x);
          x = fmaf(a1.x, b1.x, x), x = fmaf(a1.y, b1.y, x), x = fmaf(a1.z, b1.z, x);
          dot_s += fmaf(a1.w, b1.w, x);
        }
        const bs_parts<3> sf = row_parts(a0, a1), df = row_parts(b0, b1);
        xq[i] = bs_mma<2>(of, sf, xq[i]);
        xr[i] = bs_mma<2>(rf, sf, xr[i]);
        xs[i] = bs_mma<2>(uf, df, xs[i]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j <= wave) {
          const bs_parts<3> b = row_parts(us + (16 * j + m) * dvp + d);
          da[j] = bs_mma<2>(of, b, da[j]);
          dl[j] = bs_mma<2>(rf, b, dl[j]);
        }
    }
    const float4 grow = *(const float4*)(co + out0), lft = *(const float4*)(co + kChunk + out0),
                 beta = *(const float4*)(co + 2 * kChunk + out0);
    const float* gr = (const float*)&grow;
    const float* lf = (const float*)&lft;
    const float* be = (const float*)&beta;
    // terms of the state products, by rows out0 + r
    float drun[4] = {0.f, 0.f, 0.f, 0.f}, db[4] = {0.f, 0.f, 0.f, 0.f}, dtot = 0.f;
#pragma unroll
    for (int i = 0; i < CT; ++i) {
      const int64_t at = kb + (int64_t)(16 * i + m) * kChunk + out0;
      const bs_f32x4 k4 = column4<PI>(w.kt + at, DK * kChunk);
      const bs_f32x4 q4 = column4<PI>(w.qt + at, DK * kChunk);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float a = in.scale * gr[r] * xq[i][r], b = gr[r] * xr[i][r], s = lf[r] * xs[i][r];
        aq[i][r] += a;
        ak[i][r] += s - be[r] * b;
        drun[r] += q4[r] * a - k4[r] * (be[r] * b + s);
        db[r] -= k4[r] * b;
        dtot = fmaf(k4[r], s, dtot);
      }
    }
    dtot += co[3 * kChunk] * dot_s;
    __syncthreads();                // run
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float cs = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = out0 + r, jj = 16 * j + m;
        float p = 0.f, q = 0.f;
        if (j <= wave && jj <= i) {
          const float e = expf((float)(run[i] - run[jj]));
          p = in.scale * e * da[j][r];
          const float x = jj < i ? -dl[j][r] * e : 0.f;
          q = be[r] * x;
          const float both = p * qk[j][r] + q * kk[j][r];
          db[r] = fmaf(x, kk[j][r], db[r]);
          drun[r] += both;
          cs += both;
        }
        lp[i][jj] = p, lm[i][jj] = q;
      }
      cs = sum4(cs);
      if (g == 0) cols[wave][16 * j + m] = cs;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      drun[r] = sum16(drun[r]);
      db[r] = sum16(db[r]);
      if (m == 0) rows[out0 + r] = drun[r], bsum[out0 + r] = db[r];
    }
    dtot = sum4(sum16(dtot));
    if (lane == 0) tot[wave] = dtot;
    dot_v = sum4(dot_v);
    __syncthreads();
    if (g == 0 && live)
      bs_store_any(dbeta, in.beta_dtype, (sp.batch * plan.tokens + t0 + row) * in.hv + h,
                   bsum[row] + dot_v);
    if (wave == 0) {
      double x = (double)rows[lane] - cols[0][lane] - cols[1][lane] - cols[2][lane] -
                 cols[3][lane];
      if (lane == 63) x += (double)tot[0] + tot[1] + tot[2] + tot[3];
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double y = __shfl_down(x, d);
        if (lane + d < 64) x += y;
      }
      if (lane < len)
        bs_store_any(dg, in.g_dtype, (sp.batch * plan.tokens + t0 + lane) * in.hv + h, (float)x);
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int j0 = 32 * st + 8 * g;
      float sym[8], pt[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        sym[x] = lm[row][j0 + x] + lm[j0 + x][row];
        pt[x] = lp[j0 + x][row];
      }
      const bs_parts<3> pf = row_parts(&lp[row][j0]);
      const bs_parts<3> sf = bs_split8<3>(sym), tf = bs_split8<3>(pt);
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        const int64_t at = kb + (int64_t)(16 * i + m) * kChunk + j0;
        const bs_parts<PI> kf = delta_frags<PI>(w.kt + at, DK * kChunk);
        if (st <= blk) aq[i] = bs_mma<2>(pf, kf, aq[i]);
        ak[i] = bs_mma<2>(sf, kf, ak[i]);
        if (st >= blk)
          ak[i] = bs_mma<2>(tf, delta_frags<PI>(w.qt + at, DK * kChunk), ak[i]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < CT; ++i) {
    const int d = 16 * i + m;
    if (d >= in.dk) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (out0 + r < len) {
        const int64_t at = ((sp.batch * plan.tokens + t0 + out0 + r) * in.hk + hk) * in.dk + d;
        dq[at] = bs_from_f32<T>(aq[i][r]);
        dk[at] = bs_from_f32<T>(ak[i][r]);
      }
  }
}

struct GradOut { void *dq, *dk, *dv, *dg, *dbeta; float* dstate; };

template <typename T, int PI, int KS>
void launch_grad(const bs_delta_in& in, const DeltaPlan& plan, const DeltaWork& w,
                 const DeltaSizes& z, const void* go, const float* gstate, const float* keep_s,
                 const float* keep_u, const GradOut& o, hipStream_t st) {
  const unsigned extra = plan.offsets ? 1 : 0;
  grad_chain_kernel<T, PI, KS><<<dim3(z.dvp / 16, in.hv, plan.seqs + extra), 256, 0, st>>>(
      in, plan, w, (const T*)go, gstate, (T*)o.dv, o.dstate, z.dvp);
  if (plan.slots + extra == 0) return;
  const int vec = in.dv % 8 == 0 && (uintptr_t)go % 16 == 0;
  grad_chunk_kernel<T, PI, KS><<<dim3(plan.slots + extra, in.hk), 256, 0, st>>>(
      in, plan, w, (const T*)go, keep_s, keep_u, (T*)o.dq, (T*)o.dk, o.dg, o.dbeta, z.dvp, vec);
}

template <typename T, int PI>
void backward(const bs_delta_in& in, const DeltaPlan& plan, const DeltaWork& w,
              const DeltaSizes& z, const void* go, const float* gstate, const float* keep_s,
              const float* keep_u, const GradOut& o, hipStream_t st) {
  if (z.ks == 2) launch_grad<T, PI, 2>(in, plan, w, z, go, gstate, keep_s, keep_u, o, st);
  else launch_grad<T, PI, 4>(in, plan, w, z, go, gstate, keep_s, keep_u, o, st);
}

}  // namespace

extern "C" size_t bs_gated_delta_grad_workspace_size(const bs_delta_in* in, int32_t seqs,
                                                     int32_t tokens, int32_t packed) {
  static const int32_t dummy[1] = {0};
  const int32_t* off = packed ? dummy : nullptr;
  if (delta_check_chunked(in, seqs, tokens, off, "bs_gated_delta_grad_workspace_size")) return 0;
  return (size_t)delta_sizes(*in, delta_plan(seqs, tokens, off).slots, 1).bytes;
}

extern "C" int bs_gated_delta_rule_grad(const bs_delta_in* in, int32_t seqs, int32_t tokens,
                                        const int32_t* seq_offsets, const void* grad_o,
                                        const float* grad_state, const float* kept_states,
                                        const float* kept_u, void* dq, void* dk, void* dv,
                                        void* dg, void* dbeta, float* dstate, void* workspace,
                                        size_t workspace_bytes, bs_stream_t stream) {
  if (int rc = delta_check_chunked(in, seqs, tokens, seq_offsets, "bs_gated_delta_rule_grad"))
    return rc;
  if (seqs == 0 && !seq_offsets) return BS_OK;
  const DeltaPlan plan = delta_plan(seqs, tokens, seq_offsets);
  const DeltaSizes z = delta_sizes(*in, plan.slots, 1);
  BS_CHECK_ARG(tokens == 0 || (in->q && in->k && in->v && in->g && in->beta && grad_o &&
                               kept_states && kept_u && dq && dk && dv && dg && dbeta),
               "bs_gated_delta_rule_grad: NULL pointer");
  BS_CHECK_ARG(z.bytes == 0 || (workspace && workspace_bytes >= (size_t)z.bytes),
               "bs_gated_delta_rule_grad: workspace of %lld bytes needed, %lld given",
               (long long)z.bytes, (long long)(workspace ? workspace_bytes : 0));
  hipStream_t st = bs_stream(stream);
  const DeltaWork w = delta_work(workspace, z, 1);
  if (int rc = delta_prepare(*in, plan, w, z, 1, st)) return rc;
  const GradOut o = {dq, dk, dv, dg, dbeta, dstate};
  if (in->dtype == BS_BF16)
    backward<bs_bf16, 1>(*in, plan, w, z, grad_o, grad_state, kept_states, kept_u, o, st);
  else if (in->dtype == BS_F16)
    backward<bs_f16, 2>(*in, plan, w, z, grad_o, grad_state, kept_states, kept_u, o, st);
  else
    backward<float, 3>(*in, plan, w, z, grad_o, grad_state, kept_states, kept_u, o, st);
  BS_CHECK_LAUNCH();
  return BS_OK;
}
