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
//
// 4 x 2,048 tokens x 16 heads of 128 x 128 in bfloat16, the whole step 625 us.  Its kernels under
// the tracer, 643 in all: forward prepare 55 and chain 140 (it keeps the states), prepare again 58
// (all of it kept from the forward pass would hold 146 MB more a layer), grad_chain_kernel 158,
// grad_chunk_kernel 232.  The last fills its 256 registers with products in three parts and their
// cutting (16 bytes a lane spill): beside 613 for the whole step then, 687 with U's parts cut by
// every wave that takes them, 652 with the fragments' addresses kept over the heads (184 bytes
// spilled, 100 MB written and read).  Two waves a SIMD to issue from keep the matrix cores busy in
// a fifth of the cycles, in both kernels.
// Keys past 64 values in fp16 and in 32 bits do not fit the registers: grad_chain_kernel spills 180
// bytes a lane in fp16 (with 32 columns) and 248 or 344 in 32 bits, grad_chunk_kernel 80 and 220;
// the gradients of the same layer take 591 and 974 us there, 451 in bfloat16.
#include "delta_chunk.h"

namespace {

// Chunks of one sequence, value head and slice of 16 NT value columns, last to first, by two sets
// of 4 waves as in the forward pass: the first has the recurrence, the second forms dR again for the
// gradient of v and the chunk's gradients, and keeps the gradient of the state.
template <typename T, int PI, int KS, int NT>
__global__ __launch_bounds__(512, 2) void grad_chain_kernel(
    bs_delta_in in, DeltaPlan plan, DeltaWork w, const T* go, const float* gstate, T* dv,
    float* dstate, int dvp, int units, int vec) {
  constexpr int DK = KS * 32, TW = KS / 2;
  constexpr int kS = KS * NT * 128, kR = 2 * NT * 128;       // words of a part
  __shared__ __attribute__((aligned(16))) uint2 ls[3 * kS];        // dS
  __shared__ __attribute__((aligned(16))) uint2 lo[PI * kR];       // dO
  __shared__ __attribute__((aligned(16))) uint2 lg[2][3 * kR];     // scale G dO
  __shared__ __attribute__((aligned(16))) uint2 lu[3 * kR];        // dU
  __shared__ __attribute__((aligned(16))) uint2 lr[3 * kR];        // -beta G dR
  const DeltaPlace at = delta_place(units, dvp / (16 * NT));
  if (at.unit >= units) return;
  const int h = __builtin_amdgcn_readfirstlane(at.unit % in.hv);
  const int n = __builtin_amdgcn_readfirstlane(at.unit / in.hv), hk = h / (in.hv / in.hk);
  if (n >= plan.seqs) {
    zero_outside(plan, dv, in.hv, in.dv, h, at.slice * 16 * NT, 16 * NT);
    return;
  }
  const DeltaSpan sp = delta_span(plan, n);
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int role = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3), blk = wave >> 1;
  const int tok = delta_row(wave, m);
  const int64_t keys = (int64_t)in.hk * PI * kChunk * DK;
  const int64_t kb = ((int64_t)sp.slot * in.hk + hk) * PI * kChunk * DK;
  const int64_t hb = (int64_t)sp.slot * in.hv + h;
  const float* cp = w.coef + hb * kCoef;
  auto load_square = [&](const uint16_t* a, int c, bs_parts<3>* f) {
#pragma unroll
    for (int st = 0; st < 2; ++st)
      f[st] = delta_frags<3>(a + (hb + (int64_t)c * in.hv) * 3 * kSquare +
                                 delta_upper(wave, max(st, blk)) * kFrag + lane * 8, kSquare);
  };

  if (role == 0) {
    const int col = at.slice * 16 * NT + m;
    const int out0 = 32 * blk + 8 * g + 4 * (wave & 1);
    const int own = (blk * NT * 64 + lane) * 2 + (wave & 1);
    bs_f32x4 s[TW][NT];
    int d0[TW], sown[TW];
#pragma unroll
    for (int i = 0; i < TW; ++i) {
      const int t = TW * wave + i;
      d0[i] = 32 * (t >> 1) + 8 * g + 4 * (t & 1);
      sown[i] = ((t >> 1) * NT * 64 + lane) * 2 + (t & 1);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[i][j][r] = gstate && d0[i] + r < in.dk && col + 16 * j < in.dv
              ? gstate[(((int64_t)n * in.hv + h) * in.dk + d0[i] + r) * in.dv + col + 16 * j]
              : 0.f;
        delta_put<3>(ls + sown[i] + 128 * j, kS, s[i][j]);
      }
    }
    const uint16_t* kp = w.kp + kb + wave * KS * kFrag + lane * 8;
    const int64_t tb = kb + wave * TW * 2 * kFrag + lane * 8;
    const DeltaRows<T, NT> rows(go + ((sp.batch * plan.tokens + sp.first) * in.hv + h) * in.dv,
                                (int64_t)in.hv * in.dv, out0, col, in.dv);
    bs_parts<PI> kf[KS], ktf[TW][2], qtf[TW][2];
    bs_parts<3> tf[2], af[2];
    struct Values {
      typename DeltaRows<T, NT>::Raw v[NT][4];
      float total;
      float4 coef[3];
    } values[2];
    float all = 0.f;
    float4 now[3];
    auto load_keys = [&](int c) {
#pragma unroll
      for (int st = 0; st < KS; ++st)
        kf[st] = delta_frags<PI>(kp + c * keys + st * kFrag, kChunk * DK);
    };
    auto load_grad = [&](int c, Values& x) {
      const float* co = cp + (int64_t)c * in.hv * kCoef;
      rows.load(c, sp.len, x.v);
      x.coef[0] = *(const float4*)(co + kGrow * kChunk + out0);
      x.coef[1] = *(const float4*)(co + kLeft * kChunk + out0);
      x.coef[2] = *(const float4*)(co + kBeta * kChunk + out0);
      x.total = co[kTotal * kChunk];
    };
    auto load_columns = [&](int c) {
#pragma unroll
      for (int i = 0; i < 2 * TW; ++i) {
        ktf[i >> 1][i & 1] = delta_frags<PI>(w.kt + tb + c * keys + i * kFrag, kChunk * DK);
        qtf[i >> 1][i & 1] = delta_frags<PI>(w.qt + tb + c * keys + i * kFrag, kChunk * DK);
      }
    };
    // dO of the chunk that was loaded, and scale G dO, into LDS; its factors are the next ones
    auto stage = [&](int buf, const Values& v) {
      const float* gw = (const float*)&v.coef[0];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        bs_f32x4 x, y;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[r] = rows.value(v.v[j][r]);
          y[r] = in.scale * gw[r] * x[r];
        }
        delta_put<PI>(lo + own + 128 * j, kR, x);
        delta_put<3>(lg[buf] + own + 128 * j, kR, y);
      }
      now[0] = v.coef[0], now[1] = v.coef[1], now[2] = v.coef[2], all = v.total;
    };
    if (const int c = sp.chunks - 1; c >= 0) {
      load_grad(c, values[1]);
      load_grad(max(c - 1, 0), values[0]);
      load_keys(c);
      load_square(w.att, c, af);
      load_square(w.inv, c, tf);
      load_columns(c);
      stage(c & 1, values[1]);
      load_grad(max(c - 2, 0), values[1]);
    }
    wait_loads();
    __syncthreads();
    // `v` holds chunk c - 1, and then c - 3
    auto step = [&](int c, Values& v) {
      const int next = max(c - 1, 0);
      bs_f32x4 du[NT], dr[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) du[j] = dr[j] = zero4();
#pragma unroll
      for (int st = 0; st < KS; ++st)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          du[j] = bs_mma<2>(kf[st], delta_lds<3>(ls + ((st * NT + j) * 64 + lane) * 2, kS), du[j]);
      const float* lf = (const float*)&now[1];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) du[j][r] *= lf[r];
#pragma unroll
      for (int st = 0; st < 2; ++st)
        if (st >= blk) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
            du[j] = bs_mma<2>(af[st], delta_lds<PI>(lo + ((st * NT + j) * 64 + lane) * 2, kR),
                              du[j]);
        }
#pragma unroll
      for (int j = 0; j < NT; ++j) delta_put<3>(lu + own + 128 * j, kR, du[j]);
      __builtin_amdgcn_sched_barrier(0);
      load_keys(next);
      load_square(w.att, next, af);
      __syncthreads();                     // dU; dO's last readers are through
#pragma unroll
      for (int st = 0; st < 2; ++st)
        if (st >= blk) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
            dr[j] = bs_mma<2>(tf[st], delta_lds<3>(lu + ((st * NT + j) * 64 + lane) * 2, kR),
                              dr[j]);
        }
      const float* gw = (const float*)&now[0];
      const float* be = (const float*)&now[2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) dr[j][r] *= -gw[r] * be[r];
        delta_put<3>(lr + own + 128 * j, kR, dr[j]);
      }
      __builtin_amdgcn_sched_barrier(0);
      load_square(w.inv, next, tf);
      __syncthreads();                     // dR; the state's last readers are through
#pragma unroll
      for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) s[i][j] *= all;
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int at2 = ((st * NT + j) * 64 + lane) * 2;
          const bs_parts<3> a = delta_lds<3>(lg[c & 1] + at2, kR);
          const bs_parts<3> b = delta_lds<3>(lr + at2, kR);
#pragma unroll
          for (int i = 0; i < TW; ++i) {
            s[i][j] = bs_mma<2>(qtf[i][st], a, s[i][j]);
            s[i][j] = bs_mma<2>(ktf[i][st], b, s[i][j]);
          }
        }
#pragma unroll
      for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) delta_put<3>(ls + sown[i] + 128 * j, kS, s[i][j]);
      stage((c - 1) & 1, v);               // past chunk 0: what no one reads
      __builtin_amdgcn_sched_barrier(0);
      load_columns(next);
      load_grad(max(c - 3, 0), v);
      __syncthreads();                     // the state
    };
    for (int c = sp.chunks - 1; c > 0; c -= 2) {
      step(c, values[0]);
      step(c - 1, values[1]);
    }
    if (sp.chunks & 1) step(0, values[0]);
    if (dstate) {
#pragma unroll
      for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (d0[i] + r < in.dk && col + 16 * j < in.dv)
              dstate[(((int64_t)n * in.hv + h) * in.dk + d0[i] + r) * in.dv + col + 16 * j] =
                  s[i][j][r];
    }
  } else {
    const int ocol = at.slice * 16 * NT + 4 * g;
    struct Operands { bs_parts<3> t[2]; float beta; } operands[2];
    auto load = [&](int c, Operands& x) {
      load_square(w.inv, c, x.t);
      x.beta = cp[(int64_t)c * in.hv * kCoef + kBeta * kChunk + tok];
    };
    T* op = dv + ((sp.batch * plan.tokens + sp.first + tok) * in.hv + h) * in.dv + ocol;
    if (const int c = sp.chunks - 1; c >= 0) {
      load(c, operands[0]);
      load(max(c - 1, 0), operands[1]);
    }
    wait_loads();
    __syncthreads();
    auto step = [&](int c, Operands& now) {
      const int64_t sh = hb + (int64_t)c * in.hv;
#pragma unroll
      for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int t = TW * wave + i;
          const bs_f32x4 x = delta_turn(
              delta_lds<3>(ls + (((t >> 1) * NT + j) * 64 + lane) * 2, kS), t & 1, lane);
          *(bs_f32x4*)(w.ds + sh * DK * dvp + delta_kept(t, at.slice * NT + j, lane, dvp)) = x;
        }
      __syncthreads();                     // dU
      bs_f32x4 dr[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) dr[j] = zero4();
#pragma unroll
      for (int st = 0; st < 2; ++st)
        if (st >= blk) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
            dr[j] = bs_mma<2>(delta_lds<3>(lu + ((st * NT + j) * 64 + lane) * 2, kR), now.t[st],
                              dr[j]);
        }
      const float beta = now.beta;
      load(max(c - 2, 0), now);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        *(bs_f32x4*)(w.dr + sh * kChunk * dvp +
                     delta_kept(wave, at.slice * NT + j, lane, dvp)) = dr[j];
        if (c * kChunk + tok < sp.len) {
          T* p = op + (int64_t)c * kChunk * in.hv * in.dv + 16 * j;
          const int oc = ocol + 16 * j;
          bs_f32x4 y = beta * dr[j];
          // rounded to 32 bits in every form: in some of them the compiler folds the product into the
          // conversion to fp16, which then rounds once, and a row's last bit would go by how many
          // heads and sequences run beside it
#pragma unroll
          for (int r = 0; r < 4; ++r) asm volatile("" : "+v"(y[r]));
          if (vec) {
            if (oc < in.dv) bs_store4(p, y);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (oc + r < in.dv) p[r] = bs_from_f32<T>(y[r]);
          }
        }
      }
      __syncthreads();                     // dR
      __syncthreads();                     // the state
    };
    for (int c = sp.chunks - 1; c > 0; c -= 2) {
      step(c, operands[0]);
      step(c - 1, operands[1]);
    }
    if (sp.chunks & 1) step(0, operands[0]);
  }
}

__device__ __forceinline__ float sum4(float x) {      // over the 4 lane groups
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Value e (0..7) of a fragment, its parts added up.
template <int PI>
__device__ __forceinline__ float frag_value(const bs_parts<PI>& f, int e) {
  float x = 0.f;
#pragma unroll
  for (int p = PI - 1; p >= 0; --p)
    x += __uint_as_float((uint32_t)__builtin_bit_cast(bs_u16x8, f.p[p])[e] << 16);
  return x;
}

// One chunk (x) and key head (y); the value heads that share the key head are taken in turn,
// their dq and dk summed in registers.  8 waves: wave (t, half) has the tokens of tile t and half
// of the dk rows, everything transposed (rows dk, columns tokens), so that factors of a token are
// one value a lane and a token's dk lie side by side.  The exponents' gradients need no sums of
// their own: run_i multiplies q_i in dq's terms and k_i in the terms of R and L's rows, and
// divides k_i in the others, so
//   drun_i = q_i.dq_i + k_i.dkA_i - k_i.dkB_i,   dk = dkA + dkB.
template <typename T, int PI, int KS>
__global__ __launch_bounds__(512) void grad_chunk_kernel(bs_delta_in in, DeltaPlan plan,
                                                         DeltaWork w, const T* go,
                                                         const float* keep_s, const float* keep_u,
                                                         T* dq, T* dk, void* dg, void* dbeta,
                                                         int dvp, int vec) {
  constexpr int DK = KS * 32, CT = KS, HS = KS / 2;     // tiles and steps of dk of a wave
  __shared__ __attribute__((aligned(16))) float lp[kChunk][kChunk + 4];
  __shared__ __attribute__((aligned(16))) float lm[kChunk][kChunk + 4];
  __shared__ float rows[2][kChunk], betas[2][kChunk], tot[8];
  __shared__ __attribute__((aligned(16))) uint4 lst[2][2][2 * KS][3][64];    // states' parts
  __shared__ __attribute__((aligned(16))) uint4 lut[2][4][3][64];            // U's
  const int slot = blockIdx.x, hk = blockIdx.y, group = in.hv / in.hk;
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), t = wave & 3, half = wave >> 2;
  if (slot == plan.slots) {       // packed only: rows outside all sequences
    zero_outside(plan, dq, in.hk, in.dk, hk, 0, 128);
    zero_outside(plan, dk, in.hk, in.dk, hk, 0, 128);
    const int a = delta_offset(plan, 0), b = max(delta_offset(plan, plan.seqs), a);
    for (int r = tid; r < plan.tokens; r += 512)
      if (r < a || r >= b)
        for (int h = hk * group; h < (hk + 1) * group; ++h) {
          bs_store_any(dg, in.g_dtype, (int64_t)r * in.hv + h, 0.f);
          bs_store_any(dbeta, in.beta_dtype, (int64_t)r * in.hv + h, 0.f);
        }
    return;
  }
  const DeltaSpan sp = delta_span(plan, delta_owner(plan, slot));
  const int c = slot - sp.slot;
  if (c < 0 || c >= sp.chunks) return;
  const int64_t t0 = sp.first + (int64_t)c * kChunk;
  const int len = min(sp.len - c * kChunk, kChunk);
  const int64_t kb = ((int64_t)slot * in.hk + hk) * PI * kChunk * DK;
  const int blk = t >> 1, tok = delta_row(t, m);
  const bool live = tok < len;
  // tiles of columns of the masked products of this wave: j0, and j0 + 1 in the second block
  const int j0 = blk ? 2 * half : half, nj = blk ? 2 : 1;

  bs_f32x4 qk[2], kk[2], aq[CT], ak[CT];
#pragma unroll
  for (int j = 0; j < 2; ++j) qk[j] = kk[j] = zero4();
#pragma unroll
  for (int i = 0; i < CT; ++i) aq[i] = ak[i] = zero4();
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const uint16_t* p = w.kp + kb + lane * 8 + s * kFrag;
    const bs_parts<PI> qf = delta_frags<PI>(w.qp + kb + lane * 8 + (t * KS + s) * kFrag, kChunk * DK);
    const bs_parts<PI> kf = delta_frags<PI>(p + t * KS * kFrag, kChunk * DK);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (j < nj) {
        const bs_parts<PI> a = delta_frags<PI>(p + (j0 + j) * KS * kFrag, kChunk * DK);
        qk[j] = bs_mma<2>(a, qf, qk[j]);
        kk[j] = bs_mma<2>(a, kf, kk[j]);
      }
  }
  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    // the key head's fragments are addressed anew for each head: kept, the addresses spill
    int64_t kbh = kb;
    asm volatile("" : "+s"(kbh));
    const int64_t sh = (int64_t)slot * in.hv + h;
    const float* co = w.coef + sh * kCoef;
    const double* run = (const double*)(co + kRun * kChunk);
    const float* us = keep_u + sh * kChunk * dvp;
    const float* dr = w.dr + sh * kChunk * dvp;
    const float* s0 = keep_s + sh * DK * dvp;
    const float* ds = w.ds + sh * DK * dvp;
    const DeltaRow<T> gr(go + ((sp.batch * plan.tokens + t0) * in.hv + h) * in.dv,
                         (int64_t)in.hv * in.dv, tok, len, in.dv, vec & 1);
    const DeltaRow<T> vr((const T*)in.v + bs_delta_at(in.v_stride, sp.batch, t0, h),
                         in.v_stride[1], tok, len, in.dv, vec & 2);
    bs_f32x4 xq[CT], xs[CT], xr[CT], da[2], dl[2];
    float dot_s = 0.f, dot_v = 0.f;
#pragma unroll
    for (int i = 0; i < CT; ++i) xq[i] = xs[i] = xr[i] = zero4();
#pragma unroll
    for (int j = 0; j < 2; ++j) da[j] = dl[j] = zero4();
    // Steps of 32 value columns.  The parts of the states and of U are cut once for all waves: wave
    // w loads tile w of both states, the first four tile w of U, a step ahead, and leaves them in
    // LDS, two steps deep.
    float4 sw[4], rw[2], uw[2];
    uint4 gw[sizeof(T) / 2], vw[sizeof(T) / 2];
    auto load_step = [&](int e) {
      gr.raw(e + 8 * g, gw);
      vr.raw(e + 8 * g, vw);
      const float* p = delta_kept_frag(s0, min(wave, 2 * KS - 1), e >> 5, lane, dvp);
      const float* q = delta_kept_frag(ds, min(wave, 2 * KS - 1), e >> 5, lane, dvp);
      sw[0] = *(const float4*)p, sw[1] = *(const float4*)(p + 256);
      sw[2] = *(const float4*)q, sw[3] = *(const float4*)(q + 256);
      p = delta_kept_frag(dr, t, e >> 5, lane, dvp);
      rw[0] = *(const float4*)p, rw[1] = *(const float4*)(p + 256);
      p = delta_kept_frag(us, t, e >> 5, lane, dvp);
      uw[0] = *(const float4*)p, uw[1] = *(const float4*)(p + 256);
    };
    auto step = [&](int e, auto more) {
      const int buf = (e >> 5) & 1;
      if (wave < 2 * KS) {
        const bs_parts<3> a = row_parts(sw[0], sw[1]), b = row_parts(sw[2], sw[3]);
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          *(bs_bf16x8*)&lst[buf][0][wave][p][lane] = a.p[p];
          *(bs_bf16x8*)&lst[buf][1][wave][p][lane] = b.p[p];
        }
        const float* x = (const float*)sw;
#pragma unroll
        for (int i = 0; i < 8; ++i) dot_s = fmaf(x[i], x[8 + i], dot_s);
      }
      const bs_parts<PI> of = gr.template parts<PI>(gw);
      const bs_parts<3> rf = row_parts(rw[0], rw[1]);
      if (half == 0) {
        const bs_parts<3> u = row_parts(uw[0], uw[1]);
#pragma unroll
        for (int p = 0; p < 3; ++p) *(bs_bf16x8*)&lut[buf][t][p][lane] = u.p[p];
      }
      if (buf == half) {
        const float* x = (const float*)rw;
        float f[8];
        vr.values(vw, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) dot_v = fmaf(x[j], f[j], dot_v);
      }
      if (more.value) load_step(e + 32);
      __syncthreads();                // the parts of this step
      bs_parts<3> uf;
#pragma unroll
      for (int p = 0; p < 3; ++p) uf.p[p] = *(const bs_bf16x8*)&lut[buf][t][p][lane];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (j < nj) {
          bs_parts<3> a;
#pragma unroll
          for (int p = 0; p < 3; ++p) a.p[p] = *(const bs_bf16x8*)&lut[buf][j0 + j][p][lane];
          da[j] = bs_mma<2>(a, of, da[j]);
          dl[j] = bs_mma<2>(a, rf, dl[j]);
        }
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        bs_parts<3> sf, df;
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          sf.p[p] = *(const bs_bf16x8*)&lst[buf][0][half * CT + i][p][lane];
          df.p[p] = *(const bs_bf16x8*)&lst[buf][1][half * CT + i][p][lane];
        }
        xq[i] = bs_mma<2>(sf, of, xq[i]);
        xr[i] = bs_mma<2>(sf, rf, xr[i]);
        xs[i] = bs_mma<2>(df, uf, xs[i]);
      }
    };
    load_step(0);
    for (int e = 0; e + 32 < dvp; e += 32) step(e, std::true_type());
    step(dvp - 32, std::false_type());
    // the masked products of this wave, to LDS by rows
    const float grow = co[kGrow * kChunk + tok], beta = co[kBeta * kChunk + tok];
    const double run_i = run[tok];
    float db = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (j < nj) {
        const int jj = 32 * ((j0 + j) >> 1) + 8 * g + 4 * ((j0 + j) & 1);
        float p[4], q[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = jj + r <= tok ? expf((float)(run_i - run[jj + r])) : 0.f;
          const float x = jj + r < tok ? -dl[j][r] * e : 0.f;
          p[r] = in.scale * e * da[j][r];
          q[r] = beta * x;
          db = fmaf(x, kk[j][r], db);
        }
        *(float4*)&lp[tok][jj] = make_float4(p[0], p[1], p[2], p[3]);
        *(float4*)&lm[tok][jj] = make_float4(q[0], q[1], q[2], q[3]);
      }
    // factors of the state products, and what they give beta and the chunk's total
    const float fq = in.scale * grow, fr = -beta * grow, fs = co[kLeft * kChunk + tok];
    float kx = 0.f, kt = 0.f;
    bs_parts<PI> kf[HS], qf[HS];
#pragma unroll
    for (int s = 0; s < HS; ++s) {
      const int64_t at = kbh + lane * 8 + (t * KS + half * HS + s) * kFrag;
      kf[s] = delta_frags<PI>(w.kp + at, kChunk * DK);
      qf[s] = delta_frags<PI>(w.qp + at, kChunk * DK);
    }
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float k = frag_value(kf[i >> 1], 4 * (i & 1) + r);
        kx = fmaf(k, xr[i][r], kx);
        xq[i][r] *= fq, xr[i][r] *= fr, xs[i][r] *= fs;
        kt = fmaf(k, xs[i][r], kt);
      }
    db -= grow * kx;
    __syncthreads();
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int y = 32 * st + 8 * g;
      if (st <= blk) {             // rows of the masked products: this tile's tokens as i
        const bs_parts<3> pf = row_parts(&lp[tok][y]), mf = row_parts(&lm[tok][y]);
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          const bs_parts<PI> a = delta_frags<PI>(
              w.kt + kbh + lane * 8 + ((half * CT + i) * 2 + st) * kFrag, kChunk * DK);
          xq[i] = bs_mma<2>(a, pf, xq[i]);
          xr[i] = bs_mma<2>(a, mf, xr[i]);
        }
      }
      if (st >= blk) {             // columns: as j
        float p[8], q[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) p[x] = lp[y + x][tok], q[x] = lm[y + x][tok];
        const bs_parts<3> pf = bs_split8<3>(p), mf = bs_split8<3>(q);
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          const int64_t at = kbh + lane * 8 + ((half * CT + i) * 2 + st) * kFrag;
          xs[i] = bs_mma<2>(delta_frags<PI>(w.qt + at, kChunk * DK), pf, xs[i]);
          xs[i] = bs_mma<2>(delta_frags<PI>(w.kt + at, kChunk * DK), mf, xs[i]);
        }
      }
    }
    float drun = 0.f;
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int e = 4 * (i & 1) + r;
        drun = fmaf(frag_value(qf[i >> 1], e), xq[i][r], drun);
        drun = fmaf(frag_value(kf[i >> 1], e), xr[i][r] - xs[i][r], drun);
        aq[i][r] += xq[i][r];
        ak[i][r] += xr[i][r] + xs[i][r];
      }
    drun = sum4(drun);
    db = sum4(db + dot_v);
    if (g == 0) rows[half][tok] = drun, betas[half][tok] = db;
    kt = fmaf(co[kTotal * kChunk], dot_s, kt);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) kt += __shfl_xor(kt, x);
    if (lane == 0) tot[wave] = kt;
    __syncthreads();
    if (wave == 0) {
      double x = (double)rows[0][lane] + rows[1][lane];
      if (lane == 63) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x += tot[i];
      }
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double y = __shfl_down(x, d);
        if (lane + d < 64) x += y;
      }
      if (lane < len) {
        const int64_t at = (sp.batch * plan.tokens + t0 + lane) * in.hv + h;
        bs_store_any(dg, in.g_dtype, at, (float)x);
        bs_store_any(dbeta, in.beta_dtype, at, betas[0][lane] + betas[1][lane]);
      }
    }
  }
  if (!live) return;
#pragma unroll
  for (int s = 0; s < HS; ++s) {
    const int d = 32 * (half * HS + s) + 8 * g;
    const int64_t at = ((sp.batch * plan.tokens + t0 + tok) * in.hk + hk) * in.dk + d;
    T x[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = bs_from_f32<T>(aq[2 * s + (e >> 2)][e & 3]);
      y[e] = bs_from_f32<T>(ak[2 * s + (e >> 2)][e & 3]);
    }
    if (d + 8 <= in.dk) {
      __builtin_memcpy(dq + at, x, sizeof(x));
      __builtin_memcpy(dk + at, y, sizeof(y));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d + e < in.dk) dq[at + e] = x[e], dk[at + e] = y[e];
    }
  }
}

struct GradOut { void *dq, *dk, *dv, *dg, *dbeta; float* dstate; };

template <typename T, int PI, int KS>
void launch_grad(const bs_delta_in& in, const DeltaPlan& plan, const DeltaWork& w,
                 const DeltaSizes& z, const void* go, const float* gstate, const float* keep_s,
                 const float* keep_u, const GradOut& o, hipStream_t st) {
  const unsigned extra = plan.offsets ? 1 : 0;
  const int units = (plan.seqs + (int)extra) * in.hv;
  const int wide = in.dv % 4 == 0 && (uintptr_t)o.dv % (4 * sizeof(T)) == 0;
  auto run = [&](auto nt) {
    grad_chain_kernel<T, PI, KS, nt.value>
        <<<delta_grid(units, z.dvp / (16 * nt.value)), 512, 0, st>>>(
            in, plan, w, (const T*)go, gstate, (T*)o.dv, o.dstate, z.dvp, units, wide);
  };
  if (delta_wide(units, z.dvp)) run(std::integral_constant<int, 2>());
  else run(std::integral_constant<int, 1>());
  if (plan.slots + extra == 0) return;
  int vec = in.dv % 8 == 0 ? 3 : 0;           // bit 0: grad_o's rows, bit 1: v's
  if ((uintptr_t)go % 16) vec &= 2;
  if ((uintptr_t)in.v % 16) vec &= 1;
  for (int i = 0; i < 3; ++i)
    if (in.v_stride[i] % 8) vec &= 1;
  grad_chunk_kernel<T, PI, KS><<<dim3(plan.slots + extra, in.hk), 512, 0, st>>>(
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
                               (plan.slots == 0 || (kept_states && kept_u)) && dq && dk && dv &&
                               dg && dbeta),
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
