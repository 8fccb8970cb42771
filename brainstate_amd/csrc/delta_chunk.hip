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
//
// One prompt of 8,192 tokens x 32 heads of 128 x 128 in bfloat16, 401 us: prepare 107, of which the
// 258 MB it writes for chain_kernel are 51 at a large copy's rate; chain 314 under the tracer, 2.5
// us a chunk: bound by the latency of its three dependent products and barriers (the matrix cores
// are busy in 17 % of the cycles, 394 MB move).  With the output's operands cut to two parts the
// call took 373 us, and terms that cancel left their errors of 2^-15.  The same prompt in fp16 530,
// in 32 bits 737.
#include "delta_chunk.h"

namespace {

// One chunk and value head: 4 waves, wave w has tile w's rows.
// The inverse is formed by blocks of 16 tokens: the four on the diagonal by substitution, one
// column a lane, the ones below by X_ij = -X_ii sum_k L_ik X_kj in 32-bit matrix instructions.
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
  if (c < 0 || c >= sp.chunks) return;      // c < 0: ahead of the first sequence
  const int64_t t0 = sp.first + (int64_t)c * kChunk;
  const int len = min(sp.len - c * kChunk, kChunk);
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool first = h % group == 0;
  const int64_t sh = (int64_t)slot * in.hv + h;
  const int64_t kb = ((int64_t)slot * in.hk + hk) * PI * kChunk * DK;

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
    float* co = w.coef + sh * kCoef;
    co[kGrow * kChunk + lane] = expf((float)x);
    co[kLeft * kChunk + lane] = expf((float)(total - x));
    co[kBeta * kChunk + lane] = b;
    co[kTotal * kChunk + lane] = expf((float)total);
    ((double*)(co + kRun * kChunk))[lane] = x;
  }
  const int row = delta_row(wave, m);
  bs_parts<PI> qf[KS], kf[KS];
  {
    const DeltaRow<T> kr((const T*)in.k + bs_delta_at(in.k_stride, sp.batch, t0, hk),
                         in.k_stride[1], row, len, in.dk, vec);
    const DeltaRow<T> qr((const T*)in.q + bs_delta_at(in.q_stride, sp.batch, t0, hk),
                         in.q_stride[1], row, len, in.dk, vec);
    uint4 kx[KS][sizeof(T) / 2], qx[KS][sizeof(T) / 2];
#pragma unroll
    for (int s = 0; s < KS; ++s) kr.raw(32 * s + 8 * g, kx[s]);
#pragma unroll
    for (int s = 0; s < KS; ++s) qr.raw(32 * s + 8 * g, qx[s]);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 32 * s + 8 * g;
      kf[s] = kr.template parts<PI>(kx[s]);
      qf[s] = qr.template parts<PI>(qx[s]);
#pragma unroll
      for (int p = 0; p < PI; ++p) {
        *(bs_bf16x8*)&kl[p][row][d] = kf[s].p[p];
        if (first) {
          const int64_t f = kb + (int64_t)((p * 4 + wave) * KS + s) * kFrag + lane * 8;
          *(bs_bf16x8*)(w.kp + f) = kf[s].p[p];
          *(bs_bf16x8*)(w.qp + f) = qf[s].p[p];
        }
      }
    }
  }
  __syncthreads();
  // the transposed copy of what kl holds, by fragments
  auto transposed = [&](uint16_t* to) {
#pragma unroll
    for (int p = 0; p < PI; ++p)
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int f = wave * KS + i, d = delta_row(f >> 1, m), j0 = 32 * (f & 1) + 8 * g;
        bs_u16x8 r;
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = kl[p][j0 + j][d];
        *(bs_u16x8*)(to + kb + (int64_t)(p * 4 * KS + f) * kFrag + lane * 8) = r;
      }
  };
  const int i0 = 32 * (wave >> 1) + 8 * g + 4 * (wave & 1);     // rows i0 .. i0 + 3 come back
  float am[4][4];                 // the masked product, for LDS later
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) {
    const int j = delta_row(jt, m);
    bs_f32x4 kk = zero4(), qk = zero4();
    if (jt <= (wave | 1)) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        bs_parts<PI> b;
#pragma unroll
        for (int p = 0; p < PI; ++p) b.p[p] = *(const bs_bf16x8*)&kl[p][j][32 * s + 8 * g];
        kk = bs_mma<2>(kf[s], b, kk);
        qk = bs_mma<2>(qf[s], b, qk);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = i0 + r;
      const float e = j <= i ? expf((float)(run[i] - run[j])) : 0.f;
      lm[i][j] = j < i ? bt[i] * e * kk[r] : 0.f;
      if ((i >> 4) < (j >> 4)) xm[i][j] = 0.f;
      am[jt][r] = j <= i ? in.scale * e * qk[r] : 0.f;
    }
  }
  if (first) transposed(w.kt);
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
  if (BWD && first) transposed(w.qt);
  for (int d = 1; d < 4; ++d) {
    const int j = wave, i = wave + d;
    if (i < 4) {
      bs_f32x4 a = zero4(), b = zero4();
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
#pragma unroll
  for (int jt = 0; jt < 4; ++jt)
#pragma unroll
    for (int r = 0; r < 4; ++r) lm[i0 + r][delta_row(jt, m)] = am[jt][r];
  __syncthreads();
  for (int f = wave; f < 6; f += 4) {
    const int t = BWD ? (f < 4 ? f >> 1 : f - 2) : f < 2 ? f : (f + 2) >> 1;
    const int s = BWD ? (f < 4 ? f & 1 : 1) : f < 2 ? 0 : f & 1;
    const int i = delta_row(t, m), j = 32 * s + 8 * g;
    float x[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = BWD ? xm[j + e][i] : xm[i][j + e];
      y[e] = BWD ? lm[j + e][i] : lm[i][j + e];
    }
    const bs_parts<3> xp = bs_split8<3>(x), yp = bs_split8<3>(y);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      *(bs_bf16x8*)(w.inv + (sh * 3 + p) * kSquare + f * kFrag + lane * 8) = xp.p[p];
      *(bs_bf16x8*)(w.att + (sh * 3 + p) * kSquare + f * kFrag + lane * 8) = yp.p[p];
    }
  }
}

// Forward over the chunks of one sequence, value head and slice of 16 NT value columns, by two
// sets of 4 waves.  The first has the recurrence: each wave 16 tokens of a chunk and a quarter of the
// state's rows; what the others need goes through LDS, as parts and in the lane that takes it.
// The second forms from the same LDS what the recurrence does not wait for: the output and, for
// the backward pass, U and the state before the chunk, transposed (the operands of a product
// swapped; for the state, times 1), which leaves 4 neighbouring columns of a row in a lane.  So
// no wave of the recurrence waits for a store, and a SIMD has two waves to issue from: the
// recurrence's own arithmetic (products of 3 parts, splitting) leaves it idle half the time.
// Operands that do not depend on the state are loaded into registers one or two chunks ahead.
template <typename T, int PI, int KS, int NT, bool KEEP>
__global__ __launch_bounds__(512, 2) void chain_kernel(
    bs_delta_in in, DeltaPlan plan, DeltaWork w, const float* state0, float* state1, T* o,
    float* keep_s, float* keep_u, int dvp, int units, int vec) {
  constexpr int DK = KS * 32, TW = KS / 2;
  constexpr int kS = KS * NT * 128, kR = 2 * NT * 128;       // words of a part
  __shared__ __attribute__((aligned(16))) uint2 ls[3 * kS];     // the state
  __shared__ __attribute__((aligned(16))) uint2 lr[3 * kR];     // R
  __shared__ __attribute__((aligned(16))) uint2 lu[3 * kR];     // exp(total - run) U
  __shared__ __attribute__((aligned(16))) uint2 lv[3 * kR];     // U
  const DeltaPlace at = delta_place(units, dvp / (16 * NT));
  if (at.unit >= units) return;
  const int h = __builtin_amdgcn_readfirstlane(at.unit % in.hv);
  const int n = __builtin_amdgcn_readfirstlane(at.unit / in.hv), hk = h / (in.hv / in.hk);
  if (n >= plan.seqs) {
    zero_outside(plan, o, in.hv, in.dv, h, at.slice * 16 * NT, 16 * NT);
    return;
  }
  const DeltaSpan sp = delta_span(plan, n);
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int role = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3), blk = wave >> 1;
  const int tok = delta_row(wave, m);                      // the row this lane feeds
  const int64_t keys = (int64_t)in.hk * PI * kChunk * DK;  // from chunk to chunk
  const int64_t kb = ((int64_t)sp.slot * in.hk + hk) * PI * kChunk * DK;
  const int64_t hb = (int64_t)sp.slot * in.hv + h;
  const float* cp = w.coef + hb * kCoef;
  const uint16_t* ip = w.inv + hb * 3 * kSquare + lane * 8;

  if (role == 0) {
    const int col = at.slice * 16 * NT + m;
    const int out0 = 32 * blk + 8 * g + 4 * (wave & 1);    // the 4 rows it receives
    const int own = (blk * NT * 64 + lane) * 2 + (wave & 1);     // and 128 on for each column tile
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
          s[i][j][r] = state0 && d0[i] + r < in.dk && col + 16 * j < in.dv
              ? state0[(((int64_t)n * in.hv + h) * in.dk + d0[i] + r) * in.dv + col + 16 * j]
              : 0.f;
        delta_put<3>(ls + sown[i] + 128 * j, kS, s[i][j]);
      }
    }
    const uint16_t* kp = w.kp + kb + wave * KS * kFrag + lane * 8;
    const uint16_t* kt = w.kt + kb + wave * TW * 2 * kFrag + lane * 8;
    const DeltaRows<T, NT> rows((const T*)in.v + bs_delta_at(in.v_stride, sp.batch, sp.first, h),
                                in.v_stride[1], out0, col, in.dv);
    bs_parts<PI> kf[KS], ktf[TW][2];
    bs_parts<3> tf[2];
    struct Values {
      typename DeltaRows<T, NT>::Raw v[NT][4];
      float total;
      float4 grow, left, beta;
    } values[2];
    auto load_keys = [&](int c) {
#pragma unroll
      for (int st = 0; st < KS; ++st)
        kf[st] = delta_frags<PI>(kp + c * keys + st * kFrag, kChunk * DK);
    };
    auto load_values = [&](int c, Values& x) {
      const float* co = cp + (int64_t)c * in.hv * kCoef;
      rows.load(c, sp.len, x.v);
      x.grow = *(const float4*)(co + kGrow * kChunk + out0);
      x.left = *(const float4*)(co + kLeft * kChunk + out0);
      x.beta = *(const float4*)(co + kBeta * kChunk + out0);
      x.total = co[kTotal * kChunk];
    };
    auto load_inverse = [&](int c) {
#pragma unroll
      for (int st = 0; st < 2; ++st)
        tf[st] = delta_frags<3>(ip + (int64_t)c * in.hv * 3 * kSquare +
                                    delta_lower(wave, min(st, blk)) * kFrag, kSquare);
    };
    auto load_columns = [&](int c) {
#pragma unroll
      for (int i = 0; i < 2 * TW; ++i)
        ktf[i >> 1][i & 1] = delta_frags<PI>(kt + c * keys + i * kFrag, kChunk * DK);
    };
    const int last = sp.chunks - 1;
    if (sp.chunks) {
      load_values(0, values[0]);
      load_keys(0);
      load_inverse(0);
      load_columns(0);
      load_values(min(1, last), values[1]);
    }
    wait_loads();
    __syncthreads();
    auto step = [&](int c, Values& now) {
      const int next = min(c + 1, last);
      bs_f32x4 x[NT], u[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) x[j] = u[j] = zero4();
#pragma unroll
      for (int st = 0; st < KS; ++st)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          x[j] = bs_mma<2>(kf[st], delta_lds<3>(ls + ((st * NT + j) * 64 + lane) * 2, kS), x[j]);
      const float* gr = (const float*)&now.grow;
      const float* be = (const float*)&now.beta;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          x[j][r] = be[r] * fmaf(-gr[r], x[j][r], rows.value(now.v[j][r]));
        delta_put<3>(lr + own + 128 * j, kR, x[j]);
      }
      __builtin_amdgcn_sched_barrier(0);   // loads after what the others wait for
      load_keys(next);
      __syncthreads();                     // R
#pragma unroll
      for (int st = 0; st < 2; ++st)
        if (st <= blk) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
            u[j] = bs_mma<2>(tf[st], delta_lds<3>(lr + ((st * NT + j) * 64 + lane) * 2, kR), u[j]);
        }
      const float* lf = (const float*)&now.left;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) x[j][r] = lf[r] * u[j][r];
        delta_put<3>(lu + own + 128 * j, kR, x[j]);
        delta_put<3>(lv + own + 128 * j, kR, u[j]);
      }
      __builtin_amdgcn_sched_barrier(0);
      load_inverse(next);
      __syncthreads();                     // U; the state's last readers are through
#pragma unroll
      for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) s[i][j] *= now.total;
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const bs_parts<3> b = delta_lds<3>(lu + ((st * NT + j) * 64 + lane) * 2, kR);
#pragma unroll
          for (int i = 0; i < TW; ++i) s[i][j] = bs_mma<2>(ktf[i][st], b, s[i][j]);
        }
#pragma unroll
      for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) delta_put<3>(ls + sown[i] + 128 * j, kS, s[i][j]);
      __builtin_amdgcn_sched_barrier(0);
      load_columns(next);
      load_values(min(c + 2, last), now);
      __syncthreads();                     // the state
    };
    // two steps a turn, without a way out between them (see wait_loads)
    for (int c = 0; c + 1 < sp.chunks; c += 2) {
      step(c, values[0]);
      step(c + 1, values[1]);
    }
    if (sp.chunks & 1) step(last, values[0]);
    if (state1) {
#pragma unroll
      for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (d0[i] + r < in.dk && col + 16 * j < in.dv)
              state1[(((int64_t)n * in.hv + h) * in.dk + d0[i] + r) * in.dv + col + 16 * j] =
                  s[i][j][r];
    }
  } else {
    const int ocol = at.slice * 16 * NT + 4 * g;
    const uint16_t* qp = w.qp + kb + wave * KS * kFrag + lane * 8;
    const uint16_t* ap = w.att + hb * 3 * kSquare + lane * 8;
    struct Operands { bs_parts<PI> q[KS]; bs_parts<3> a[2]; float scale; } operands[2];
    auto load = [&](int c, Operands& x) {
      const int64_t ch = (int64_t)c * in.hv;
#pragma unroll
      for (int st = 0; st < KS; ++st)
        x.q[st] = delta_frags<PI>(qp + c * keys + st * kFrag, kChunk * DK);
#pragma unroll
      for (int st = 0; st < 2; ++st)
        x.a[st] = delta_frags<3>(ap + ch * 3 * kSquare +
                                     delta_lower(wave, min(st, blk)) * kFrag, kSquare);
      x.scale = in.scale * cp[ch * kCoef + kGrow * kChunk + tok];
    };
    const int last = sp.chunks - 1;
    if (sp.chunks) {
      load(0, operands[0]);
      load(min(1, last), operands[1]);
    }
    T* op = o + ((sp.batch * plan.tokens + sp.first + tok) * in.hv + h) * in.dv + ocol;
    wait_loads();
    __syncthreads();
    // loads two chunks ahead: a load is not seen to arrive before the stores issued before it
    auto step = [&](int c, Operands& now) {
      const int64_t sh = hb + (int64_t)c * in.hv;
      __syncthreads();                     // R: from here the recurrence leaves the state alone
      bs_f32x4 y[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) y[j] = zero4();
#pragma unroll
      for (int st = 0; st < KS; ++st)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          y[j] = bs_mma<2>(delta_lds<3>(ls + ((st * NT + j) * 64 + lane) * 2, kS), now.q[st], y[j]);
#pragma unroll
      for (int j = 0; j < NT; ++j) y[j] *= now.scale;
      if (KEEP) {
#pragma unroll
        for (int i = 0; i < TW; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const int t = TW * wave + i;
            const bs_f32x4 x = delta_turn(
                delta_lds<3>(ls + (((t >> 1) * NT + j) * 64 + lane) * 2, kS), t & 1, lane);
            *(bs_f32x4*)(keep_s + sh * DK * dvp + delta_kept(t, at.slice * NT + j, lane, dvp)) = x;
          }
      }
      __syncthreads();                     // U
#pragma unroll
      for (int st = 0; st < 2; ++st)
        if (st <= blk) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
            y[j] = bs_mma<2>(delta_lds<3>(lv + ((st * NT + j) * 64 + lane) * 2, kR), now.a[st],
                             y[j]);
        }
      load(min(c + 2, last), now);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (KEEP) {
          const bs_f32x4 u = delta_turn(delta_lds<3>(lv + ((blk * NT + j) * 64 + lane) * 2, kR),
                                        wave & 1, lane);
          *(bs_f32x4*)(keep_u + sh * kChunk * dvp +
                       delta_kept(wave, at.slice * NT + j, lane, dvp)) = u;
        }
        if (c * kChunk + tok < sp.len) {
          T* p = op + (int64_t)c * kChunk * in.hv * in.dv + 16 * j;
          const int oc = ocol + 16 * j;
          if (vec) {
            if (oc < in.dv) bs_store4(p, y[j]);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (oc + r < in.dv) p[r] = bs_from_f32<T>(y[j][r]);
          }
        }
      }
      __syncthreads();                     // the state
    };
    // two steps a turn, without a way out between them (see wait_loads)
    for (int c = 0; c + 1 < sp.chunks; c += 2) {
      step(c, operands[0]);
      step(c + 1, operands[1]);
    }
    if (sp.chunks & 1) step(last, operands[0]);
  }
}

template <typename T, int PI, int KS>
void launch_prepare(const bs_delta_in& in, const DeltaPlan& plan, const DeltaWork& w,
                    int backward, hipStream_t st) {
  const dim3 grid(plan.slots, in.hv);
  int vec = in.dk % 8 == 0 && (uintptr_t)in.q % 16 == 0 && (uintptr_t)in.k % 16 == 0;
  for (int i = 0; i < 3; ++i) vec = vec && in.q_stride[i] % 8 == 0 && in.k_stride[i] % 8 == 0;
  if (backward) prepare_kernel<T, PI, KS, true><<<grid, 256, 0, st>>>(in, plan, w, vec);
  else prepare_kernel<T, PI, KS, false><<<grid, 256, 0, st>>>(in, plan, w, vec);
}

template <typename T, int PI, int KS>
void launch_chain(const bs_delta_in& in, const DeltaPlan& plan, const DeltaWork& w,
                  const DeltaSizes& z, const float* s0, float* s1, void* o, float* keep_s,
                  float* keep_u, hipStream_t st) {
  const int units = (plan.seqs + (plan.offsets ? 1 : 0)) * in.hv;
  const int vec = in.dv % 4 == 0 && (uintptr_t)o % (4 * sizeof(T)) == 0;
  auto run = [&](auto nt, auto keep) {
    chain_kernel<T, PI, KS, nt.value, keep.value>
        <<<delta_grid(units, z.dvp / (16 * nt.value)), 512, 0, st>>>(
            in, plan, w, s0, s1, (T*)o, keep_s, keep_u, z.dvp, units, vec);
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  if (delta_wide(units, z.dvp)) {
    if (keep_s) run(Two(), std::true_type());
    else run(Two(), std::false_type());
  } else {
    if (keep_s) run(One(), std::true_type());
    else run(One(), std::false_type());
  }
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
  // a chunk's rows are addressed in 32 bits
  for (const int64_t* st : {in->q_stride, in->k_stride, in->v_stride})
    BS_CHECK_ARG(st[1] >= 0 && st[1] < (1 << 23) && in->hv * in->dv < (1 << 23),
                 "%s: %lld elements from token to token", who, (long long)st[1]);
  const int64_t slots = offsets ? (int64_t)tokens / kChunk + seqs
                                : (int64_t)seqs * ((tokens + kChunk - 1) / kChunk);
  // launches of 512 threads a slot, or a unit and slice of 32 columns (16 only where those are at
  // most one a CU), have fewer than 2^32 threads; past that the count wraps without an error
  BS_CHECK_ARG(slots < (1 << 23) - 1 && in->hv <= 65535 &&
                   (((int64_t)seqs + 1) * in->hv + 7) * ((in->dv + 31) / 32) < 1 << 23,
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
  BS_CHECK_ARG(!kept_states == !kept_u,
               "bs_gated_delta_rule: one of kept_states and kept_u is NULL");
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
