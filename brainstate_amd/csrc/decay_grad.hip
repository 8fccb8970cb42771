// Gradients of decay attention: three walks (decay.h) over the chunks, in one launch.  With dS_t
// the gradient of the state before what o_t takes from it, without token t's own part,
//
//   dq_t = scale S_t do_t:                     the forward walk of queries do, keys v, values k
//   dv_t = (dS_t + scale q_t do_t^T)^T k_t:    a walk from the last token, queries k, keys q, values do
//   dk_t = (dS_t + scale q_t do_t^T) v_t:      the same of queries v, keys do, values q
//   dg_t = sum_{t <= i < e} (A_i + sum_j P_ij - B_i - sum_j P_ji) + <S_e, dS_e>
//
// for any end e of tokens [s, e) around t, where P_ij = scale exp(run_i - run_j) (q_i.k_j) (do_i.v_j)
// within them, A_i is q_i's product with the part of dq_i that comes from S_s, and B_i k_i's with the
// part of dk_i from dS_e: the derivative of every decay that an output or a write of t .. e - 1
// passes.  It is a difference of sums that grow with the tokens between t and e, so e is the end of
// t's chunk (the forward call saves its states there, and the walk of dv multiplies them with dS).  Both
// sums of P are of the same 32-bit numbers, added in 64 bits: what cancels of them leaves nothing.  A_i,
// B_i and <S_e, dS_e> are 32-bit sums over a head's values, added over the tokens in 64; each is off by
// some 2^-24 of its factors' norms, which is what is left where the others cancel.  300 tokens, heads
// of 64 that fade by 0.003 to 12 a token: 1e-7 to 6e-7 of a head's gradient, no more in fast heads than
// in slow ones, since all terms fade with them.  An infinity or NaN reaches dg of its whole chunk.
// 4 x 2,048 tokens, 16 heads of 128 x 128 in bf16: the three walks 248 us beside 72 of the forward one,
// each bound by what its waves issue (decay_chunk.hip); sums and scan 50, decays 5.  One launch, so that
// a walk's last workgroups run beside the next one's first.
//
// The states of the first walk and of dk's are the transposes of the other two's, which only changes
// how the carried ones are read.
#include "decay.h"
#include "decay_slots.h"

namespace {

struct GradWork {
  void* carry;
  float *start;                // [segs][hv][dk][dv]: dS at the segments' ends
  double *x, *y;               // [hv][rows]: A + sum P_ij - sum P_ji, and B
  float* edge;                 // [slots][hv]: <S, dS> at the chunks' ends
  float *dq, *dk;              // [rows][hv][dk] where heads share keys
  float *final;                // [seqs][hv][dk][dv], with a gradient of the final states
  double* sums;                // [slots][hv]: dg's sums where g has one value a head
};

int64_t align16(int64_t n) { return (n + 15) / 16 * 16; }

// Splits `ws`, or only counts its bytes where it is NULL.
int64_t work_of(const bs_delta_in& in, const DecayPlan& plan, int seqs, int64_t rows, bool decays,
                void* ws, GradWork* w) {
  char* p = (char*)ws;
  auto take = [&](int64_t bytes) {
    char* r = p;
    p += align16(bytes);
    return r;
  };
  const int64_t state = (int64_t)in.hv * in.dk * in.dv * 4, slots = decays ? plan.seq.slots : 0;
  w->carry = take(decay_carry_bytes(in, plan));
  w->start = (float*)take(plan.carry ? plan.segs * state : 0);
  const int64_t shared = in.hk < in.hv ? rows * in.hv * in.dk * 4 : 0;
  w->dq = (float*)take(shared);
  w->dk = (float*)take(shared);
  w->x = (double*)take(decays ? rows * in.hv * 8 : 0);
  w->y = (double*)take(decays ? rows * in.hv * 8 : 0);
  w->edge = (float*)take(slots * in.hv * 4);
  w->sums = (double*)take(slots * in.hv * 8);
  w->final = (float*)take(decays ? seqs * state : 0);
  return p - (char*)ws;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

struct GradIn {
  const double *x, *y;
  const float *edge, *final, *grad_state;
  void* dg;
  double* sums;
  int64_t rows;
  int n;                       // dk dv
};

// dg of a chunk and head: one wave, lane = row from the chunk's end.
__global__ __launch_bounds__(64) void decays_kernel(DecayPlan plan, GradIn in) {
  const int slot = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  if (slot >= plan.seq.slots) {
    auto zero = [&](auto* p) { zero_outside(plan.seq, p, plan.hv, 1, h, 0, 1); };
    if (plan.g_dtype == BS_F32) zero((float*)in.dg);
    else if (plan.g_dtype == BS_BF16) zero((bs_bf16*)in.dg);
    else zero((bs_f16*)in.dg);
    return;
  }
  Chunks chunks(plan.seq, slot, slot + 1, 1);
  DecayChunk c;
  double sum = 0.0;
  if (chunks.next(plan.seq, c, [](int) {})) {
    double base = 0.0;
    if (!c.first) {
      base = in.edge[(int64_t)slot * plan.hv + h];
    } else if (in.grad_state) {              // the states after the sequence
      const int64_t at = ((int64_t)c.seq * plan.hv + h) * in.n;
      for (int i = lane; i < in.n; i += 64)
        base += (double)in.final[at + i] * (double)in.grad_state[at + i];
      base = wave_sum(base);
    }
    const int64_t token = c.token + c.rows - 1 - lane, row = c.batch * plan.seq.tokens + token;
    const bool live = lane < c.rows;
    double x = 0.0;
    if (live) x = in.x[h * in.rows + row] - in.y[h * in.rows + row];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double y = __shfl_up(x, d);
      if (lane >= d) x += y;
    }
    if (live) {
      // the clamp of log decays has no slope below its bound
      const float g = bs_load_any(plan.g, plan.g_dtype,
                                  bs_delta_at(plan.g_stride, c.batch, token, h));
      const double r = g < BS_DELTA_G_MIN ? 0.0 : base + x;
      if (in.sums) sum = r;
      else bs_store_any(in.dg, plan.g_dtype, row * plan.hv + h, (float)r);
    }
  }
  if (in.sums) {
    sum = wave_sum(sum);
    if (lane == 0) in.sums[(int64_t)slot * plan.hv + h] = sum;
  }
}

// dg of heads: the chunks' sums in their order.
__global__ __launch_bounds__(64) void heads_kernel(const double* sums, int slots, int hv, void* dg,
                                                   int dtype) {
  const int h = blockIdx.x;
  double s = 0.0;
  for (int i = threadIdx.x; i < slots; i += 64) s += sums[(int64_t)i * hv + h];
  s = wave_sum(s);
  if (threadIdx.x == 0) bs_store_any(dg, dtype, h, (float)s);
}

// Gradients of shared keys: sums over the heads that share one, in their order.
template <typename T>
__global__ __launch_bounds__(256) void shared_kernel(const float* dq, const float* dk, T* q, T* k,
                                                     int64_t n, int group, int d) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * 256) {
    const int64_t at = i / d * group * d + i % d;
    const float* p = (blockIdx.y ? dk : dq) + at;
    float s = 0.f;
    for (int j = 0; j < group; ++j) s += p[(int64_t)j * d];
    (blockIdx.y ? k : q)[i] = bs_from_f32<T>(s);
  }
}

int64_t rows_of(int seqs, int tokens, const int32_t* offsets) {
  return offsets ? tokens : (int64_t)seqs * tokens;
}

}  // namespace

extern "C" size_t bs_decay_attention_grad_workspace_size(const bs_delta_in* in, int32_t seqs,
                                                         int32_t tokens, int32_t packed,
                                                         int32_t decays) {
  static const int32_t dummy[1] = {0};
  const int32_t* off = packed ? dummy : nullptr;
  if (decay_check(in, seqs, tokens, off, "bs_decay_attention_grad_workspace_size")) return 0;
  GradWork w;
  return (size_t)work_of(*in, decay_plan(*in, seqs, tokens, off), seqs,
                         rows_of(seqs, tokens, off), decays, nullptr, &w);
}

extern "C" int bs_decay_attention_grad(const bs_delta_in* in, int32_t seqs, int32_t tokens,
                                       const int32_t* seq_offsets, const void* grad_o,
                                       const float* grad_state, const float* initial_state,
                                       const void* kept, void* dq, void* dk, void* dv,
                                       void* dg, int32_t dg_heads, float* dstate, void* workspace,
                                       size_t workspace_bytes, bs_stream_t stream) {
  static const char* who = "bs_decay_attention_grad";
  if (int rc = decay_check(in, seqs, tokens, seq_offsets, who)) return rc;
  hipStream_t st = bs_stream(stream);
  const DecayPlan plan = decay_plan(*in, seqs, tokens, seq_offsets);
  const int64_t rows = rows_of(seqs, tokens, seq_offsets);
  GradWork w;
  const size_t need = (size_t)work_of(*in, plan, seqs, rows, dg != nullptr, nullptr, &w);
  BS_CHECK_ARG(rows == 0 || (in->q && in->k && in->v && in->g && grad_o && dq && dk && dv),
               "%s: NULL pointer", who);
  BS_CHECK_ARG(kept || !decay_kept_bytes(*in, plan, dg ? 2 : 1), "%s: kept is NULL", who);
  BS_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
               "%s: workspace of %zu bytes needed, %zu given", who, need,
               workspace ? workspace_bytes : (size_t)0);
  work_of(*in, plan, seqs, rows, dg != nullptr, workspace, &w);
  const int64_t states = (int64_t)seqs * in->hv * in->dk * in->dv;
  if (plan.seq.slots == 0 && dstate && states) decay_keep(grad_state, dstate, states, st);
  const int group = in->hv / in->hk;
  auto op = [](const void* p, const int64_t* s, int rep) {
    return DecayOperand{p, {s[0], s[1], s[2]}, rep};
  };
  const int64_t go_stride[3] = {(int64_t)tokens * in->hv * in->dv, (int64_t)in->hv * in->dv,
                                in->dv};
  const DecayOperand q = op(in->q, in->q_stride, group), k = op(in->k, in->k_stride, group),
                     v = op(in->v, in->v_stride, 1), go = op(grad_o, go_stride, 1),
                     none = op(nullptr, go_stride, 1);
  const int dkn = in->dk, dvn = in->dv;
  DecayRun r[3] = {decay_run(*in, k, q, go, none, dkn, dvn), decay_run(*in, v, go, q, dg ? k : none, dvn, dkn),
                   decay_run(*in, go, v, k, dg ? q : none, dvn, dkn)};
  for (int i = 0; i < 2; ++i) {
    r[i].back = 1, r[i].grow_scale = 1.f, r[i].add_scale = in->scale;
    r[i].first.p = const_cast<float*>(grad_state);
    r[i].start.p = w.start;
  }
  r[0].o = dv, r[0].last.p = dstate;
  r[0].vec_o = dvn % 8 == 0 && (uintptr_t)dv % 16 == 0;
  r[1].o = group > 1 ? (void*)w.dk : dk, r[2].o = group > 1 ? (void*)w.dq : dq;
  r[1].dots = w.y, r[2].dots = w.x, r[2].pairs = dg != nullptr;
  r[2].first.p = const_cast<float*>(initial_state);
  r[2].start.p = (float*)const_cast<void*>(kept);
  if (dg) {
    r[0].saved = decay_kept_saved(*in, plan, const_cast<void*>(kept)), r[0].edge = w.edge;
    if (grad_state) r[2].last.p = w.final;
  }
  for (int i = 1; i < 3; ++i) {
    r[i].o_f32 = group > 1, r[i].rows = rows;
    r[i].vec_o = dkn % 8 == 0 && (uintptr_t)r[i].o % 16 == 0;
    for (DecayState* s : {&r[i].first, &r[i].start, &r[i].last}) s->row = 1, s->col = dvn;
  }
  if (plan.carry) decay_carry(r[0], plan, in->dtype, w.carry, st);
  decay_walk(r, 3, plan, in->dtype, st);
  BS_CHECK_LAUNCH();
  if (dg) {
    const GradIn gi = {w.x, w.y, w.edge, w.final, grad_state, dg, dg_heads ? w.sums : nullptr,
                       rows, dkn * dvn};
    const unsigned grid = plan.seq.slots + (plan.seq.offsets && !dg_heads ? 1 : 0);
    if (grid) decays_kernel<<<dim3(grid, in->hv), 64, 0, st>>>(plan, gi);
    if (dg_heads)
      heads_kernel<<<in->hv, 64, 0, st>>>(w.sums, plan.seq.slots, in->hv, dg, in->g_dtype);
  }
  if (group > 1 && rows) {
    const int64_t n = rows * in->hk * dkn, blocks = (n + 255) / 256;
    const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536), 2);
    auto sum = [&](auto t) {
      using T = decltype(t);
      shared_kernel<<<grid, 256, 0, st>>>(w.dq, w.dk, (T*)dq, (T*)dk, n, group, dkn);
    };
    if (in->dtype == BS_F32) sum(float());
    else if (in->dtype == BS_BF16) sum(bs_bf16());
    else sum(bs_f16());
  }
  BS_CHECK_LAUNCH();
  return BS_OK;
}
