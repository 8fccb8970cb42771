// Plan and operands of decay attention over whole sequences (decay_chunk.hip, decay_grad.hip).
#pragma once

#include "delta_chunk.h"

using bs_f32x16 = __attribute__((__vector_size__(16 * sizeof(float)))) float;

// One walk over the chunks of sequences: with queries q and keys k of `dc` values and values v of
// `dv`, in processing order,
//
//   o_i = grow_scale exp(run_i) S0^T q_i + att_scale sum_{j <= i} exp(run_i - run_j) (q_i.k_j) v_j
//   S   = exp(total) S0 + add_scale sum_j exp(total - run_j) k_j v_j^T
//
// The gradients are such walks too, with the operands exchanged, two of them from the last token to
// the first (decay_grad.hip).
struct DecayOperand {
  const void* p;
  int64_t stride[3];          // of batch, token and head, in elements
  int rep;                    // value heads to one of its heads
};

struct DecayState {           // element (r, c) of sequence or segment n's state of head h lies at
  float* p;                   // ((n hv + h) dc dv) + r row + c col
  int row, col;
};

struct DecayRun {
  DecayOperand q, k, v;
  DecayOperand dot;           // rows like o's whose product with o's first term goes to dots, or
                              // p = NULL
  DecayState first;           // states before the sequences, p = NULL for zeros
  DecayState last;            // and after them, p = NULL if not wanted
  DecayState start;           // states before the segments that go on with a sequence
  void* o;                    // [.., hv, dv] of the operands' type, or in 32 bits (o_f32)
  double* dots;               // [hv][rows], rows of all sequences
  int pairs;                  // dots have the second term's too, less what it gives as key: with
                              // P_ij = att_ij (dot_i.v_j), sum_j P_ij - sum_j P_ji
  float* save;                // states before the chunks but a sequence's first, see decay_saved;
  const float* saved;         // from the last token to the first: the ones that a run has saved,
  float* edge;                // [slots][hv]: and their product with the state at a chunk's end
  int64_t rows;
  int dc, dv, back, o_f32;
  int vec, vec_o;             // operands' rows start on 16 bytes and end on 8 values, and o's
  float att_scale, grow_scale, add_scale;
};

// A segment is `per` slots (delta_chunk.h) side by side, walked by one workgroup for each head; a
// sequence that goes on in the next segment is carried there by sum_kernel and scan_kernel.
struct DecayPlan {
  DeltaPlan seq;
  int per, segs, carry, hv;
  const void* g;
  int64_t g_stride[3];
  int g_dtype;
};

// What the segment leaves to the one that is processed next.
struct DecayLink {
  int seq;                    // the sequence that goes on, or -1
  int first;                  // whether it begins in this segment
};

// A chunk: sequence, batch row, its first token and rows, and whether it is the sequence's first
// or last in processing order.
struct DecayChunk {
  int seq, slot, rows, first, last;
  int64_t batch, token;
  int next_g;                 // back: whether a token follows the chunk in its sequence
};

// Values of a saved state: its columns in tiles of 32, in the order of the registers.
static inline __host__ __device__ int decay_saved(int dc, int dv) {
  return (dc + 31) / 32 * ((dv + 31) / 32) * 1024;
}

DecayPlan decay_plan(const bs_delta_in& in, int seqs, int tokens, const int32_t* offsets);
int decay_check(const bs_delta_in* in, int seqs, int tokens, const int32_t* offsets,
                const char* who);
// What the forward call keeps for the gradients: the segments' states and, for those of the decays,
// a state a chunk (at decay_kept_saved); `keep` is enum-like: 0 nothing, 1 without them, 2 with.
int64_t decay_kept_bytes(const bs_delta_in& in, const DecayPlan& plan, int keep);
float* decay_kept_saved(const bs_delta_in& in, const DecayPlan& plan, void* kept);
// Decays and links of the segments: the workspace of one run's carry.
int64_t decay_carry_bytes(const bs_delta_in& in, const DecayPlan& plan);
// Fills run.start (sums, then their scan over the segments); `scratch` holds decays and links.
void decay_carry(const DecayRun& run, const DecayPlan& plan, int dtype, void* scratch,
                 hipStream_t st);
// The walks, all in one launch.
void decay_walk(const DecayRun* runs, int n, const DecayPlan& plan, int dtype, hipStream_t st);
DecayRun decay_run(const bs_delta_in& in, const DecayOperand& q, const DecayOperand& k,
                   const DecayOperand& v, const DecayOperand& dot, int dc, int dv);
// Copies n floats, zeros from NULL.
void decay_keep(const float* from, float* to, int64_t n, hipStream_t st);
