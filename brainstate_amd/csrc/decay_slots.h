// The chunks of a segment on the device (decay_chunk.hip, decay_grad.hip).
#pragma once

#include "decay.h"

// The slots of a segment in processing order, those with a chunk.
struct Chunks {
  int slot, end, step, back;
  DeltaSpan span;
  __device__ __forceinline__ Chunks(const DeltaPlan& p, int from, int to, int b) {
    back = b, step = b ? -1 : 1;
    slot = b ? to - 1 : from;
    end = b ? from - 1 : to;
    span.slot = -1, span.chunks = 0;
  }
  // `empty`: called for a sequence without tokens
  template <typename F>
  __device__ __forceinline__ bool next(const DeltaPlan& p, DecayChunk& c, F&& empty) {
    for (; slot != end; slot += step) {
      if (slot < span.slot || slot >= span.slot + span.chunks) {
        span = delta_span(p, delta_owner(p, slot));
        if (span.chunks == 0 && slot == span.slot) empty(span.seq);
      }
      const int k = slot - span.slot;
      if (k < 0 || k >= span.chunks) continue;
      c.seq = span.seq, c.slot = slot, c.batch = span.batch;
      c.token = span.first + (int64_t)k * kChunk;
      c.rows = min(span.len - k * kChunk, kChunk);
      c.next_g = k < span.chunks - 1;
      c.first = back ? k == span.chunks - 1 : k == 0;
      c.last = back ? k == 0 : k == span.chunks - 1;
      slot += step;
      return true;
    }
    return false;
  }
};

// What the segment [from, to) leaves to the next one, and the slots it takes.
__device__ __forceinline__ DecayLink link_of(const DeltaPlan& p, int back, int& from, int& to) {
  const int edge = back ? from : to - 1;
  const DeltaSpan s = delta_span(p, delta_owner(p, edge));
  const int k = edge - s.slot;
  if (k < 0 || k >= s.chunks || k == (back ? 0 : s.chunks - 1)) return {-1, 0};
  const int first = back ? s.slot + s.chunks <= to : s.slot >= from;
  if (back) to = min(to, s.slot + s.chunks);
  else from = max(from, s.slot);
  return {s.seq, first};
}
