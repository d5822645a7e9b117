// Sliding-window attention with sinks: launches of sliding_fwd.hip and sliding_bwd.hip for
// the C-ABI entry points.
#pragma once

#include <hip/hip_runtime.h>

struct SlidingArgs {
  const void *q, *k, *v, *o, *go;     // q, o, go [B, T, H, D]; k, v [B, T, G, D]
  void *out, *dq, *dk, *dv;           // contiguous
  float *lse, *delta;                 // [B, H, T]: log2 of a row's sum of exp2; rowsum(go o)
  float* part;                        // partial sums of the sinks' gradients
  const int* lengths;                 // [B] or NULL
  long qb, qt, qh, kb, kt, kh, vb, vt, vh;  // strides of q, k, v in elements
  int B, T, H, G, D, W, S;
  int narrow;                         // W + S <= kNarrow
  float scale, scale2;                // scale, scale * log2(e)
};

constexpr int kSinkChunk = 1024;  // queries of one partial sum of the sinks' gradients
constexpr int kMaxSinks = 64;
constexpr int kNarrow = 64;

// Partial sums a sink's gradient is made of: its near queries, then (chunk, head).
inline int sliding_sink_slots(int T, int H, int G, int W, int S) {
  return S > 0 && T > W ? 1 + (T - W + kSinkChunk - 1) / kSinkChunk * (H / G) : 0;
}

hipError_t hattn_sliding_fwd_launch(const SlidingArgs& p, int dtype, hipStream_t stream);
hipError_t hattn_sliding_bwd_launch(const SlidingArgs& p, int dtype, hipStream_t stream);
