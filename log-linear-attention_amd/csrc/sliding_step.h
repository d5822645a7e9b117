// Sliding-window attention's token step and cache: launches of sliding_step.hip for the
// C-ABI entry points.
#pragma once

#include <hip/hip_runtime.h>

constexpr int kStepSplits = 256;  // workgroups that one row and key head's slots are cut into, at most

struct SlidingStepArgs {
  const void *q, *k, *v;  // step: q [B, H, D], k, v [B, G, D]
  void *kc, *vc;          // [B, G, S + W, D]
  int* counts;            // [B]: tokens that each row has seen
  void* o;                // [B, H, D]
  float *part, *stat;     // [B, H, splits, D], [B, H, splits, 2]
  int B, H, G, D, W, S, splits, rblocks;
  float scale2;           // scale * log2(e)
};

hipError_t hattn_sliding_step_launch(const SlidingStepArgs& p, int dtype, hipStream_t stream);
hipError_t hattn_sliding_cache_launch(const SlidingStepArgs& p, int T, const long* strides,
                                      const int* lengths, hipStream_t stream);
