// Gated linear recurrence: launches of recurrence.hip for the C-ABI entry points.
#pragma once

#include <hip/hip_runtime.h>

struct RecurrenceArgs {
  const void *x, *g, *go;             // [B, T, D]; step [B, D]; go: gradient of o
  const float *h0, *ght;              // [B, D] or NULL: state before, gradient of the state after
  const int* lengths;                 // [B] or NULL
  void *o, *dx, *dg;                  // [B, T, D]; step o [B, D]
  float *ht, *dh0;                    // [B, D] or NULL; step: the state
  float* carry;                       // [B, nseg, D]: the state that enters each segment
  void* ws;                           // nseg * B * strips * 64 vec words of 8 bytes where nseg > 1
  int B, T, D, vec, strips, nseg;     // vec channels a lane, strips of 64 lanes
};

// Tokens of a segment where a lane has vec channels.
int hattn_recurrence_segment(int vec);
hipError_t hattn_recurrence_launch(int what, const RecurrenceArgs& p, int dtype_x, int dtype_g,
                                   hipStream_t stream);
