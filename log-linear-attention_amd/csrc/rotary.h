// Rotary positions: launch of rotary.hip for the C-ABI entry point.
#pragma once

#include <hip/hip_runtime.h>

struct RotaryArgs {
  const void* x[2];              // [B, T, heads, D]; the second may have no heads
  void* y[2];                    // contiguous
  long xb[2], xt[2], xh[2];      // strides of x in elements
  int heads[2];
  const void* freqs;             // [pairs], radians a token
  const void* pos;               // position of (b, t) at pb * b + pt * t; NULL: t
  long pb, pt;
  long N;                        // B * T
  int T, D, pairs;
  int freq64, pos64;             // freqs are doubles, positions 64-bit
  int from;                      // positions are of each row's first token
  int tokens, cols;              // tokens a workgroup; lanes of a head
  float scale, sign;             // sign -1: the inverse rotation
};

// Elements that a lane moves at once: 16 bytes where `wide`.
inline int rotary_vec(int bytes, bool wide) { return wide ? 16 / bytes : 1; }
inline size_t rotary_lds(int tokens, int pairs) { return (size_t)tokens * (pairs * 8 + 16); }

hipError_t hattn_rotary_launch(const RotaryArgs& p, int dtype, bool interleaved, bool wide,
                               hipStream_t stream);
