// A cache of keys and values in 8 bits: launches of quant_cache.hip, quant_few.hip and
// quant_chunk.hip for the C-ABI entry points.
#pragma once

#include <hip/hip_runtime.h>

constexpr int kQuantBlock = 64;   // tokens that share a scale
constexpr int kQuantSplits = 256; // parts that one row's tokens are cut into, at most

struct QuantArgs {
  const void *q, *k, *v;          // q [B, T, H, D]; k, v [B, T, G, D]: the new tokens
  long qb, qt, qh, kb, kt, kh, vb, vt, vh;  // their strides in elements
  const int* lengths;             // [B] or NULL: new tokens of each row
  unsigned char *kc, *vc;         // [B, G, cap, D]: e4m3 codes
  float *ks, *vs;                 // [B, G, cap / 64]
  int* counts;                    // [B]: tokens that each row has had
  void *o, *ko, *vo;              // o [B, T, H, D]; read: ko, vo [B, n, G, D]
  float *part, *stat;             // [B, T, H, splits, D], [B, T, H, splits, 2]
  int* held;                      // [B], where `coming`: tokens with the new one, -1 without a slot
  int B, T, H, G, D, cap;
  int start, n;                   // read: slots [start, start + n)
  int blocks;                     // append, read: blocks of a row, at most
  int coming;                     // one token a row enters the cache in the attention itself
  int splits, rblocks;            // attention: parts of a row's tokens, blocks of its queries
  float scale2;                   // scale * log2(e)
};

// Counts of tokens past the capacity stay below INT_MAX.
hipError_t hattn_quant_append_launch(const QuantArgs& p, int dtype, hipStream_t stream);
// One token a row; the counts advance in the same launch.
hipError_t hattn_quant_token_launch(const QuantArgs& p, int dtype, hipStream_t stream);
hipError_t hattn_quant_read_launch(const QuantArgs& p, int dtype, hipStream_t stream);
// Blocks of 16 or 32 queries (few: 32 where there are more than 16) or 128 (chunk) of a row and key
// head.  With `coming` (at most 16 queries)
// the token enters the cache, and the join advances the counts.
hipError_t hattn_quant_few_launch(const QuantArgs& p, int dtype, hipStream_t stream);
hipError_t hattn_quant_chunk_launch(const QuantArgs& p, int dtype, hipStream_t stream);
hipError_t hattn_quant_join_launch(const QuantArgs& p, int dtype, hipStream_t stream);
