// A cache of keys and values in 8 bits: what its kernels share.
//
// A code is a number of e4m3 (4 bits of significand from 2^-6 to 448, steps of 2^-9 below, NaN, no
// infinities), and a value is its code times the scale of its block of 64 tokens of a head.  The
// scale is 2^e with the least e for which 448 * 2^e holds every finite value of the block,
// so dividing by it is exact, and a code has one rounding.  A block that grows past
// its scale gets a larger power of two: codes are floating-point numbers, so dividing the old
// ones by a power of two is exact but for those that fall below 2^-6.
//
// e is at least -100 (smaller values are 0) and at most what keeps 448 * 2^e finite in the
// inputs' type (7 in fp16, 119 in bf16; larger values become 448 * 2^e).  Infinities and NaN
// become NaN and do not count for the scale.
#pragma once

#include "common.h"
#include "quant_cache.h"

namespace hattn {

template <typename E>
struct Half;
template <>
struct Half<__bf16> {
  static constexpr unsigned kInf = 0x7f80;
  static constexpr int kMost = 119;
  static constexpr float kSlack = 8.f, kLift = 0.f, kPart = 0x1p-40f;
};
template <>
struct Half<_Float16> {
  static constexpr unsigned kInf = 0x7c00;
  static constexpr int kMost = 7;
  static constexpr float kSlack = 4.f, kLift = 11.f, kPart = 1.f;
};

// The running maximum m of a query's scores (powers of two) is taken again only where a score passes
// it by more than kSlack, so that most tiles do not rescale the sums; probabilities are
// 2^(s - m + kLift), at most 2^15.  In fp16 the lift keeps those down to 2^-25 of the largest out of
// the subnormal numbers: of many tokens of little weight each, the sum would be off.
// Weights of up to 2^kSlack of 2^30 tokens come to 2^38 before they are divided by their sum: in bf16,
// whose values go to 2^128, partial results are held times kPart.

// The magnitude of a 16-bit number as an integer of the same order; 0 where it is not finite.
template <typename E>
__device__ __forceinline__ unsigned finite_bits(unsigned x) {
  x &= 0x7fff;
  return x < Half<E>::kInf ? x : 0;
}

// The scale's exponent for a largest magnitude.  448 = 1.75 * 2^8.
template <typename E>
__device__ __forceinline__ int scale_exponent(unsigned bits) {
  const unsigned f = __builtin_bit_cast(
      unsigned, from16<E>(__builtin_bit_cast(__bf16, (unsigned short)bits)));
  const int e = (int)(f >> 23) - 127 - 8 + ((f & 0x7fffff) > 0x600000);
  return f == 0 ? -100 : min(max(e, -100), Half<E>::kMost);
}
__device__ __forceinline__ float power(int e) {
  return __builtin_bit_cast(float, (unsigned)(e + 127) << 23);
}

// Two 16-bit numbers (the halves of x) as codes, in the halves of the result that HI picks.
template <typename E, bool HI>
__device__ __forceinline__ int codes2(unsigned x, float inverse, int old) {
  float y[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const unsigned short h = (unsigned short)(x >> 16 * i);
    const float f = from16<E>(__builtin_bit_cast(__bf16, h)) * inverse;
    y[i] = (h & 0x7fff) < Half<E>::kInf ? fminf(fmaxf(f, -448.f), 448.f) : __builtin_nanf("");
  }
  return __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], old, HI);
}
template <typename E>
__device__ __forceinline__ uint2 codes8(uint4 x, float inverse) {
  int lo = codes2<E, false>(x.x, inverse, 0), hi = codes2<E, false>(x.z, inverse, 0);
  lo = codes2<E, true>(x.y, inverse, lo);
  hi = codes2<E, true>(x.w, inverse, hi);
  return uint2{(unsigned)lo, (unsigned)hi};
}

// Codes under a scale that is larger by 1 / ratio.
__device__ __forceinline__ unsigned rescale4(unsigned x, float ratio) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
  const int r = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * ratio, lo[1] * ratio, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * ratio, hi[1] * ratio, r, true);
}

// Four codes as 16-bit numbers (exact in either type).
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
template <typename E>
__device__ __forceinline__ bf16x4 widen4(unsigned x) {
  if constexpr (__is_same(E, _Float16)) {
    const bf16x2 a = __builtin_bit_cast(bf16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, false));
    const bf16x2 b = __builtin_bit_cast(bf16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, true));
    return bf16x4{a[0], a[1], b[0], b[1]};
  } else {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, true);
    return bf16x4{a[0], a[1], b[0], b[1]};
  }
}
template <typename E>
__device__ __forceinline__ bf16x8 widen8(unsigned lo, unsigned hi) {
  const bf16x4 a = widen4<E>(lo), b = widen4<E>(hi);
  return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

__device__ __forceinline__ unsigned wave_max(unsigned x) {
#pragma unroll
  for (int k = 1; k < 64; k *= 2) x = max(x, (unsigned)__shfl_xor((int)x, k, 64));
  return x;
}

// The larger of the halves' finite magnitudes.
template <typename E>
__device__ __forceinline__ unsigned top2(unsigned x) {
  return max(finite_bits<E>(x & 0xffff), finite_bits<E>(x >> 16));
}
// One new token of row b and key head g enters slot n0, by one wave: its codes, the block's scales,
// and where these grow the block's older codes.
template <typename E>
__device__ __forceinline__ void token_codes(const QuantArgs& p, int b, int g, int n0) {
  const int lane = threadIdx.x & 63, lo = n0 % kQuantBlock, first = n0 - lo;
  const long bg = (long)b * p.G + g, block = bg * (p.cap / kQuantBlock) + first / kQuantBlock;
  const bool mine = 2 * lane < p.D;
  float* const scale[2] = {p.ks + block, p.vs + block};
  unsigned char* const codes[2] = {p.kc + (bg * p.cap + first) * p.D, p.vc + (bg * p.cap + first) * p.D};
  const __bf16* const x[2] = {(const __bf16*)p.k + b * p.kb + g * p.kh,
                              (const __bf16*)p.v + b * p.vb + g * p.vh};
  unsigned y[2], top[2];
  float was[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    y[i] = mine ? *(const unsigned*)(x[i] + 2 * lane) : 0;
    was[i] = lo > 0 ? *scale[i] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) top[i] = wave_max(top2<E>(y[i]));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float now = fmaxf(power(scale_exponent<E>(top[i])), was[i]);
    const int c = codes2<E, false>(y[i], 1.f / now, 0);
    if (mine) *(unsigned short*)(codes[i] + lo * p.D + 2 * lane) = (unsigned short)c;
    if (lane == 0) *scale[i] = now;
    if (lo > 0 && now > was[i]) {
      const float ratio = was[i] / now;
      for (int at = 16 * lane; at < lo * p.D; at += 1024) {
        uint4 old = *(const uint4*)(codes[i] + at);
        old = uint4{rescale4(old.x, ratio), rescale4(old.y, ratio), rescale4(old.z, ratio),
                    rescale4(old.w, ratio)};
        *(uint4*)(codes[i] + at) = old;
      }
    }
  }
}

// What a row has: tokens in its cache (none where the count has passed the capacity: `full`), and
// its new tokens.  `coming`: its one new token is not counted yet.
struct QuantRow {
  int n, fresh;
  bool full;
  __device__ __forceinline__ QuantRow(const QuantArgs& p, int b, bool coming = false) {
    const int c = max(p.counts[b], 0);
    full = c > p.cap - coming;
    n = full ? 0 : c + coming;
    fresh = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  }
  // One new token, from what the attention's kernel noted.
  __device__ __forceinline__ explicit QuantRow(int held) : n(max(held, 0)), fresh(1), full(held < 0) {}
  // The slots that query t of the new ones sees end before this.
  __device__ __forceinline__ int end(int t) const {
    return t < fresh ? max(n - fresh + t + 1, 0) : 0;
  }
};

// Tokens of one part of a row that has n: whole blocks.
__device__ __forceinline__ int part_tokens(int n, int splits) {
  return ((n + splits - 1) / splits + kQuantBlock - 1) / kQuantBlock * kQuantBlock;
}

}  // namespace hattn
