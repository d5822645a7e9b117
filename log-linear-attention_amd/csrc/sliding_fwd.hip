// Sliding-window attention forward: o = softmax(scale q k^T) v over the visible keys.
//
// A workgroup has 128 queries of one head, a wave 32 of them, and walks the list of their
// keys in tiles of 32.  One pass with the running maximum m and sum l of each row (both in
// the row's lane):
//   S^T = K Q^T,  P = exp2(c S - m),  O^T += V^T P^T,  c = scale log2(e).
// The accumulators are rescaled only where a row's maximum has grown by more than 8
// (powers of two) since it was last taken, so that most tiles skip that pass; P is then
// at most 2^8, and as exact in 16 bits as one below 1.  P is rounded to the inputs' type, which
// the matrix instructions take: o's error against 64 bits is 1.35 times that of one rounding.
//
// K and V lie in two buffers each, filled one tile ahead by asynchronous loads.  The tiles in
// the middle of the list, which all queries of the block see whole, have a loop of their own
// without masks.
//
// Tiles of 32 keys leave registers for three waves on a SIMD (D 128: 10 registers are spilled,
// outside the loop without masks) or four (D 64), whose products run beside each other's
// softmax: 552 us at B 1, T 16384, 16 heads of 128 in 4 groups, window 4096 (871 TFLOP/s),
// 210 us at B 4, T 8192, 16 heads of 64, window 1024 (613 TFLOP/s); tiles of 64 and two waves
// take 553 and 213 us.  The vector instructions bound it
// at D 64 (the matrix units are busy 29% of the time); at D 128 also the card's power: on
// zeros the same instructions take a fifth less time.
#include "sliding_device.h"

namespace hattn {

template <typename E, int DP>
__global__ __launch_bounds__(256, DP == 64 ? 4 : 3) void sliding_fwd_kernel(SlidingArgs p) {
  constexpr int BN = 32;
  // apart, not indexed, so that the compiler sees which of them a load in flight writes
  __shared__ __attribute__((aligned(16))) __bf16 K0[BN * DP], K1[BN * DP], V0[BN * DP], V1[BN * DP];
  const int lane = threadIdx.x & 63, ln = lane & 31, hf = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = p.H / p.G, nblk = (p.T + 127) / 128;
  const long item = work_item((long)p.B * p.H * nblk);
  if (item < 0) return;
  const int r = item % R, blk = item / R % nblk, bg = item / R / nblk;
  const int b = bg / p.G, g = bg % p.G, h = g * R + r, t0 = blk * 128;
  const int len = row_length(p, b);
  const int tw = t0 + 32 * wave, t = tw + ln;
  __bf16* out = (__bf16*)p.out + (((long)b * p.T + t) * p.H + h) * p.D;
  float* lse = p.lse ? p.lse + ((long)b * p.H + h) * p.T + t : nullptr;

  floatx16 acc[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = zero16();
  if (t0 >= len) {
    if (t < p.T) store_t<E, DP>(out, acc, 0.f, false, p.D);
    return;
  }
  const __bf16* k = (const __bf16*)p.k + b * p.kb + g * p.kh;
  const __bf16* v = (const __bf16*)p.v + b * p.vb + g * p.vh;
  bf16x8 qf[DP / 16];
  load_frags<DP>((const __bf16*)p.q + b * p.qb + h * p.qh + min(t, len - 1) * p.qt, p.D, qf);
  const KeyList<BN> keys(t0, 128, len, p.W, p.S);
  const int tiles = keys.tiles();
  const TileLoad<DP, BN, 4> tile(p.D);

  float m = -3e38f, l = 0.f;  // below every score; not -inf, whose difference is NaN
  const auto part = [&](auto MASK, int j, int kt, int kind, const __bf16* K, const __bf16* V)
                        __attribute__((always_inline)) {
    floatx16 s = zero16();
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) s = mfma32<E>(row_frag<DP>(K, 32 * kt, c), qf[c], s);
    if constexpr (MASK.value) {
      if (kind != kFull) {
        const TileMask seen(keys, j, t, p.W, p.S);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool in = seen(32 * kt + 8 * (i >> 2) + (i & 3));
          s[i] = in ? s[i] : -INFINITY;
        }
      }
    }
    float top = fmaxf(s[0], s[1]);
#pragma unroll
    for (int i = 2; i < 16; i += 2) top = max3(top, s[i], s[i + 1]);
    top = fmaxf(top, __shfl_xor(top, 32, 64)) * p.scale2;
    if (__any(top > m + 8.f)) {
      const float m2 = fmaxf(m, top), shrink = exp2_(m - m2);
      m = m2;
      l *= shrink;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) acc[dt] *= shrink;
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = exp2_(s[i] * p.scale2 - m);
      sum += s[i];
    }
    l += sum;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const bf16x8 pf = pack8<E>(s, c);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
        acc[dt] = mfma32<E>(tr32<DP>(V, 32 * kt + 16 * c, 32 * dt), pf, acc[dt]);
    }
  };
  const auto step = [&](auto MASK, int j, const __bf16* K, const __bf16* V, __bf16* Kl, __bf16* Vl)
                        __attribute__((always_inline)) {
    tile_barrier();
    if (j + 1 < tiles) {
      keys.load(tile, j + 1, k, p.kt, Kl);
      keys.load(tile, j + 1, v, p.vt, Vl);
    }
    int kind = kFull;
    if constexpr (MASK.value) kind = tile_kind(keys, j, tw, p.W, p.S);
    if (kind == kSkip) return;
#pragma unroll
    for (int kt = 0; kt < BN / 32; ++kt) part(MASK, j, kt, kind, K, V);
  };
  keys.load(tile, 0, k, p.kt, K0);
  keys.load(tile, 0, v, p.vt, V0);
  int j = 0;
  const auto pairs = [&](auto MASK) __attribute__((always_inline)) {
    step(MASK, j, K0, V0, K1, V1);
    if (j + 1 < tiles) step(MASK, j + 1, K1, V1, K0, V0);
  };
  const int lo = keys.first_whole(t0, 128, p.W), hi = keys.end_whole(t0);
  for (; j < tiles && !(j >= lo && j + 2 <= hi); j += 2) pairs(Bool<true>());
  for (; j + 2 <= hi; j += 2) pairs(Bool<false>());
  for (; j < tiles; j += 2) pairs(Bool<true>());
  l += __shfl_xor(l, 32, 64);
  if (t < p.T) store_t<E, DP>(out, acc, 1.f / l, t < len, p.D);
  if (lse && t < len && hf == 0) *lse = m + log2f(l);
}

}  // namespace hattn

hipError_t hattn_sliding_fwd_launch(const SlidingArgs& p, int dtype, hipStream_t stream) {
  using namespace hattn;
  const dim3 grid((unsigned)work_grid((long)p.B * p.H * ((p.T + 127) / 128)));
#define GO(E, DP) hipLaunchKernelGGL((sliding_fwd_kernel<E, DP>), grid, dim3(256), 0, stream, p)
  if (dtype == 1) {
    if (p.D <= 64) GO(_Float16, 64);
    else GO(_Float16, 128);
  } else {
    if (p.D <= 64) GO(__bf16, 64);
    else GO(__bf16, 128);
  }
#undef GO
  return hipGetLastError();
}
