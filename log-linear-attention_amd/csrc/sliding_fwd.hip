// Sliding-window attention forward: o = softmax(scale q k^T) v over the visible keys.
//
// A workgroup has 128 queries of one head, a wave 32 of them, and walks the list of
// their keys in tiles of 64, double-buffered in LDS by asynchronous loads.  One pass
// with the running maximum m and sum l of each row (both in the row's lane):
//   S^T = K Q^T,  P = exp2(c S - m),  O^T += V^T P^T,  c = scale log2(e).
// The accumulators are rescaled only where a row's maximum has grown by more than 8
// (powers of two) since it was last taken, so that most tiles skip that pass; P is then
// at most 2^8, and as exact in 16 bits as one below 1.
#include "sliding_device.h"

namespace hattn {

template <typename E, int DP>
__global__ __launch_bounds__(256, 2) void sliding_fwd_kernel(SlidingArgs p) {
  __shared__ __attribute__((aligned(16))) __bf16 K0[64 * DP], V0[64 * DP], K1[64 * DP], V1[64 * DP];
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
    if (t < p.T) store_t<E, DP>(out, acc, 0.f, p.D);
    return;
  }
  const __bf16* k = (const __bf16*)p.k + b * p.kb + g * p.kh;
  const __bf16* v = (const __bf16*)p.v + b * p.vb + g * p.vh;
  bf16x8 qf[DP / 16];
  load_frags<DP>((const __bf16*)p.q + b * p.qb + h * p.qh + min(t, len - 1) * p.qt, p.D, qf);
  const KeyList keys(t0, len, p.W, p.S);
  const int tiles = (keys.n + 63) / 64;

  const auto stage = [&](int j, __bf16* K, __bf16* V) __attribute__((always_inline)) {
    constexpr int RPI = 512 / DP, N = DP / 32;  // rows a load, loads a wave
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = wave * N + i, row = at * RPI + lane / (DP / 8);
      const long pos = keys.pos(min(64 * j + row, keys.n - 1));
      load_rows<DP>(k + pos * p.kt, row, p.D, K + at * 512);
      load_rows<DP>(v + pos * p.vt, row, p.D, V + at * 512);
    }
  };

  float m = -1e30f, l = 0.f;
  const auto step = [&](int j, const __bf16* K, const __bf16* V, __bf16* Kn, __bf16* Vn)
                        __attribute__((always_inline)) {
    tile_barrier();
    if (j + 1 < tiles) stage(j + 1, Kn, Vn);
    const int kind = tile_kind(keys, j, tw, p.W, p.S);
    if (kind == kSkip) return;
    floatx16 s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      s[kt] = zero16();
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) s[kt] = mfma32<E>(row_frag<DP>(K, 32 * kt, c), qf[c], s[kt]);
    }
    if (kind == kMask) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int slot = 64 * j + 32 * kt + 8 * (i >> 2) + 4 * hf + (i & 3);
          const int pos = keys.pos(slot);
          const bool seen = slot < keys.n && pos <= t && (pos + p.W > t || pos < p.S);
          s[kt][i] = seen ? s[kt][i] : -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = fmaxf(top, s[i >> 4][i & 15]);
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
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[kt][i] = exp2_(s[kt][i] * p.scale2 - m);
        sum += s[kt][i];
      }
    l += sum;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bf16x8 pf = pack8<E>(s[kt], c);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
          acc[dt] = mfma32<E>(tr32<DP>(V, 32 * kt + 16 * c, 32 * dt), pf, acc[dt]);
      }
  };
  // the two buffers are four arrays and the loop is unrolled by two, so that the compiler
  // sees that the loads in flight write none of the arrays that are read meanwhile
  stage(0, K0, V0);
  for (int j = 0; j < tiles; j += 2) {
    step(j, K0, V0, K1, V1);
    if (j + 1 < tiles) step(j + 1, K1, V1, K0, V0);
  }
  l += __shfl_xor(l, 32, 64);
  if (t < p.T) store_t<E, DP>(out, acc, t < len ? 1.f / l : 0.f, p.D);
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
