// Attention of a chunk of queries over a cache in 8 bits.
//
// The queries of a row that share a key head, query t of head r as t * R + r, are cut into
// blocks of 128, a wave 32 of them, so that a block's heads share each tile of keys.  One pass over the slots
// that any of the block sees, in tiles of 32, with the running maximum m and sum l of each
// query (both in the query's lane):
//   S^T = K Q^T,  P = exp2(c ks S - m),  O^T += vs V^T P^T,  c = scale log2(e)
// on the codes.  Codes are exact in 16 bits: the workgroup widens each tile once, between the
// registers that its bytes come to, one tile ahead, and LDS, in the layout of sliding_device.h.
// A tile has one scale of K, which multiplies its scores.  Its scale of V is folded into P's
// exponent in bf16, whose range holds it; in fp16, whose range does not, it multiplies the tile's part
// of the sum.
//
// Where blocks are few, a row's slots are cut over workgroups too, whose partial results
// quant_few.hip's second kernel joins.
#include "quant_device.h"
#include "sliding_device.h"

namespace hattn {

template <typename E, int DP>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void quant_chunk_kernel(QuantArgs p) {
  constexpr int BN = 32;
  constexpr bool FOLD = !__is_same(E, _Float16);
  __shared__ __attribute__((aligned(16))) __bf16 K0[BN * DP], K1[BN * DP], V0[BN * DP], V1[BN * DP];
  const int lane = threadIdx.x & 63, ln = lane & 31, hf = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = p.H / p.G;
  const long item = work_item((long)p.B * p.G * p.rblocks * p.splits);
  if (item < 0) return;
  const int split = item % p.splits;
  // the last queries, which see the most, first
  const int blk = p.rblocks - 1 - (int)(item / p.splits % p.rblocks);
  const int bg = (int)(item / p.splits / p.rblocks), b = bg / p.G, g = bg % p.G;
  const QuantRow row(p, b);
  const int each = part_tokens(row.n, p.splits);
  const int from = (int)min((long)split * each, (long)row.n);
  const int q0 = blk * 128, qw = q0 + 32 * wave, query = qw + ln;
  const int t = query / R, r = query - t * R, end = row.end(t);
  // what the block, and the wave, see at most, and what each of the wave's queries sees; blocks
  // and waves of padding see nothing
  const int to = q0 / R < row.fresh ? min(from + each, row.end(min((q0 + 127) / R, row.fresh - 1))) : 0;
  const int most = qw / R < row.fresh ? row.end(min((qw + 31) / R, row.fresh - 1)) : 0;
  const int least = row.end(qw / R);
  const bool mine = t < p.T;
  const long at = ((long)b * p.T + t) * p.H + g * R + r;

  floatx16 acc[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = zero16();
  float m = -3e38f, l = 0.f;  // below every score; not -inf, whose difference is NaN

  if (from < to) {
    const unsigned char* kc = p.kc + (long)bg * p.cap * p.D;
    const unsigned char* vc = p.vc + (long)bg * p.cap * p.D;
    const float* ks = p.ks + (long)bg * (p.cap / kQuantBlock);
    const float* vs = p.vs + (long)bg * (p.cap / kQuantBlock);
    bf16x8 qf[DP / 16];
    load_frags<DP>((const __bf16*)p.q + b * p.qb + min(t, row.fresh - 1) * p.qt +
                       (g * R + (t < row.fresh ? r : 0)) * p.qh, p.D, qf);

    // 16 bytes of one slot's K or V: with D 128 both from every thread, else one
    constexpr int PIECES = DP / 16, N = DP / 64;
    const int rw = threadIdx.x / PIECES % BN, pc = threadIdx.x % PIECES;
    uint4 raw[N];
    const auto fetch = [&](int s0) __attribute__((always_inline)) {
      const long o = (long)min(s0 + rw, to - 1) * p.D + 16 * pc;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool isv = N == 2 ? i == 1 : threadIdx.x >= BN * PIECES;
        raw[i] = 16 * pc < p.D ? *(const uint4*)((isv ? vc : kc) + o) : uint4{};
      }
    };
    const auto put = [&](__bf16* K, __bf16* V) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool isv = N == 2 ? i == 1 : threadIdx.x >= BN * PIECES;
        __bf16* X = (isv ? V : K) + rw * DP;
        *(bf16x8*)(X + ((2 * pc) ^ swizzle<DP>(rw)) * 8) = widen8<E>(raw[i].x, raw[i].y);
        *(bf16x8*)(X + ((2 * pc + 1) ^ swizzle<DP>(rw)) * 8) = widen8<E>(raw[i].z, raw[i].w);
      }
    };
    const auto part = [&](auto MASK, int s0, const __bf16* K, const __bf16* V)
                          __attribute__((always_inline)) {
      const float kscale = ks[s0 / kQuantBlock] * p.scale2, vscale = vs[s0 / kQuantBlock];
      floatx16 s = zero16();
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) s = mfma32<E>(row_frag<DP>(K, 0, c), qf[c], s);
      if constexpr (MASK.value) {
        const int up = end - s0 - 4 * hf;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 8 * (i >> 2) + (i & 3) < up ? s[i] : -INFINITY;
      }
      float top = fmaxf(s[0], s[1]);
#pragma unroll
      for (int i = 2; i < 16; i += 2) top = max3(top, s[i], s[i + 1]);
      top = fmaxf(top, __shfl_xor(top, 32, 64)) * kscale;
      if (__any(top > m + 8.f)) {
        const float m2 = fmaxf(m, top), shrink = exp2_(m - m2);
        m = m2;
        l *= shrink;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) acc[dt] *= shrink;
      }
      const float base = FOLD ? m - log2f(vscale) : m;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = exp2_(fmaf(s[i], kscale, -base));
        sum += s[i];
      }
      l += FOLD ? sum / vscale : sum;
      const bf16x8 pf[2] = {pack8<E>(s, 0), pack8<E>(s, 1)};
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        floatx16 o = FOLD ? acc[dt] : zero16();
#pragma unroll
        for (int c = 0; c < 2; ++c) o = mfma32<E>(tr32<DP>(V, 16 * c, 32 * dt), pf[c], o);
        if constexpr (FOLD) {
          acc[dt] = o;
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[dt][i] = fmaf(o[i], vscale, acc[dt][i]);
        }
      }
    };
    const auto step = [&](int s0, const __bf16* K, const __bf16* V, __bf16* Kn, __bf16* Vn)
                          __attribute__((always_inline)) {
      __syncthreads();
      const bool more = s0 + BN < to;
      if (more) fetch(s0 + BN);
      if (s0 + BN <= least) part(Bool<false>(), s0, K, V);
      else if (s0 < most) part(Bool<true>(), s0, K, V);
      if (more) put(Kn, Vn);
    };
    fetch(from);
    put(K0, V0);
    for (int s0 = from; s0 < to; s0 += 2 * BN) {
      step(s0, K0, V0, K1, V1);
      if (s0 + BN < to) step(s0 + BN, K1, V1, K0, V0);
    }
    l += __shfl_xor(l, 32, 64);
  }

  if (p.splits == 1) {
    if (!mine) return;
    __bf16* o = (__bf16*)p.o + at * p.D;
    if (row.full && t < row.fresh) {
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] = __builtin_nanf("");
      store_t<E, DP>(o, acc, 1.f, true, p.D);
    } else {
      store_t<E, DP>(o, acc, 1.f / l, end > 0, p.D);
    }
    return;
  }
  // the join reads the parts that hold tokens of the row, whether this block sees them or not
  if (!mine || from >= row.n) return;
  const long to_part = at * p.splits + split;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 32 * dt + 8 * i + 4 * hf;
      floatx4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = acc[dt][4 * i + j];
      if (d < p.D) *(floatx4*)(p.part + to_part * p.D + d) = x;
    }
  if (hf == 0) {
    p.stat[2 * to_part] = m;
    p.stat[2 * to_part + 1] = l;
  }
}

}  // namespace hattn

hipError_t hattn_quant_chunk_launch(const QuantArgs& p, int dtype, hipStream_t stream) {
  using namespace hattn;
  const dim3 grid((unsigned)work_grid((long)p.B * p.G * p.rblocks * p.splits));
#define GO(E, DP) hipLaunchKernelGGL((quant_chunk_kernel<E, DP>), grid, dim3(256), 0, stream, p)
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
