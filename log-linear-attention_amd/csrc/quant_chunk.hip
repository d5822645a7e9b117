// Attention of a chunk of queries over a cache in 8 bits.
//
// The queries of a row that share a key head, query t of head r as t * R + r, are cut into
// blocks of 128, a wave 32 of them, so that a block's heads share each tile of keys.  One pass over
// the slots that any of the block sees, in tiles of 64, with the running maximum m and sum l of each
// query (both in the query's lane):
//   S^T = K Q^T,  P = exp2(c ks S - m),  O^T += vs V^T P^T,  c = scale log2(e)
// on the codes.  Codes are exact in 16 bits: the workgroup widens each tile once, between the
// registers that its bytes come to, one tile ahead, and LDS, in the layout of sliding_device.h.
// Tiles that all of the block's queries see whole have a loop without masks.
//
// 2048 queries of 32 heads of 128 after 30000 tokens take 931 to 954 us (1.12 to 1.09 PFLOP/s, of the 1.2
// that a large product reaches): the matrix units are busy in 53% of the cycles and the vector units, with
// the softmax, in 40%, at the clock that the card's power leaves.  In fp16 1012 us.  With heads of 64 608 us (0.86
// PFLOP/s; 36% and 49%), and 4 prompts of up to 4005 tokens of 16 heads of 64 149 us (0.60 PFLOP/s):
// there a CU has work for 60% of the time.  D = 80, 96 and 112 run the products of 128: 904 us and 917
// for the first two.  Tiles of 32, with a barrier each, took a tenth more; waves take priority during their
// products: without that 5% more.
//
// A block of 64 slots has one scale of K, which multiplies its scores, and one of V, which is folded into
// P's exponent.  In bf16 its range holds that.  In fp16 the sums are in units of a scale near
// the block's own (at least 2^-40: smaller values are 0 in the result), so that P is folded by
// at most 2^-8, which its lift makes up for.  In bf16 a workgroup that comes across a scale above 2^80 has its
// sums in units of 2^40, so that they stay finite, and a loop of its own (a test in each tile costs 1 to
// 2%).  Scales below 2^-60 are out of P's range there: their blocks count for the sum of the weights alone,
// their values, below 2^-52, as 0.
//
// Where blocks are few, a row's slots are cut over workgroups too, whose partial results
// quant_few.hip's second kernel joins.
#include "quant_device.h"
#include "sliding_device.h"

namespace hattn {

// x of lanes ln and ln + 32, in both; x comes from a vector instruction, not from a matrix product.
struct Halves {
  float lo, hi;
  __device__ __forceinline__ explicit Halves(float x) {
    lo = hi = x;
    // as assembly: the compiler takes the builtin's two results for one.  The instruction reads
    // what vector instructions wrote two states ago at the latest.
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(lo), "+v"(hi));
  }
};

constexpr float kLeastUnit = 0x1p-40f;                                 // fp16
constexpr float kLarge = 0x1p80f, kUnit = 0x1p40f, kLeast = 0x1p-60f;  // bf16

template <typename E, int DP>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void quant_chunk_kernel(QuantArgs p) {
  constexpr int BN = kQuantBlock, N = BN * DP / 2048;  // 16-byte pieces of K and V that a thread widens
  constexpr bool UNITS = __is_same(E, _Float16);
  // apart, not indexed, so that the compiler sees which of them is written
  __shared__ __attribute__((aligned(16))) __bf16 K0[BN * DP], K1[BN * DP], V0[BN * DP], V1[BN * DP];
  const int lane = threadIdx.x & 63, ln = lane & 31, hf = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = p.H / p.G;
  const long place = work_item((long)p.B * p.G * p.rblocks * p.splits);
  if (place < 0) return;
  const unsigned item = (unsigned)place;  // below 2^24
  const int split = item % (unsigned)p.splits;
  // the last queries, which see the most, first
  const int blk = p.rblocks - 1 - (int)(item / (unsigned)p.splits % (unsigned)p.rblocks);
  const int bg = (int)(item / (unsigned)p.splits / (unsigned)p.rblocks), b = bg / p.G, g = bg % p.G;
  const QuantRow row(p, b);
  const int each = part_tokens(row.n, p.splits);
  const int from = (int)min((long)split * each, (long)row.n);
  const int q0 = blk * 128, qw = q0 + 32 * wave, query = qw + ln;
  const int t = query / R, r = query - t * R, end = row.end(t);
  // what the block, and the wave, see at most; blocks and waves of padding see nothing
  const int to = q0 / R < row.fresh ? min(from + each, row.end(min((q0 + 127) / R, row.fresh - 1))) : 0;
  const int most = qw / R < row.fresh ? row.end(min((qw + 31) / R, row.fresh - 1)) : 0;
  const bool mine = t < p.T;
  const long at = ((long)b * p.T + t) * p.H + g * R + r;

  floatx16 acc[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = zero16();
  float m = -3e38f, l = 0.f;  // below every score; not -inf, whose difference is NaN
  float vunit = 1.f;          // what acc is in units of

  if (from < to) {
    const unsigned char* kc = p.kc + (long)bg * p.cap * p.D;
    const unsigned char* vc = p.vc + (long)bg * p.cap * p.D;
    const float* ks = p.ks + (long)bg * (p.cap / kQuantBlock);
    const float* vs = p.vs + (long)bg * (p.cap / kQuantBlock);
    bf16x8 qf[DP / 16];
    load_frags<DP>((const __bf16*)p.q + b * p.qb + min(t, row.fresh - 1) * p.qt +
                       (g * R + (t < row.fresh ? r : 0)) * p.qh, p.D, qf);

    // pieces pc of slots rw, rw + 4096 / DP, .. of a block: first K's, then V's
    constexpr int PIECES = DP / 16, ROWS = 256 / PIECES;
    const int rw = threadIdx.x / PIECES, pc = threadIdx.x % PIECES;
    uint4 raw[N];
    float kscale = ks[from / kQuantBlock], vscale = vs[from / kQuantBlock], knext, vnext;
    if (UNITS) vunit = fmaxf(vscale, kLeastUnit);
    // slots past the end read the last one, and pieces past D the row's first: Q is zero there, or the
    // result is not stored
    const auto fetch = [&](int s0) __attribute__((always_inline)) {
      knext = ks[s0 / kQuantBlock];
      vnext = vs[s0 / kQuantBlock];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const long o = (long)min(s0 + rw + i % (N / 2) * ROWS, to - 1) * p.D;
        raw[i] = *(const uint4*)((i < N / 2 ? kc : vc) + o + (16 * pc < p.D ? 16 * pc : 0));
      }
    };
    const auto put = [&](__bf16* K, __bf16* V) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = rw + i % (N / 2) * ROWS;
        __bf16* X = (i < N / 2 ? K : V) + r * DP;
        *(bf16x8*)(X + ((2 * pc) ^ swizzle<DP>(r)) * 8) = widen8<E>(raw[i].x, raw[i].y);
        *(bf16x8*)(X + ((2 * pc + 1) ^ swizzle<DP>(r)) * 8) = widen8<E>(raw[i].z, raw[i].w);
      }
      kscale = knext;
      vscale = vnext;
    };
    const auto part = [&](auto MASK, auto LARGE, int s0, const __bf16* K, const __bf16* V)
                          __attribute__((always_inline)) {
      float unit = kscale * p.scale2;
      floatx16 s[2];
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        bf16x8 kf[DP / 16];
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) kf[c] = row_frag<DP>(K, 32 * h, c);
        __builtin_amdgcn_sched_barrier(0);
        s[h] = zero16();
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) s[h] = mfma32<E>(kf[c], qf[c], s[h]);
      }
      if constexpr (MASK.value) {  // behind the product with unit, which may be 0
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int up = end - s0 - 32 * h - 4 * hf;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[h][i] = 8 * (i >> 2) + (i & 3) < up ? s[h][i] * unit : -INFINITY;
        }
        unit = 1.f;
      }
      __builtin_amdgcn_s_setprio(0);
      float top = fmaxf(s[0][0], s[0][1]);
#pragma unroll
      for (int i = 2; i < 16; i += 2) top = max3(top, s[0][i], s[0][i + 1]);
      float top1 = fmaxf(s[1][0], s[1][1]);
#pragma unroll
      for (int i = 2; i < 16; i += 2) top1 = max3(top1, s[1][i], s[1][i + 1]);
      const Halves both(fmaxf(top, top1));
      top = fmaxf(both.lo, both.hi) * unit;
      if (__any(top > m + Half<E>::kSlack)) {
        const float m2 = fmaxf(m, top), shrink = exp2_(m - m2);
        m = m2;
        l *= shrink;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) acc[dt] *= shrink;
      }
      if (UNITS && __any(vscale > vunit || (vscale < vunit * 0x1p-8f && vunit > kLeastUnit))) {
        const float next = fmaxf(vscale, kLeastUnit), by = fminf(vunit / next, 3e38f);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) acc[dt] *= by;
        vunit = next;
      }
      float ratio = UNITS ? vscale * __builtin_amdgcn_rcpf(vunit) : vscale;
      if constexpr (LARGE.value) {
        ratio *= 1.f / kUnit;
        if (vscale < kLeast) {  // the weights' sum, and P = 0
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            l += exp2_(fmaf(s[0][i], unit, -m)) + exp2_(fmaf(s[1][i], unit, -m));
            s[0][i] = s[1][i] = -INFINITY;
          }
          ratio = unit = 1.f;
        }
      }
      const float base = m - Half<E>::kLift - __builtin_amdgcn_logf(ratio);
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[h][i] = exp2_(fmaf(s[h][i], unit, -base));
          sum += s[h][i];
        }
      }
      l = fmaf(sum, __builtin_amdgcn_rcpf(ratio), l);
      __builtin_amdgcn_s_setprio(1);
      const bf16x8 pf[4] = {pack8<E>(s[0], 0), pack8<E>(s[0], 1), pack8<E>(s[1], 0), pack8<E>(s[1], 1)};
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          acc[dt] = mfma32<E>(tr32<DP>(V, 16 * c, 32 * dt), pf[c], acc[dt]);
      __builtin_amdgcn_s_setprio(0);
    };
    const auto step = [&](auto MASK, auto LARGE, int s0, const __bf16* K, const __bf16* V, __bf16* Kn,
                          __bf16* Vn) __attribute__((always_inline)) {
      __syncthreads();
      const bool more = s0 + BN < to;
      if (more) fetch(s0 + BN);
      if (!MASK.value || s0 < most) part(MASK, LARGE, s0, K, V);
      if (more) put(Kn, Vn);
    };
    float largest = 0.f;  // of the scales of V
    if constexpr (!UNITS) {
      const int end_block = (to - 1) / kQuantBlock;
      int i = from / kQuantBlock + lane;
      largest = vs[min(i, end_block)];
      while ((i += 64) <= end_block) largest = fmaxf(largest, vs[i]);
    }
    fetch(from);
    put(K0, V0);
    const bool large = !UNITS && __any(largest > kLarge);
    int s0 = from;
    const auto pair = [&](auto MASK, auto LARGE) __attribute__((always_inline)) {
      step(MASK, LARGE, s0, K0, V0, K1, V1);
      if (!MASK.value || s0 + BN < to) step(MASK, LARGE, s0 + BN, K1, V1, K0, V0);
    };
    if (!large) {
      // blocks that all queries see whole, in pairs, then those that need masks
      for (const int whole = min(row.end(q0 / R), to); s0 + 2 * BN <= whole; s0 += 2 * BN)
        pair(Bool<false>(), Bool<false>());
      for (; s0 < to; s0 += 2 * BN) pair(Bool<true>(), Bool<false>());
    } else if constexpr (!UNITS) {
      vunit = kUnit;
      for (bool odd = false; s0 < to; s0 += BN, odd = !odd)
        step(Bool<true>(), Bool<true>(), s0, odd ? K1 : K0, odd ? V1 : V0, odd ? K0 : K1, odd ? V0 : V1);
    }
    const Halves both(l);
    l = both.lo + both.hi;
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
      store_t<E, DP>(o, acc, vunit / l, end > 0, p.D);
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
      for (int j = 0; j < 4; ++j) x[j] = acc[dt][4 * i + j] * (vunit * Half<E>::kPart);
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
