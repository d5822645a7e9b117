// Attention of a few queries over a cache in 8 bits: one token a row, or some drafted ones.
//
// The queries of a row that share a key head, query t of head r as t * R + r, are the columns of
// 16x16x32 products, 16 to a workgroup:
//   S^T[slot][query] = K Q^T,  P = exp2(c ks S - m),  O^T[d][query] += vs V^T P^T
// on the codes themselves, which are exact in 16 bits: the scale ks of a block of keys multiplies
// its scores, and vs the block's part of the sum.  P is rounded to the inputs' type.
//
// The cache is read once, which bounds it.  A row's slots are cut over workgroups (by its own
// count, read on the device), whose partial results a second kernel joins; a wave walks
// blocks of 64 slots, which have one scale.  Both K and V come straight into registers, K in 16
// bytes of a slot's row a lane (two steps of a product over d; Q is laid out alike), V in
// 8 bytes of each of 8 slots (4 where D <= 64), which become operands over the slots by byte
// permutations.  No wave waits for another before the end.
#include "quant_device.h"

namespace hattn {

// The four 4-byte rows of a 4 x 4 block, transposed.
__device__ __forceinline__ void transpose4(const unsigned (&a)[4], unsigned (&t)[4]) {
  const unsigned x0 = __builtin_amdgcn_perm(a[1], a[0], 0x05010400);
  const unsigned x1 = __builtin_amdgcn_perm(a[1], a[0], 0x07030602);
  const unsigned y0 = __builtin_amdgcn_perm(a[3], a[2], 0x05010400);
  const unsigned y1 = __builtin_amdgcn_perm(a[3], a[2], 0x07030602);
  t[0] = __builtin_amdgcn_perm(y0, x0, 0x05040100);
  t[1] = __builtin_amdgcn_perm(y0, x0, 0x07060302);
  t[2] = __builtin_amdgcn_perm(y1, x1, 0x05040100);
  t[3] = __builtin_amdgcn_perm(y1, x1, 0x07060302);
}

template <typename E, int DP>
__global__ __launch_bounds__(256, 2) void quant_few_kernel(QuantArgs p) {
  constexpr int W = DP / 64;   // words of a slot's V that a lane holds; 16-byte pieces of its K
  __shared__ __attribute__((aligned(16))) float part[4 * 16 * DP];
  __shared__ float sm[4][16], sl[4][16];
  const int lane = threadIdx.x & 63, ln = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = p.H / p.G;
  long item = blockIdx.x;
  const int split = item % p.splits;
  item /= p.splits;
  const int rb = item % p.rblocks, bg = (int)(item / p.rblocks), b = bg / p.G, g = bg % p.G;
  const QuantRow row(p, b);
  const int each = part_tokens(row.n, p.splits);
  const int from = (int)min((long)split * each, (long)row.n), to = min(from + each, row.n);
  const int col = rb * 16 + ln, t = col / R, r = col - t * R;  // this lane's query
  const int end = row.end(t), least = row.end(rb * 16 / R);    // the block's first sees least
  if (from >= to) return;                                      // nor does the join read it

  bf16x8 qf[W][2];
#pragma unroll
  for (int s = 0; s < W; ++s)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int d = 64 * s + 16 * lq + 8 * h;
      qf[s][h] = t < row.fresh && d < p.D
                     ? *(const bf16x8*)((const __bf16*)p.q + b * p.qb + t * p.qt +
                                        (g * R + r) * p.qh + d)
                     : bf16x8{};
    }
  const unsigned char* kc = p.kc + (long)bg * p.cap * p.D;
  const unsigned char* vc = p.vc + (long)bg * p.cap * p.D;
  const float* ks = p.ks + (long)bg * (p.cap / kQuantBlock);
  const float* vs = p.vs + (long)bg * (p.cap / kQuantBlock);

  uint4 K[4][W];
  unsigned V[2][2][4][W];
  // slots past the end read the last one
  const auto load_k = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      const unsigned char* at = kc + (long)min(s0 + 16 * kt + ln, to - 1) * p.D;
#pragma unroll
      for (int s = 0; s < W; ++s) {
        const int d = 64 * s + 16 * lq;
        K[kt][s] = d < p.D ? *(const uint4*)(at + d) : uint4{};
      }
    }
  };
  const auto load_v = [&](int s0) __attribute__((always_inline)) {
    const int d = 4 * W * ln;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int slot = min(s0 + 32 * c + 16 * h + 4 * lq + i, to - 1);
          const unsigned char* at = vc + (long)slot * p.D + (d < p.D ? d : 0);
          if constexpr (W == 2) {
            const uint2 x = *(const uint2*)at;
            V[c][h][i][0] = x.x;
            V[c][h][i][1] = x.y;
          } else {
            V[c][h][i][0] = *(const unsigned*)at;
          }
        }
  };

  float m = -3e38f, l = 0.f;  // below every score; not -inf, whose difference is NaN
  floatx4 acc[DP / 16];       // element d = 4 W (4 lq + i) + n of acc[n][i]
#pragma unroll
  for (int n = 0; n < DP / 16; ++n) acc[n] = zero4();
  int s0 = from + kQuantBlock * wave;
  if (s0 < to) {
    load_k(s0);
    load_v(s0);
  }
  for (; s0 < to; s0 += 4 * kQuantBlock) {
    const float kscale = ks[s0 / kQuantBlock] * p.scale2, vscale = vs[s0 / kQuantBlock];
    floatx4 s[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      s[kt] = zero4();
#pragma unroll
      for (int c = 0; c < W; ++c) {
        const uint4 x = K[kt][c];
        s[kt] = mfma16<E>(widen8<E>(x.x, x.y), qf[c][0], s[kt]);
        s[kt] = mfma16<E>(widen8<E>(x.z, x.w), qf[c][1], s[kt]);
      }
    }
    if (s0 + 4 * kQuantBlock < to) load_k(s0 + 4 * kQuantBlock);
    const bool whole = s0 + kQuantBlock <= min(least, to);  // every query sees the block whole
    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[kt][i] *= kscale;
        if (!whole) s[kt][i] = s0 + 16 * kt + 4 * lq + i < end ? s[kt][i] : -INFINITY;
        top = fmaxf(top, s[kt][i]);
      }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top > m + 8.f)) {
      const float m2 = fmaxf(m, top), shrink = __builtin_amdgcn_exp2f(m - m2);
      m = m2;
      l *= shrink;
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) acc[n] *= shrink;
    }
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[kt][i] = __builtin_amdgcn_exp2f(s[kt][i] - m);
        l += s[kt][i];
      }
    const bf16x8 pf[2] = {cat8e<E>(s[0], s[1]), cat8e<E>(s[2], s[3])};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      floatx4 o[4];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        unsigned lo[4], hi[4], a[4], z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] = V[c][0][i][w];
          z[i] = V[c][1][i][w];
        }
        transpose4(a, lo);
        transpose4(z, hi);
#pragma unroll
        for (int n = 0; n < 4; ++n)
          o[n] = mfma16<E>(widen8<E>(lo[n], hi[n]), pf[c], c ? o[n] : zero4());
      }
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[4 * w + n][i] = fmaf(o[n][i], vscale, acc[4 * w + n][i]);
    }
    if (s0 + 4 * kQuantBlock < to) load_v(s0 + 4 * kQuantBlock);
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // the four waves' results; 4-element piece c of a query lies at c ^ query
  float* mine = part + wave * 16 * DP + ln * DP;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int piece = W * (4 * lq + i) + w;
      floatx4 x;
#pragma unroll
      for (int n = 0; n < 4; ++n) x[n] = acc[4 * w + n][i];
      *(floatx4*)(mine + (piece ^ ln) * 4) = x;
    }
  if (lq == 0) {
    sm[wave][ln] = m;
    sl[wave][ln] = l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * DP / 4; i += 256) {
    const int c = i / (DP / 4), d4 = i % (DP / 4), query = rb * 16 + c, tq = query / R;
    if (tq >= p.T || 4 * d4 >= p.D) continue;
    float top = sm[0][c];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, sm[w][c]);
    floatx4 o = zero4();
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w][c] - top);
      const floatx4 x = *(const floatx4*)(part + (w * 16 + c) * DP + (d4 ^ c) * 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = fmaf(x[k], f, o[k]);
      sum += sl[w][c] * f;
    }
    const long at = ((((long)b * p.T + tq) * p.H + g * R + query - tq * R)) * p.splits + split;
    *(floatx4*)(p.part + at * p.D + 4 * d4) = o;
    if (d4 == 0) {
      p.stat[2 * at] = top;
      p.stat[2 * at + 1] = sum;
    }
  }
}

// Joins a query's partial results, those of the parts that have tokens: groups of lanes that hold
// 4 elements each take every n-th part, and the groups' sums meet in LDS, in order.
template <typename E>
__global__ __launch_bounds__(256) void quant_join_kernel(QuantArgs p) {
  __shared__ float share[kQuantSplits];
  __shared__ floatx4 sums[256];
  const long query = blockIdx.x, bt = query / p.H;
  const int b = (int)(bt / p.T), t = (int)(bt - (long)b * p.T), lane = threadIdx.x & 63;
  const QuantRow row(p, b);
  __bf16* o = (__bf16*)p.o + query * p.D;
  if (row.end(t) == 0) {  // it sees nothing
    const float none = row.full && t < row.fresh ? __builtin_nanf("") : 0.f;
    if (threadIdx.x < p.D) o[threadIdx.x] = to16<E>(none);
    return;
  }
  const int each = part_tokens(row.n, p.splits), live = (row.n + each - 1) / each;
  const float* stat = p.stat + query * p.splits * 2;
  // every wave takes the maximum and the sum, a part a lane
  float top = -INFINITY, sum = 0.f;
  for (int s = lane; s < live; s += 64) top = fmaxf(top, stat[2 * s]);
#pragma unroll
  for (int k = 1; k < 64; k *= 2) top = fmaxf(top, __shfl_xor(top, k, 64));
  for (int s = lane; s < live; s += 64) {
    const float f = __builtin_amdgcn_exp2f(stat[2 * s] - top);
    if (threadIdx.x < 64) share[s] = f;
    sum += stat[2 * s + 1] * f;
  }
#pragma unroll
  for (int k = 1; k < 64; k *= 2) sum += __shfl_xor(sum, k, 64);
  __syncthreads();
  const int pieces = p.D / 4, groups = 256 / pieces;
  const int group = threadIdx.x / pieces, c = threadIdx.x - group * pieces;
  floatx4 x = zero4();
  if (group < groups) {
    const float* part = p.part + query * p.splits * p.D + 4 * c;
#pragma unroll 4
    for (int s = group; s < live; s += groups) {
      const floatx4 y = *(const floatx4*)(part + (long)s * p.D);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = fmaf(y[i], share[s], x[i]);
    }
    sums[threadIdx.x] = x;
  }
  __syncthreads();
  if (group != 0) return;
  for (int s = 1; s < min(groups, live); ++s) x += sums[s * pieces + c];
  bf16x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = to16<E>(x[i] / sum);
  *(bf16x4*)(o + 4 * c) = y;
}

}  // namespace hattn

hipError_t hattn_quant_few_launch(const QuantArgs& p, int dtype, hipStream_t stream) {
  using namespace hattn;
  const dim3 grid((unsigned)((long)p.B * p.G * p.rblocks * p.splits));
#define GO(E, DP) hipLaunchKernelGGL((quant_few_kernel<E, DP>), grid, dim3(256), 0, stream, p)
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

hipError_t hattn_quant_join_launch(const QuantArgs& p, int dtype, hipStream_t stream) {
  using namespace hattn;
  const dim3 grid((unsigned)((long)p.B * p.T * p.H));
  if (dtype == 1)
    hipLaunchKernelGGL((quant_join_kernel<_Float16>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((quant_join_kernel<__bf16>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}
