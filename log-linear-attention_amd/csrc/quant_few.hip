// Attention of a few queries over a cache in 8 bits: one token a row, or some drafted ones.
//
// The queries of a row that share a key head, query t of head r as t * R + r, are the columns of
// 16x16x32 products, 16 or 32 to a workgroup:
//   S^T[slot][query] = K Q^T,  P = exp2(c ks S - m),  O^T[d][query] += vs V^T P^T
// on the codes themselves, which are exact in 16 bits: the scale ks of a block of keys multiplies
// its scores, and vs the block's part of the sum.  P is rounded to the inputs' type.
//
// The cache is read once, which bounds it: 64 rows of up to 9000 tokens, 32 heads of 128 in 8 groups, 115
// us (5.2 TB/s); one row of 262000, 4 key heads, 50 us (5.3 TB/s).  A row's slots are cut over
// workgroups (by its own count, read on the device), whose partial results a second kernel joins
// (6 to 8 us); a wave walks blocks of 64 slots, which have one scale, the next block's bytes in
// flight.  Both K and V come straight into registers, K in 16 bytes of a slot's row a lane (two
// steps of a product over d; Q is laid out alike), V in 8 bytes of each of 8 slots (4 where D <= 64),
// which become operands over the slots by byte permutations.  No wave waits for another before
// the end.
//
// A step's token is taken in by the one wave that walks its block, before its walk: a launch of
// its own took 3 to 5 us.
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

template <typename E, int DP, int NB, bool COMING>
__global__ __launch_bounds__(256, 2) void quant_few_kernel(QuantArgs p) {
  constexpr int W = DP / 64;   // words of a slot's V that a lane holds; 16-byte pieces of its K
  __shared__ __attribute__((aligned(16))) float part[4 * 16 * DP];
  __shared__ float sm[4][16 * NB], sl[4][16 * NB];
  const int lane = threadIdx.x & 63, ln = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = p.H / p.G;
  unsigned item = blockIdx.x;  // 32-bit divisions: 64-bit ones are hundreds of instructions
  const int split = item % (unsigned)p.splits;
  item /= (unsigned)p.splits;
  const int rb = item % (unsigned)p.rblocks, bg = (int)(item / (unsigned)p.rblocks);
  const int b = (unsigned)bg / (unsigned)p.G, g = bg - b * p.G;
  const QuantRow row(p, b, COMING);
  // for the join, which advances the counts
  if (COMING && split == 0 && g == 0 && threadIdx.x == 0) p.held[b] = row.full ? -1 : row.n;
  const int each = part_tokens(row.n, p.splits);
  const int from = (int)min((long)split * each, (long)row.n);
  const int first = rb * 16 * NB, last = min(first + 16 * NB, row.fresh * R) - 1;
  // nor does the join read parts without tokens, and queries of padding
  if (from >= row.n || first > last) return;
  const int least = row.end((unsigned)first / (unsigned)R);  // its first query's
  // Up to what the last one sees; a part behind that holds nothing, which the join reads.
  const int to = min(from + each, row.end((unsigned)last / (unsigned)R));
  if constexpr (COMING) {
    // by the wave that walks the new token's block, which no other reads
    if (to == row.n && ((to - 1 - from) / kQuantBlock & 3) == wave) {
      token_codes<E>(p, b, g, row.n - 1);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
  }

  int end[NB];
  bf16x8 qf[NB][W][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int query = first + 16 * nb + ln, t = (unsigned)query / (unsigned)R, r = query - t * R;
    end[nb] = row.end(t);
#pragma unroll
    for (int s = 0; s < W; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int d = 64 * s + 16 * lq + 8 * h;
        qf[nb][s][h] = t < row.fresh && d < p.D
                           ? *(const bf16x8*)((const __bf16*)p.q + b * p.qb + t * p.qt +
                                              (g * R + r) * p.qh + d)
                           : bf16x8{};
      }
  }
  const unsigned char* kc = p.kc + (long)bg * p.cap * p.D;
  const unsigned char* vc = p.vc + (long)bg * p.cap * p.D;
  const float* ks = p.ks + (long)bg * (p.cap / kQuantBlock);
  const float* vs = p.vs + (long)bg * (p.cap / kQuantBlock);

  uint4 K[4][W];
  unsigned V[2][2][4][W];
  float kscale, vscale;
  // Slots past the end read the last one, and pieces past D the row's first (Q is zero there, or
  // the result is not stored).
  const auto load_k = [&](int s0) __attribute__((always_inline)) {
    kscale = ks[s0 / kQuantBlock];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      const unsigned char* at = kc + (long)min(s0 + 16 * kt + ln, to - 1) * p.D;
#pragma unroll
      for (int s = 0; s < W; ++s) {
        const int d = 64 * s + 16 * lq;
        K[kt][s] = *(const uint4*)(at + (d < p.D ? d : 0));
      }
    }
  };
  const auto load_v = [&](int s0) __attribute__((always_inline)) {
    const int d = 4 * W * ln;
    vscale = vs[s0 / kQuantBlock];
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

  float m[NB], l[NB];
  floatx4 acc[NB][DP / 16];  // element d = 4 W (4 lq + i) + n of acc[..][n][i]
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb] = -3e38f;  // below every score; not -inf, whose difference is NaN
    l[nb] = 0.f;
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) acc[nb][n] = zero4();
  }
  int s0 = from + kQuantBlock * wave;
  if (s0 < to) {
    load_k(s0);
    load_v(s0);
  }
  for (; s0 < to; s0 += 4 * kQuantBlock) {
    const float unit = kscale * p.scale2;
    floatx4 s[NB][4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[nb][kt] = zero4();
#pragma unroll
      for (int c = 0; c < W; ++c) {
        const uint4 x = K[kt][c];
        const bf16x8 lo = widen8<E>(x.x, x.y), hi = widen8<E>(x.z, x.w);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          s[nb][kt] = mfma16<E>(lo, qf[nb][c][0], s[nb][kt]);
          s[nb][kt] = mfma16<E>(hi, qf[nb][c][1], s[nb][kt]);
        }
      }
    }
    if (s0 + 4 * kQuantBlock < to) load_k(s0 + 4 * kQuantBlock);
    const bool whole = s0 + kQuantBlock <= min(least, to);  // every query sees the block whole
    bf16x8 pf[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float top = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = s[nb][kt][i] * unit;
          if (!whole) x = s0 + 16 * kt + 4 * lq + i < end[nb] ? x : -INFINITY;
          s[nb][kt][i] = x;
          top = fmaxf(top, x);
        }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__any(top > m[nb] + Half<E>::kSlack)) {
        const float m2 = fmaxf(m[nb], top), shrink = __builtin_amdgcn_exp2f(m[nb] - m2);
        m[nb] = m2;
        l[nb] *= shrink;
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) acc[nb][n] *= shrink;
      }
      const float base = m[nb] - Half<E>::kLift;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[nb][kt][i] = __builtin_amdgcn_exp2f(s[nb][kt][i] - base);
          l[nb] += s[nb][kt][i];
        }
      pf[nb][0] = cat8e<E>(s[nb][0], s[nb][1]);
      pf[nb][1] = cat8e<E>(s[nb][2], s[nb][3]);
    }
    const float unit_v = vscale * Half<E>::kPart;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      floatx4 o[NB][4];
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
        for (int n = 0; n < 4; ++n) {
          const bf16x8 x = widen8<E>(lo[n], hi[n]);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            o[nb][n] = mfma16<E>(x, pf[nb][c], c ? o[nb][n] : zero4());
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[nb][4 * w + n][i] = fmaf(o[nb][n][i], unit_v, acc[nb][4 * w + n][i]);
    }
    if (s0 + 4 * kQuantBlock < to) load_v(s0 + 4 * kQuantBlock);
  }

  // the four waves' results, 16 queries at a time; 4-element piece c of a query lies at c ^ query
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    l[nb] += __shfl_xor(l[nb], 16, 64);
    l[nb] += __shfl_xor(l[nb], 32, 64);
    const int queries = p.T * R - first - 16 * nb;  // the others hold nothing
    if (nb > 0) __syncthreads();
    if (ln < queries) {
      float* mine = part + wave * 16 * DP + ln * DP;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const int piece = W * (4 * lq + i) + w;
          floatx4 x;
#pragma unroll
          for (int n = 0; n < 4; ++n) x[n] = acc[nb][4 * w + n][i];
          *(floatx4*)(mine + (piece ^ ln) * 4) = x;
        }
      if (lq == 0) {
        sm[wave][16 * nb + ln] = m[nb];
        sl[wave][16 * nb + ln] = l[nb];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(queries, 16) * (DP / 4); i += 256) {
      const int c = i / (DP / 4), d4 = i % (DP / 4), at = 16 * nb + c;
      if (4 * d4 >= p.D) continue;
      float top = sm[0][at];
#pragma unroll
      for (int w = 1; w < 4; ++w) top = fmaxf(top, sm[w][at]);
      floatx4 o = zero4();
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(sm[w][at] - top);
        const floatx4 x = *(const floatx4*)(part + (w * 16 + c) * DP + (d4 ^ c) * 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = fmaf(x[k], f, o[k]);
        sum += sl[w][at] * f;
      }
      const unsigned query = first + at, t = query / (unsigned)R;
      const long to_part =
          ((((long)b * p.T + t) * p.H + g * R + query - t * R)) * p.splits + split;
      *(floatx4*)(p.part + to_part * p.D + 4 * d4) = o;
      if (d4 == 0) {
        p.stat[2 * to_part] = top;
        p.stat[2 * to_part + 1] = sum;
      }
    }
  }
}

// Joins a query's partial results, those of the parts that have tokens, and counts a step's new
// tokens (no other workgroup reads the counts then): groups of lanes that hold
// 4 elements each take every n-th part, and the groups' sums meet in LDS, in order.
template <typename E>
__global__ __launch_bounds__(256) void quant_join_kernel(QuantArgs p) {
  __shared__ float share[kQuantSplits];
  __shared__ floatx4 sums[256];
  const unsigned bt = blockIdx.x / (unsigned)p.H;
  const long query = blockIdx.x;
  const int b = (int)(bt / (unsigned)p.T), t = (int)(bt - (unsigned)b * p.T), lane = threadIdx.x & 63;
  const QuantRow row = p.coming ? QuantRow(p.held[b]) : QuantRow(p, b);
  if (p.coming && blockIdx.x == bt * p.H && blockIdx.y == 0 && threadIdx.x == 0)
    p.counts[b] = min(max(p.counts[b], 0), 0x7ffffffe) + 1;
  __bf16* o = (__bf16*)p.o + query * p.D;
  if (row.end(t) == 0) {  // it sees nothing
    const float none = row.full && t < row.fresh ? __builtin_nanf("") : 0.f;
    if (threadIdx.x < p.D && blockIdx.y == 0) o[threadIdx.x] = to16<E>(none);
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
  const int per = 32 / gridDim.y, c0 = blockIdx.y * per;
  const int pieces = min(p.D / 4 - c0, per), groups = 256 / pieces;
  const int group = threadIdx.x / (unsigned)pieces, c = threadIdx.x - group * pieces;
  floatx4 x = zero4();
  if (group < groups) {
    const float* part = p.part + query * p.splits * p.D + 4 * (c0 + c);
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
  for (int i = 0; i < 4; ++i) y[i] = to16<E>(x[i] / (sum * Half<E>::kPart));
  *(bf16x4*)(o + 4 * (c0 + c)) = y;
}

}  // namespace hattn

hipError_t hattn_quant_few_launch(const QuantArgs& p, int dtype, hipStream_t stream) {
  using namespace hattn;
  const dim3 grid((unsigned)((long)p.B * p.G * p.rblocks * p.splits));
  const long queries = (long)p.T * (p.H / p.G);
#define RUN(E, DP, NB, C) \
  hipLaunchKernelGGL((quant_few_kernel<E, DP, NB, C>), grid, dim3(256), 0, stream, p)
#define GO(E, DP)                             \
  if (queries > 16) RUN(E, DP, 2, false);     \
  else if (p.coming) RUN(E, DP, 1, true);     \
  else RUN(E, DP, 1, false);
#define PICK(E)   \
  if (p.D <= 64) { \
    GO(E, 64)     \
  } else {        \
    GO(E, 128)    \
  }
  if (dtype == 1) {
    PICK(_Float16)
  } else {
    PICK(__bf16)
  }
#undef PICK
#undef GO
#undef RUN
  return hipGetLastError();
}

hipError_t hattn_quant_join_launch(const QuantArgs& p, int dtype, hipStream_t stream) {
  using namespace hattn;
  // where there are many parts, 64 elements a workgroup (256 parts of 32 queries: 6.6 us, with all
  // 128 elements 8.2; 4 parts of 2048 queries: 9.8, with all 6.2)
  const dim3 grid((unsigned)((long)p.B * p.T * p.H), p.D > 64 && p.splits > 32 ? 2 : 1);
  if (dtype == 1)
    hipLaunchKernelGGL((quant_join_kernel<_Float16>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((quant_join_kernel<__bf16>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}
