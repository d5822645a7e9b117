// Sliding-window attention, one token per row against its cache, and the cache's filling.
//
// The cache of a row and key head is sinks + window slots: slot s < S holds token s, slot
// S + i the last token p >= S with p - S = i modulo W.  After the new token is in, the slots
// [0, min(count + 1, S + W)) are exactly the tokens that it sees, and softmax does not ask
// for their order, so the step is plain attention over one run of slots.
//
// The step reads K and V once per key head, which bounds it: the heads of a group share a
// workgroup as the 16 columns of its products, and a row's slots are cut over several
// workgroups (by its own count, read on the device) whose partial results a second kernel
// joins.  Each wave walks its own tiles of 32 slots: K comes straight into operand
// registers, V through a buffer of the wave's own in LDS, both one tile ahead, and no wave
// waits for another before the end.
//
// P is rounded to the inputs' type, as in the forward.  150 us at B 64, 32 heads of 128 in 8 groups, window 4096, 9000 tokens seen at most: 5.6 TB/s.
//
//   S^T[slot][head] = K Q^T,  P = exp2(c S - m),  O^T[d][head] += V^T P^T
// (16x16x32 MFMAs in the layouts of common.h).  The new token is read from the inputs, by
// every workgroup; one of them writes it into its slot, which no other reads.  The counts
// advance in the second kernel.
#include "common.h"
#include "sliding_step.h"

namespace hattn {

// As the tiles of sliding_device.h, for reads of 4 rows x 16 columns by each 16 lanes: 8 rows, two
// pieces meet every bank once.
template <int DP>
__device__ __forceinline__ int swizzle16(int row) {
  if constexpr (DP == 128) return (row & 7) << 1;
  else return (row >> 1 & 3) << 1;
}

// Rows r0 + 4 lq + j and r0 + 16 + 4 lq + j (j = 0..3) of column c0 + ln.
template <int DP>
__device__ __forceinline__ bf16x8 tr16(const __bf16* X, int c0) {
  const int lane = threadIdx.x & 63, row = 4 * (lane >> 4) + (lane >> 2 & 3);
  const int col = c0 + 4 * (lane & 3);
  const __bf16* at = X + row * DP + (col >> 3 ^ swizzle16<DP>(row)) * 8 + (col & 7);
  const bf16x4 lo = ds_read_tr(at), hi = ds_read_tr(at + 16 * DP);  // swizzle16 has period 8
  return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

template <typename E, int DP>
__global__ __launch_bounds__(256, 2) void sliding_step_kernel(SlidingStepArgs p) {
  __shared__ __attribute__((aligned(16))) __bf16 V0[4 * 32 * DP], V1[4 * 32 * DP];
  __shared__ float sm[4][16], sl[4][16];
  const int lane = threadIdx.x & 63, ln = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = p.H / p.G;
  int item = blockIdx.x;
  const int split = item % p.splits;
  item /= p.splits;
  const int rb = item % p.rblocks, bg = item / p.rblocks, b = bg / p.G, g = bg % p.G;
  const int count = max(p.counts[b], 0);
  const int fresh = count < p.S ? count : p.S + (count - p.S) % p.W;
  const int n = min(count, p.S + p.W - 1) + 1;
  const int each = ((n + p.splits - 1) / p.splits + 31) & ~31;
  const int from = split * each, to = min(from + each, n);
  const int head = rb * 16 + ln;  // of the group; columns past R are zero and not stored
  const long cache = (long)bg * (p.S + p.W) * p.D;
  const __bf16 *kc = (const __bf16*)p.kc + cache, *vc = (const __bf16*)p.vc + cache;
  const __bf16 *kn = (const __bf16*)p.k + (long)bg * p.D, *vn = (const __bf16*)p.v + (long)bg * p.D;

  if (split == 0 && rb == 0)
    for (int i = threadIdx.x; i < p.D; i += 256) {
      ((__bf16*)p.kc)[cache + (long)fresh * p.D + i] = kn[i];
      ((__bf16*)p.vc)[cache + (long)fresh * p.D + i] = vn[i];
    }

  bf16x8 qf[DP / 32];
#pragma unroll
  for (int s = 0; s < DP / 32; ++s) {
    const int d = 32 * s + 8 * lq;
    qf[s] = head < R && d < p.D
                ? *(const bf16x8*)((const __bf16*)p.q + ((long)b * p.H + g * R + head) * p.D + d)
                : bf16x8{};
  }

  struct KTile {
    bf16x8 f[2][DP / 32];
  };
  // slots past the end read the last one; pieces past D read the row's first
  const auto load = [&](int s0, KTile& K, __bf16* V) __attribute__((always_inline)) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int slot = min(s0 + 16 * kt + ln, to - 1);
      const __bf16* row = slot == fresh ? kn : kc + (long)slot * p.D;
#pragma unroll
      for (int s = 0; s < DP / 32; ++s) {
        const int d = 32 * s + 8 * lq;
        K.f[kt][s] = *(const bf16x8*)(row + (d < p.D ? d : 0));
      }
    }
    constexpr int RPI = 512 / DP;
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
      const int rw = i * RPI + lane / (DP / 8), slot = min(s0 + rw, to - 1);
      const __bf16* row = slot == fresh ? vn : vc + (long)slot * p.D;
      const int c = lane % (DP / 8) ^ swizzle16<DP>(rw);
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(row + (c * 8 < p.D ? c * 8 : 0)),
          (__attribute__((address_space(3))) void*)(V + wave * 32 * DP + i * 512), 16, 0, 0);
    }
  };
  float m = -3e38f, l = 0.f;  // below every score; not -inf, whose difference is NaN
  floatx4 acc[DP / 16];
#pragma unroll
  for (int dt = 0; dt < DP / 16; ++dt) acc[dt] = zero4();
  const auto step = [&](int s0, const KTile& K, const __bf16* V) __attribute__((always_inline)) {
    floatx4 s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      s[kt] = zero4();
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) s[kt] = mfma16<E>(K.f[kt][c], qf[c], s[kt]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s[kt][i] = s0 + 16 * kt + 4 * lq + i < to ? s[kt][i] * p.scale2 : -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                      fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top > m + 8.f)) {
      const float m2 = fmaxf(m, top), shrink = __builtin_amdgcn_exp2f(m - m2);
      m = m2;
      l *= shrink;
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt) acc[dt] *= shrink;
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[kt][i] = __builtin_amdgcn_exp2f(s[kt][i] - m);
        l += s[kt][i];
      }
    const bf16x8 pf = cat8e<E>(s[0], s[1]);
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt)
      acc[dt] = mfma16<E>(tr16<DP>(V + wave * 32 * DP, 16 * dt), pf, acc[dt]);
  };
  KTile Ka, Kb;
  const int s0 = from + 32 * wave;
  if (s0 < to) load(s0, Ka, V0);
  for (int s = s0; s < to; s += 256) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this tile; the next is issued below
    if (s + 128 < to) load(s + 128, Kb, V1);
    step(s, Ka, V0);
    if (s + 128 >= to) break;
    __builtin_amdgcn_s_waitcnt(0x0f70);
    if (s + 256 < to) load(s + 256, Ka, V0);
    step(s + 128, Kb, V1);
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // the four waves' results, through V0 (32 DP 16-bit values = 16 DP floats a wave)
  __syncthreads();
  float* mine = (float*)V0 + wave * 16 * DP;
#pragma unroll
  for (int dt = 0; dt < DP / 16; ++dt)
    *(floatx4*)(mine + ln * DP + ((4 * dt + lq) ^ ln % (DP / 16)) * 4) = acc[dt];
  if (lq == 0) {
    sm[wave][ln] = m;
    sl[wave][ln] = l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * DP / 4; i += 256) {
    const int r = i / (DP / 4), d4 = i % (DP / 4);
    if (rb * 16 + r >= R || 4 * d4 >= p.D) continue;
    float top = sm[0][r];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, sm[w][r]);
    floatx4 o = zero4();
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w][r] - top);
      const float* at = (const float*)V0 + (w * 16 + r) * DP + (d4 ^ r % (DP / 16)) * 4;
      o += *(const floatx4*)at * f;
      sum += sl[w][r] * f;
    }
    const long row = ((long)b * p.H + g * R + rb * 16 + r) * p.splits + split;
    *(floatx4*)(p.part + row * p.D + 4 * d4) = o;
    if (d4 == 0) {
      p.stat[2 * row] = top;
      p.stat[2 * row + 1] = sum;
    }
  }
}

// Joins a head's partial results and advances its row's count; one thread an element.
template <typename E>
__global__ __launch_bounds__(128) void sliding_step_join_kernel(SlidingStepArgs p) {
  __shared__ float share[kStepSplits];
  const long row = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const float* stat = p.stat + row * p.splits * 2;
  // both waves take the maximum and the sum, a split a lane
  float top = -INFINITY, sum = 0.f;
  for (int s = lane; s < p.splits; s += 64) top = fmaxf(top, stat[2 * s]);
#pragma unroll
  for (int k = 1; k < 64; k *= 2) top = fmaxf(top, __shfl_xor(top, k, 64));
  for (int s = lane; s < p.splits; s += 64) {
    const float f = __builtin_amdgcn_exp2f(stat[2 * s] - top);
    if (threadIdx.x < 64) share[s] = f;
    sum += stat[2 * s + 1] * f;
  }
#pragma unroll
  for (int k = 1; k < 64; k *= 2) sum += __shfl_xor(sum, k, 64);
  __syncthreads();
  const int d = threadIdx.x;
  if (d < p.D) {
    const float* part = p.part + row * p.splits * p.D + d;
    float x = 0.f, y[8];
    for (int s = 0; s < p.splits; s += 8) {
#pragma unroll
      for (int u = 0; u < 8; ++u) y[u] = s + u < p.splits ? part[(s + u) * p.D] * share[s + u] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) x += y[u];
    }
    ((__bf16*)p.o)[row * p.D + d] = to16<E>(x / sum);
  }
  if (row % p.H == 0 && threadIdx.x == 0) p.counts[row / p.H] = max(p.counts[row / p.H], 0) + 1;
}

// Cache of the last tokens of each row of a batch of prompts: one thread for 8 values of K
// and of V.  Slots that no token fills are zero.
__global__ __launch_bounds__(256) void sliding_cache_kernel(SlidingStepArgs p, int T, long kb,
                                                            long kt, long kh, long vb, long vt,
                                                            long vh, const int* lengths) {
  const int pieces = p.D / 8, slots = p.S + p.W;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)p.B * p.G * slots * pieces) return;
  const int c = i % pieces, slot = i / pieces % slots;
  const long bg = i / pieces / slots, b = bg / p.G, g = bg % p.G;
  const int len = lengths ? min(max(lengths[b], 0), T) : T;
  int at = slot;
  if (slot >= p.S) {
    const int back = (len - 1 - slot) % p.W;
    at = len - 1 - (back < 0 ? back + p.W : back);
  }
  const bool held = at < len && at >= (slot < p.S ? 0 : p.S);
  uint4 k{}, v{};
  if (held) {
    k = *(const uint4*)((const __bf16*)p.k + b * kb + at * kt + g * kh + 8 * c);
    v = *(const uint4*)((const __bf16*)p.v + b * vb + at * vt + g * vh + 8 * c);
  }
  ((uint4*)p.kc)[i] = k;
  ((uint4*)p.vc)[i] = v;
  if (g == 0 && slot == 0 && c == 0) p.counts[b] = len;
}

}  // namespace hattn

hipError_t hattn_sliding_step_launch(const SlidingStepArgs& p, int dtype, hipStream_t stream) {
  using namespace hattn;
  const dim3 grid((unsigned)((long)p.B * p.G * p.rblocks * p.splits));
#define GO(E, DP) hipLaunchKernelGGL((sliding_step_kernel<E, DP>), grid, dim3(256), 0, stream, p)
  if (dtype == 1) {
    if (p.D <= 64) GO(_Float16, 64);
    else GO(_Float16, 128);
  } else {
    if (p.D <= 64) GO(__bf16, 64);
    else GO(__bf16, 128);
  }
#undef GO
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const dim3 rows((unsigned)((long)p.B * p.H));
  if (dtype == 1)
    hipLaunchKernelGGL((sliding_step_join_kernel<_Float16>), rows, dim3(128), 0, stream, p);
  else
    hipLaunchKernelGGL((sliding_step_join_kernel<__bf16>), rows, dim3(128), 0, stream, p);
  return hipGetLastError();
}

hipError_t hattn_sliding_cache_launch(const SlidingStepArgs& p, int T, const long* strides,
                                      const int* lengths, hipStream_t stream) {
  const long n = (long)p.B * p.G * (p.S + p.W) * (p.D / 8);
  hipLaunchKernelGGL(hattn::sliding_cache_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0,
                     stream, p, T, strides[0], strides[1], strides[2], strides[3], strides[4],
                     strides[5], lengths);
  return hipGetLastError();
}
