// A cache of keys and values in 8 bits: tokens entering it and coming back.
//
// Appending, a workgroup makes one block of 64 tokens of one head of K or V: the new tokens
// stay in registers between the block's maximum and their codes, so that each value is read
// once and each code written once, which bounds it.  Where the block has older tokens and its
// scale grows, their codes are made again.  4 rows of up to 8192 tokens, 8 heads of 128: 29 us
// (5.6 TB/s), and 5 us for the counts, which advance in a launch of their own, when nothing reads them
// any more; with the codes written through the caches both took 38 us.
#include "quant_device.h"

namespace hattn {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

template <typename E>
__device__ __forceinline__ unsigned top8(uint4 x) {
  return max(max(top2<E>(x.x), top2<E>(x.y)), max(top2<E>(x.z), top2<E>(x.w)));
}

// 2^PC lanes for the 8-element pieces of a token.
template <typename E, int PC>
__global__ __launch_bounds__(256) void quant_append_kernel(QuantArgs p) {
  constexpr int ROWS = 256 >> PC, N = ROWS >= kQuantBlock ? 1 : kQuantBlock / ROWS;
  __shared__ unsigned tops[4];
  unsigned item = blockIdx.x;  // 32-bit divisions: 64-bit ones are hundreds of instructions
  const bool isv = item & 1;
  item >>= 1;
  const int j = item % (unsigned)p.blocks;
  const int bg = (int)(item / (unsigned)p.blocks);
  const int b = (unsigned)bg / (unsigned)p.G, g = bg - b * p.G;
  const int n0 = max(p.counts[b], 0);
  const int fresh = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const long first = ((long)(n0 / kQuantBlock) + j) * kQuantBlock;  // the block's first slot
  const long end = min((long)n0 + fresh, (long)p.cap);              // of the tokens that are kept
  if (first >= end || n0 >= end) return;
  const int lo = (int)max((long)n0 - first, 0L), hi = (int)min(end - first, (long)kQuantBlock);
  float* scale = (isv ? p.vs : p.ks) + (long)bg * (p.cap / kQuantBlock) + first / kQuantBlock;
  unsigned char* codes = (isv ? p.vc : p.kc) + ((long)bg * p.cap + first) * p.D;
  const long st = isv ? p.vt : p.kt;
  const __bf16* x = (const __bf16*)(isv ? p.v : p.k) + b * (isv ? p.vb : p.kb) +
                    g * (isv ? p.vh : p.kh) + (first - n0) * st;  // row 0 of the block
  const int d = 8 * (threadIdx.x & ((1 << PC) - 1)), row0 = threadIdx.x >> PC;

  const float was = lo > 0 ? *scale : 0.f;
  uint4 y[N];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int row = row0 + i * ROWS;
    y[i] = row >= lo && row < hi && d < p.D ? *(const uint4*)(x + row * st + d) : uint4{};
  }
#pragma unroll
  for (int i = 0; i < N; ++i) top = max(top, top8<E>(y[i]));
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  const float now = fmaxf(power(scale_exponent<E>(top)), was), inverse = 1.f / now;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int row = row0 + i * ROWS;
    if (row >= lo && row < hi && d < p.D)
      __builtin_nontemporal_store(__builtin_bit_cast(u32x2, codes8<E>(y[i], inverse)),
                                  (u32x2*)(codes + row * p.D + d));
  }
  if (threadIdx.x == 0) *scale = now;
  if (lo > 0 && now > was) {
    const float ratio = was / now;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = row0 + i * ROWS;
      if (row < lo && d < p.D) {
        uint2* at = (uint2*)(codes + row * p.D + d);
        const uint2 c = *at;
        *at = uint2{rescale4(c.x, ratio), rescale4(c.y, ratio)};
      }
    }
  }
}

__global__ __launch_bounds__(256) void quant_advance_kernel(QuantArgs p) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= p.B) return;
  const int fresh = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  p.counts[b] = (int)min((long)max(p.counts[b], 0) + fresh, 0x7fffffffL);
}

// One token: a workgroup makes a row's codes of all heads, a wave one head at a time, and then
// advances the row's count, which no other workgroup reads.
template <typename E>
__global__ __launch_bounds__(1024) void quant_token_kernel(QuantArgs p) {
  const int b = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int n0 = max(p.counts[b], 0);
  if (n0 < p.cap)
    for (int i = wave; i < p.G; i += waves) token_codes<E>(p, b, i, n0);
  __syncthreads();
  if (threadIdx.x == 0) p.counts[b] = min(n0, 0x7ffffffe) + 1;
}

// A workgroup has one block of a head of K or V, so that its scale is one number.  2^PC lanes for the
// pieces of a token, which are 16 bytes of the result: neighbours write whole lines, past the caches.
// 8 rows of 16000 tokens, 8 heads of 128, in bf16: 115 us (5.8 TB/s); through the caches 125, and
// with 32 bytes of the result a lane 144.
template <typename T, int PC>
__global__ __launch_bounds__(256) void quant_read_kernel(QuantArgs p) {
  constexpr int V = 16 / sizeof(T), ROWS = 256 >> PC, N = ROWS >= kQuantBlock ? 1 : kQuantBlock / ROWS;
  unsigned item = blockIdx.x;
  const bool isv = item & 1;
  item >>= 1;
  const int j = item % (unsigned)p.blocks;
  const int bg = (int)(item / (unsigned)p.blocks);
  const int b = (unsigned)bg / (unsigned)p.G, g = bg - b * p.G;
  const int first = (p.start / kQuantBlock + j) * kQuantBlock;
  const int count = p.counts[b], end = min(p.start + p.n, first + kQuantBlock);
  const float scale = (isv ? p.vs : p.ks)[(long)bg * (p.cap / kQuantBlock) + first / kQuantBlock];
  const unsigned char* codes = (isv ? p.vc : p.kc) + (long)bg * p.cap * p.D;
  T* out = (T*)(isv ? p.vo : p.ko);
  const int d = V * (threadIdx.x & ((1 << PC) - 1)), slot0 = first + (threadIdx.x >> PC);
  if (d >= p.D) return;
  unsigned x[N][V / 4];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int slot = slot0 + i * ROWS;
    const bool held = slot >= p.start && slot < end && slot < count;
    const unsigned* at = (const unsigned*)(codes + (long)slot * p.D + d);
    if constexpr (V == 8) {
      const uint2 y = held ? *(const uint2*)at : uint2{};
      x[i][0] = y.x;
      x[i][1] = y.y;
    } else {
      x[i][0] = held ? *at : 0;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int slot = slot0 + i * ROWS;
    if (slot < p.start || slot >= end) continue;
    struct alignas(16) Out {
      T v[V];
    } y;
#pragma unroll
    for (int k = 0; k < V / 4; ++k) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)x[i][k], false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)x[i][k], true);
      const float f[4] = {lo[0], lo[1], hi[0], hi[1]};
      // slots that hold no token are zero whatever the scale there
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y.v[4 * k + e] = from_f32<T>(slot < count ? f[e] * scale : 0.f);
    }
    T* to = out + (((long)b * p.n + slot - p.start) * p.G + g) * p.D + d;
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, y), (u32x4*)to);
  }
}

}  // namespace hattn

hipError_t hattn_quant_append_launch(const QuantArgs& p, int dtype, hipStream_t stream) {
  using namespace hattn;
  const dim3 grid((unsigned)((long)p.B * p.G * p.blocks * 2));
#define GO(E, PC) hipLaunchKernelGGL((quant_append_kernel<E, PC>), grid, dim3(256), 0, stream, p)
#define PICK(E)             \
  if (p.D <= 16) GO(E, 1);  \
  else if (p.D <= 32) GO(E, 2); \
  else if (p.D <= 64) GO(E, 3); \
  else GO(E, 4);
  if (dtype == 1) {
    PICK(_Float16)
  } else {
    PICK(__bf16)
  }
#undef PICK
#undef GO
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  hipLaunchKernelGGL(quant_advance_kernel, dim3((unsigned)((p.B + 255) / 256)), dim3(256), 0, stream,
                     p);
  return hipGetLastError();
}

hipError_t hattn_quant_token_launch(const QuantArgs& p, int dtype, hipStream_t stream) {
  using namespace hattn;
  const dim3 grid((unsigned)p.B), block(64 * (p.G < 16 ? p.G : 16));
  if (dtype == 1)
    hipLaunchKernelGGL((quant_token_kernel<_Float16>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((quant_token_kernel<__bf16>), grid, block, 0, stream, p);
  return hipGetLastError();
}

hipError_t hattn_quant_read_launch(const QuantArgs& p, int dtype, hipStream_t stream) {
  using namespace hattn;
  const dim3 grid((unsigned)((long)p.B * p.G * p.blocks * 2));
#define GO(T, PC) hipLaunchKernelGGL((quant_read_kernel<T, PC>), grid, dim3(256), 0, stream, p)
#define PICK(T, PC)                 \
  if (p.D <= 16) GO(T, PC);         \
  else if (p.D <= 32) GO(T, PC + 1); \
  else if (p.D <= 64) GO(T, PC + 2); \
  else GO(T, PC + 3);
  if (dtype == 0) {
    PICK(__bf16, 1)
  } else if (dtype == 1) {
    PICK(_Float16, 1)
  } else {
    PICK(float, 2)
  }
#undef PICK
#undef GO
  return hipGetLastError();
}
