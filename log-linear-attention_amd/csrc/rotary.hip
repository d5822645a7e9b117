// Rotary positions: every pair (a, b) of the first 2 `pairs` elements of a head turns by
// pos * freq, and the others stay:
//   a' = scale (a cos - b sin),  b' = scale (a sin + b cos)
// with pairs (i, i + pairs) or, interleaved, (2 i, 2 i + 1).  The backward is the inverse
// rotation (sign -1) with the same scale.
//
// The angle is taken in turns and in 64 bits, and reduced to [-1/2, 1/2] before it is rounded
// to 32: at position 10^6 an angle in 32 bits would be off by 0.06.
//
// Each element is read and written once, which bounds it: 4 x 8192 tokens of 32 heads of 64 in bf16 take
// 53 us (5.0 TB/s), 32768 tokens of 40 heads of 128 114 us (5.9 TB/s).  The sines of a workgroup's tokens
// are made once, in LDS, for all of their heads; then the lanes run along the heads, two
// 16-byte pieces each, whose elements are pairs of each other (interleaved: pairs in
// themselves).  Where heads, pairs, strides and addresses are not all whole pieces, the pieces are one
// element, at a third of the rate (9 heads of 82: 1.7 TB/s; 20 of 80 elements turned: 1.4).
#include "common.h"
#include "rotary.h"

namespace hattn {

constexpr int kAhead = 2;

template <typename T, int V>
struct alignas(sizeof(T) * V) Piece {
  T v[V];
};

// (a, b) turned by r = (cos, sin): which product is rounded is written out, so that the results do not
// depend on the variant that a tensor's alignment picks.
template <typename T>
__device__ __forceinline__ void turned(T& a, T& b, float2 r) {
  const float f = to_f32(a), g = to_f32(b);
  a = from_f32<T>(fmaf(f, r.x, -g * r.y));
  b = from_f32<T>(fmaf(f, r.y, g * r.x));
}

template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs p) {
  extern __shared__ __attribute__((aligned(16))) char shared[];
  float2* cs = (float2*)shared;                        // [tokens][pairs]
  long* at = (long*)(cs + p.tokens * p.pairs);         // [2][tokens]: offsets of x
  const long n0 = (long)blockIdx.x * p.tokens;
  const int tokens = (int)min((long)p.tokens, p.N - n0);
  for (int i = threadIdx.x; i < tokens * p.pairs; i += 256) {
    const int tt = i / p.pairs, j = i - tt * p.pairs;
    const long n = n0 + tt, b = n / p.T, t = n - b * p.T;
    long pos = t;
    if (p.pos) {
      const long o = b * p.pb + (p.from ? 0 : t * p.pt);
      pos = (p.pos64 ? ((const long*)p.pos)[o] : (long)((const int*)p.pos)[o]) + (p.from ? t : 0);
    }
    const double f = p.freq64 ? ((const double*)p.freqs)[j] : (double)((const float*)p.freqs)[j];
    const double turns = (double)pos * f * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = float2{c * p.scale, s * p.scale * p.sign};
    if (j == 0) {
      at[tt] = b * p.xb[0] + t * p.xt[0];
      at[p.tokens + tt] = b * p.xb[1] + t * p.xt[1];
    }
  }
  __syncthreads();

  const int heads = p.heads[0] + p.heads[1], rot = 2 * p.pairs;
  const int col = threadIdx.x % p.cols, rows = 256 / p.cols;
  // The lane's two pieces: each in its own half of the pairs or of what stays, so that neighbours
  // read on; single elements that are interleaved lie together.
  const int turning = p.pairs / V, col2 = col - turning;  // lanes with pairs
  const int staying = ((p.D - rot) / V + 1) / 2;
  const bool turn = col < turning;
  const int a = !turn ? rot + V * col2 : INTER && V == 1 ? 2 * col : V * col;
  const int b = !turn ? a + V * staying : INTER && V == 1 ? a + 1 : a + p.pairs;
  if (!turn && col2 >= staying) return;
  const bool two = b < p.D;
  int h = threadIdx.x / p.cols, tt = h / heads;
  h -= tt * heads;
  const int dt = rows / heads, dh = rows - dt * heads;
  typedef Piece<T, V> P;
  // kAhead heads at once: their loads are in flight together
  while (tt < tokens) {
    P u[kAhead], v[kAhead];
    int token[kAhead];
    T* y[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      token[k] = tt < tokens ? tt : -1;
      u[k] = v[k] = P{};
      if (tt < tokens) {
        const int w = h >= p.heads[0], hw = w ? h - p.heads[0] : h;
        const T* x = (const T*)p.x[w] + at[w * p.tokens + tt] + hw * p.xh[w];
        y[k] = (T*)p.y[w] + ((n0 + tt) * p.heads[w] + hw) * p.D;
        u[k] = *(const P*)(x + a);
        if (two) v[k] = *(const P*)(x + b);
      }
      tt += dt;
      h += dh;
      if (h >= heads) {
        h -= heads;
        ++tt;
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (token[k] < 0) break;
      if (turn) {
        const float2* angle = cs + token[k] * p.pairs + (INTER ? a / 2 : a);
        if constexpr (INTER && V > 1) {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            turned(u[k].v[2 * i], u[k].v[2 * i + 1], angle[i]);
            turned(v[k].v[2 * i], v[k].v[2 * i + 1], angle[p.pairs / 2 + i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) turned(u[k].v[i], v[k].v[i], angle[i]);
        }
      }
      *(P*)(y[k] + a) = u[k];
      if (two) *(P*)(y[k] + b) = v[k];
    }
  }
}

}  // namespace hattn

hipError_t hattn_rotary_launch(const RotaryArgs& p, int dtype, bool interleaved, bool wide,
                               hipStream_t stream) {
  using namespace hattn;
  const dim3 grid((unsigned)((p.N + p.tokens - 1) / p.tokens));
  const size_t lds = rotary_lds(p.tokens, p.pairs);
#define GO(T, V, I) hipLaunchKernelGGL((rotary_kernel<T, V, I>), grid, dim3(256), lds, stream, p)
#define PICK(T, V)                \
  if (wide) {                     \
    if (interleaved) GO(T, V, true); \
    else GO(T, V, false);         \
  } else {                        \
    if (interleaved) GO(T, 1, true); \
    else GO(T, 1, false);         \
  }
  if (dtype == 0) {
    PICK(__bf16, 8)
  } else if (dtype == 1) {
    PICK(_Float16, 8)
  } else {
    PICK(float, 4)
  }
#undef PICK
#undef GO
  return hipGetLastError();
}
