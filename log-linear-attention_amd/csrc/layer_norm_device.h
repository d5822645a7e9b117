// Row access, sums and the choice of a row's spread, shared by layer_norm.hip and
// layer_norm_bwd.hip.
#pragma once

#include "common.h"
#include "layer_norm.h"

namespace hattn {

// One element of a parameter whose type is known at run time.
__device__ __forceinline__ float load_param(const void* p, int dtype, int i) {
  if (dtype == 0) return (float)((const __bf16*)p)[i];
  if (dtype == 1) return (float)((const _Float16*)p)[i];
  return ((const float*)p)[i];
}
__device__ __forceinline__ void store_param(void* p, int dtype, int i, float x) {
  if (dtype == 0) ((__bf16*)p)[i] = (__bf16)x;
  else if (dtype == 1) ((_Float16*)p)[i] = (_Float16)x;
  else ((float*)p)[i] = x;
}

template <typename T, int VEC>
__device__ __forceinline__ void load_row(const T* p, float (&out)[VEC]) {
  if constexpr (VEC == 1) {
    out[0] = to_f32<T>(p[0]);
  } else if constexpr (sizeof(T) == 2) {
    static_assert(VEC == 8);
    const uint4 r = *(const uint4*)p;
    T e[8];
    __builtin_memcpy(e, &r, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = to_f32<T>(e[i]);
  } else {
    const floatx4 a = ((const floatx4*)p)[0], b = ((const floatx4*)p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[i] = a[i];
      out[4 + i] = b[i];
    }
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_row(T* p, const float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    p[0] = from_f32<T>(x[0]);
  } else if constexpr (sizeof(T) == 2) {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
    uint4 r;
    __builtin_memcpy(&r, e, 16);
    *(uint4*)p = r;
  } else {
    ((floatx4*)p)[0] = floatx4{x[0], x[1], x[2], x[3]};
    ((floatx4*)p)[1] = floatx4{x[4], x[5], x[6], x[7]};
  }
}

// VEC elements of a row as they lie in memory, so that a load can be in flight over other work.
template <typename T, int VEC>
struct RawRow {
  T x[VEC];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC == 1) {
      x[0] = p[0];
    } else if constexpr (sizeof(T) == 2) {
      const uint4 r = *(const uint4*)p;
      __builtin_memcpy(x, &r, 16);
    } else {
      const floatx4 a = ((const floatx4*)p)[0], b = ((const floatx4*)p)[1];
      __builtin_memcpy(x, &a, 16);
      __builtin_memcpy(x + 4, &b, 16);
    }
  }
  __device__ __forceinline__ void get(float (&out)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = to_f32<T>(x[i]);
  }
};

// VEC elements of a parameter from element `at` on, x in each where there is none.
template <int VEC>
__device__ __forceinline__ void load_params(const void* p, int dtype, int at, int n, float x,
                                            float (&out)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) out[i] = x;
  if (!p || at >= n) return;
  if constexpr (VEC == 8) {
    if ((uintptr_t)p % 16 == 0) {  // n is a multiple of 8, so the eight are there
      if (dtype == 0) load_row<__bf16, 8>((const __bf16*)p + at, out);
      else if (dtype == 1) load_row<_Float16, 8>((const _Float16*)p + at, out);
      else load_row<float, 8>((const float*)p + at, out);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) out[i] = load_param(p, dtype, at + i);
}

// Sum over the 64 lanes, in every lane.
__device__ __forceinline__ float wave_sum(float x) { return sum_lq(row_sum16(x)); }

// Sums of NV values over the NW waves that share a row (NW = 1: over the wave).
// red: NW * NV floats of LDS; the caller alternates two of them, so that one
// barrier per call is enough.
template <int NW, int NV>
__device__ __forceinline__ void row_sums(float (&x)[NV], float* red) {
#pragma unroll
  for (int v = 0; v < NV; ++v) x[v] = wave_sum(x[v]);
  if constexpr (NW > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int v = 0; v < NV; ++v) red[wave * NV + v] = x[v];
    __syncthreads();
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float s = red[v];
#pragma unroll
      for (int w = 1; w < NW; ++w) s += red[w * NV + v];
      x[v] = s;
    }
  }
}

// Workgroups of the backward at most, each of which writes one partial row of the parameters'
// gradients: 1024 where a wave has its own rows, 512 where four waves share one.
constexpr int kNormBwdGrid1 = 1024, kNormBwdGrid4 = 512;

// How a row of n elements is spread over lanes: VEC elements a lane and load
// (8, or 1 where rows do not start on 16 bytes), NW waves of the workgroup's
// four on one row, CH loads a lane.  One wave a row up to 2048 elements; four
// where the row is longer or the rows are too few to fill the card with waves.
struct NormShape {
  int vec, nw, ch;
};
inline NormShape norm_shape(long rows, int n, bool vec) {
  if (!vec) return {1, 4, n <= 1024 ? 4 : n <= 4096 ? 16 : 64};
  const int nw = n > 2048 || rows <= 1024 ? 4 : 1;
  const int need = (n + 512 * nw - 1) / (512 * nw);
  return {8, nw, need <= 4 ? need : need <= 6 ? 6 : 8};
}

}  // namespace hattn

// Calls F.template operator()<VEC, NW, CH>() for a shape of norm_shape().
#define HATTN_NORM_DISPATCH(sh, CALL)                              \
  do {                                                             \
    if ((sh).vec == 1) {                                           \
      if ((sh).ch == 4) { CALL(1, 4, 4); }                         \
      else if ((sh).ch == 16) { CALL(1, 4, 16); }                  \
      else { CALL(1, 4, 64); }                                     \
    } else if ((sh).nw == 1) {                                     \
      if ((sh).ch == 1) { CALL(8, 1, 1); }                         \
      else if ((sh).ch == 2) { CALL(8, 1, 2); }                    \
      else if ((sh).ch == 3) { CALL(8, 1, 3); }                    \
      else { CALL(8, 1, 4); }                                      \
    } else {                                                       \
      if ((sh).ch == 1) { CALL(8, 4, 1); }                         \
      else if ((sh).ch == 2) { CALL(8, 4, 2); }                    \
      else if ((sh).ch == 3) { CALL(8, 4, 3); }                    \
      else if ((sh).ch == 4) { CALL(8, 4, 4); }                    \
      else if ((sh).ch == 6) { CALL(8, 4, 6); }                    \
      else { CALL(8, 4, 8); }                                      \
    }                                                              \
  } while (0)
