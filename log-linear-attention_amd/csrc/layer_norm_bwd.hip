// Layer norm backward.  With hat = (s - mean) rstd and t = dy weight:
//   dx = rstd (t - mean(t) - hat mean(t hat)) + ds,  dweight = sum_rows dy hat,
//   dbias = sum_rows dy.
// ds is the gradient that reaches s past the norm (the residual stream); the same dx
// is the gradient of x and of the residual.  Each wave keeps its columns' parameter
// sums in registers over all its rows; they are joined per workgroup in LDS and
// written as one partial row, and a second kernel adds the partial rows in a fixed
// order, so that no atomic decides the result.  Bound by the bytes: 109 us and 6 for the
// join (4.9 TB/s) at 65536 rows of 1024 in bf16 with a residual, 49 and 5 (4.6) at 8190 rows
// of 2304 in fp32.
#include "layer_norm_device.h"

namespace hattn {

template <typename TX, typename TS, bool DS, int VEC, int NW, int CH>
__global__ __launch_bounds__(256) void layer_norm_bwd_kernel(
    const TS* __restrict__ s, const void* __restrict__ weight, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, const TX* __restrict__ dy, const TS* __restrict__ ds,
    TX* __restrict__ dx, TS* __restrict__ dres, float* __restrict__ part, long rows, int n,
    int dtype_w) {
  __shared__ float red[2][2 * NW];
  extern __shared__ float cols[];  // NW = 1: the waves' parameter sums
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int RPB = 4 / NW;
  const int first = (NW == 1 ? lane : (int)threadIdx.x) * VEC;
  constexpr int STEP = 64 * NW * VEC;
  float w[CH][VEC], dw[CH][VEC], db[CH][VEC];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    load_params<VEC>(weight, dtype_w, first + c * STEP, n, 1.f, w[c]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[c][i] = db[c][i] = 0.f;
  }
  const float inv_n = 1.f / (float)n;
  int turn = 0;
  // Where four waves share a row, s and dy of the next one are in flight over the barrier of
  // this one's sums (57 -> 49 us at 8190 rows of 2304 in fp32); waves with rows of their own
  // fill the time better with more of them (110 us at 65536 rows of 1024, 133 with the rows
  // ahead).
  // Long rows have no registers for it.
  constexpr bool AHEAD = NW > 1 && CH * VEC <= 32;
  RawRow<TS, VEC> sn[CH];
  RawRow<TX, VEC> dyn[CH];
  float mean = 0.f, rstd = 0.f;
  const auto fetch = [&](long row) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (first + c * STEP < n) {
        sn[c].load(s + row * n + first + c * STEP);
        dyn[c].load(dy + row * n + first + c * STEP);
      }
    mean = mean_in[row];
    rstd = rstd_in[row];
  };
  const long step = (long)gridDim.x * RPB;
  long row = (long)blockIdx.x * RPB + (NW == 1 ? wave : 0);
  if (AHEAD && row < rows) fetch(row);
  for (; row < rows; row += step, turn ^= 1) {
    const long base = row * n;
    if constexpr (!AHEAD) {
      mean = mean_in[row];
      rstd = rstd_in[row];
    }
    const float mu = mean, rs = rstd;
    float h[CH][VEC], t[CH][VEC], sum[2] = {0.f, 0.f};
    RawRow<TS, VEC> dsn[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = first + c * STEP;
      if (at < n) {
        if constexpr (AHEAD) {
          sn[c].get(h[c]);
          dyn[c].get(t[c]);
          if constexpr (DS) dsn[c].load(ds + base + at);
        } else {
          load_row<TS, VEC>(s + base + at, h[c]);
          load_row<TX, VEC>(dy + base + at, t[c]);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          h[c][i] = (h[c][i] - mu) * rs;
          dw[c][i] += t[c][i] * h[c][i];
          db[c][i] += t[c][i];
          t[c][i] *= w[c][i];
          sum[0] += t[c][i];
          sum[1] += t[c][i] * h[c][i];
        }
      }
    }
    if (AHEAD && row + step < rows) fetch(row + step);
    row_sums<NW>(sum, red[turn]);
    const float c1 = sum[0] * inv_n, c2 = sum[1] * inv_n;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = first + c * STEP;
      if (at < n) {
        float o[VEC];
        if constexpr (DS && AHEAD) dsn[c].get(o);
        else if constexpr (DS) load_row<TS, VEC>(ds + base + at, o);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          o[i] = (DS ? o[i] : 0.f) + rs * (t[c][i] - c1 - h[c][i] * c2);
        if (dx) store_row<TX, VEC>(dx + base + at, o);
        if (dres) store_row<TS, VEC>(dres + base + at, o);
      }
    }
  }
  if (!part) return;
  float* out = part + (long)blockIdx.x * 2 * n;
  if constexpr (NW == 1) {
    // the four waves hold the same columns: joined in LDS, wave after wave
    for (int k = 0; k < 4; ++k) {
      if (wave == k)
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const int at = c * 64 * VEC + i * 64 + lane;  // lane-contiguous slots
            cols[at] = (k ? cols[at] : 0.f) + dw[c][i];
            cols[CH * 64 * VEC + at] = (k ? cols[CH * 64 * VEC + at] : 0.f) + db[c][i];
          }
      __syncthreads();
    }
    if (wave == 0)
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          dw[c][i] = cols[c * 64 * VEC + i * 64 + lane];
          db[c][i] = cols[CH * 64 * VEC + c * 64 * VEC + i * 64 + lane];
        }
    if (wave != 0) return;
  }
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int at = first + c * STEP + i;
      if (at < n) {
        out[at] = dw[c][i];
        out[n + at] = db[c][i];
      }
    }
}

// Adds the partial rows: 16 columns a workgroup, 16 row lanes each.
__global__ __launch_bounds__(256) void layer_norm_bwd_join_kernel(const float* __restrict__ part,
                                                                  void* __restrict__ dweight,
                                                                  void* __restrict__ dbias,
                                                                  int nparts, int n, int dtype_w) {
  __shared__ float sm[16][17];
  const int col = blockIdx.x * 16 + (threadIdx.x & 15), r = threadIdx.x >> 4;
  float a = 0.f;
  if (col < 2 * n) {
    // eight loads in flight: the sum is short and waits for memory
    float x[8];
    for (int p = r; p < nparts; p += 128) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p + 16 * i < nparts ? part[(long)(p + 16 * i) * 2 * n + col] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) a += x[i];
    }
  }
  sm[r][threadIdx.x & 15] = a;
  __syncthreads();
  if (r == 0 && col < 2 * n) {
    float t = 0.f;
    for (int k = 0; k < 16; ++k) t += sm[k][threadIdx.x & 15];
    if (col < n) {
      if (dweight) store_param(dweight, dtype_w, col, t);
    } else if (dbias) {
      store_param(dbias, dtype_w, col - n, t);
    }
  }
}

static long norm_bwd_grid(long rows, const NormShape& sh) {
  const long want = (rows + 4 / sh.nw - 1) / (4 / sh.nw);
  const long most = sh.nw == 1 ? kNormBwdGrid1 : kNormBwdGrid4;
  return want < most ? want : most;
}

template <typename TX, typename TS, bool DS>
static hipError_t launch_bwd(const void* s, const void* weight, const float* mean,
                             const float* rstd, const void* dy, const void* ds, void* dx,
                             void* dres, void* dweight, void* dbias, float* ws, long rows, int n,
                             int dtype_w, hipStream_t stream) {
  const uintptr_t bits =
      (uintptr_t)s | (uintptr_t)dy | (uintptr_t)ds | (uintptr_t)dx | (uintptr_t)dres;
  const NormShape sh = norm_shape(rows, n, n % 8 == 0 && bits % 16 == 0);
  const int grid = (int)norm_bwd_grid(rows, sh);
  float* part = dweight || dbias ? ws : nullptr;
  const size_t smem = sh.nw == 1 ? (size_t)2 * sh.ch * 64 * sh.vec * 4 : 0;
#define CALL(VEC, NW, CH)                                                                       \
  hipLaunchKernelGGL((layer_norm_bwd_kernel<TX, TS, DS, VEC, NW, CH>), dim3(grid), dim3(256),   \
                     smem, stream, (const TS*)s, weight, mean, rstd, (const TX*)dy,             \
                     (const TS*)ds, (TX*)dx, (TS*)dres, part, rows, n, dtype_w)
  HATTN_NORM_DISPATCH(sh, CALL);
#undef CALL
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  if (part)
    hipLaunchKernelGGL(layer_norm_bwd_join_kernel, dim3((2 * n + 15) / 16), dim3(256), 0, stream,
                       part, dweight, dbias, grid, n, dtype_w);
  return hipGetLastError();
}

}  // namespace hattn

size_t hattn_layer_norm_bwd_ws_bytes(long rows, int n) {
  // the larger grid of the two that the tensors' alignment leaves open
  const long most = rows > 1024 && n <= 2048 ? hattn::kNormBwdGrid1 : hattn::kNormBwdGrid4;
  return (size_t)(rows < most ? rows : most) * 2 * n * sizeof(float);
}

hipError_t hattn_layer_norm_bwd_launch(const void* s, const void* weight, const float* mean,
                                       const float* rstd, const void* dy, const void* ds, void* dx,
                                       void* dres, void* dweight, void* dbias, float* ws, long rows,
                                       int n, int dtype_x, int dtype_s, int dtype_w,
                                       hipStream_t stream) {
  using namespace hattn;
#define GO(TX, TS, DS)                                                                         \
  return launch_bwd<TX, TS, DS>(s, weight, mean, rstd, dy, ds, dx, dres, dweight, dbias, ws,   \
                                rows, n, dtype_w, stream)
  if (dtype_s == 2 && dtype_x != 2) {
    if (dtype_x == 0) {
      if (ds) GO(__bf16, float, true);
      GO(__bf16, float, false);
    }
    if (ds) GO(_Float16, float, true);
    GO(_Float16, float, false);
  }
  if (dtype_x == 0) {
    if (ds) GO(__bf16, __bf16, true);
    GO(__bf16, __bf16, false);
  }
  if (dtype_x == 1) {
    if (ds) GO(_Float16, _Float16, true);
    GO(_Float16, _Float16, false);
  }
  if (ds) GO(float, float, true);
  GO(float, float, false);
#undef GO
}
