// Gated linear recurrence per channel, h_t = a_t h_{t-1} + x_t with a_t = exp(g_t),
// its gradient, and its single-token step.
//
// Backward, with e_{t} = a_t dh_t the gradient that reaches h_{t-1}:
//   dh_t = do_t + e_{t+1},  dx_t = dh_t,  dg_t = dh_t a_t h_{t-1}.
// Both directions compose affine maps h -> A h + X, which is associative:
//   (A2, X2) o (A1, X1) = (A2 A1, A2 X1 + X2).
//
// A lane owns one channel, a wave 32 tokens of 64 channels held in registers, a
// workgroup 256 tokens (a segment).  Inside the workgroup the waves' maps meet in
// LDS; between the segments of a channel the workgroup publishes its map in a word
// {A, X} and then walks back over the words before it until one has A = 0.  A
// segment whose state is known replaces its word by {0, h}, so the walk is short, and
// the data is read once and written once: bound by the bytes.
//
// A word is 64 bits wide and is written and read by one atomic access of device
// scope, so it is its own flag: kEmpty (a NaN pattern that publish() never writes)
// until it holds a map.  A workgroup waits only for workgroups that come before it
// in the order of dispatch; the wait is bounded, and one that gives up makes its
// outputs NaN.
#include "common.h"
#include "recurrence.h"

namespace hattn {

constexpr int kTok = 32;                 // tokens a wave
constexpr int kWaves = 8;                // waves a workgroup
constexpr int kSeg = kTok * kWaves;      // tokens a segment
constexpr unsigned long long kEmpty = ~0ull;
constexpr int kSpins = 1 << 20;          // rounds of a wait, about a second

struct Map {
  float A, X;
};

__device__ __forceinline__ float no_payload(float x) {
  return x != x ? __builtin_bit_cast(float, 0x7fc00000u) : x;
}

__device__ __forceinline__ void publish(unsigned long long* w, float A, float X) {
  const unsigned lo = __builtin_bit_cast(unsigned, no_payload(A));
  const unsigned hi = __builtin_bit_cast(unsigned, no_payload(X));
  __hip_atomic_store(w, (unsigned long long)hi << 32 | lo, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ unsigned long long word(const unsigned long long* w) {
  return __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float apply(unsigned long long w, float h) {
  const float A = __builtin_bit_cast(float, (unsigned)w);
  const float X = __builtin_bit_cast(float, (unsigned)(w >> 32));
  return A == 0.f ? X : A * h + X;
}

// The state that enters this segment from the words of the `before` segments before
// it (w[0], w[step], ..): back to the nearest one whose words all have A = 0, or to
// the first segment and `base`, then their maps forward from there.  The state is
// built in the order of the tokens wherever the walk starts, so its bits do not
// depend on which words were already replaced.
__device__ __forceinline__ float look_back(const unsigned long long* w, long step, int before,
                                           float base, bool live) {
  constexpr int N = 8;
  const float nan = __builtin_bit_cast(float, 0x7fc00000u);
  int n = 0;  // words walked back over
  for (int spin = 0; n < before; ++spin) {
    if (spin >= kSpins) return nan;
    unsigned long long got[N];
#pragma unroll
    for (int i = 0; i < N; ++i) got[i] = live && n + i < before ? word(w + (n + i) * step) : 0ull;
    int used = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (used == i && !found && n + i < before && !__any(got[i] == kEmpty)) {
        ++used;
        found = __all((unsigned)got[i] << 1 == 0);
      }
    n += used;
    if (found) break;
    if (used == 0) __builtin_amdgcn_s_sleep(1);
  }
  float h = base;
  while (n > 0) {
    unsigned long long got[N];
#pragma unroll
    for (int i = 0; i < N; ++i) got[i] = live && i < n ? word(w + (n - 1 - i) * step) : 0ull;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) h = apply(got[i], h);
    n -= N;
  }
  return h;
}

__global__ void fill_empty_kernel(unsigned long long* w, long n) {
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x)
    w[i] = kEmpty;
}

// blockIdx.x = segment * units + unit, unit = batch * strips + strip of 64 channels:
// every unit's first segment is dispatched first.
struct Place {
  int b, d, seg, len;
  long unit;
  bool live;
};
__device__ __forceinline__ Place place(const RecurrenceArgs& p, bool backward) {
  Place at;
  const int units = p.B * p.strips;
  const int u = blockIdx.x % units, s = blockIdx.x / units;
  at.seg = backward ? p.nseg - 1 - s : s;
  at.unit = u;
  at.b = u / p.strips;
  at.d = (u % p.strips) * 64 + (threadIdx.x & 63);
  at.live = at.d < p.D;
  at.len = p.lengths ? min(max(p.lengths[at.b], 0), p.T) : p.T;
  return at;
}

template <typename TX, typename TG>
__global__ __launch_bounds__(64 * kWaves, 4) void recurrence_fwd_kernel(RecurrenceArgs p) {
  __shared__ Map maps[kWaves][64];
  __shared__ float enter[64];
  const Place at = place(p, false);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = at.seg * kSeg + wave * kTok;
  const long base = (long)at.b * p.T * p.D;
  const TX* x = (const TX*)p.x + base;
  const TG* g = (const TG*)p.g + base;
  const int d = at.live ? at.d : p.D - 1;

  float a[kTok], v[kTok];
  if (t0 < p.T) {
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      // rows past the end read the last one; what they read is not used
      const long row = (long)min(t0 + i, p.T - 1) * p.D + d;
      v[i] = to_f32<TX>(x[row]);
      a[i] = to_f32<TG>(g[row]);
    }
  }
  float A = 1.f, X = 0.f;
#pragma unroll
  for (int i = 0; i < kTok; ++i) {
    const bool in = t0 + i < at.len;
    a[i] = in ? fexp(a[i]) : 1.f;
    v[i] = in ? v[i] : 0.f;
    X = a[i] * X + v[i];
    A *= a[i];
  }
  maps[wave][lane] = Map{A, X};
  __syncthreads();
  if (wave == 0) {
    Map m = maps[0][lane];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) {
      const Map n = maps[k][lane];
      m = Map{n.A * m.A, n.A * m.X + n.X};
    }
    const float h0 = p.h0 && at.live ? p.h0[(long)at.b * p.D + d] : 0.f;
    const long stride = (long)p.B * p.strips * 64;
    unsigned long long* w = (unsigned long long*)p.ws + at.seg * stride + at.unit * 64 + lane;
    const bool last = at.seg == p.nseg - 1;
    if (at.live && !last && at.seg > 0) publish(w, m.A, m.X);
    const float h = look_back(w - stride, -stride, at.seg, h0, at.live);
    // as apply(): A = 0 ends a walk, so nothing before such a segment reaches past it
    const float out = m.A == 0.f ? m.X : m.A * h + m.X;
    if (at.live && !last) publish(w, 0.f, out);
    if (at.live && last && p.ht) p.ht[(long)at.b * p.D + d] = out;
    if (at.live && p.carry) p.carry[((long)at.b * p.nseg + at.seg) * p.D + d] = h;
    enter[lane] = h;
  }
  __syncthreads();
  float h = enter[lane];
  for (int k = 0; k < wave; ++k) h = maps[k][lane].A * h + maps[k][lane].X;
  TX* o = (TX*)p.o + base;
#pragma unroll
  for (int i = 0; i < kTok; ++i) {
    h = a[i] * h + v[i];
    if (at.live && t0 + i < p.T) o[(long)(t0 + i) * p.D + d] = from_f32<TX>(t0 + i < at.len ? h : 0.f);
  }
}

template <typename TX, typename TG>
__global__ __launch_bounds__(64 * kWaves) void recurrence_bwd_kernel(RecurrenceArgs p) {
  __shared__ Map fwd[kWaves][64], bwd[kWaves][64];
  __shared__ float enter[64];
  const Place at = place(p, true);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = at.seg * kSeg + wave * kTok;
  const long base = (long)at.b * p.T * p.D;
  const TX *x = (const TX*)p.x + base, *go = (const TX*)p.go + base;
  const TG* g = (const TG*)p.g + base;
  const int d = at.live ? at.d : p.D - 1;

  float a[kTok], v[kTok], q[kTok];
  if (t0 < p.T) {
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      const long row = (long)min(t0 + i, p.T - 1) * p.D + d;
      a[i] = to_f32<TG>(g[row]);
      q[i] = to_f32<TX>(go[row]);
      v[i] = to_f32<TX>(x[row]);
    }
  }
  float A = 1.f, X = 0.f, E = 0.f;
#pragma unroll
  for (int i = 0; i < kTok; ++i) {
    const bool in = t0 + i < at.len;
    a[i] = in ? fexp(a[i]) : 1.f;
    v[i] = in ? v[i] : 0.f;
    q[i] = in ? q[i] : 0.f;
    X = a[i] * X + v[i];
    A *= a[i];
  }
#pragma unroll
  for (int i = kTok - 1; i >= 0; --i) E = a[i] * (q[i] + E);
  fwd[wave][lane] = Map{A, X};
  bwd[wave][lane] = Map{A, E};
  __syncthreads();
  if (wave == 0) {
    Map m = bwd[kWaves - 1][lane];
#pragma unroll
    for (int k = kWaves - 2; k >= 0; --k) {
      const Map n = bwd[k][lane];
      m = Map{n.A * m.A, n.A * m.X + n.X};
    }
    const float end = p.ght && at.live ? p.ght[(long)at.b * p.D + d] : 0.f;
    const long stride = (long)p.B * p.strips * 64;
    unsigned long long* w = (unsigned long long*)p.ws + at.seg * stride + at.unit * 64 + lane;
    const int after = p.nseg - 1 - at.seg;
    if (at.live && after > 0 && at.seg > 0) publish(w, m.A, m.X);
    const float e = look_back(w + stride, stride, after, end, at.live);
    const float out = m.A == 0.f ? m.X : m.A * e + m.X;
    if (at.live && at.seg > 0) publish(w, 0.f, out);
    if (at.live && at.seg == 0 && p.dh0) p.dh0[(long)at.b * p.D + d] = out;
    enter[lane] = e;
  }
  // the state that enters this wave's tokens, while wave 0 looks ahead
  float h = p.carry[((long)at.b * p.nseg + at.seg) * p.D + d];
  for (int k = 0; k < wave; ++k) h = fwd[k][lane].A * h + fwd[k][lane].X;
#pragma unroll
  for (int i = 0; i < kTok; ++i) {
    const float was = h;
    h = a[i] * h + v[i];
    v[i] = was;
  }
  __syncthreads();
  float e = enter[lane];
  for (int k = kWaves - 1; k > wave; --k) e = bwd[k][lane].A * e + bwd[k][lane].X;
  TX* dx = (TX*)p.dx + base;
  TG* dg = (TG*)p.dg + base;
#pragma unroll
  for (int i = kTok - 1; i >= 0; --i) {
    const float dh = q[i] + e;
    e = a[i] * dh;
    if (at.live && t0 + i < p.T) {
      const long row = (long)(t0 + i) * p.D + d;
      const bool in = t0 + i < at.len;
      dx[row] = from_f32<TX>(in ? dh : 0.f);
      dg[row] = from_f32<TG>(in ? e * v[i] : 0.f);
    }
  }
}

template <typename TX, typename TG>
__global__ __launch_bounds__(256) void recurrence_step_kernel(float* __restrict__ h,
                                                              const TX* __restrict__ x,
                                                              const TG* __restrict__ g,
                                                              TX* __restrict__ o, long n) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const float y = fexp(to_f32<TG>(g[i])) * h[i] + to_f32<TX>(x[i]);
  h[i] = y;
  o[i] = from_f32<TX>(y);
}

template <typename TX, typename TG>
static hipError_t launch(int what, const RecurrenceArgs& p, hipStream_t stream) {
  if (what == 2) {
    const long n = (long)p.B * p.D;
    hipLaunchKernelGGL((recurrence_step_kernel<TX, TG>), dim3((unsigned)((n + 255) / 256)),
                       dim3(256), 0, stream, p.ht, (const TX*)p.x, (const TG*)p.g, (TX*)p.o, n);
    return hipGetLastError();
  }
  const long units = (long)p.B * p.strips;
  if (p.nseg > 1) {
    const long n = units * 64 * p.nseg;
    const long want = (n + 1023) / 1024;
    hipLaunchKernelGGL(fill_empty_kernel, dim3((unsigned)(want < 1024 ? want : 1024)), dim3(256), 0,
                       stream, (unsigned long long*)p.ws, n);
  }
  const dim3 grid((unsigned)(units * p.nseg));
  if (what == 0)
    hipLaunchKernelGGL((recurrence_fwd_kernel<TX, TG>), grid, dim3(64 * kWaves), 0, stream, p);
  else
    hipLaunchKernelGGL((recurrence_bwd_kernel<TX, TG>), grid, dim3(64 * kWaves), 0, stream, p);
  return hipGetLastError();
}

}  // namespace hattn

int hattn_recurrence_segments(int T) { return (T + hattn::kSeg - 1) / hattn::kSeg; }

// what: 0 forward, 1 backward, 2 step
hipError_t hattn_recurrence_launch(int what, const RecurrenceArgs& p, int dtype_x, int dtype_g,
                                   hipStream_t stream) {
  using namespace hattn;
  if (dtype_g == 2) {
    if (dtype_x == 0) return launch<__bf16, float>(what, p, stream);
    if (dtype_x == 1) return launch<_Float16, float>(what, p, stream);
    return launch<float, float>(what, p, stream);
  }
  if (dtype_x == 0) return launch<__bf16, __bf16>(what, p, stream);
  return launch<_Float16, _Float16>(what, p, stream);
}
