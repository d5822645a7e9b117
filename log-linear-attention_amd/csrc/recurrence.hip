// Gated linear recurrence per channel, h_t = a_t h_{t-1} + x_t with a_t = exp(g_t),
// its gradient, and its single-token step.
//
// Backward, with e_{t} = a_t dh_t the gradient that reaches h_{t-1}:
//   dh_t = do_t + e_{t+1},  dx_t = dh_t,  dg_t = dh_t a_t h_{t-1}.
// Both directions compose affine maps h -> A h + X, which is associative:
//   (A2, X2) o (A1, X1) = (A2 A1, A2 X1 + X2).
//
// A lane owns one channel in 32 bits, or two next to each other in 16 bits (where D is even):
// a wave reads rows of 256 bytes (rows of 128 take 98 and not 91 us forward, 158 and not
// 133 backward, at B 4, T 8192, D 2048 in bf16).  A wave holds 32 or 16 tokens in registers, a
// workgroup eight times as many (a segment); registers are held to 128, so that a second
// workgroup on the CU loads and stores while the first waits (the backward with one channel a
// lane then spills 1 to 12 of them).
//
// Inside the workgroup the waves' maps meet in LDS; between the segments of a channel the
// workgroup publishes its map in a word {A, X} and then walks back over the words before it
// until one holds a state.  A segment whose state is known replaces its word by {kState, h}, so
// the walk is short, and the data is read once and written once: bound by the bytes (forward
// 4.4 TB/s and backward 5.0 at the shape above, forward 5.6 at B 1, T 131072, D 1024 in fp32).
//
// A word is 64 bits wide and is written and read by one atomic access of device
// scope, so it is its own flag: kEmpty (a NaN pattern that publish() never writes)
// until it holds a map.  No map drops what comes before it: a state that is not finite passes
// it as it passes the tokens, also where the product of decays that are not zero falls below
// fp32's range, which is kept as its smallest number (compose() below).  Segments are handed out by one counter in the order of the walk, so
// a workgroup waits only for workgroups that already run, wherever and whenever the card
// starts them and whatever else runs beside (each XCD starts its own share of a grid in order,
// which does not order the whole).  The wait is bounded all the same, and one that gives up
// makes its outputs NaN.
#include "common.h"
#include "recurrence.h"

namespace hattn {

constexpr int kWaves = 8;                // waves a workgroup
template <int VEC>
constexpr int kTok = 32 / VEC;           // tokens a wave
constexpr unsigned long long kEmpty = ~0ull;
constexpr unsigned kState = 0x7fc00001u;  // in place of A: the word holds a state (a NaN pattern too)
constexpr int kSpins = 1 << 20;          // rounds of a wait, about a second

struct Map {
  float A, X;
};

__device__ __forceinline__ float no_payload(float x) {
  return x != x ? __builtin_bit_cast(float, 0x7fc00000u) : x;
}

__device__ __forceinline__ void put_word(unsigned long long* w, unsigned lo, float X) {
  const unsigned hi = __builtin_bit_cast(unsigned, no_payload(X));
  __hip_atomic_store(w, (unsigned long long)hi << 32 | lo, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void publish(unsigned long long* w, Map m) {
  put_word(w, __builtin_bit_cast(unsigned, no_payload(m.A)), m.X);
}
__device__ __forceinline__ void publish_state(unsigned long long* w, float h) {
  put_word(w, kState, h);
}

__device__ __forceinline__ unsigned long long word(const unsigned long long* w) {
  return __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float apply(Map m, float h) { return __builtin_fmaf(m.A, h, m.X); }
__device__ __forceinline__ float apply(unsigned long long w, float h) {
  const float X = __builtin_bit_cast(float, (unsigned)(w >> 32));
  return (unsigned)w == kState ? X : apply(Map{__builtin_bit_cast(float, (unsigned)w), X}, h);
}

// A product of decays, `zero` where one of them is zero.  One that only underflowed is kept as
// the smallest number, so that infinity stays infinity; it adds at most 5e-7 to a state whose
// predecessor is 3e38.
__device__ __forceinline__ float no_underflow(float A, bool zero) {
  return A == 0.f && !zero ? __builtin_bit_cast(float, 1u) : A;
}
template <int TOK, int VEC>
__device__ __forceinline__ float no_underflow(float A, const float (&a)[TOK][VEC], int e) {
  if (!__any(A == 0.f)) return A;
  bool zero = false;
#pragma unroll
  for (int i = 0; i < TOK; ++i) zero |= a[i][e] == 0.f;
  return no_underflow(A, zero);
}
// n after m
__device__ __forceinline__ Map compose(Map n, Map m) {
  return Map{no_underflow(n.A * m.A, n.A == 0.f || m.A == 0.f), apply(n, m.X)};
}

// The state that enters this segment from the words of the `before` segments before
// it (w[0], w[step], ..): back to the nearest one whose words all hold a state, or to
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
        found = __all(!live || (unsigned)got[i] == kState);
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

// The counter of the segments lies in the first word of the last segment of the walk, which
// no other segment reads.
__device__ __host__ __forceinline__ long counter_word(const RecurrenceArgs& p, bool backward) {
  return backward ? 0 : (long)(p.nseg - 1) * p.B * p.strips * 64 * p.vec;
}

__global__ void fill_empty_kernel(unsigned long long* w, long n, long counter) {
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x)
    w[i] = i == counter ? 0 : kEmpty;
}

// The workgroup's item = step of the walk * units + unit, unit = batch * strips + strip of 64
// lanes: every unit's first segment comes first.  Items past the last are only handed out where
// another call resets the counter meanwhile: such a workgroup does nothing.
__device__ __forceinline__ unsigned take_item(const RecurrenceArgs& p, bool backward) {
  if (p.nseg == 1) return blockIdx.x;
  __shared__ unsigned ticket;
  if (threadIdx.x == 0)
    ticket = __hip_atomic_fetch_add(
        (unsigned*)((unsigned long long*)p.ws + counter_word(p, backward)), 1u, __ATOMIC_RELAXED,
        __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(ticket);
}
struct Place {
  int b, d, seg, len;
  long unit;
  bool live;  // all of a lane's channels are there or none
};
template <int VEC>
__device__ __forceinline__ Place place(const RecurrenceArgs& p, unsigned item, bool backward) {
  Place at;
  const int units = p.B * p.strips;
  const int u = item % units, s = item / units;
  at.seg = backward ? p.nseg - 1 - s : s;
  at.unit = u;
  at.b = u / p.strips;
  at.d = ((u % p.strips) * 64 + (threadIdx.x & 63)) * VEC;
  at.live = at.d < p.D;
  at.len = p.lengths ? min(max(p.lengths[at.b], 0), p.T) : p.T;
  return at;
}

// VEC values of a row, and their store.
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[VEC]) {
  typedef T TV __attribute__((ext_vector_type(VEC)));
  if constexpr (VEC == 1) {
    out[0] = to_f32<T>(p[0]);
  } else {
    const TV x = *(const TV*)p;
#pragma unroll
    for (int e = 0; e < VEC; ++e) out[e] = to_f32<T>(x[e]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[VEC]) {
  typedef T TV __attribute__((ext_vector_type(VEC)));
  if constexpr (VEC == 1) {
    p[0] = from_f32<T>(x[0]);
  } else {
    TV y;
#pragma unroll
    for (int e = 0; e < VEC; ++e) y[e] = from_f32<T>(x[e]);
    *(TV*)p = y;
  }
}

template <typename TX, typename TG, int VEC>
__global__ __launch_bounds__(64 * kWaves, 4) void recurrence_fwd_kernel(RecurrenceArgs p) {
  constexpr int TOK = kTok<VEC>;
  __shared__ Map maps[kWaves][VEC][64];
  __shared__ float enter[VEC][64];
  const unsigned item = take_item(p, false);
  if (item >= gridDim.x) return;
  const Place at = place<VEC>(p, item, false);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = (at.seg * kWaves + wave) * TOK;
  const int d = at.live ? at.d : 0;
  const long base = (long)at.b * p.T * p.D + d;
  const TX* x = (const TX*)p.x + base;
  const TG* g = (const TG*)p.g + base;

  float a[TOK][VEC], v[TOK][VEC];
  if (t0 < p.T) {
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      // rows past the end read the last one; what they read is not used
      const long row = (long)min(t0 + i, p.T - 1) * p.D;
      load_vec<TX, VEC>(x + row, v[i]);
      load_vec<TG, VEC>(g + row, a[i]);
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    float A = 1.f, X = 0.f;
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      const bool in = t0 + i < at.len;
      a[i][e] = in ? fexp(a[i][e]) : 1.f;
      v[i][e] = in ? v[i][e] : 0.f;
      X = a[i][e] * X + v[i][e];
      A *= a[i][e];
    }
    maps[wave][e][lane] = Map{no_underflow(A, a, e), X};
  }
  __syncthreads();
  // the first waves join the maps, one for each of a lane's channels
  if (wave < VEC) {
    const int e = wave;
    Map m = maps[0][e][lane];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) m = compose(maps[k][e][lane], m);
    const float h0 = p.h0 && at.live ? p.h0[(long)at.b * p.D + d + e] : 0.f;
    const long stride = (long)p.B * p.strips * 64 * VEC;
    unsigned long long* w =
        (unsigned long long*)p.ws + at.seg * stride + (at.unit * VEC + e) * 64 + lane;
    const bool last = at.seg == p.nseg - 1;
    if (at.live && !last && at.seg > 0) publish(w, m);
    const float h = look_back(w - stride, -stride, at.seg, h0, at.live);
    const float out = apply(m, h);
    if (at.live && !last) publish_state(w, out);
    if (at.live && last && p.ht) p.ht[(long)at.b * p.D + d + e] = out;
    if (at.live && p.carry) p.carry[((long)at.b * p.nseg + at.seg) * p.D + d + e] = h;
    enter[e][lane] = h;
  }
  __syncthreads();
  float h[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    h[e] = enter[e][lane];
    for (int k = 0; k < wave; ++k) h[e] = apply(maps[k][e][lane], h[e]);
  }
  TX* o = (TX*)p.o + base;
#pragma unroll
  for (int i = 0; i < TOK; ++i) {
    float y[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      h[e] = a[i][e] * h[e] + v[i][e];
      y[e] = t0 + i < at.len ? h[e] : 0.f;
    }
    if (at.live && t0 + i < p.T) store_vec<TX, VEC>(o + (long)(t0 + i) * p.D, y);
  }
}

template <typename TX, typename TG, int VEC>
__global__ __launch_bounds__(64 * kWaves, 4) void recurrence_bwd_kernel(RecurrenceArgs p) {
  constexpr int TOK = kTok<VEC>;
  __shared__ Map fwd[kWaves][VEC][64], bwd[kWaves][VEC][64];
  __shared__ float enter[VEC][64];
  const unsigned item = take_item(p, true);
  if (item >= gridDim.x) return;
  const Place at = place<VEC>(p, item, true);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = (at.seg * kWaves + wave) * TOK;
  const int d = at.live ? at.d : 0;
  const long base = (long)at.b * p.T * p.D + d;
  const TX *x = (const TX*)p.x + base, *go = (const TX*)p.go + base;
  const TG* g = (const TG*)p.g + base;

  float a[TOK][VEC], v[TOK][VEC], q[TOK][VEC];
  if (t0 < p.T) {
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      const long row = (long)min(t0 + i, p.T - 1) * p.D;
      load_vec<TG, VEC>(g + row, a[i]);
      load_vec<TX, VEC>(go + row, q[i]);
      load_vec<TX, VEC>(x + row, v[i]);
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    float A = 1.f, X = 0.f, E = 0.f;
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      const bool in = t0 + i < at.len;
      a[i][e] = in ? fexp(a[i][e]) : 1.f;
      v[i][e] = in ? v[i][e] : 0.f;
      q[i][e] = in ? q[i][e] : 0.f;
      X = a[i][e] * X + v[i][e];
      A *= a[i][e];
    }
#pragma unroll
    for (int i = TOK - 1; i >= 0; --i) E = a[i][e] * (q[i][e] + E);
    A = no_underflow(A, a, e);
    fwd[wave][e][lane] = Map{A, X};
    bwd[wave][e][lane] = Map{A, E};
  }
  __syncthreads();
  if (wave < VEC) {
    const int e = wave;
    Map m = bwd[kWaves - 1][e][lane];
#pragma unroll
    for (int k = kWaves - 2; k >= 0; --k) m = compose(bwd[k][e][lane], m);
    const float end = p.ght && at.live ? p.ght[(long)at.b * p.D + d + e] : 0.f;
    const long stride = (long)p.B * p.strips * 64 * VEC;
    unsigned long long* w =
        (unsigned long long*)p.ws + at.seg * stride + (at.unit * VEC + e) * 64 + lane;
    const int after = p.nseg - 1 - at.seg;
    if (at.live && after > 0 && at.seg > 0) publish(w, m);
    const float in = look_back(w + stride, stride, after, end, at.live);
    const float out = apply(m, in);
    if (at.live && at.seg > 0) publish_state(w, out);
    if (at.live && at.seg == 0 && p.dh0) p.dh0[(long)at.b * p.D + d + e] = out;
    enter[e][lane] = in;
  }
  // the state that enters this wave's tokens, while the first waves look ahead
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    float h = p.carry[((long)at.b * p.nseg + at.seg) * p.D + d + e];
    for (int k = 0; k < wave; ++k) h = apply(fwd[k][e][lane], h);
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      const float was = h;
      h = a[i][e] * h + v[i][e];
      v[i][e] = was;
    }
  }
  __syncthreads();
  float s[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    s[e] = enter[e][lane];
    for (int k = kWaves - 1; k > wave; --k) s[e] = apply(bwd[k][e][lane], s[e]);
  }
  TX* dx = (TX*)p.dx + base;
  TG* dg = (TG*)p.dg + base;
#pragma unroll
  for (int i = TOK - 1; i >= 0; --i) {
    const bool in = t0 + i < at.len;
    float y[VEC], z[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float dh = q[i][e] + s[e];
      s[e] = a[i][e] * dh;
      y[e] = in ? dh : 0.f;
      z[e] = in ? s[e] * v[i][e] : 0.f;
    }
    if (at.live && t0 + i < p.T) {
      store_vec<TX, VEC>(dx + (long)(t0 + i) * p.D, y);
      store_vec<TG, VEC>(dg + (long)(t0 + i) * p.D, z);
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

template <typename TX, typename TG, int VEC>
static hipError_t launch_scan(int what, const RecurrenceArgs& p, hipStream_t stream) {
  const long units = (long)p.B * p.strips;
  if (p.nseg > 1) {
    const long n = units * 64 * VEC * p.nseg;
    const long want = (n + 1023) / 1024;
    hipLaunchKernelGGL(fill_empty_kernel, dim3((unsigned)(want < 1024 ? want : 1024)), dim3(256), 0,
                       stream, (unsigned long long*)p.ws, n, counter_word(p, what == 1));
  }
  const dim3 grid((unsigned)(units * p.nseg)), block(64 * kWaves);
  if (what == 0)
    hipLaunchKernelGGL((recurrence_fwd_kernel<TX, TG, VEC>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((recurrence_bwd_kernel<TX, TG, VEC>), grid, block, 0, stream, p);
  return hipGetLastError();
}

template <typename TX, typename TG>
static hipError_t launch(int what, const RecurrenceArgs& p, hipStream_t stream) {
  if (what == 2) {
    const long n = (long)p.B * p.D;
    hipLaunchKernelGGL((recurrence_step_kernel<TX, TG>), dim3((unsigned)((n + 255) / 256)),
                       dim3(256), 0, stream, p.ht, (const TX*)p.x, (const TG*)p.g, (TX*)p.o, n);
    return hipGetLastError();
  }
  if constexpr (sizeof(TX) == 2)
    if (p.vec == 2) return launch_scan<TX, TG, 2>(what, p, stream);
  return launch_scan<TX, TG, 1>(what, p, stream);
}

}  // namespace hattn

int hattn_recurrence_segment(int vec) { return (32 / vec) * hattn::kWaves; }

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
