// Sliding-window attention backward.  With P = exp2(c S - lse) and delta = rowsum(go o):
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q.
//
// Two kernels make S and dP again, one with a row's queries (dQ), one with a block's keys
// in registers (dK, dV), seven products where one kernel would do with five: but every
// sum has one owner and one order, and dQ needs no atomics.  All heads that share a key
// are summed in its workgroup.
//
// A sink is seen by every query, a key by W of them, so the sinks' far queries (those
// whose window does not reach them) are cut into chunks of kSinkChunk queries and one
// head, each with its own partial sums in 32 bits; the near queries' sum is one more,
// and a last kernel adds them in order.
//
// P and dS are rounded to the inputs' type, which the matrix instructions take: dV's error
// against 64 bits is 1.4 times that of one rounding.  delta is taken from the rounded o, whose
// half step is a small part of dP where many keys share the weight.  In a window of up to
// kNarrow keys, and for the first queries of any (whose gradients are the largest), it is not,
// and there dQ's kernel first takes delta = sum P dP in a pass of its own: dQ's error is then
// 1.42 times that of one rounding, and not up to 1.9 times.
//
// Measured at B 1, T 16384, 16 heads of 128 in 4 groups, window 4096, and at B 4, T 8192, 16
// heads of 64, window 1024: dQ 762 and 277 us (946 and 697 TFLOP/s of its three products), dK
// and dV 1290 and 337 us (746 and 765 of its four), the sinks 30 and 26.  dQ is bound as the
// forward is.  dK and dV hold two accumulators and two operands, 372 registers at D 128: one
// wave a SIMD, whose products wait for its own vector instructions.
//
// A query that sees one key has P = 1 and dS = 0 whatever its scores: dP - delta is not
// left to cancel there.
#include <climits>

#include "sliding_device.h"

namespace hattn {

template <typename E, int DP>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void sliding_bwd_q_kernel(SlidingArgs p) {
  constexpr int BN = 32;
  __shared__ __attribute__((aligned(16))) __bf16 K0[BN * DP], V0[BN * DP], K1[BN * DP], V1[BN * DP];
  const int lane = threadIdx.x & 63, ln = lane & 31, hf = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = p.H / p.G, nblk = (p.T + 127) / 128;
  const long item = work_item((long)p.B * p.H * nblk);
  if (item < 0) return;
  const int r = item % R, blk = item / R % nblk, bg = item / R / nblk;
  const int b = bg / p.G, g = bg % p.G, h = g * R + r, t0 = blk * 128;
  const int len = row_length(p, b);
  const int tw = t0 + 32 * wave, t = tw + ln;
  const long row = ((long)b * p.T + t) * p.H + h;
  __bf16* dq = (__bf16*)p.dq + row * p.D;

  floatx16 acc[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = zero16();
  if (t0 >= len) {
    if (t < p.T) store_t<E, DP>(dq, acc, 0.f, false, p.D);
    return;
  }
  const __bf16* k = (const __bf16*)p.k + b * p.kb + g * p.kh;
  const __bf16* v = (const __bf16*)p.v + b * p.vb + g * p.vh;
  const int tc = min(t, len - 1);  // rows past the end read the last one
  const long rc = (((long)b * p.T + tc) * p.H + h) * p.D, stat = ((long)b * p.H + h) * p.T;
  bf16x8 qf[DP / 16], gf[DP / 16];
  load_frags<DP>((const __bf16*)p.q + b * p.qb + h * p.qh + tc * p.qt, p.D, qf);
  load_frags<DP>((const __bf16*)p.go + rc, p.D, gf);
  const bool narrow = p.narrow || t0 == 0;
  float delta = 0.f;
  if (!narrow) {
    bf16x8 of[DP / 16];
    load_frags<DP>((const __bf16*)p.o + rc, p.D, of);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta += from16<E>(gf[s][j]) * from16<E>(of[s][j]);
    delta += __shfl_xor(delta, 32, 64);
    if (hf == 0 && t < len) p.delta[stat + t] = delta;
  }
  const float lse = p.lse[stat + tc];
  const bool alone = t == 0 || (p.W == 1 && p.S == 0);
  float sum = 0.f;
  const KeyList<BN> keys(t0, 128, len, p.W, p.S);
  const int tiles = keys.tiles();

  const TileLoad<DP, BN, 4> tile(p.D);
  const auto stage = [&](int j, __bf16* K, __bf16* V) __attribute__((always_inline)) {
    keys.load(tile, j, k, p.kt, K);
    keys.load(tile, j, v, p.vt, V);
  };
  // DELTA: only the sum of P dP over the keys
  const auto step = [&](auto MASK, auto DELTA, int j, const __bf16* K, const __bf16* V, __bf16* Kn,
                        __bf16* Vn) __attribute__((always_inline)) {
    tile_barrier();
    if (j + 1 < tiles) stage(j + 1, Kn, Vn);
    int kind = kFull;
    if constexpr (MASK.value) kind = tile_kind(keys, j, tw, p.W, p.S);
    if (kind == kSkip) return;
#pragma unroll
    for (int kt = 0; kt < BN / 32; ++kt) {
      floatx16 s = zero16(), dp = zero16();
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) s = mfma32<E>(row_frag<DP>(K, 32 * kt, c), qf[c], s);
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) dp = mfma32<E>(row_frag<DP>(V, 32 * kt, c), gf[c], dp);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[i] = exp2_(s[i] * p.scale2 - lse) * (DELTA.value ? dp[i] : dp[i] - delta);
      if constexpr (MASK.value) {
        if (kind == kMask) {
          const TileMask seen(keys, j, t, p.W, p.S);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[i] = (seen(32 * kt + 8 * (i >> 2) + (i & 3)) & !alone) ? s[i] : 0.f;
        }
      }
      if constexpr (DELTA.value) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += s[i];
        continue;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bf16x8 sf = pack8<E>(s, c);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
          acc[dt] = mfma32<E>(tr32<DP>(K, 32 * kt + 16 * c, 32 * dt), sf, acc[dt]);
      }
    }
  };
  stage(0, K0, V0);
  int j = 0;
  const auto pairs = [&](auto MASK, auto DELTA) __attribute__((always_inline)) {
    step(MASK, DELTA, j, K0, V0, K1, V1);
    if (j + 1 < tiles) step(MASK, DELTA, j + 1, K1, V1, K0, V0);
  };
  if (narrow) {
    for (; j < tiles; j += 2) pairs(Bool<true>(), Bool<true>());
    delta = sum + __shfl_xor(sum, 32, 64);
    if (hf == 0 && t < len) p.delta[stat + t] = delta;
    __syncthreads();
    stage(0, K0, V0);
    j = 0;
  }
  // where each query sees one key, every tile is masked
  const int lo = keys.first_whole(t0, 128, p.W), hi = alone ? 0 : keys.end_whole(t0);
  for (; j < tiles && !(j >= lo && j + 2 <= hi); j += 2) pairs(Bool<true>(), Bool<false>());
  for (; j + 2 <= hi; j += 2) pairs(Bool<false>(), Bool<false>());
  for (; j < tiles; j += 2) pairs(Bool<true>(), Bool<false>());
  if (t < p.T) store_t<E, DP>(dq, acc, p.scale, t < len, p.D);
}

// dK and dV.  SINKS false: 128 keys a workgroup, 32 a wave, over the queries whose window
// holds them, 64 at a time.  SINKS true: the same 32 sinks in all four waves, over 128 far
// queries at a time, 32 a wave; the waves' sums meet in LDS at the end.
template <typename E, int DP, bool SINKS>
__global__ __launch_bounds__(256, DP == 64 && !SINKS ? 2 : 1) void sliding_bwd_kv_kernel(
    SlidingArgs p) {
  constexpr int QT = SINKS ? 128 : 64;
  __shared__ __attribute__((aligned(16))) __bf16 Q0[QT * DP], O0[QT * DP], Q1[QT * DP], O1[QT * DP];
  __shared__ __attribute__((aligned(16))) float st0[2 * QT], st1[2 * QT];
  const int lane = threadIdx.x & 63, ln = lane & 31, hf = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = p.H / p.G;
  const int chunks = SINKS ? (p.T - p.W + kSinkChunk - 1) / kSinkChunk : 1;
  const int nblk = SINKS ? (p.S + 31) / 32 * chunks * R : (p.T + 127) / 128;
  const long item = work_item((long)p.B * p.G * nblk);
  if (item < 0) return;
  const int bg = item / nblk, b = bg / p.G, g = bg % p.G;
  int blk = item % nblk;
  const int len = row_length(p, b);
  int key0, first, end, heads = R, h0 = g * R, slot = 0;
  if constexpr (SINKS) {
    h0 += blk % R;
    heads = 1;
    const int chunk = blk / R % chunks;
    slot = 1 + chunk * R + blk % R;
    key0 = blk / R / chunks * 32;
    first = p.W + chunk * kSinkChunk;
    end = min(first + kSinkChunk, len);
  } else {
    key0 = blk * 128;
    first = key0;
    end = min(key0 + 128 + min(p.W, p.T) - 1, len);
  }
  const int kw = SINKS ? key0 : key0 + 32 * wave, key = kw + ln;
  const int kc = max(0, min(key, len - 1));  // keys past the end read the last one
  bf16x8 kf[DP / 16], vf[DP / 16];
  load_frags<DP>((const __bf16*)p.k + b * p.kb + g * p.kh + kc * p.kt, p.D, kf);
  load_frags<DP>((const __bf16*)p.v + b * p.vb + g * p.vh + kc * p.vt, p.D, vf);
  floatx16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) dk[dt] = dv[dt] = zero16();
  const bool alone = p.W == 1 && p.S == 0;  // every query sees one key
  const int per = end > first ? (end - first + QT - 1) / QT : 0;  // tiles of one head
  const int tiles = per * heads;

  const TileLoad<DP, QT, 4> tile(p.D);
  const auto stage = [&](int j, __bf16* Q, __bf16* O, float* st) __attribute__((always_inline)) {
    const int h = h0 + j / per, tq = first + j % per * QT;
    const __bf16* q = (const __bf16*)p.q + b * p.qb + h * p.qh;
    const __bf16* go = (const __bf16*)p.go + ((long)b * p.T * p.H + h) * p.D;
    tile.run(q, p.qt, tq, end - 1, Q);
    tile.run(go, (long)p.H * p.D, tq, end - 1, O);
    // lse and delta of the tile's rows, 64 values a wave
    if (wave < 2 * QT / 64) {
      const int i = 64 * wave + lane;
      const float* src = (i < QT ? p.lse : p.delta) + ((long)b * p.H + h) * p.T;
      const int t = min(tq + i % QT, end - 1);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + t),
                                       (__attribute__((address_space(3))) void*)(st + 64 * wave), 4,
                                       0, 0);
    }
  };
  const auto step = [&](int j, const __bf16* Q, const __bf16* O, const float* st, __bf16* Qn,
                        __bf16* On, float* stn) __attribute__((always_inline)) {
    tile_barrier();
    if (j + 1 < tiles) stage(j + 1, Qn, On, stn);
    const int tq = first + j % per * QT;
#pragma unroll
    for (int u = 0; u < (SINKS ? 1 : 2); ++u) {
      // the queries tw .. tw + 31 against the wave's keys
      const int q0 = SINKS ? 32 * wave : 32 * u, tw = tq + q0;
      if (tw >= end || (!SINKS && (tw + 31 < kw || tw >= kw + 31 + p.W))) continue;
      const bool mask = alone || tw == 0 || tw + 31 >= end ||
                        (SINKS ? tw - kw - 31 < p.W : tw < kw + 31 || tw + 31 >= kw + p.W);
      floatx16 s = zero16(), dp = zero16();
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) s = mfma32<E>(row_frag<DP>(Q, q0, c), kf[c], s);
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) dp = mfma32<E>(row_frag<DP>(O, q0, c), vf[c], dp);
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const floatx4 lse = *(const floatx4*)(st + q0 + 8 * i4 + 4 * hf);
        const floatx4 delta = *(const floatx4*)(st + QT + q0 + 8 * i4 + 4 * hf);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[4 * i4 + i] = exp2_(s[4 * i4 + i] * p.scale2 - lse[i]);
          dp[4 * i4 + i] = s[4 * i4 + i] * (dp[4 * i4 + i] - delta[i]);
        }
      }
      if (mask) {
        // query tw + 4 hf + place sees the key from place >= low on, up to place <= up
        const int from = tw + 4 * hf, up = SINKS ? end - 1 - from : min(end, key + p.W) - 1 - from;
        const int low = SINKS ? key + p.W - from : key - from, one = alone ? INT_MAX : -from;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int place = 8 * (i >> 2) + (i & 3);
          const bool seen = (place >= low) & (place <= up);
          s[i] = seen ? s[i] : 0.f;
          dp[i] = (seen & (place > one)) ? dp[i] : 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bf16x8 pf = pack8<E>(s, c), sf = pack8<E>(dp, c);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) {
          dv[dt] = mfma32<E>(tr32<DP>(O, q0 + 16 * c, 32 * dt), pf, dv[dt]);
          dk[dt] = mfma32<E>(tr32<DP>(Q, q0 + 16 * c, 32 * dt), sf, dk[dt]);
        }
      }
    }
  };
  if (tiles > 0) stage(0, Q0, O0, st0);
  for (int j = 0; j < tiles; j += 2) {
    step(j, Q0, O0, st0, Q1, O1, st1);
    if (j + 1 < tiles) step(j + 1, Q1, O1, st1, Q0, O0, st0);
  }

  const bool live = key < len;  // the others' sums are zero, or 0 times what is not finite
  // row (slot, b, g, key) of the partial sums: D of dK, D of dV
  float* part = p.part + ((((long)slot * p.B + b) * p.G + g) * p.S + key) * 2 * p.D;
  const auto put = [&](const floatx16(&acc)[DP / 32], float* dst) __attribute__((always_inline)) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * dt + 8 * i + 4 * hf;
        if (d < p.D)
          *(floatx4*)(dst + d) = live ? floatx4{acc[dt][4 * i], acc[dt][4 * i + 1],
                                                acc[dt][4 * i + 2], acc[dt][4 * i + 3]}
                                      : floatx4{};
      }
  };
  if constexpr (SINKS) {
    // the waves' sums, wave after wave, through Q0 (16 KB at least: 32 keys of DP floats)
    float* sum = (float*)Q0;
    const auto join = [&](floatx16(&acc)[DP / 32]) __attribute__((always_inline)) {
      for (int w = 0; w < 4; ++w) {
        __syncthreads();
        if (wave == w)
#pragma unroll
          for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float* at = sum + (dt * 16 + i) * 64 + lane;
              if (w > 0) acc[dt][i] += *at;
              if (w < 3) *at = acc[dt][i];
            }
      }
    };
    join(dk);
    join(dv);
    if (wave == 3 && key < p.S) {
      put(dk, part);
      put(dv, part + p.D);
    }
  } else {
    if (key >= p.T) return;
    if (p.part && key < p.S) {
      put(dk, part);
      put(dv, part + p.D);
      return;
    }
    const long row = (((long)b * p.T + key) * p.G + g) * p.D;
    store_t<E, DP>((__bf16*)p.dk + row, dk, p.scale, live, p.D);
    store_t<E, DP>((__bf16*)p.dv + row, dv, 1.f, live, p.D);
  }
}

// Adds the partial sums of the sinks' gradients: one thread an element of dK or dV.
template <typename E>
__global__ __launch_bounds__(256) void sliding_bwd_sinks_kernel(SlidingArgs p, int slots) {
  const long n = (long)p.B * p.G * p.S * 2 * p.D, i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float x = 0.f, y[8];
  for (int s = 0; s < slots; s += 8) {  // eight loads in flight: the sum waits for memory
#pragma unroll
    for (int u = 0; u < 8; ++u) y[u] = s + u < slots ? p.part[(s + u) * n + i] : 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) x += y[u];
  }
  const int d = i % p.D, which = i / p.D % 2, key = i / (2 * p.D) % p.S;
  const long bg = i / (2 * p.D) / p.S, b = bg / p.G, g = bg % p.G;
  const long at = ((b * p.T + key) * p.G + g) * p.D + d;
  if (which == 0) ((__bf16*)p.dk)[at] = to16<E>(x * p.scale);
  else ((__bf16*)p.dv)[at] = to16<E>(x);
}

template <typename E, int DP>
static hipError_t launch_bwd(const SlidingArgs& p, hipStream_t stream) {
  const long nblk = (p.T + 127) / 128;
  const int slots = sliding_sink_slots(p.T, p.H, p.G, p.W, p.S);
  hipLaunchKernelGGL((sliding_bwd_q_kernel<E, DP>), dim3((unsigned)work_grid(p.B * p.H * nblk)),
                     dim3(256), 0, stream, p);
  hipLaunchKernelGGL((sliding_bwd_kv_kernel<E, DP, false>),
                     dim3((unsigned)work_grid(p.B * p.G * nblk)), dim3(256), 0, stream, p);
  if (slots > 0) {
    const long items = (long)p.B * p.G * ((p.S + 31) / 32) * (slots - 1);
    hipLaunchKernelGGL((sliding_bwd_kv_kernel<E, DP, true>), dim3((unsigned)work_grid(items)),
                       dim3(256), 0, stream, p);
    const long n = (long)p.B * p.G * p.S * 2 * p.D;
    hipLaunchKernelGGL((sliding_bwd_sinks_kernel<E>), dim3((unsigned)((n + 255) / 256)), dim3(256),
                       0, stream, p, slots);
  }
  return hipGetLastError();
}

}  // namespace hattn

hipError_t hattn_sliding_bwd_launch(const SlidingArgs& p, int dtype, hipStream_t stream) {
  using namespace hattn;
  if (dtype == 1)
    return p.D <= 64 ? launch_bwd<_Float16, 64>(p, stream) : launch_bwd<_Float16, 128>(p, stream);
  return p.D <= 64 ? launch_bwd<__bf16, 64>(p, stream) : launch_bwd<__bf16, 128>(p, stream);
}
