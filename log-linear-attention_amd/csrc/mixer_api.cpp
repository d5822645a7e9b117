// C-ABI entry points of the hybrid stack's mixers and norm (declared in
// include/hattn.h): layer norm, gated linear recurrence, sliding-window attention.
// All checks are made here, on the host; the kernels assume what they establish.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "api_common.h"
#include "layer_norm.h"
#include "recurrence.h"
#include "sliding.h"
#include "sliding_step.h"

using namespace hattn_api;

namespace {

const float kLog2e = 1.4426950408889634f;

// The attention kernels address the rows of one tile by 32-bit offsets.
const long long kMaxTokenStride = 1LL << 24;

// Slots of a cache: the step rounds its runs of slots up, by 32 in each of 256.
const long long kMaxSlots = INT_MAX - (1 << 14);

// Whether n work items, `per` a workgroup (or workgroups in groups of `per`), make a launch: it
// holds at most 2^32 - 1 threads.
bool fits(double n, int per, int threads) { return std::ceil(n / per) * threads < 4294967296.0; }

int check_dtype(int code, const char* what) {
  if (code < HATTN_BF16 || code > HATTN_FP32)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "%s: dtype code %d", what, code);
  return HATTN_OK;
}

bool aligned(std::initializer_list<const void*> ps, size_t n) {
  uintptr_t bits = 0;
  for (const void* p : ps) bits |= (uintptr_t)p;
  return bits % n == 0;
}

int norm_checks(long long rows, int n, int dtype_x, int dtype_r, int dtype_w, bool residual) {
  if (rows <= 0 || n <= 0) return fail(HATTN_ERR_VALUE, "non-positive dimension");
  if (n > kLayerNormMaxN)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "n=%d above %d", n, kLayerNormMaxN);
  if (int st = check_dtype(dtype_x, "x")) return st;
  if (int st = check_dtype(dtype_w, "weight")) return st;
  if (residual && dtype_r != dtype_x && dtype_r != HATTN_FP32)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "residual of dtype code %d with x of %d", dtype_r, dtype_x);
  return HATTN_OK;
}

// 16-bit channels go two to a lane where D is even.
RecurrenceArgs recurrence_shape(int B, int T, int D, int dtype_x) {
  RecurrenceArgs p{};
  p.B = B; p.T = T; p.D = D;
  p.vec = dtype_x != HATTN_FP32 && D % 2 == 0 ? 2 : 1;
  p.strips = (D - 1) / (64 * p.vec) + 1;
  const int tokens = hattn_recurrence_segment(p.vec);
  p.nseg = (T - 1) / tokens + 1;
  return p;
}

int recurrence_types(int B, int T, int D, int dtype_x, int dtype_g) {
  if (B <= 0 || T <= 0 || D <= 0) return fail(HATTN_ERR_VALUE, "non-positive dimension");
  if (int st = check_dtype(dtype_x, "x")) return st;
  if (dtype_g != dtype_x && dtype_g != HATTN_FP32)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "g of dtype code %d with x of %d", dtype_g, dtype_x);
  return HATTN_OK;
}

int recurrence_checks(int B, int T, int D, int dtype_x, int dtype_g) {
  if (int st = recurrence_types(B, T, D, dtype_x, dtype_g)) return st;
  if (T > (1 << 30)) return fail(HATTN_ERR_NOT_IMPLEMENTED, "T=%d above 2^30", T);
  const RecurrenceArgs p = recurrence_shape(B, T, D, dtype_x);
  if (!fits((double)p.B * p.strips * p.nseg, 1, 512))
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "B=%d T=%d D=%d: 2^23 workgroups or more", B, T, D);
  return HATTN_OK;
}

size_t recurrence_ws(const RecurrenceArgs& p) {
  return p.nseg > 1 ? (size_t)p.nseg * p.B * p.strips * 64 * p.vec * 8 : 0;
}

// The scan's tensors: rows of vec channels are read at once.
int recurrence_tensors(const RecurrenceArgs& p, std::initializer_list<const void*> xs,
                       std::initializer_list<const void*> gs, int dtype_x, int dtype_g,
                       size_t ws_bytes) {
  const auto bytes = [](int code) { return code == HATTN_FP32 ? 4 : 2; };
  for (const void* q : xs)
    if (!q) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  for (const void* q : gs)
    if (!q) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  if (!aligned(xs, bytes(dtype_x) * p.vec) || !aligned(gs, bytes(dtype_g) * p.vec))
    return fail(HATTN_ERR_VALUE, "tensor not aligned to %d of its elements", p.vec);
  const size_t need = recurrence_ws(p);
  if (need > 0 && (!p.ws || ws_bytes < need || !aligned({p.ws}, 8)))
    return fail(HATTN_ERR_VALUE, "workspace of %zu bytes, %zu needed", ws_bytes, need);
  return HATTN_OK;
}

int sliding_checks(int B, int H, int G, int D, int window, int sinks, float scale, int dtype) {
  if (B <= 0 || H <= 0 || G <= 0 || D <= 0) return fail(HATTN_ERR_VALUE, "non-positive dimension");
  if (H % G != 0) return fail(HATTN_ERR_VALUE, "H=%d is not a multiple of G=%d", H, G);
  if (window < 1) return fail(HATTN_ERR_VALUE, "window=%d below 1", window);
  if (sinks < 0) return fail(HATTN_ERR_VALUE, "sinks=%d below 0", sinks);
  if (!(scale > 0.f) || !(scale <= 1e30f)) return fail(HATTN_ERR_VALUE, "scale must be positive and finite");
  if (sinks > kMaxSinks)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "sinks=%d above %d", sinks, kMaxSinks);
  if (D % 8 != 0 || D > 128)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "D=%d is not a multiple of 8 up to 128", D);
  if (dtype != HATTN_BF16 && dtype != HATTN_FP16)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "dtype code %d (bf16 or fp16 only)", dtype);
  if ((long long)H * D >= kMaxTokenStride)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "H=%d D=%d: a token of 2^24 elements or more", H, D);
  return HATTN_OK;
}

// Strides in elements, batch / token / head of q, k, v: 16-byte rows.
int stride_checks(const long long* st, int n) {
  for (int i = 0; i < n; ++i)
    if (st[i] % 8 != 0 || st[i] < 0)
      return fail(HATTN_ERR_VALUE, "stride %lld is not a multiple of 8 elements", st[i]);
  for (int i = 1; i < n; i += 3)
    if (st[i] >= kMaxTokenStride)
      return fail(HATTN_ERR_NOT_IMPLEMENTED, "token stride %lld of 2^24 elements or more", st[i]);
  return HATTN_OK;
}

// Workgroups of the forward (and of dQ's kernel), and with `train` of the backward's others.
int sliding_grids(int B, int T, int H, int G, int D, int window, int sinks, bool train) {
  const long long rows = T / 128 + (T % 128 != 0);
  const int W = std::min(window, T), S = std::min(sinks, T);
  const long long far = S > 0 ? (T - W) / kSinkChunk + ((T - W) % kSinkChunk != 0) : 0;
  bool ok = T <= INT_MAX / 2 && fits((double)B * H * rows, 8, 8 * 256);
  if (train && far > 0)
    ok = ok && fits((double)B * H * far * ((S + 31) / 32), 8, 8 * 256) &&
         fits((double)B * G * S * 2 * D, 256, 256);
  return ok ? HATTN_OK
            : fail(HATTN_ERR_NOT_IMPLEMENTED, "B=%d T=%d H=%d: 2^24 workgroups or more", B, T, H);
}

int sliding_fill(SlidingArgs& p, const void* q, const void* k, const void* v, const int* lengths,
                 const long long* strides, int B, int T, int H, int G, int D, int window, int sinks,
                 float scale, int dtype, bool train) {
  if (T <= 0) return fail(HATTN_ERR_VALUE, "non-positive dimension");
  if (int st = sliding_checks(B, H, G, D, window, sinks, scale, dtype)) return st;
  if (int st = sliding_grids(B, T, H, G, D, window, sinks, train)) return st;
  if (!q || !k || !v || !strides) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  if (int st = stride_checks(strides, 9)) return st;
  p = SlidingArgs{};
  p.q = q; p.k = k; p.v = v; p.lengths = lengths;
  p.qb = strides[0]; p.qt = strides[1]; p.qh = strides[2];
  p.kb = strides[3]; p.kt = strides[4]; p.kh = strides[5];
  p.vb = strides[6]; p.vt = strides[7]; p.vh = strides[8];
  p.B = B; p.T = T; p.H = H; p.G = G; p.D = D;
  p.W = std::min(window, T);  // a window of T keys holds every earlier one
  p.S = std::min(sinks, T);
  p.narrow = p.W + p.S <= kNarrow;
  p.scale = scale;
  p.scale2 = scale * kLog2e;
  return HATTN_OK;
}

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

size_t sliding_bwd_delta(int B, int T, int H) { return up16((size_t)B * H * T * sizeof(float)); }

// Workgroups that one row and key head's slots are cut into: enough that the card has
// 1024 of them, where each keeps at least 128 slots (a tile for each of its waves).
int step_splits(int B, int H, int G, int slots) {
  const long base = (long)B * G * ((H / G + 15) / 16);
  const long want = (1024 + base - 1) / base, most = (slots + 127) / 128;
  return (int)std::max(1L, std::min({want, most, (long)kStepSplits}));
}

}  // namespace

extern "C" {

int hattn_layer_norm_fwd(const void* x, const void* residual, const void* weight, const void* bias,
                         void* y, void* s, float* mean, float* rstd, long long rows, int n,
                         float eps, int dtype_x, int dtype_r, int dtype_w, void* stream) {
  if (int st = norm_checks(rows, n, dtype_x, dtype_r, dtype_w, residual != nullptr)) return st;
  if (!x || !y || (residual && !s) || !mean != !rstd) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  return check_hip(hattn_layer_norm_fwd_launch(x, residual, weight, bias, y, s, mean, rstd,
                                               (long)rows, n, eps, dtype_x, dtype_r, dtype_w,
                                               (hipStream_t)stream),
                   "hattn_layer_norm_fwd launch");
}

size_t hattn_layer_norm_bwd_workspace(long long rows, int n) {
  if (rows <= 0 || n <= 0 || n > kLayerNormMaxN) return 0;
  return hattn_layer_norm_bwd_ws_bytes((long)rows, n);
}

int hattn_layer_norm_bwd(const void* s, const void* weight, const float* mean, const float* rstd,
                         const void* dy, const void* ds, void* dx, void* dresidual, void* dweight,
                         void* dbias, long long rows, int n, int dtype_x, int dtype_s, int dtype_w,
                         void* ws, size_t ws_bytes, void* stream) {
  if (int st = norm_checks(rows, n, dtype_x, dtype_s, dtype_w, true)) return st;
  if (!s || !mean || !rstd || !dy) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  if (dweight || dbias) {
    const size_t need = hattn_layer_norm_bwd_ws_bytes((long)rows, n);
    if (!ws || ws_bytes < need)
      return fail(HATTN_ERR_VALUE, "workspace of %zu bytes, %zu needed", ws_bytes, need);
  }
  return check_hip(hattn_layer_norm_bwd_launch(s, weight, mean, rstd, dy, ds, dx, dresidual, dweight,
                                               dbias, (float*)ws, (long)rows, n, dtype_x, dtype_s,
                                               dtype_w, (hipStream_t)stream),
                   "hattn_layer_norm_bwd launch");
}

int hattn_gated_recurrence_segments(int T, int D, int dtype_x) {
  return recurrence_checks(1, T, D, dtype_x, dtype_x) == HATTN_OK
             ? recurrence_shape(1, T, D, dtype_x).nseg : 0;
}

size_t hattn_gated_recurrence_workspace(int B, int T, int D, int dtype_x) {
  return recurrence_checks(B, T, D, dtype_x, dtype_x) == HATTN_OK
             ? recurrence_ws(recurrence_shape(B, T, D, dtype_x)) : 0;
}

int hattn_gated_recurrence_fwd(const void* x, const void* g, const float* h0, const int* lengths,
                               void* o, float* ht, float* carry, int B, int T, int D, int dtype_x,
                               int dtype_g, void* ws, size_t ws_bytes, void* stream) {
  if (int st = recurrence_checks(B, T, D, dtype_x, dtype_g)) return st;
  RecurrenceArgs p = recurrence_shape(B, T, D, dtype_x);
  p.x = x; p.g = g; p.h0 = h0; p.lengths = lengths; p.o = o; p.ht = ht; p.carry = carry; p.ws = ws;
  if (int st = recurrence_tensors(p, {x, o}, {g}, dtype_x, dtype_g, ws_bytes)) return st;
  return check_hip(hattn_recurrence_launch(0, p, dtype_x, dtype_g, (hipStream_t)stream),
                   "hattn_gated_recurrence_fwd launch");
}

int hattn_gated_recurrence_bwd(const void* x, const void* g, const float* carry,
                               const int* lengths, const void* dout, const float* dht, void* dx,
                               void* dg, float* dh0, int B, int T, int D, int dtype_x, int dtype_g,
                               void* ws, size_t ws_bytes, void* stream) {
  if (int st = recurrence_checks(B, T, D, dtype_x, dtype_g)) return st;
  if (!carry) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  RecurrenceArgs p = recurrence_shape(B, T, D, dtype_x);
  p.x = x; p.g = g; p.go = dout; p.ght = dht; p.lengths = lengths; p.dx = dx; p.dg = dg;
  p.dh0 = dh0; p.carry = const_cast<float*>(carry); p.ws = ws;
  if (int st = recurrence_tensors(p, {x, dout, dx}, {g, dg}, dtype_x, dtype_g, ws_bytes)) return st;
  return check_hip(hattn_recurrence_launch(1, p, dtype_x, dtype_g, (hipStream_t)stream),
                   "hattn_gated_recurrence_bwd launch");
}

int hattn_gated_recurrence_step(float* state, const void* x, const void* g, void* o, int B, int D,
                                int dtype_x, int dtype_g, void* stream) {
  if (int st = recurrence_types(B, 1, D, dtype_x, dtype_g)) return st;
  if (!fits((double)B * D, 256, 256))
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "B=%d D=%d: 2^32 channels or more", B, D);
  if (!state || !x || !g || !o) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  RecurrenceArgs p{};
  p.x = x; p.g = g; p.o = o; p.ht = state;
  p.B = B; p.T = 1; p.D = D;
  return check_hip(hattn_recurrence_launch(2, p, dtype_x, dtype_g, (hipStream_t)stream),
                   "hattn_gated_recurrence_step launch");
}

int hattn_sliding_fwd(const void* q, const void* k, const void* v, const int* lengths,
                      const long long* strides, void* o, float* lse, int B, int T, int H, int G,
                      int D, int window, int sinks, float scale, int dtype, void* stream) {
  SlidingArgs p;
  // with lse a backward follows: what it refuses is refused here
  if (int st = sliding_fill(p, q, k, v, lengths, strides, B, T, H, G, D, window, sinks, scale, dtype,
                            lse != nullptr))
    return st;
  if (!o) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  if (!aligned({q, k, v, o}, 16)) return fail(HATTN_ERR_VALUE, "tensor not aligned to 16 bytes");
  p.out = o;
  p.lse = lse;
  return check_hip(hattn_sliding_fwd_launch(p, dtype, (hipStream_t)stream),
                   "hattn_sliding_fwd launch");
}

size_t hattn_sliding_bwd_workspace(int B, int T, int H, int G, int D, int window, int sinks) {
  if (B <= 0 || T <= 0 || D <= 0 || window < 1 || sinks < 0 || G <= 0 || H < G) return 0;
  const int S = std::min(sinks, T);
  if (S > kMaxSinks || sliding_grids(B, T, H, G, D, window, sinks, true)) return 0;
  return sliding_bwd_delta(B, T, H) + (size_t)sliding_sink_slots(T, H, G, std::min(window, T), S) *
                                          B * G * S * 2 * D * sizeof(float);
}

int hattn_sliding_bwd(const void* q, const void* k, const void* v, const int* lengths,
                      const long long* strides, const void* o, const float* lse, const void* dout,
                      void* dq, void* dk, void* dv, int B, int T, int H, int G, int D, int window,
                      int sinks, float scale, int dtype, void* ws, size_t ws_bytes, void* stream) {
  SlidingArgs p;
  if (int st = sliding_fill(p, q, k, v, lengths, strides, B, T, H, G, D, window, sinks, scale, dtype,
                            true))
    return st;
  if (!o || !lse || !dout || !dq || !dk || !dv) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  if (!aligned({q, k, v, o, dout, dq, dk, dv, ws}, 16))
    return fail(HATTN_ERR_VALUE, "tensor not aligned to 16 bytes");
  const size_t need = hattn_sliding_bwd_workspace(B, T, H, G, D, window, sinks);
  if (!ws || ws_bytes < need)
    return fail(HATTN_ERR_VALUE, "workspace of %zu bytes, %zu needed", ws_bytes, need);
  p.o = o; p.go = dout; p.lse = const_cast<float*>(lse);
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.delta = (float*)ws;
  if (sliding_sink_slots(T, H, G, p.W, p.S) > 0)
    p.part = (float*)((char*)ws + sliding_bwd_delta(B, T, H));
  return check_hip(hattn_sliding_bwd_launch(p, dtype, (hipStream_t)stream),
                   "hattn_sliding_bwd launch");
}

int hattn_sliding_cache_fill(const void* k, const void* v, const int* lengths,
                             const long long* strides, void* k_cache, void* v_cache, int* counts,
                             int B, int T, int G, int D, int window, int sinks, int dtype,
                             void* stream) {
  if (T <= 0) return fail(HATTN_ERR_VALUE, "non-positive dimension");
  if (int st = sliding_checks(B, G, G, D, window, sinks, 1.f, dtype)) return st;
  if ((long long)window + sinks > INT_MAX ||
      !fits((double)B * G * ((double)sinks + window) * (D / 8), 256, 256))
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "B=%d G=%d window=%d: a cache of 2^32 pieces or more", B, G,
                window);
  if (!k || !v || !strides || !k_cache || !v_cache || !counts)
    return fail(HATTN_ERR_VALUE, "null tensor pointer");
  if (int st = stride_checks(strides, 6)) return st;
  if (!aligned({k, v, k_cache, v_cache}, 16))
    return fail(HATTN_ERR_VALUE, "tensor not aligned to 16 bytes");
  SlidingStepArgs p{};
  p.k = k; p.v = v; p.kc = k_cache; p.vc = v_cache; p.counts = counts;
  p.B = B; p.G = G; p.D = D; p.W = window; p.S = sinks;
  long st[6];
  for (int i = 0; i < 6; ++i) st[i] = (long)strides[i];
  return check_hip(hattn_sliding_cache_launch(p, T, st, lengths, (hipStream_t)stream),
                   "hattn_sliding_cache_fill launch");
}

size_t hattn_sliding_step_workspace(int B, int H, int G, int D, int window, int sinks) {
  if (B <= 0 || G <= 0 || H < G || D <= 0 || window < 1 || sinks < 0 ||
      (long long)window + sinks > kMaxSlots)
    return 0;
  return (size_t)B * H * step_splits(B, H, G, window + sinks) * (D + 2) * sizeof(float);
}

int hattn_sliding_step(const void* q, const void* k, const void* v, void* k_cache, void* v_cache,
                       int* counts, void* o, int B, int H, int G, int D, int window, int sinks,
                       float scale, int dtype, void* ws, size_t ws_bytes, void* stream) {
  if (int st = sliding_checks(B, H, G, D, window, sinks, scale, dtype)) return st;
  if ((long long)window + sinks > kMaxSlots)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "window=%d too large", window);
  const int splits = step_splits(B, H, G, window + sinks), rblocks = (H / G + 15) / 16;
  if (!fits((double)B * G * rblocks * splits, 1, 256) || !fits((double)B * H, 1, 128))
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "B=%d H=%d: too many rows", B, H);
  if (!q || !k || !v || !k_cache || !v_cache || !counts || !o)
    return fail(HATTN_ERR_VALUE, "null tensor pointer");
  if (!aligned({q, k, v, k_cache, v_cache, ws}, 16))
    return fail(HATTN_ERR_VALUE, "tensor not aligned to 16 bytes");
  const size_t need = hattn_sliding_step_workspace(B, H, G, D, window, sinks);
  if (!ws || ws_bytes < need)
    return fail(HATTN_ERR_VALUE, "workspace of %zu bytes, %zu needed", ws_bytes, need);
  SlidingStepArgs p{};
  p.q = q; p.k = k; p.v = v; p.kc = k_cache; p.vc = v_cache; p.counts = counts; p.o = o;
  p.B = B; p.H = H; p.G = G; p.D = D; p.W = window; p.S = sinks;
  p.splits = splits;
  p.rblocks = rblocks;
  p.scale2 = scale * kLog2e;
  p.part = (float*)ws;
  p.stat = p.part + (size_t)B * H * p.splits * D;
  return check_hip(hattn_sliding_step_launch(p, dtype, (hipStream_t)stream),
                   "hattn_sliding_step launch");
}

}  // extern "C"
