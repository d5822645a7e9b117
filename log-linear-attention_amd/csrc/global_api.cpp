// C-ABI entry points of a hybrid stack's global attention (declared in include/hattn.h): rotary
// positions, the cache in 8 bits, attention over it.  All checks are made here, on the host;
// the kernels assume what they establish.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "api_common.h"
#include "quant_cache.h"
#include "rotary.h"

using namespace hattn_api;

namespace {

const float kLog2e = 1.4426950408889634f;
const int kRotaryMaxD = 512;
const int kMaxCapacity = 1 << 30;

// Whether n workgroups make a launch: it holds at most 2^32 - 1 threads.
bool fits(double n, int threads) { return n * threads < 4294967296.0; }

bool aligned(std::initializer_list<const void*> ps, size_t n) {
  uintptr_t bits = 0;
  for (const void* p : ps) bits |= (uintptr_t)p;
  return bits % n == 0;
}

// Strides in elements: 16-byte rows.
int stride_checks(const long long* st, int n) {
  for (int i = 0; i < n; ++i)
    if (st[i] % 8 != 0 || st[i] < 0)
      return fail(HATTN_ERR_VALUE, "stride %lld is not a multiple of 8 elements", st[i]);
  return HATTN_OK;
}

int cache_checks(int B, int G, int D, int capacity) {
  if (B <= 0 || G <= 0 || D <= 0 || capacity <= 0)
    return fail(HATTN_ERR_VALUE, "non-positive dimension");
  if (capacity % kQuantBlock != 0)
    return fail(HATTN_ERR_VALUE, "capacity=%d is not a multiple of %d", capacity, kQuantBlock);
  if (D % 16 != 0 || D > 128)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "D=%d is not a multiple of 16 up to 128", D);
  if (capacity > kMaxCapacity)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "capacity=%d above 2^30", capacity);
  if ((double)B * G > INT_MAX) return fail(HATTN_ERR_NOT_IMPLEMENTED, "B=%d G=%d: too many rows", B, G);
  return HATTN_OK;
}

int half_check(int dtype) {
  if (dtype != HATTN_BF16 && dtype != HATTN_FP16)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "dtype code %d (bf16 or fp16 only)", dtype);
  return HATTN_OK;
}

int cache_tensors(const void* kc, const void* vc, const void* ks, const void* vs, const void* counts) {
  if (!kc || !vc || !ks || !vs || !counts) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  if (!aligned({kc, vc}, 16)) return fail(HATTN_ERR_VALUE, "cache not aligned to 16 bytes");
  return HATTN_OK;
}

QuantArgs cache_args(const void* kc, const void* vc, const float* ks, const float* vs,
                     const int* counts, int B, int G, int D, int capacity) {
  QuantArgs p{};
  p.kc = (unsigned char*)kc; p.vc = (unsigned char*)vc;
  p.ks = (float*)ks; p.vs = (float*)vs;
  p.counts = (int*)counts;
  p.B = B; p.G = G; p.D = D; p.cap = capacity;
  return p;
}

// Blocks that T tokens from any place on can touch.
int touched(int T) { return (T + kQuantBlock - 2) / kQuantBlock + 1; }

// How a call's queries are cut: blocks of 16 or 32 where a row and key head has at most kFewQueries
// (4 rows of up to 32000 tokens, 8 key heads of 128: 64 queries take 63 us so and 87 as part of
// a block of 128, 128 queries 115 and 90),
// else of 128; and parts of a row's tokens, enough that the card has work.  With few rows a workgroup's
// start counts, and 1024 of them (512 with two blocks of queries each) are best: 4 rows of 8000
// to 32000 tokens, 8 key heads of 128: 43 us with 1024, 46 with 2048, 52 with 4096.  With many rows,
// whose lengths differ, more even out the end: 64 rows of up to 9000 tokens 128, 126, 127 us.
struct Cut {
  bool few;
  int rblocks, splits;
};
const int kFewQueries = 64;
Cut cut(int B, int T, int H, int G, int capacity) {
  Cut c;
  const long queries = (long)T * (H / G);
  c.few = queries <= kFewQueries;
  c.rblocks = (int)(c.few ? (queries + 31) / 32 : (queries + 127) / 128);
  const long base = (long)B * G * c.rblocks;
  const long target = !c.few || queries > 16 ? 512 : base < 128 ? 1024 : 2048;
  const long want = (target + base - 1) / base;
  const long most = (capacity + 255) / 256;
  c.splits = (int)std::max(1L, std::min({want, most, (long)kQuantSplits}));
  return c;
}

bool joins(const Cut& c) { return c.few || c.splits > 1; }

int attention_checks(int B, int T, int H, int G, int D, int capacity, float scale, int dtype) {
  if (T <= 0 || H <= 0) return fail(HATTN_ERR_VALUE, "non-positive dimension");
  if (int st = cache_checks(B, G, D, capacity)) return st;
  if (H % G != 0) return fail(HATTN_ERR_VALUE, "H=%d is not a multiple of G=%d", H, G);
  if (!(scale > 0.f) || !(scale <= 1e30f)) return fail(HATTN_ERR_VALUE, "scale must be positive and finite");
  if (int st = half_check(dtype)) return st;
  if ((double)T * (H / G) > (double)(INT_MAX / 2))
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "T=%d H=%d: 2^30 queries of a key head or more", T, H);
  const Cut c = cut(B, T, H, G, capacity);
  if (!fits((double)B * G * c.rblocks * c.splits + 8, 256) ||
      (joins(c) && !fits((double)B * T * H, 512)))
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "B=%d T=%d H=%d: 2^24 workgroups or more", B, T, H);
  return HATTN_OK;
}

// Workspace in floats: the parts, their maxima and sums, and the rows' tokens during a step.
size_t part_floats(int B, int T, int H, const Cut& c, int D) { return (size_t)B * T * H * c.splits * D; }
size_t workspace_bytes(int B, int T, int H, const Cut& c, int D) {
  return (part_floats(B, T, H, c, D) + (size_t)B * T * H * c.splits * 2 + B) * sizeof(float);
}

// The attention's launches on tensors that have been checked.
int attend(QuantArgs& p, const void* q, const long long* strides, void* o, int T, int H, float scale,
           int dtype, void* ws, size_t ws_bytes, hipStream_t stream) {
  const Cut c = cut(p.B, T, H, p.G, p.cap);
  p.q = q;
  p.qb = strides[0]; p.qt = strides[1]; p.qh = strides[2];
  p.o = o;
  p.T = T; p.H = H;
  p.splits = c.splits; p.rblocks = c.rblocks;
  p.scale2 = scale * kLog2e;
  p.part = (float*)ws;
  p.stat = p.part + part_floats(p.B, T, H, c, p.D);
  p.held = (int*)(p.stat + (size_t)p.B * T * H * c.splits * 2);
  if (int st = check_hip(c.few ? hattn_quant_few_launch(p, dtype, stream)
                               : hattn_quant_chunk_launch(p, dtype, stream),
                         "attention over a cache launch"))
    return st;
  return joins(c) ? check_hip(hattn_quant_join_launch(p, dtype, stream), "join launch") : HATTN_OK;
}

int workspace_check(const void* ws, size_t bytes, size_t need) {
  if (need > 0 && (!ws || bytes < need || !aligned({ws}, 16)))
    return fail(HATTN_ERR_VALUE, "workspace of %zu bytes, %zu needed, aligned to 16", bytes, need);
  return HATTN_OK;
}

}  // namespace

extern "C" {

int hattn_rotary(const void* q, const void* k, const long long* strides, void* q_out, void* k_out,
                 const void* freqs, int freqs64, const void* positions, int positions64,
                 long long position_batch, long long position_token, int per_row, int B, int T, int H,
                 int G, int D, int pairs, int interleaved, float scale, int inverse, int dtype,
                 void* stream) {
  if (B <= 0 || T <= 0 || H <= 0 || G < 0 || D <= 0 || pairs <= 0)
    return fail(HATTN_ERR_VALUE, "non-positive dimension");
  if (2LL * pairs > D) return fail(HATTN_ERR_VALUE, "%d pairs in heads of %d", pairs, D);
  if (!(std::fabs(scale) <= 1e30f)) return fail(HATTN_ERR_VALUE, "scale must be finite");
  if (dtype < HATTN_BF16 || dtype > HATTN_FP32)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "dtype code %d", dtype);
  if (D > kRotaryMaxD) return fail(HATTN_ERR_NOT_IMPLEMENTED, "D=%d above %d", D, kRotaryMaxD);
  if ((double)H + G > 1 << 20) return fail(HATTN_ERR_NOT_IMPLEMENTED, "H=%d G=%d: above 2^20", H, G);
  if (!q || !q_out || (G > 0 && (!k || !k_out)) || !strides || !freqs)
    return fail(HATTN_ERR_VALUE, "null tensor pointer");
  const int bytes = dtype == HATTN_FP32 ? 4 : 2, vec = 16 / bytes;
  if (!aligned({q, q_out, G > 0 ? k : q, G > 0 ? k_out : q_out}, bytes) ||
      !aligned({freqs}, freqs64 ? 8 : 4) ||
      !aligned({positions}, positions64 ? 8 : 4))
    return fail(HATTN_ERR_VALUE, "tensor not aligned to its elements");
  RotaryArgs p{};
  p.x[0] = q; p.x[1] = k;
  p.y[0] = q_out; p.y[1] = k_out;
  p.heads[0] = H; p.heads[1] = G;
  // pieces of 16 bytes where every one of them starts on 16 bytes and none holds both a pair and
  // an element that stays
  bool wide = D % vec == 0 && pairs % vec == 0 &&
              aligned({q, q_out, G > 0 ? k : q, G > 0 ? k_out : q_out}, 16);
  for (int i = 0; i < 2; ++i) {
    p.xb[i] = strides[3 * i]; p.xt[i] = strides[3 * i + 1]; p.xh[i] = strides[3 * i + 2];
    if (p.heads[i] > 0) wide = wide && p.xb[i] % vec == 0 && p.xt[i] % vec == 0 && p.xh[i] % vec == 0;
  }
  p.freqs = freqs; p.freq64 = freqs64;
  p.pos = positions; p.pos64 = positions64;
  p.pb = position_batch; p.pt = position_token;
  p.from = per_row;
  p.N = (long)B * T;
  p.T = T; p.D = D; p.pairs = pairs;
  p.scale = scale;
  p.sign = inverse ? -1.f : 1.f;
  const int v = rotary_vec(bytes, wide), lanes = pairs / v + ((D - 2 * pairs) / v + 1) / 2;
  p.cols = 1;
  while (p.cols < lanes) p.cols *= 2;
  // One round of kAhead heads a lane, so that many workgroups, in their several phases, share a CU
  // (4 x 8192 tokens of 32 heads of 64 in bf16: 53 us; with twice the tokens 5 more, half of them 1),
  // but at least 1024 workgroups where the tokens allow it, and sines of at most 8 KB.  Single
  // elements take four rounds (2 x 16384 tokens of 9 heads of 82: 52 us, with one 68).
  const long heads = (long)H + G;
  p.tokens = (int)std::max(1L, std::min({(wide ? 512 : 2048) / (heads * p.cols), (long)(1024 / pairs), p.N / 1024}));
  if (!fits(std::ceil((double)p.N / p.tokens), 256))
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "B=%d T=%d: 2^24 workgroups or more", B, T);
  return check_hip(hattn_rotary_launch(p, dtype, interleaved != 0, wide, (hipStream_t)stream),
                   "hattn_rotary launch");
}

int hattn_quant_cache_append(const void* k, const void* v, const int* lengths,
                             const long long* strides, void* k_codes, void* v_codes, float* k_scale,
                             float* v_scale, int* counts, int B, int T, int G, int D, int capacity,
                             int dtype, void* stream) {
  if (T <= 0) return fail(HATTN_ERR_VALUE, "non-positive dimension");
  if (int st = cache_checks(B, G, D, capacity)) return st;
  if (int st = half_check(dtype)) return st;
  if (T > capacity) return fail(HATTN_ERR_VALUE, "T=%d tokens for a capacity of %d", T, capacity);
  if (!fits((double)B * G * touched(T) * 2, 256))
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "B=%d T=%d G=%d: 2^24 workgroups or more", B, T, G);
  if (!k || !v || !strides) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  if (int st = cache_tensors(k_codes, v_codes, k_scale, v_scale, counts)) return st;
  if (!aligned({k, v}, 16)) return fail(HATTN_ERR_VALUE, "tensor not aligned to 16 bytes");
  if (int st = stride_checks(strides, 6)) return st;
  QuantArgs p = cache_args(k_codes, v_codes, k_scale, v_scale, counts, B, G, D, capacity);
  p.k = k; p.v = v; p.lengths = lengths;
  p.kb = strides[0]; p.kt = strides[1]; p.kh = strides[2];
  p.vb = strides[3]; p.vt = strides[4]; p.vh = strides[5];
  p.T = T;
  p.blocks = touched(T);
  return check_hip(hattn_quant_append_launch(p, dtype, (hipStream_t)stream),
                   "hattn_quant_cache_append launch");
}

int hattn_quant_cache_read(const void* k_codes, const void* v_codes, const float* k_scale,
                           const float* v_scale, const int* counts, void* k, void* v, int B, int G,
                           int D, int capacity, int start, int n, int dtype, void* stream) {
  if (int st = cache_checks(B, G, D, capacity)) return st;
  if (n <= 0 || start < 0 || start > capacity - n)
    return fail(HATTN_ERR_VALUE, "slots [%d, %d + %d) of %d", start, start, n, capacity);
  if (dtype < HATTN_BF16 || dtype > HATTN_FP32)
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "dtype code %d", dtype);
  const int blocks = (start % kQuantBlock + n - 1) / kQuantBlock + 1;
  if (!fits((double)B * G * blocks * 2, 256))
    return fail(HATTN_ERR_NOT_IMPLEMENTED, "B=%d G=%d n=%d: 2^24 workgroups or more", B, G, n);
  if (!k || !v) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  if (int st = cache_tensors(k_codes, v_codes, k_scale, v_scale, counts)) return st;
  if (!aligned({k, v}, 16)) return fail(HATTN_ERR_VALUE, "tensor not aligned to 16 bytes");
  QuantArgs p = cache_args(k_codes, v_codes, k_scale, v_scale, counts, B, G, D, capacity);
  p.ko = k; p.vo = v;
  p.start = start; p.n = n;
  p.blocks = blocks;
  return check_hip(hattn_quant_read_launch(p, dtype, (hipStream_t)stream),
                   "hattn_quant_cache_read launch");
}

size_t hattn_quant_cache_attention_workspace(int B, int T, int H, int G, int D, int capacity) {
  if (attention_checks(B, T, H, G, D, capacity, 1.f, HATTN_BF16)) return 0;
  const Cut c = cut(B, T, H, G, capacity);
  return joins(c) ? workspace_bytes(B, T, H, c, D) : 0;
}

int hattn_quant_cache_attention(const void* q, const int* lengths, const long long* strides,
                                const void* k_codes, const void* v_codes, const float* k_scale,
                                const float* v_scale, const int* counts, void* o, int B, int T, int H,
                                int G, int D, int capacity, float scale, int dtype, void* ws,
                                size_t ws_bytes, void* stream) {
  if (int st = attention_checks(B, T, H, G, D, capacity, scale, dtype)) return st;
  if (!q || !strides || !o) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  if (int st = cache_tensors(k_codes, v_codes, k_scale, v_scale, counts)) return st;
  if (!aligned({q, o}, 16)) return fail(HATTN_ERR_VALUE, "tensor not aligned to 16 bytes");
  if (int st = stride_checks(strides, 3)) return st;
  if (int st = workspace_check(ws, ws_bytes, hattn_quant_cache_attention_workspace(B, T, H, G, D, capacity)))
    return st;
  QuantArgs p = cache_args(k_codes, v_codes, k_scale, v_scale, counts, B, G, D, capacity);
  p.lengths = lengths;
  return attend(p, q, strides, o, T, H, scale, dtype, ws, ws_bytes, (hipStream_t)stream);
}

int hattn_quant_cache_step(const void* q, const void* k, const void* v, const long long* strides,
                           void* k_codes, void* v_codes, float* k_scale, float* v_scale, int* counts,
                           void* o, int B, int H, int G, int D, int capacity, float scale, int dtype,
                           void* ws, size_t ws_bytes, void* stream) {
  if (int st = attention_checks(B, 1, H, G, D, capacity, scale, dtype)) return st;
  if (!fits(B, 1024)) return fail(HATTN_ERR_NOT_IMPLEMENTED, "B=%d: too many rows", B);
  if (!q || !k || !v || !strides || !o) return fail(HATTN_ERR_VALUE, "null tensor pointer");
  if (int st = cache_tensors(k_codes, v_codes, k_scale, v_scale, counts)) return st;
  if (!aligned({q, k, v, o}, 16)) return fail(HATTN_ERR_VALUE, "tensor not aligned to 16 bytes");
  if (int st = stride_checks(strides, 9)) return st;
  if (int st = workspace_check(ws, ws_bytes, hattn_quant_cache_attention_workspace(B, 1, H, G, D, capacity)))
    return st;
  QuantArgs p = cache_args(k_codes, v_codes, k_scale, v_scale, counts, B, G, D, capacity);
  p.k = k; p.v = v;
  p.kb = strides[3]; p.kt = strides[4]; p.kh = strides[5];
  p.vb = strides[6]; p.vt = strides[7]; p.vh = strides[8];
  p.T = 1;
  // Where one workgroup has all queries of a key head, it takes in the token too: a launch less
  // (with 17 to 32 queries the kernel has no registers left for it)
  p.coming = H / G <= 16;
  if (!p.coming)
    if (int st = check_hip(hattn_quant_token_launch(p, dtype, (hipStream_t)stream),
                           "hattn_quant_cache_step launch"))
      return st;
  return attend(p, q, strides, o, 1, H, scale, dtype, ws, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
