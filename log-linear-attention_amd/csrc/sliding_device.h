// Sliding-window attention with sinks: what its kernels share.
//
// Query t sees key s where s <= t and (t - s < W or s < S): a window of W keys that
// ends with the query's own, and the first S tokens (the sinks).
//
// All products are 32x32x16 MFMAs, lane = 32 hf + ln (ln in [0, 32), hf in {0, 1}):
//   A operand : lane holds A[m = ln][k = 8 hf + j], j = 0..7
//   B operand : lane holds B[k = 8 hf + j][n = ln]
//   C / D     : lane holds D[m = 8 (i >> 2) + 4 hf + (i & 3)][n = ln], i = 0..15
// The scores are computed with the softmax's row as n, so a row's maximum, sum and
// scale live in one lane (and its partner at ln + 32).  Registers 8 s .. 8 s + 7 of
// such a D tile are then the B operand of a product over m, with the order of m
//   16 s + 8 (j >> 2) + 4 hf + (j & 3)
// in which tr32() reads the other operand, transposed, from its tile in LDS: the
// probabilities never leave their registers.
//
// A tile in LDS is rows of DP (64 or 128) 16-bit values with no padding, as the
// asynchronous loads write it; 16-byte piece c of row r lies at piece c ^ swizzle(r),
// so that both the reads along rows (32 rows, one piece) and the transposed reads
// (4 rows, four pieces) meet every bank once.
#pragma once

#include "common.h"
#include "sliding.h"

namespace hattn {

typedef float floatx16 __attribute__((ext_vector_type(16)));

template <typename E>
__device__ __forceinline__ floatx16 mfma32(bf16x8 a, bf16x8 b, floatx16 c) {
  if constexpr (__is_same(E, _Float16))
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                   __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ floatx16 zero16() {
  floatx16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// max(a, b, c) as one instruction: fmaxf would first quiet each operand by one of its own.
// A NaN operand is ignored.  The compiler places no wait between a matrix product and inline
// assembly that reads it, so `a` comes from an ordinary instruction that has read b's and c's
// product before.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Eight values (registers 8 s .. 8 s + 7 of a D tile) as a 16-bit operand.
template <typename E>
__device__ __forceinline__ bf16x8 pack8(const floatx16& x, int s) {
  bf16x8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = to16<E>(x[8 * s + j]);
  return r;
}

template <int DP>
__device__ __forceinline__ int swizzle(int row) {
  if constexpr (DP == 128) return (row & 3) << 2 | (row >> 2 & 3);
  else return (row >> 1 & 1) << 2 | (row >> 2 & 3);
}

// A operand [m = row][k = d] from a tile: row r0 + ln, elements 16 s + 8 hf ..
template <int DP>
__device__ __forceinline__ bf16x8 row_frag(const __bf16* X, int r0, int s) {
  const int lane = threadIdx.x & 63, row = r0 + (lane & 31);
  return *(const bf16x8*)(X + row * DP + ((2 * s + (lane >> 5)) ^ swizzle<DP>(row)) * 8);
}

// A operand [m = d][k = row] from the same tile: column d0 + ln, rows r0 + 4 hf + {0..3}
// and r0 + 8 + 4 hf + {0..3}.
template <int DP>
__device__ __forceinline__ bf16x8 tr32(const __bf16* X, int r0, int d0) {
  const int lane = threadIdx.x & 63;
  const int row = r0 + 4 * (lane >> 5) + (lane >> 2 & 3);
  const int col = d0 + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
  const bf16x4 lo = ds_read_tr(X + row * DP + (col >> 3 ^ swizzle<DP>(row)) * 8 + (col & 7));
  const bf16x4 hi =
      ds_read_tr(X + (row + 8) * DP + (col >> 3 ^ swizzle<DP>(row + 8)) * 8 + (col & 7));
  return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// Asynchronous loads of a tile of ROWS rows by the workgroup's NW waves.  A load fills
// 1 KB of LDS, lane i the 16 bytes at 16 i: 512 / DP rows.  Pieces past D read the row's
// first: the other operand is zero there, or the result is not stored.
template <int DP, int ROWS, int NW>
struct TileLoad {
  static constexpr int RPI = 512 / DP, N = ROWS / RPI / NW;  // rows a load, loads a wave
  int wave;
  unsigned piece[N];  // bytes into its row that this lane reads
  __device__ __forceinline__ explicit TileLoad(int D)
      : wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % NW) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (threadIdx.x & 63) % (DP / 8) ^ swizzle<DP>(row(i));
      piece[i] = c * 8 < D ? c * 16 : 0;
    }
  }
  __device__ __forceinline__ int row(int i) const {
    return (wave * N + i) * RPI + (threadIdx.x & 63) / (DP / 8);
  }
  // src: the row of this lane's load i, as bytes from a base that all lanes share
  __device__ __forceinline__ void load(const char* base, unsigned src, int i, __bf16* X) const {
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)(base + (src + piece[i])),
        (__attribute__((address_space(3))) void*)(X + (wave * N + i) * 512), 16, 0, 0);
  }
  // rows first .. first + ROWS - 1 of a matrix with a token stride of `stride` elements; those
  // past `last` read it
  __device__ __forceinline__ void run(const __bf16* base, long stride, int first, int last,
                                      __bf16* X) const {
    const char* at = (const char*)(base + first * stride);
#pragma unroll
    for (int i = 0; i < N; ++i)
      load(at, (unsigned)min(row(i), last - first) * (unsigned)(2 * stride), i, X);
  }
};

// Waits for this wave's asynchronous loads, then for the other waves.
__device__ __forceinline__ void tile_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
}

// The B operand rows of one matrix, kept in registers: row `src` of this lane (ln),
// zero past D.
template <int DP>
__device__ __forceinline__ void load_frags(const __bf16* src, int D, bf16x8 (&f)[DP / 16]) {
  const int hf = threadIdx.x >> 5 & 1;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int d = 16 * s + 8 * hf;
    f[s] = d < D ? *(const bf16x8*)(src + d) : bf16x8{};
  }
}

// Stores a transposed result: X[d][row = ln], acc tile dt has d = 32 dt + 8 (i >> 2) +
// 4 hf + (i & 3); dst: this lane's row.  Rows that are not live are zero, whatever acc holds (a
// padded row's lane repeats the last live one, which need not be finite).
template <typename E, int DP>
__device__ __forceinline__ void store_t(__bf16* dst, const floatx16 (&acc)[DP / 32], float scale,
                                        bool live, int D) {
  const int hf = threadIdx.x >> 5 & 1;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 32 * dt + 8 * i + 4 * hf;
      bf16x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = to16<E>(live ? acc[dt][4 * i + j] * scale : 0.f);
      if (d < D) *(bf16x4*)(dst + d) = x;
    }
}

// Work items in an order in which neighbours share their keys; each of the eight XCDs
// (workgroups are handed to them in turn) takes one run of it, so that the neighbours
// share an L2.  The grid is 8 ceil(n / 8); -1: no work.
__device__ __forceinline__ long work_item(long n) {
  const long per = (n + 7) / 8, i = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  return (blockIdx.x >> 3) < per && i < n ? i : -1;
}
inline long work_grid(long n) { return (n + 7) / 8 * 8; }

__device__ __forceinline__ int row_length(const SlidingArgs& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
}

// The keys of `block` queries from t0 on, as one list without holes: the sinks that lie
// before the window, then the window [lo, hi); tiles of BN keys.
template <int BN>
struct KeyList {
  int ns, lo, n;
  __device__ __forceinline__ KeyList(int t0, int block, int len, int W, int S) {
    lo = max(0, t0 - W + 1);
    ns = min(S, lo);
    n = ns + min(len, t0 + block) - lo;
  }
  __device__ __forceinline__ int pos(int slot) const {
    return slot < ns ? slot : slot - ns + lo;
  }
  // The tiles that all of the block's queries see whole, from the first to before the end
  // (none where the end is not above the first).
  __device__ __forceinline__ int first_whole(int t0, int block, int W) const {
    return (ns + max(0, t0 + block - W - lo) + BN - 1) / BN;
  }
  __device__ __forceinline__ int end_whole(int t0) const { return (ns + t0 + 1 - lo) / BN; }
  __device__ __forceinline__ int tiles() const { return (n + BN - 1) / BN; }
  // Starts the loads of keys BN j .. BN j + BN - 1 of the list.  Tiles with sinks may have a
  // hole between them and the window.
  template <typename Tile>
  __device__ __forceinline__ void load(const Tile& tile, int j, const __bf16* x, long stride,
                                       __bf16* X) const {
    if (BN * j < ns) {
#pragma unroll
      for (int i = 0; i < tile.N; ++i)
        tile.load((const char*)(x + pos(min(BN * j + tile.row(i), n - 1)) * stride), 0, i, X);
    } else {
      tile.run(x, stride, BN * j - ns + lo, n - 1 - ns + lo, X);
    }
  }
};

// What a wave's 32 queries from tw on need of tile j of the list.
enum { kSkip, kFull, kMask };
template <int BN>
__device__ __forceinline__ int tile_kind(const KeyList<BN>& keys, int j, int tw, int W, int S) {
  const int s0 = BN * j, s1 = min(s0 + BN - 1, keys.n - 1);
  const int first = keys.pos(s0), last = keys.pos(s1), near = keys.pos(max(s0, keys.ns));
  if (first > tw + 31 || (first >= S && last + W <= tw)) return kSkip;
  return s1 < s0 + BN - 1 || last > tw || near + W <= tw + 31 ? kMask : kFull;
}

// Which keys of a masked tile this lane's query t sees, by the key's place 8 (i >> 2) + (i & 3)
// + 32 kt after BN j + 4 hf: from the window's first (low < place) or as a sink (place < sink),
// up to its own (place <= up).  Sinks are the list's first S slots, whether they lie before
// the window or in it, and the hole after them lies before every query.
struct TileMask {
  int up, low, sink;
  template <int BN>
  __device__ __forceinline__ TileMask(const KeyList<BN>& keys, int j, int t, int W, int S) {
    const int from = BN * j + 4 * (threadIdx.x >> 5 & 1), at = from + keys.lo - keys.ns;
    up = min(t - at, keys.n - 1 - from);
    low = t - W - at;
    sink = S - from;
  }
  __device__ __forceinline__ bool operator()(int place) const {
    return (place <= up) & ((place > low) | (place < sink));
  }
};

template <bool B>
struct Bool {
  static constexpr bool value = B;
};

}  // namespace hattn
