// y = x w^T with x and w in e4m3, a 32-bit scale per 128 columns of a row of x and
// per 128 x 128 block of w, on the matrix cores (16x16x128, the full 8-bit rate).
//
// One instruction is one block of 128 columns for 16 outputs and 16 rows of x, so
// each starts from zero and is folded into the sum with its two scales:
//   acc += p * (xs[t, b] * ws[n / 128, b])
// The product is taken as W X^T: a lane then holds one row of x (its column) and four
// neighbouring outputs, so the fold has one factor a lane, which serves every output
// of a 128-block, and the outputs leave in 8-byte stores.  Which 32 of a block's 128
// columns a lane holds does not matter as long as both operands agree: a lane takes
// the 16-byte pieces g and g + 4 of its row (g = lane / 16), so that a load of 64
// lanes covers 64 bytes in a row of each of 16 rows.
//
// The instruction adds products by eights of neighbouring columns, cut off 13 bits below
// the eight's largest, and the eights' sums in 32 bits (measured: beside 2^16 - 2^16 a
// product of 2^3 arrives and one of 2^2 does not, but 2^-7 does from another eight).  The
// operands' own rounding to e4m3 is 2^-4, so the cuts stay far below it: of four million
// random outputs of one block the worst was 2^-16 of its sum of magnitudes off.
#include <algorithm>
#include <type_traits>

#include "layer.h"

namespace moe {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma_e4m3(i32x8 a, i32x8 b) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ i32x8 pieces(u32x4_t lo, u32x4_t hi) {
  const i32x4 a = __builtin_bit_cast(i32x4, lo), b = __builtin_bit_cast(i32x4, hi);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Outputs n .. n + 3 of row t, those below N.
template <class T>
__device__ __forceinline__ void store_outputs(const LinearArgs &a, int t, int n, f32x4 v) {
  if (n >= a.N) return;
  uint16_t *const y = a.y + (int64_t)t * a.N + n;
  if (a.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) v[i] += T::load(a.bias[n + i]);
  }
  const uint32_t lo = T::store(v[0]) | (T::store(v[1]) << 16);
  const uint32_t hi = T::store(v[2]) | (T::store(v[3]) << 16);
  if (n + 3 < a.N) {
    typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
    *reinterpret_cast<u32x2_any *>(y) = (u32x2_any){lo, hi};
  } else {
    y[0] = (uint16_t)lo;
    if (n + 1 < a.N) y[1] = (uint16_t)(lo >> 16);
    if (n + 2 < a.N) y[2] = (uint16_t)hi;
  }
}

// ---------------------------------------------------------------------------
// Few rows (T <= 16 TT): bound by the weights' bytes, and by latency below some 20
// MB of them.  A workgroup's 8 waves share 16 NT outputs and take every 8th block of
// columns, so that together they read 1 KB of a weight row at a time; their sums are
// added in a fixed order through LDS.  XT: x in 16 bits (TT = 1) is quantised on the
// way into the registers, 4 lanes a block, which costs less than a launch before.  One row
// of 2048 x 5120 (10.5 MB) takes 7.4 us, of 2048 x 151936 70 us (4.4 TB/s).
// ---------------------------------------------------------------------------
constexpr int kThinWaves = 8;
template <class T, class XT, int TT, int NT>
__global__ __launch_bounds__(64 * kThinWaves) void linear_thin_kernel(LinearArgs a) {
  constexpr bool kX16 = !__is_same(XT, uint8_t);
  __shared__ f32x4 part[kThinWaves][TT * NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = lane & 15, g = lane >> 4;
  const int blocks = (a.K + kFp8Block - 1) / kFp8Block;
  const int n0 = blockIdx.x * 16 * NT;
  const uint8_t *w[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) w[j] = a.w + (int64_t)min(n0 + 16 * j + row, a.N - 1) * a.K;
  int t[TT];
#pragma unroll
  for (int i = 0; i < TT; ++i) t[i] = min(16 * i + row, a.T - 1);
  f32x4 acc[TT][NT];
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const u32x4_t none = {0, 0, 0, 0};
  // One block's operands as they come: 16 bytes a piece, of x in 16 bits two for one.
  struct Operands {
    u32x4_t w[NT][2], x[TT][kX16 ? 4 : 2];
    float xs[TT], ws;
  };
  auto load = [&](Operands &o, int b) __attribute__((always_inline)) {
    const int k[2] = {b * kFp8Block + 16 * g, b * kFp8Block + 16 * g + 64};
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const bool in = k[p] < a.K;   // (K is whole pieces)
#pragma unroll
      for (int j = 0; j < NT; ++j)
        o.w[j][p] =
            in ? __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(w[j] + k[p])) : none;
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        if constexpr (kX16) {
          const uint16_t *x = reinterpret_cast<const uint16_t *>(a.x) + t[i] * a.x_stride + k[p];
#pragma unroll
          for (int e = 0; e < 2; ++e)
            o.x[i][2 * p + e] = in ? *reinterpret_cast<const u32x4_any *>(x + 8 * e) : none;
        } else {
          const uint8_t *x = a.x + t[i] * a.x_stride + k[p];
          o.x[i][p] = in ? *reinterpret_cast<const u32x4_t *>(x) : none;
        }
      }
    }
    // (16 NT outputs lie in one block of 128)
    o.ws = a.ws[(int64_t)(n0 / kFp8Block) * blocks + b];
    if constexpr (!kX16) {
#pragma unroll
      for (int i = 0; i < TT; ++i) o.xs[i] = a.xs[(int64_t)t[i] * blocks + b];
    }
  };
  auto multiply = [&](const Operands &o) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      i32x8 xf;
      float xs = o.xs[i];
      if constexpr (kX16) {
        float v[4][8];
        uint32_t m = __float_as_uint(kFp8Least);
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const uint32_t pair = o.x[i][e / 8][e % 8 / 2];
          v[e / 8][e % 8] = XT::load(e & 1 ? pair >> 16 : pair & 0xffffu);
          m = max(m, __float_as_uint(v[e / 8][e % 8]) & 0x7fffffffu);
        }
        m = max(m, (uint32_t)__shfl_xor((int)m, 16));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32));
        u32x4_t c[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint2 q = to_fp8(v[e], m);
          c[e / 2][2 * (e & 1)] = q.x;
          c[e / 2][2 * (e & 1) + 1] = q.y;
        }
        xf = pieces(c[0], c[1]);
        xs = fp8_scale(m);
      } else {
        xf = pieces(o.x[i][0], o.x[i][1]);
      }
      const float f = xs * o.ws;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const f32x4 p = mfma_e4m3(pieces(o.w[j][0], o.w[j][1]), xf);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(p[e], f, acc[i][j][e]);
      }
    }
  };
  for (int b = wave; b < blocks; b += kThinWaves) {
    Operands o;
    load(o, b);
    multiply(o);
  }
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
  __syncthreads();
  for (int q = wave; q < TT * NT; q += kThinWaves) {
    f32x4 v = part[0][q][lane];
#pragma unroll
    for (int k = 1; k < kThinWaves; ++k) v += part[k][q][lane];
    const int tt = 16 * (q / NT) + row;
    if (tt < a.T) store_outputs<T>(a, tt, n0 + 16 * (q % NT) + 4 * g, v);
  }
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup's WT x WN waves take a tile of 16 RT WT rows by 16 RN WN
// outputs, each wave 16 RT x 16 RN of it.  The tile's block of 128 columns of x and of w
// goes straight to LDS a block ahead, 16-byte pieces permuted within a row (two rows of
// 128 bytes span the banks) so that 16 rows' reads of a piece meet no conflict.  The
// scales of the lane's rows are a block ahead in registers.  8192 x 4096 x 8192 takes 284
// us, 1.94 PFLOP/s (a large library product of unscaled blocks: 2.78); 4096 x 2048 x 5120 54
// us, 1.6, with the matrix unit busy 30 % of the cycles: the reads of the operands from
// LDS and the folds, four multiply-adds a product, go between.
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

template <class T, int RT, int RN, int WT, int WN>
__device__ __forceinline__ void linear_tile(const LinearArgs &a, int t0, int n0, char *lds_x0,
                                            char *lds_x1, char *lds_w0, char *lds_w1) {
  constexpr int W = WT * WN;
  constexpr int kT = 16 * RT * WT, kN = 16 * RN * WN;
  constexpr int kLoadsX = kT / 8 / W, kLoadsW = kN / 8 / W;   // a wave's, 8 rows each
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blocks = (a.K + kFp8Block - 1) / kFp8Block;
  const int last = a.K / 16 - 1;               // the last piece of a row

  // Rows past the end are the last one again, and not stored.
  const int sub = lane / 8, piece = lane % 8;
  uint32_t xo[kLoadsX], wo[kLoadsW];
  const uint8_t *const x0 = a.x + min(t0, a.T - 1) * a.x_stride;
  const uint8_t *const w0 = a.w + (int64_t)min(n0, a.N - 1) * a.K;
#pragma unroll
  for (int i = 0; i < kLoadsX; ++i)
    xo[i] = (uint32_t)(min((i * W + wave) * 8 + sub, a.T - 1 - t0) * a.x_stride);
#pragma unroll
  for (int i = 0; i < kLoadsW; ++i)
    wo[i] = (uint32_t)(min((i * W + wave) * 8 + sub, a.N - 1 - n0) * a.K);
  // The k-th load of block b: rows of x, then of w.  (A piece past K is the row's last
  // one again; x's are zeroed where they are used.)
  const int pc = piece ^ ((wave * 4 + sub / 2) & 7);
  auto fetch = [&](int b, int k, char *to_x, char *to_w) __attribute__((always_inline)) {
    const uint32_t at = 16 * min(b * 8 + pc, last);
    if (k < kLoadsX)
      __builtin_amdgcn_global_load_lds((global_void *)(x0 + (xo[k % kLoadsX] + at)),
                                       (lds_void *)(to_x + (k * W + wave) * 1024), 16, 0, 0);
    else
      __builtin_amdgcn_global_load_lds((global_void *)(w0 + (wo[(k - kLoadsX) % kLoadsW] + at)),
                                       (lds_void *)(to_w + ((k - kLoadsX) * W + wave) * 1024), 16,
                                       0, 0);
  };
  const int row = lane & 15, g = lane >> 4;
  const int tw = (wave % WT) * 16 * RT, nw = (wave / WT) * 16 * RN;   // the wave's share
  const float *xs[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
    xs[i] = a.xs + (int64_t)min(t0 + tw + 16 * i + row, a.T - 1) * blocks;
  // (16 RN outputs lie in one block of 128)
  const float *ws = a.ws + (int64_t)(min(n0 + nw, a.N - 1) / kFp8Block) * blocks;
  float sc[RT], sw = ws[0];
#pragma unroll
  for (int i = 0; i < RT; ++i) sc[i] = xs[i][0];
  f32x4 acc[RT][RN];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  // Where a lane reads in a tile, but for the block of 16 rows: one value each, so that
  // the compiler keeps sight of which array is read.
  const int f = (row >> 1) & 7;
  int x_at = (tw + row) * kFp8Block + (g ^ f) * 16, w_at = (nw + row) * kFp8Block + (g ^ f) * 16;
  asm("" : "+v"(x_at), "+v"(w_at));
  auto frag = [&](const char *tile, int at, int r) __attribute__((always_inline)) {
    return pieces(*reinterpret_cast<const u32x4_t *>(tile + at + r * 16 * kFp8Block),
                  *reinterpret_cast<const u32x4_t *>(tile + (at ^ 64) + r * 16 * kFp8Block));
  };
  auto block = [&](int b, const char *in_x, const char *in_w, char *to_x, char *to_w)
      __attribute__((always_inline)) {
    issue_order_fence();
    __builtin_amdgcn_s_waitcnt(loads_left(0));
    __syncthreads();   // block b has landed, and block b - 1 is read
    issue_order_fence();
    float f[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) f[i] = sc[i] * sw;
    const bool end = b + 1 == blocks;
    const int next = min(b + 1, blocks - 1);   // (the last block again, not used)
#pragma unroll
    for (int i = 0; i < RT; ++i) sc[i] = xs[i][next];
    sw = ws[next];
    constexpr int kAhead = 3;   // outputs' operands under way
    i32x8 xf[RT], wf[kAhead];
    wf[0] = frag(in_w, w_at, 0);
#pragma unroll
    for (int i = 0; i < RT; ++i) xf[i] = frag(in_x, x_at, i);
#pragma unroll
    for (int j = 1; j < kAhead - 1 && j < RN; ++j) wf[j] = frag(in_w, w_at, j);
    if (end && a.K % kFp8Block) {
      const int left = (a.K % kFp8Block) / 16;
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if ((e < 4 ? g : g + 4) >= left) xf[i][e] = 0;
    }
    // A product is folded while the two after it run; the next block's loads and the
    // next outputs' operand go between.
    constexpr int kLag = 2, kMul = RT * RN, kLoads = kLoadsX + kLoadsW;
    constexpr int kEach = (2 * kLoads + kMul - 1) / kMul;   // (gone by the half)
    f32x4 p[kLag + 1];
#pragma unroll
    for (int u = 0; u < kMul + kLag; ++u) {
      const int j = u / RT, i = u % RT;
      if (u < kMul) {
        if (i == 0 && j + kAhead - 1 < RN)
          wf[(j + kAhead - 1) % kAhead] = frag(in_w, w_at, j + kAhead - 1);
        p[u % (kLag + 1)] = mfma_e4m3(wf[j % kAhead], xf[i]);
#pragma unroll
        for (int k = kEach * u; k < kEach * (u + 1) && k < kLoads; ++k) fetch(next, k, to_x, to_w);
      }
      if (u >= kLag) {
        const int v = u - kLag, vj = v / RT, vi = v % RT;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[vi][vj][e] = fmaf(p[v % (kLag + 1)][e], f[vi], acc[vi][vj][e]);
          asm volatile("" : "+v"(acc[vi][vj][e]));   // (here, between the products)
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int k = 0; k < kLoadsX + kLoadsW; ++k) fetch(0, k, lds_x0, lds_w0);
  for (int b = 0; b < blocks; b += 2) {
    block(b, lds_x0, lds_w0, lds_x1, lds_w1);
    if (b + 1 < blocks) block(b + 1, lds_x1, lds_w1, lds_x0, lds_w0);
  }
  // Each wave turns its share round through LDS, a block of 16 rows at a time, so that a
  // row's outputs leave in whole pieces of 16 bytes.
  issue_order_fence();
  __builtin_amdgcn_s_waitcnt(loads_left(0));
  __syncthreads();
  constexpr int kCols = 16 * RN, kPad = kCols + 8;   // (16 bytes more a row: other banks)
  static_assert(W / 2 * 16 * kPad * 2 <= kT * kFp8Block, "the waves' boxes fit two tiles of x");
  uint16_t *const box =
      reinterpret_cast<uint16_t *>(wave < W / 2 ? lds_x0 : lds_x1) + wave % (W / 2) * 16 * kPad;
  float bias[RN][4];
#pragma unroll
  for (int j = 0; j < RN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + nw + 16 * j + 4 * g + e;
      bias[j][e] = a.bias != nullptr ? T::load(a.bias[min(n, a.N - 1)]) : 0.f;
    }
#pragma unroll
  for (int i = 0; i < RT; ++i) {
#pragma unroll
    for (int j = 0; j < RN; ++j) {
      const f32x4 v = acc[i][j];
      const uint32_t lo = T::store(v[0] + bias[j][0]) | (T::store(v[1] + bias[j][1]) << 16);
      const uint32_t hi = T::store(v[2] + bias[j][2]) | (T::store(v[3] + bias[j][3]) << 16);
      *reinterpret_cast<uint2 *>(box + row * kPad + 16 * j + 4 * g) = make_uint2(lo, hi);
    }
    issue_order_fence();   // (a wave's own LDS operations stay in order)
    constexpr int kEach = kCols / 8;   // pieces a row
#pragma unroll
    for (int q = 0; q < 16 * kEach / 64; ++q) {
      const int r = (q * 64 + lane) / kEach, c = (q * 64 + lane) % kEach * 8;
      const u32x4_t v = *reinterpret_cast<const u32x4_t *>(box + r * kPad + c);
      const int t = t0 + tw + 16 * i + r, n = n0 + nw + c;
      uint16_t *const y = a.y + (int64_t)t * a.N + n;
      if (t < a.T && n + 8 <= a.N) {
        *reinterpret_cast<u32x4_any *>(y) = v;
      } else if (t < a.T) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < a.N) y[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
      }
    }
    issue_order_fence();
  }
}

// One workgroup a tile.  kQuarters: tiles from `whole` on are cut into four, a workgroup
// each, which the same waves take.
template <class T, int RT, int RN, int WT, int WN, bool kQuarters>
__global__ __launch_bounds__(64 * WT * WN, 2) void linear_tile_kernel(LinearArgs a, int t_tiles,
                                                                      int tiles, int whole) {
  constexpr int kT = 16 * RT * WT, kN = 16 * RN * WN;
  // (an array of its own for each tile: loads to one are under way while another is
  // read, which the compiler waits for unless it tells them apart)
  __shared__ __align__(1024) char lds_x0[kT * kFp8Block], lds_x1[kT * kFp8Block];
  __shared__ __align__(1024) char lds_w0[kN * kFp8Block], lds_w1[kN * kFp8Block];
  // Neighbouring workgroups go to the 8 dies in turn: each die takes a run of tiles, and
  // within bands of 8 row tiles all of an output tile before the next, so that the tiles
  // a die has at once read few rows of x and of w.
  const bool quarter = kQuarters && (int)blockIdx.x >= whole;
  const int i = quarter ? blockIdx.x - whole : blockIdx.x;
  const int total = quarter ? gridDim.x - whole : whole, each = total / 8, more = total % 8;
  const int die = i % 8;
  const int at = die * each + min(die, more) + i / 8;
  const int tile = quarter ? whole + at / 4 : at;
  const int n_tiles = tiles / t_tiles, band = tile / (8 * n_tiles), in = tile % (8 * n_tiles);
  const int wide = min(8, t_tiles - band * 8);
  int t0 = (band * 8 + in % wide) * kT, n0 = (in / wide) * kN;
  if constexpr (kQuarters) {
    if (quarter) {
      t0 += at % 4 / 2 * (kT / 2);
      n0 += at % 2 * (kN / 2);
      if (t0 < a.T && n0 < a.N)
        linear_tile<T, RT / 2, RN / 2, WT, WN>(a, t0, n0, lds_x0, lds_x1, lds_w0, lds_w1);
      return;
    }
  }
  linear_tile<T, RT, RN, WT, WN>(a, t0, n0, lds_x0, lds_x1, lds_w0, lds_w1);
}

// A tile takes the blocks of 128 columns one after another, some 0.5 us each, whatever its
// rows; the thin kernel's waves share them, and its time goes with outputs and sets of 16
// rows.  Behind 16 rows it runs while sets times outputs stay below this (thin against tile
// at 2048 x 5120 weights: 20 rows 8.7 us and 10.6, 32: 10.0 and 10.6, 40: 11.7 and 10.9, 64:
// 15.9 and 11.6; 4096 x 2880, 37 rows: 9.9 and 17; 4096 x 16384, 20 rows: 28 and 19).
constexpr int kThinRows = 64;
constexpr int kThinWork = 12288;
// Up to this many rows it takes x in 16 bits, one set of them: as fast as codes made by a
// launch before (16 rows, 2048 columns: 5120 outputs 12.2 us against 11.2 for the two,
// 16384 15.1 and 15.5, 65536 37.9 and 40.5; one row the same), and a launch less to issue.
constexpr int kFusedRows = 16;

bool linear_takes_16(int T) { return T <= kFusedRows; }

static bool is_thin(int T, int N) {
  return T <= 16 || (T <= kThinRows && (int64_t)((T + 15) / 16) * N <= kThinWork);
}

// Four sets of 16 outputs a workgroup read x and its scales once for them (one row, 2048
// columns: 16384 outputs 11.7 us against 13.4 with one set, 32768 19.4 against 22.7); below
// a thousand sets the workgroups are too few for that (5120 outputs 8.7 against 7.5).
template <class T, class XT, int TT>
static void thin_go(const LinearArgs &a, hipStream_t s) {
  const int sets = (a.N + 15) / 16;
  const dim3 b(64 * kThinWaves);
  if constexpr (TT == 1) {
    if (sets >= 1024) {
      hipLaunchKernelGGL((linear_thin_kernel<T, XT, 1, 4>), dim3((sets + 3) / 4), b, 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((linear_thin_kernel<T, XT, TT, 1>), dim3(sets), b, 0, s, a);
}

template <class T>
static void linear_go(const LinearArgs &a, int x_dtype, hipStream_t s) {
  if (is_thin(a.T, a.N)) {
    if (x_dtype == MOE_DTYPE_BF16) thin_go<T, Bf16, 1>(a, s);
    else if (x_dtype == MOE_DTYPE_F16) thin_go<T, F16, 1>(a, s);
    else if (a.T <= 16) thin_go<T, uint8_t, 1>(a, s);
    else if (a.T <= 32) thin_go<T, uint8_t, 2>(a, s);
    else if (a.T <= 48) thin_go<T, uint8_t, 3>(a, s);
    else thin_go<T, uint8_t, 4>(a, s);
    return;
  }
  // The larger tile reads less per product; the smaller one spreads over more CUs.  A CU
  // has two of either of the smaller ones at once, so each runs while its tiles fit that
  // (4096 x 4096 weights, 512 rows: 25.7 us with 64, 30.8 with 128; 768: 37.9 and 30.8; 2048:
  // 51.2 with 128, 62.7 with 256; 2304: 76.9 and 60.4; 8192 rows of 8192 outputs: 430 and 284).
  // Nor is a tile higher than the rows need.
  auto tiles = [&](int rows) {
    return (int64_t)((a.T + rows - 1) / rows) * ((a.N + rows - 1) / rows);
  };
  constexpr int kCus = 256;
  if (a.T <= 64 || tiles(64) <= 2 * kCus) {
    const int n = (int)tiles(64);
    hipLaunchKernelGGL((linear_tile_kernel<T, 2, 2, 2, 2, false>), dim3(n), dim3(256), 0, s, a,
                       (a.T + 63) / 64, n, n);
  } else if (a.T <= 128 || tiles(128) <= 2 * kCus) {
    const int n = (int)tiles(128);
    hipLaunchKernelGGL((linear_tile_kernel<T, 4, 4, 2, 2, false>), dim3(n), dim3(256), 0, s, a,
                       (a.T + 127) / 128, n, n);
  } else {
    // A last round in which a quarter of the CUs or fewer would have a tile is spread over
    // all of them (4096 x 2048 x 5120, 320 tiles: 54.6 us against 66.4; 4352 x 4096 x 4096,
    // 272: 94.7 against 125.1).
    const int n = (int)tiles(256), rest = n % kCus;
    const int whole = n > kCus && rest * 4 <= kCus ? n - rest : n;
    hipLaunchKernelGGL((linear_tile_kernel<T, 4, 8, 4, 2, true>), dim3(whole + (n - whole) * 4),
                       dim3(512), 0, s, a, (a.T + 255) / 256, n, whole);
  }
}

void launch_linear(const LinearArgs &a, int x_dtype, int out_dtype, hipStream_t s) {
  if (out_dtype == MOE_DTYPE_BF16) linear_go<Bf16>(a, x_dtype, s);
  else linear_go<F16>(a, x_dtype, s);
}

}  // namespace moe
