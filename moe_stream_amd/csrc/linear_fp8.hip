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
#include <algorithm>

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
// way into the registers, 4 lanes a block, which costs less than a launch before.
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
#pragma unroll 2
  for (int b = wave; b < blocks; b += kThinWaves) {
    const int k0 = b * kFp8Block + 16 * g, k1 = k0 + 64;
    const bool in0 = k0 < a.K, in1 = k1 < a.K;   // (K is whole pieces)
    i32x8 wf[NT], xf[TT];
    float sc[TT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
      wf[j] = pieces(in0 ? __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(w[j] + k0)) : none,
                     in1 ? __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(w[j] + k1)) : none);
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      if constexpr (kX16) {
        const uint16_t *x = reinterpret_cast<const uint16_t *>(a.x) + t[i] * a.x_stride;
        float v[4][8];
        load8<XT>(x + k0, in0 ? 8 : 0, v[0]);
        load8<XT>(x + k0 + 8, in0 ? 8 : 0, v[1]);
        load8<XT>(x + k1, in1 ? 8 : 0, v[2]);
        load8<XT>(x + k1 + 8, in1 ? 8 : 0, v[3]);
        uint32_t m = __float_as_uint(kFp8Least);
#pragma unroll
        for (int e = 0; e < 32; ++e) m = max(m, __float_as_uint(v[e / 8][e % 8]) & 0x7fffffffu);
        m = max(m, (uint32_t)__shfl_xor((int)m, 16));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32));
        u32x4_t lo, hi;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint2 c = to_fp8(v[e], m), d = to_fp8(v[2 + e], m);
          lo[2 * e] = c.x;
          lo[2 * e + 1] = c.y;
          hi[2 * e] = d.x;
          hi[2 * e + 1] = d.y;
        }
        xf[i] = pieces(lo, hi);
        sc[i] = fp8_scale(m);
      } else {
        const uint8_t *x = a.x + t[i] * a.x_stride;
        xf[i] = pieces(in0 ? *reinterpret_cast<const u32x4_t *>(x + k0) : none,
                       in1 ? *reinterpret_cast<const u32x4_t *>(x + k1) : none);
        sc[i] = a.xs[(int64_t)t[i] * blocks + b];
      }
    }
    // (16 NT outputs lie in one block of 128)
    const float ws = a.ws[(int64_t)(n0 / kFp8Block) * blocks + b];
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const float f = sc[i] * ws;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const f32x4 p = mfma_e4m3(wf[j], xf[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(p[e], f, acc[i][j][e]);
      }
    }
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
// Many rows: a workgroup's 4 waves take a tile of 2 * 16 R rows by as many outputs,
// each a quarter of it.  The tile's block of 128 columns of x and of w goes straight
// to LDS a block ahead, 16-byte pieces permuted within a row (two rows of 128 bytes
// span the banks) so that 16 rows' reads of a piece meet no conflict.  The scales of
// the lane's rows are a block ahead in registers.
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

template <class T, int R>
__global__ __launch_bounds__(256, 2) void linear_tile_kernel(LinearArgs a, int t_tiles) {
  constexpr int kRows = 32 * R;                // of x, and of w
  constexpr int kBytes = kRows * kFp8Block;
  constexpr int kLoads = kRows / 8 / 4;        // a wave's loads of x, and of w: 8 rows each
  __shared__ __align__(1024) char lds[2][2][kBytes];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // neighbouring workgroups go to the 8 dies in turn: each die takes a run of tiles,
  // all row tiles of an output tile before the next, so its weights stay in its cache
  const int total = gridDim.x, each = total / 8, more = total % 8;
  const int die = blockIdx.x % 8;
  const int tile = die * each + min(die, more) + blockIdx.x / 8;
  const int t0 = (tile % t_tiles) * kRows, n0 = (tile / t_tiles) * kRows;
  const int blocks = (a.K + kFp8Block - 1) / kFp8Block;
  const int last = a.K / 16 - 1;               // the last piece of a row

  const int sub = lane / 8, piece = lane % 8;
  auto fetch = [&](int b, int buf) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = (i * 4 + wave) * 8 + sub;
      // (a piece past K is the row's last one again; x's are zeroed where they are used)
      const int64_t k = 16 * (int64_t)min(b * 8 + (piece ^ ((row >> 1) & 7)), last);
      const uint8_t *gx = a.x + min(t0 + row, a.T - 1) * a.x_stride + k;
      const uint8_t *gw = a.w + (int64_t)min(n0 + row, a.N - 1) * a.K + k;
      __builtin_amdgcn_global_load_lds((global_void *)gx,
                                       (lds_void *)(&lds[buf][0][(i * 4 + wave) * 1024]), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((global_void *)gw,
                                       (lds_void *)(&lds[buf][1][(i * 4 + wave) * 1024]), 16, 0, 0);
    }
  };
  const int row = lane & 15, g = lane >> 4;
  const int tw = (wave & 1) * 16 * R, nw = (wave >> 1) * 16 * R;   // the wave's quarter
  const float *xs[R];
#pragma unroll
  for (int i = 0; i < R; ++i) xs[i] = a.xs + (int64_t)min(t0 + tw + 16 * i + row, a.T - 1) * blocks;
  const float *ws = a.ws + (int64_t)(min(n0 + nw, a.N - 1) / kFp8Block) * blocks;
  float sc[R], sw = ws[0];
#pragma unroll
  for (int i = 0; i < R; ++i) sc[i] = xs[i][0];
  f32x4 acc[R][R];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  auto frag = [&](const char *tile_lds, int r) {
    const int f = (r >> 1) & 7;
    const char *p = tile_lds + r * kFp8Block;
    return pieces(*reinterpret_cast<const u32x4_t *>(p + ((g ^ f) * 16)),
                  *reinterpret_cast<const u32x4_t *>(p + (((g + 4) ^ f) * 16)));
  };
  fetch(0, 0);
  for (int b = 0; b < blocks; ++b) {
    __syncthreads();   // block b has landed, and block b - 1 is read
    float f[R];
#pragma unroll
    for (int i = 0; i < R; ++i) f[i] = sc[i] * sw;
    if (b + 1 < blocks) {
      fetch(b + 1, (b + 1) & 1);
#pragma unroll
      for (int i = 0; i < R; ++i) sc[i] = xs[i][b + 1];
      sw = ws[b + 1];
    }
    i32x8 xf[R];
#pragma unroll
    for (int i = 0; i < R; ++i) xf[i] = frag(lds[b & 1][0], tw + 16 * i + row);
    if (b + 1 == blocks && a.K % kFp8Block) {
      const int left = (a.K % kFp8Block) / 16;
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if ((e < 4 ? g : g + 4) >= left) xf[i][e] = 0;
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const i32x8 wf = frag(lds[b & 1][1], nw + 16 * j + row);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const f32x4 p = mfma_e4m3(wf, xf[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(p[e], f[i], acc[i][j][e]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int t = t0 + tw + 16 * i + row;
    if (t < a.T) {
#pragma unroll
      for (int j = 0; j < R; ++j) store_outputs<T>(a, t, n0 + nw + 16 * j + 4 * g, acc[i][j]);
    }
  }
}

constexpr int kThinRows = 64;   // up to this many rows of x the thin kernel runs
constexpr int kFusedRows = 16;  // and up to this many it takes x in 16 bits

bool linear_takes_16(int T) { return T <= kFusedRows; }

template <class T, class XT, int TT>
static void thin_go(const LinearArgs &a, hipStream_t s) {
  const int n_tiles = (a.N + 15) / 16;
  if (n_tiles >= 2048)
    hipLaunchKernelGGL((linear_thin_kernel<T, XT, TT, 4>), dim3((n_tiles + 3) / 4),
                       dim3(64 * kThinWaves), 0, s, a);
  else
    hipLaunchKernelGGL((linear_thin_kernel<T, XT, TT, 1>), dim3(n_tiles), dim3(64 * kThinWaves),
                       0, s, a);
}

template <class T>
static void linear_go(const LinearArgs &a, int x_dtype, hipStream_t s) {
  if (a.T <= kThinRows) {
    if (x_dtype == MOE_DTYPE_BF16) thin_go<T, Bf16, 1>(a, s);
    else if (x_dtype == MOE_DTYPE_F16) thin_go<T, F16, 1>(a, s);
    else if (a.T <= 16) thin_go<T, uint8_t, 1>(a, s);
    else if (a.T <= 32) thin_go<T, uint8_t, 2>(a, s);
    else thin_go<T, uint8_t, 4>(a, s);
    return;
  }
  auto tiles = [&](int rows, int *t_tiles) {
    *t_tiles = (a.T + rows - 1) / rows;
    return *t_tiles * ((a.N + rows - 1) / rows);
  };
  int tt;
  const int n = tiles(128, &tt);
  if (n >= 256) {
    hipLaunchKernelGGL((linear_tile_kernel<T, 4>), dim3(n), dim3(256), 0, s, a, tt);
  } else {
    const int m = tiles(64, &tt);
    hipLaunchKernelGGL((linear_tile_kernel<T, 2>), dim3(m), dim3(256), 0, s, a, tt);
  }
}

void launch_linear(const LinearArgs &a, int x_dtype, int out_dtype, hipStream_t s) {
  if (out_dtype == MOE_DTYPE_BF16) linear_go<Bf16>(a, x_dtype, s);
  else linear_go<F16>(a, x_dtype, s);
}

}  // namespace moe
