// Device helpers and launchers of the operators around the expert block: norm,
// 8-bit product, rotary positions and paged attention.
#pragma once

#include "common.h"
#include "paged.h"

namespace moe {

// 16 bytes at any 2-byte (or 1-byte) address: rows of odd length start anywhere,
// and global memory takes such an access in one instruction.
typedef u32x4_t __attribute__((aligned(2))) u32x4_any;
typedef uint64_t __attribute__((aligned(1))) u64_any;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// s_waitcnt's argument for "at most n vector memory loads are under way", the other
// counts as they are: what a barrier needs before it where loads go straight to LDS.
constexpr int loads_left(int n) { return 0x0f70 | (n & 15) | (n >> 4) << 14; }

// The 16-bit types: conversions round to nearest even, NaN stays NaN.
struct Bf16 {
  static constexpr int kType = MOE_DTYPE_BF16;
  static __device__ __forceinline__ float load(uint32_t b) { return bf16_to_f32(b); }
  static __device__ __forceinline__ uint32_t store(float f) {
    return __builtin_bit_cast(uint16_t, (__bf16)f);
  }
};
struct F16 {
  static constexpr int kType = MOE_DTYPE_F16;
  static __device__ __forceinline__ float load(uint32_t b) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)b);
  }
  static __device__ __forceinline__ uint32_t store(float f) {
    return __builtin_bit_cast(uint16_t, (_Float16)f);
  }
};

// Eight elements from p, of which the first n exist (n < 1: none); the others are zero.
__device__ __forceinline__ u32x4_t bits8(const uint16_t *p, int n) {
  u32x4_t w = {0, 0, 0, 0};
  if (n >= 8) {
    w = *reinterpret_cast<const u32x4_any *>(p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) w[i / 2] |= (uint32_t)p[i] << (16 * (i & 1));
  }
  return w;
}
// The first n of eight elements to p.
__device__ __forceinline__ void put8(uint16_t *p, int n, u32x4_t w) {
  if (n >= 8) {
    *reinterpret_cast<u32x4_any *>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
  }
}
template <class T>
__device__ __forceinline__ void widen8(u32x4_t w, float v[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = T::load(w[i] & 0xffffu);
    v[2 * i + 1] = T::load(w[i] >> 16);
  }
}
template <class T>
__device__ __forceinline__ u32x4_t narrow8(const float v[8]) {
  u32x4_t w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = T::store(v[2 * i]) | (T::store(v[2 * i + 1]) << 16);
  return w;
}
template <class T>
__device__ __forceinline__ void load8(const uint16_t *p, int n, float v[8]) {
  widen8<T>(bits8(p, n), v);
}
template <class T>
__device__ __forceinline__ void store8(uint16_t *p, int n, const float v[8]) {
  put8(p, n, narrow8<T>(v));
}

// --- e4m3 with a scale per 128 values ----------------------------------------
constexpr int kFp8Block = 128;
constexpr float kFp8Max = 448.f;
constexpr float kFp8Least = 1e-30f;   // a block's largest magnitude counts as at least this

// The largest |v| of a 128-value block spread over 16 consecutive lanes, 8 values
// each, as float bits: their unsigned order is the order of magnitudes, with
// infinity and then NaN above all of them, so neither is lost.
__device__ __forceinline__ uint32_t block_most(const float v[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  m = max(m, (uint32_t)dpp_i<kDppQuadXor1>((int)m));
  m = max(m, (uint32_t)dpp_i<kDppQuadXor2>((int)m));
  m = max(m, (uint32_t)dpp_i<kDppHalfMirror>((int)m));
  m = max(m, (uint32_t)dpp_i<kDppMirror>((int)m));
  return max(m, __float_as_uint(kFp8Least));
}

// Eight values to e4m3 (two words), v * 448 / most rounded to nearest even.  For
// values of 16 bits 448 v has at most 14 significant bits, and the quotient is
// corrected by its remainder, so one that lies halfway between two codes is seen
// to lie there.  A block whose `most` is not finite is NaN as a whole (and so is
// its scale or what the scale multiplies).
__device__ __forceinline__ uint2 to_fp8(const float v[8], uint32_t most) {
  if (most >= 0x7f800000u) return make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
  const float m = __uint_as_float(most);
  const float mant = __builtin_amdgcn_frexp_mantf(m);   // [0.5, 1)
  const int e = -__builtin_amdgcn_frexp_expf(m);
  const float r = __builtin_amdgcn_rcpf(mant);
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = __builtin_amdgcn_ldexpf(v[i], e) * kFp8Max;
    const float t = a * r;
    q[i] = fmaf(fmaf(-t, mant, a), r, t);
  }
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}
__device__ __forceinline__ float fp8_scale(uint32_t most) {
  return __uint_as_float(most) / kFp8Max;
}
// n (1..8) codes of to_fp8's eight to any address
__device__ __forceinline__ void store_fp8(uint8_t *p, int n, uint2 c) {
  if (n >= 8) {
    *reinterpret_cast<u64_any *>(p) = ((uint64_t)c.y << 32) | c.x;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
  }
}

// --- norm (rows.hip) -----------------------------------------------------------
constexpr int kNormMaxWidth = 16384;
struct NormArgs {
  const uint16_t *x, *res, *weight;
  int64_t x_stride, res_stride;
  uint16_t *y, *sum;
  uint8_t *q;
  float *scales;
  int T, D;
  float eps;
};
void launch_norm(const NormArgs &a, int dtype, hipStream_t s);
// x [T, K] of 16 bits -> codes [T, K] and scales [T, ceil(K / 128)]
void launch_to_fp8(const uint16_t *x, int64_t x_stride, int dtype, int T, int K, uint8_t *q,
                   float *scales, hipStream_t s);

// --- the paged cache's view ------------------------------------------------------
struct KvArgs {
  uint16_t *k, *v;              // [n_pages, heads, page, dim]
  const int32_t *table;         // [n_seqs, width]
  const int32_t *starts;        // [n_seqs + 1]
  const int32_t *lens;          // [n_seqs]
  int32_t n_pages, heads, page_shift, dim, n_seqs, width;
  int32_t total;                // rows of the batch
};
__device__ __forceinline__ SeqSpan kv_span(const KvArgs &kv, int s) {
  return seq_span(kv.starts[s], kv.starts[s + 1], kv.lens[s], kv.total,
                  kv.width << kv.page_shift);
}

// The sequence of row t on one wave: each step probes 64 of the row starts that
// are left, so 4,096 sequences take two.  -1: t is behind the last sequence (or
// the starts are not ascending).
__device__ __forceinline__ int find_seq(const KvArgs &kv, int t, int lane) {
  int lo = 0, hi = kv.n_seqs;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int i = lo + lane * step;
    const bool le = i < hi && kv.starts[i] <= t;
    const int n = __popcll(__ballot(le));
    if (n == 0) return -1;
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
  }
  const SeqSpan s = kv_span(kv, lo);
  return t >= s.first && t < s.first + s.rows ? lo : -1;
}

struct RopeArgs {
  KvArgs kv;
  const uint16_t *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;   // token and head strides, elements
  const double *freqs;
  const uint16_t *qw, *kw;
  uint16_t *out;                                // [total, heads, dim]
  int32_t heads, rot;
  float mscale, eps;
};
void launch_rope(const RopeArgs &a, int dtype, bool interleaved, hipStream_t s);

// --- paged attention (attn.hip) ---------------------------------------------------
struct AttnArgs {
  KvArgs kv;
  const uint16_t *q;
  int64_t q_st, q_sh;
  const float *sinks;
  uint16_t *out;
  int32_t heads, window;
  float scale;
};
bool attn_supported(int dim, int heads, int kv_heads);
bool attn_fits(const KvArgs &kv, int heads, int window);
size_t attn_workspace(const KvArgs &kv, int heads, int window);
void launch_attn(const AttnArgs &a, int dtype, void *ws, hipStream_t s);

// --- 8-bit product (linear_fp8.hip) -----------------------------------------------
struct LinearArgs {
  const uint8_t *x, *w;      // (x may hold 16-bit elements, see linear_takes_16)
  int64_t x_stride;          // elements
  const float *xs, *ws;
  const uint16_t *bias;
  uint16_t *y;
  int32_t T, K, N;
};
bool linear_takes_16(int T);   // whether x of T rows may come in 16 bits
void launch_linear(const LinearArgs &a, int x_dtype, int out_dtype, hipStream_t s);

}  // namespace moe
