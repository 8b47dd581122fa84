// Operators that pass over rows once: the root-mean-square norm behind the
// residual's addition, and the rotary positions of new tokens on their way into
// the paged cache.  Both are bound by the bytes they move (a few operations an
// element), and by latency for a handful of rows.
#include <algorithm>

#include "layer.h"

namespace moe {

// ---------------------------------------------------------------------------
// h = round(x + r);  y = h * rsqrt(mean(h^2) + eps) * w.  WPR waves hold one row
// in registers, 8 elements a lane and step, so the row is read once; the sum of
// squares is 32-bit throughout.  h is rounded to the row's type before the norm,
// because that is the residual stream the next layer reads.  y is rounded once:
// to the row's type, or to e4m3 straight from 32 bits.  Bound by bytes: 8192 rows of
// 2880 with residual to 8 bits move 166 MB in 32 us, 5.2 TB/s, a large copy's rate; one
// row takes 1.9 us, little over an empty kernel.
// ---------------------------------------------------------------------------
template <class T, int WPR, int NIT, bool FP8>
__global__ __launch_bounds__(256) void norm_kernel(NormArgs a) {
  constexpr int NT = 64 * WPR;
  __shared__ float part[4];
  const int wave = threadIdx.x >> 6;
  const int t = blockIdx.x * (4 / WPR) + wave / WPR;
  const int c0 = threadIdx.x % NT;
  const bool live = t < a.T;
  const int64_t row = live ? t : 0;
  float h[NIT][8];
  float ss = 0.f;
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    const int e = (c0 + it * NT) * 8, n = a.D - e;
    load8<T>(a.x + row * a.x_stride + e, n, h[it]);
  }
  if (a.res != nullptr) {
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int e = (c0 + it * NT) * 8, n = a.D - e;
      float r[8];
      load8<T>(a.res + row * a.res_stride + e, n, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[it][i] = T::load(T::store(h[it][i] + r[i]));
      if (a.sum != nullptr && live && n > 0) store8<T>(a.sum + row * a.D + e, n, h[it]);
    }
  }
#pragma unroll
  for (int it = 0; it < NIT; ++it)
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(h[it][i], h[it][i], ss);
  ss = group_sum<64>(ss);
  if (WPR > 1) {
    if ((threadIdx.x & 63) == 0) part[wave] = ss;
    __syncthreads();
    ss = WPR == 4 ? (part[0] + part[1]) + (part[2] + part[3])
                  : part[wave & ~1] + part[wave | 1];
  }
  if (!live) return;
  const float inv = 1.f / sqrtf(ss / (float)a.D + a.eps);
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    const int c = c0 + it * NT, e = c * 8, n = a.D - e;
    float w[8];
    load8<T>(a.weight + e, n, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = h[it][i] * inv * w[i];
    if (FP8) {
      const uint32_t most = block_most(w);   // (every lane of the 16 takes part)
      if (n > 0) {
        store_fp8(a.q + row * a.D + e, n, to_fp8(w, most));
        if (c % 16 == 0)
          a.scales[row * ((a.D + kFp8Block - 1) / kFp8Block) + c / 16] = fp8_scale(most);
      }
    } else if (n > 0) {
      store8<T>(a.y + row * a.D + e, n, w);
    }
  }
}

template <class T, int WPR, int NIT>
static void norm_go(const NormArgs &a, hipStream_t s) {
  const dim3 g((a.T + 4 / WPR - 1) / (4 / WPR)), b(256);
  if (a.q != nullptr)
    hipLaunchKernelGGL((norm_kernel<T, WPR, NIT, true>), g, b, 0, s, a);
  else
    hipLaunchKernelGGL((norm_kernel<T, WPR, NIT, false>), g, b, 0, s, a);
}

template <class T>
static void norm_type(const NormArgs &a, hipStream_t s) {
  // Many rows of up to 4096 columns: one or two waves a row, so that a workgroup has more
  // rows under way.  8192 rows of 2880: 35.5 us with two waves a row (5.3 TB/s), 37.8 with
  // one, 37.0 with four; of 1024: 11.8 with one, 14.0 with four.  At 2048 rows the two are
  // even (10.0 us at 2880 columns); at 1024, 7.9 against four waves' 7.2, and one row takes
  // a third of the steps with four.
  if (a.T >= 2048 && a.D <= 4096) {
    const int nit = (a.D + 511) / 512;
    if (nit <= 1) norm_go<T, 1, 1>(a, s);
    else if (nit <= 2) norm_go<T, 1, 2>(a, s);
    else if (nit <= 4) norm_go<T, 2, 2>(a, s);
    else if (nit <= 6) norm_go<T, 2, 3>(a, s);
    else norm_go<T, 2, 4>(a, s);
    return;
  }
  const int nit = (a.D + 2047) / 2048;
  if (nit <= 1) norm_go<T, 4, 1>(a, s);
  else if (nit <= 2) norm_go<T, 4, 2>(a, s);
  else if (nit <= 4) norm_go<T, 4, 4>(a, s);
  else norm_go<T, 4, 8>(a, s);
}

void launch_norm(const NormArgs &a, int dtype, hipStream_t s) {
  if (dtype == MOE_DTYPE_BF16) norm_type<Bf16>(a, s);
  else norm_type<F16>(a, s);
}

// ---------------------------------------------------------------------------
// Rows of 16 bits to e4m3 with a scale per 128 columns: 16 lanes a block.
// ---------------------------------------------------------------------------
template <class T>
__global__ __launch_bounds__(256) void to_fp8_kernel(const uint16_t *x, int64_t x_stride, int K,
                                                     int blocks, int64_t items, uint8_t *q,
                                                     float *scales) {
  const int64_t item = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;   // (row, block)
  const int64_t at = min(item, items - 1);
  const int64_t t = at / blocks;
  const int b = (int)(at % blocks);
  const int e = b * kFp8Block + (threadIdx.x % 16) * 8, n = K - e;
  float v[8];
  load8<T>(x + t * x_stride + e, n, v);
  const uint32_t most = block_most(v);
  if (item >= items) return;
  if (n > 0) store_fp8(q + t * K + e, n, to_fp8(v, most));
  if (threadIdx.x % 16 == 0) scales[at] = fp8_scale(most);
}

void launch_to_fp8(const uint16_t *x, int64_t x_stride, int dtype, int T, int K, uint8_t *q,
                   float *scales, hipStream_t s) {
  const int blocks = (K + kFp8Block - 1) / kFp8Block;
  const int64_t items = (int64_t)T * blocks;
  const dim3 g((unsigned)((items + 15) / 16)), b(256);
  if (dtype == MOE_DTYPE_BF16)
    hipLaunchKernelGGL((to_fp8_kernel<Bf16>), g, b, 0, s, x, x_stride, K, blocks, items, q, scales);
  else
    hipLaunchKernelGGL((to_fp8_kernel<F16>), g, b, 0, s, x, x_stride, K, blocks, items, q, scales);
}

// ---------------------------------------------------------------------------
// Rotary positions.  A row at position p turns its pair i by p * freq[i]:
//   (a, b) -> m (a cos - b sin, b cos + a sin)
// with pairs (i, i + rot/2) or, interleaved, (2i, 2i + 1) of the first `rot`
// dims of a head; the others pass.  The angle is taken in 64 bits and reduced to
// a fraction of a turn there: at position 2^20 a 32-bit product would be off by
// 2^-4 radians.  The workgroup's tokens have their cosines and sines in LDS, once
// for all heads.  Keys and values go straight to their page; a token whose place
// is outside the table, the pages or the batch is left out and flagged.  Bound by
// bytes when there are many (4096 tokens of 80 heads of 64: 84 MB in 16.8 us, 5.0
// TB/s), by the chain of look-up, angle and rotation for few (61 tokens: 6.3 us).
// ---------------------------------------------------------------------------
constexpr int kRopeMaxDim = 512;
struct Pieces {
  u32x4_t a, b;   // a lane's two runs of a head's row
};

template <class T, int TOK, bool INTER>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, int lph_log2) {
  __shared__ float2 turn[TOK][kRopeMaxDim / 2];
  __shared__ int pos_s[TOK], entry_s[TOK], here_s[TOK];
  const KvArgs &kv = a.kv;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t0 = blockIdx.x * TOK;
  const int half = a.rot / 2;
  const int lph = 1 << lph_log2;              // lanes a head
  const int u = threadIdx.x & (lph - 1);
  const int groups = 256 >> lph_log2;
  const int nh = a.heads + 2 * kv.heads;
  const int D = kv.dim;
  const int ru = (half + 7) / 8;              // units of 8 pairs; then units of 16 passing dims
  const bool rotates = u < ru;
  int oa, ob, na, nb;                         // this lane's two runs of up to 8 elements
  if (rotates) {
    oa = INTER ? 16 * u : 8 * u;
    ob = INTER ? oa + 8 : half + 8 * u;
    na = INTER ? a.rot - oa : half - oa;
    nb = INTER ? a.rot - ob : na;
  } else {
    oa = a.rot + 16 * (u - ru);
    ob = oa + 8;
    na = D - oa;
    nb = D - ob;
  }
  na = max(0, min(na, 8));
  nb = max(0, min(nb, 8));
  // Head h of token k: the query's heads, then the keys', then the values'.  Its row is
  // read two heads ahead, the first ones before the token's place is known.
  const int items = TOK * nh;
  auto fetch = [&](int item) __attribute__((always_inline)) {
    const int k = min(item, items - 1) / nh, h = min(item, items - 1) % nh;
    const int64_t t = min(t0 + k, kv.total - 1);
    const int hk = h - a.heads, hv = hk - kv.heads;
    const uint16_t *src = hk < 0   ? a.q + t * a.q_st + h * a.q_sh
                          : hv < 0 ? a.k + t * a.k_st + hk * a.k_sh
                                   : a.v + t * a.v_st + hv * a.v_sh;
    Pieces p;
    p.a = bits8(src + oa, na);
    p.b = bits8(src + ob, nb);
    return p;
  };
  const int first = threadIdx.x >> lph_log2;
  Pieces now = fetch(first), next = fetch(first + groups);
  if (wave < TOK) {
    const int t = t0 + wave;
    const int s = t < kv.total ? find_seq(kv, t, lane) : -1;
    if (lane == 0) {
      int pos = 0, entry = -1;
      if (s >= 0) {
        const SeqSpan sp = kv_span(kv, s);
        pos = sp.base + (t - sp.first);
        if (pos >= 0) entry = kv.table[(int64_t)s * kv.width + (pos >> kv.page_shift)];
        if (!sp.ok || entry < 0 || entry >= kv.n_pages) flag_error_bits(kErrBadBatch);
      }
      here_s[wave] = s >= 0;
      pos_s[wave] = pos;
      entry_s[wave] = entry;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < TOK * half; i += 256) {
    const int k = i / half, p = i % half;
    double turns = (double)pos_s[k] * (a.freqs[p] * 0.15915494309189533577);
    turns -= rint(turns);
    float sn, cs;
    sincospif(2.f * (float)turns, &sn, &cs);
    turn[k][p] = make_float2(cs * a.mscale, sn * a.mscale);
  }
  __syncthreads();
  for (int item = first; item < items; item += groups) {
    const Pieces in = now;
    now = next;
    if (item + 2 * groups < items) next = fetch(item + 2 * groups);
    const int k = item / nh, h = item % nh, t = t0 + k;
    if (!here_s[k]) continue;
    const int hk = h - a.heads, hv = hk - kv.heads;
    uint16_t *dst = hk < 0 ? a.out : hv < 0 ? kv.k : kv.v;
    int64_t at = ((int64_t)t * a.heads + h) * D;
    if (hk >= 0)
      at = page_row(entry_s[k], kv.n_pages, kv.heads, hv < 0 ? hk : hv, kv.page_shift, pos_s[k], D);
    if (at < 0) continue;
    if (hv >= 0) {                            // a value head: as it is
      put8(dst + at + oa, na, in.a);
      put8(dst + at + ob, nb, in.b);
      continue;
    }
    float va[8], vb[8];
    widen8<T>(in.a, va);
    widen8<T>(in.b, vb);
    const uint16_t *w = hk < 0 ? a.qw : a.kw;
    if (w != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(va[i], va[i], fmaf(vb[i], vb[i], ss));
      for (int m = 1; m < lph; m <<= 1) ss += __shfl_xor(ss, m);
      const float inv = 1.f / sqrtf(ss / (float)D + a.eps);
      float wa[8], wb[8];
      load8<T>(w + oa, na, wa);
      load8<T>(w + ob, nb, wb);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        va[i] = va[i] * inv * wa[i];
        vb[i] = vb[i] * inv * wb[i];
      }
    }
    if (rotates) {
      if (INTER) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 ta = turn[k][8 * u + i], tb = turn[k][8 * u + 4 + i];
          const float x0 = va[2 * i], x1 = va[2 * i + 1], y0 = vb[2 * i], y1 = vb[2 * i + 1];
          va[2 * i] = x0 * ta.x - x1 * ta.y;
          va[2 * i + 1] = x1 * ta.x + x0 * ta.y;
          vb[2 * i] = y0 * tb.x - y1 * tb.y;
          vb[2 * i + 1] = y1 * tb.x + y0 * tb.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 c = turn[k][8 * u + i];
          const float x = va[i], y = vb[i];
          va[i] = x * c.x - y * c.y;
          vb[i] = y * c.x + x * c.y;
        }
      }
    }
    put8(dst + at + oa, na, narrow8<T>(va));
    put8(dst + at + ob, nb, narrow8<T>(vb));
  }
}

template <class T, bool INTER>
static void rope_go(const RopeArgs &a, hipStream_t s) {
  const int units = (a.rot / 2 + 7) / 8 + (a.kv.dim - a.rot + 15) / 16;
  int lg = 0;
  while ((1 << lg) < units) ++lg;
  // Four tokens a workgroup share its look-up from 2048 tokens on (4096 tokens of 80 heads
  // of 64: 17.1 us against 20.2 with one; 2048: 12.3 against 13.3).  Fewer tokens need the
  // workgroups (1024 tokens: 10.4 us against 8.4; 61: 10.4 against 6.3).
  if (a.kv.total >= 2048)
    hipLaunchKernelGGL((rope_kernel<T, 4, INTER>), dim3((a.kv.total + 3) / 4), dim3(256), 0, s, a,
                       lg);
  else
    hipLaunchKernelGGL((rope_kernel<T, 1, INTER>), dim3(a.kv.total), dim3(256), 0, s, a, lg);
}

void launch_rope(const RopeArgs &a, int dtype, bool interleaved, hipStream_t s) {
  if (dtype == MOE_DTYPE_BF16) {
    if (interleaved) rope_go<Bf16, true>(a, s);
    else rope_go<Bf16, false>(a, s);
  } else {
    if (interleaved) rope_go<F16, true>(a, s);
    else rope_go<F16, false>(a, s);
  }
}

}  // namespace moe
