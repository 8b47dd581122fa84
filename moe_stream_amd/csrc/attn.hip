// Attention of new tokens over the paged cache.
#include "layer.h"

namespace moe {

// One wave per (row, head): 64 keys a step, a key a lane for the scores and
// dim / 64 columns a lane for the output, with the running maximum and sum of the
// softmax.
template <class T, int D>
__global__ __launch_bounds__(256) void attn_rows_kernel(AttnArgs a) {
  const KvArgs &kv = a.kv;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (int64_t)kv.total * a.heads) return;
  const int t = (int)(item / a.heads), h = (int)(item % a.heads);
  const int s = find_seq(kv, t, lane);
  if (s < 0) return;
  const SeqSpan sp = kv_span(kv, s);
  if (!sp.ok && lane == 0) flag_error_bits(kErrBadBatch);
  const int hk = h / (a.heads / kv.heads);
  int lo, hi;
  seen_keys(sp.base + (t - sp.first), sp.len, a.window, &lo, &hi);
  const uint16_t *q = a.q + t * a.q_st + h * a.q_sh;
  const float sink = a.sinks ? a.sinks[h] : -INFINITY;
  float m = fmaxf(sink, -3e38f), l = sink > -INFINITY ? 1.f : 0.f, o[D / 64] = {};
  for (int j0 = lo; j0 < hi; j0 += 64) {
    const int j = j0 + lane;
    int64_t at = -1;
    if (j < hi) {
      const int entry = kv.table[(int64_t)s * kv.width + (j >> kv.page_shift)];
      at = page_row(entry, kv.n_pages, kv.heads, hk, kv.page_shift, j, D);
      if (at < 0) flag_error_bits(kErrBadBatch);
    }
    float z = -INFINITY;
    if (at >= 0) {
      float d = 0.f;
      for (int e = 0; e < D; ++e) d = fmaf(T::load(q[e]), T::load(kv.k[at + e]), d);
      z = d * a.scale;
    }
    const float m1 = fmaxf(m, wave_max(z));
    const float f = expf(m - m1), p = at >= 0 ? expf(z - m1) : 0.f;
    l = l * f + group_sum<64>(p);
    for (int i = 0; i < D / 64; ++i) o[i] *= f;
    for (int j = 0; j < 64; ++j) {
      const int64_t vat = __shfl(at, j);
      const float pj = __shfl(p, j);
      if (vat < 0) continue;
      for (int i = 0; i < D / 64; ++i)
        o[i] = fmaf(pj, T::load(kv.v[vat + i * 64 + lane]), o[i]);
    }
    m = m1;
  }
  for (int i = 0; i < D / 64; ++i)
    a.out[((int64_t)t * a.heads + h) * D + i * 64 + lane] =
        (uint16_t)T::store(l == 0.f ? 0.f : o[i] / l);
}

bool attn_supported(int dim, int heads, int kv_heads) {
  return (dim == 64 || dim == 128) && heads % kv_heads == 0 && heads / kv_heads <= 64;
}
size_t attn_workspace(const KvArgs &, int) { return 256; }

template <class T>
static void attn_go(const AttnArgs &a, hipStream_t s) {
  const dim3 g((unsigned)(((int64_t)a.kv.total * a.heads + 3) / 4)), b(256);
  if (a.kv.dim == 64)
    hipLaunchKernelGGL((attn_rows_kernel<T, 64>), g, b, 0, s, a);
  else
    hipLaunchKernelGGL((attn_rows_kernel<T, 128>), g, b, 0, s, a);
}

void launch_attn(const AttnArgs &a, int dtype, void *, hipStream_t s) {
  if (dtype == MOE_DTYPE_BF16) attn_go<Bf16>(a, s);
  else attn_go<F16>(a, s);
}

}  // namespace moe
