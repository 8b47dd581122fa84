// C ABI of the operators around the expert block: argument checks and launches.

namespace {

bool is16(int32_t dtype) { return dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F16; }

// The host's part of a paged batch's checks; what the device arrays hold is
// bounded by the kernels.
int make_kv_args(const moe_kv_view *v, int32_t T, moe::KvArgs *kv) {
  if (!v) return fail(MOE_ERR_INVALID, "kv view is NULL");
  if (!v->k || !v->v || !v->table || !v->starts || !v->lens)
    return fail(MOE_ERR_INVALID, "NULL k/v/table/starts/lens");
  if (!is16(v->dtype)) return fail(MOE_ERR_INVALID, "unknown cache dtype %d", v->dtype);
  if (v->n_pages <= 0 || v->kv_heads <= 0 || v->n_seqs <= 0 || v->table_width <= 0)
    return fail(MOE_ERR_INVALID, "n_pages=%d kv_heads=%d n_seqs=%d table_width=%d must be positive",
                v->n_pages, v->kv_heads, v->n_seqs, v->table_width);
  int shift = 4;
  while (shift < 8 && (1 << shift) != v->page_size) ++shift;
  if ((1 << shift) != v->page_size)
    return fail(MOE_ERR_INVALID, "page_size=%d must be a power of two in [16, 256]",
                v->page_size);
  if ((int64_t)v->table_width * v->page_size > (1 << 30))
    return fail(MOE_ERR_INVALID, "table_width=%d pages of %d pass 2^30 positions",
                v->table_width, v->page_size);
  if (v->head_dim <= 0 || v->head_dim % 2 || v->head_dim > moe::kRopeMaxDim)
    return fail(MOE_ERR_INVALID, "head_dim=%d must be even, in [2, %d]", v->head_dim,
                moe::kRopeMaxDim);
  if (T < 0 || T >= (1 << 24)) return fail(MOE_ERR_INVALID, "T=%d outside [0, 2^24)", T);
  kv->k = static_cast<uint16_t *>(v->k);
  kv->v = static_cast<uint16_t *>(v->v);
  kv->table = v->table;
  kv->starts = v->starts;
  kv->lens = v->lens;
  kv->n_pages = v->n_pages;
  kv->heads = v->kv_heads;
  kv->page_shift = shift;
  kv->dim = v->head_dim;
  kv->n_seqs = v->n_seqs;
  kv->width = v->table_width;
  kv->total = T;
  return MOE_OK;
}

}  // namespace

extern "C" {

int moe_add_rms_norm(const void *x, int64_t x_stride, const void *residual,
                     int64_t residual_stride, const void *weight, int32_t dtype, int32_t T,
                     int32_t width, float eps, void *y, uint8_t *q, float *scales, void *sum,
                     void *stream) {
  if (!is16(dtype)) return fail(MOE_ERR_INVALID, "unknown dtype %d", dtype);
  if (T < 0 || T >= (1 << 24)) return fail(MOE_ERR_INVALID, "T=%d outside [0, 2^24)", T);
  if (width <= 0 || width > moe::kNormMaxWidth)
    return fail(MOE_ERR_INVALID, "width=%d outside [1, %d]", width, moe::kNormMaxWidth);
  if (!(eps >= 0.f)) return fail(MOE_ERR_INVALID, "eps=%g must not be negative", eps);
  if (T == 0) return MOE_OK;
  if ((y != nullptr) == (q != nullptr) || (q != nullptr) != (scales != nullptr))
    return fail(MOE_ERR_INVALID, "give y, or q with scales");
  if (sum && !residual) return fail(MOE_ERR_INVALID, "sum given without residual");
  if (!x || !weight) return fail(MOE_ERR_INVALID, "NULL x/weight");
  if (x_stride < width || (residual && residual_stride < width))
    return fail(MOE_ERR_INVALID, "row strides %lld, %lld below width %d", (long long)x_stride,
                (long long)residual_stride, width);
  moe::NormArgs a;
  a.x = static_cast<const uint16_t *>(x);
  a.res = static_cast<const uint16_t *>(residual);
  a.weight = static_cast<const uint16_t *>(weight);
  a.x_stride = x_stride;
  a.res_stride = residual_stride;
  a.y = static_cast<uint16_t *>(y);
  a.sum = static_cast<uint16_t *>(sum);
  a.q = q;
  a.scales = scales;
  a.T = T;
  a.D = width;
  a.eps = eps;
  (void)hipGetLastError();
  moe::launch_norm(a, dtype, static_cast<hipStream_t>(stream));
  MOE_HIP(hipGetLastError());
  return MOE_OK;
}

// codes [T, K] and scales [T, ceil(K / 128)] of a 16-bit x
static size_t linear_codes_bytes(int32_t T, int32_t K) {
  return ((size_t)T * K + 255) & ~(size_t)255;
}
static size_t linear_scales_bytes(int32_t T, int32_t K) {
  return ((size_t)T * ((K + moe::kFp8Block - 1) / moe::kFp8Block) * 4 + 255) & ~(size_t)255;
}

size_t moe_linear_fp8_workspace(int32_t T, int32_t K, int32_t N, int32_t x_dtype) {
  if (T <= 0 || K <= 0 || N <= 0 || x_dtype == MOE_DTYPE_E4M3 || moe::linear_takes_16(T)) return 0;
  return linear_codes_bytes(T, K) + linear_scales_bytes(T, K);
}

int moe_linear_fp8(const void *x, int32_t x_dtype, int64_t x_stride, const float *x_scales,
                   const uint8_t *w, const float *w_scales, const void *bias, int32_t T,
                   int32_t K, int32_t N, int32_t out_dtype, void *y, void *workspace,
                   size_t workspace_bytes, void *stream) {
  const bool x8 = x_dtype == MOE_DTYPE_E4M3;
  if (!x8 && !is16(x_dtype)) return fail(MOE_ERR_INVALID, "unknown x dtype %d", x_dtype);
  if (!is16(out_dtype)) return fail(MOE_ERR_INVALID, "unknown output dtype %d", out_dtype);
  if (T < 0 || T >= (1 << 24)) return fail(MOE_ERR_INVALID, "T=%d outside [0, 2^24)", T);
  if (K <= 0 || K % 16 || K > (1 << 20))
    return fail(MOE_ERR_INVALID, "K=%d must be a multiple of 16 in [16, 2^20]", K);
  if (N <= 0 || N > (1 << 22)) return fail(MOE_ERR_INVALID, "N=%d outside [1, 2^22]", N);
  if (T == 0) return MOE_OK;
  if ((int64_t)T * ((K + moe::kFp8Block - 1) / moe::kFp8Block) >= (1 << 28))
    return fail(MOE_ERR_INVALID, "T=%d rows of K=%d pass one launch", T, K);
  // (tiles of 256, or their quarters, in one launch of 512 threads each; a tile's rows of
  // x lie within 32 bits)
  if ((int64_t)((T + 255) / 256) * ((N + 255) / 256) >= (1 << 22))
    return fail(MOE_ERR_INVALID, "T=%d rows of N=%d outputs pass one launch", T, N);
  if (x8 && T > 1 && x_stride > (1 << 23))
    return fail(MOE_ERR_INVALID, "e4m3 x stride %lld passes 2^23", (long long)x_stride);
  if (x8 != (x_scales != nullptr))
    return fail(MOE_ERR_INVALID, "x_scales go with an e4m3 x, and only with one");
  if (!x || !w || !w_scales || !y) return fail(MOE_ERR_INVALID, "NULL x/w/w_scales/y");
  if (x_stride < K) return fail(MOE_ERR_INVALID, "x stride %lld below K=%d", (long long)x_stride, K);
  if (!aligned(w, 16) || (x8 && (!aligned(x, 16) || x_stride % 16)))
    return fail(MOE_ERR_INVALID, "e4m3 rows of x and w must be 16-byte aligned");
  const size_t need = moe_linear_fp8_workspace(T, K, N, x_dtype);
  if (need && (!workspace || !aligned(workspace, 256)))
    return fail(MOE_ERR_INVALID, "workspace NULL or not 256-byte aligned");
  if (workspace_bytes < need)
    return fail(MOE_ERR_INVALID, "workspace %zu < %zu bytes", workspace_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  char *ws = static_cast<char *>(workspace);
  moe::LinearArgs a;
  a.x = static_cast<const uint8_t *>(x);
  a.x_stride = x_stride;
  a.xs = x_scales;
  (void)hipGetLastError();
  if (need) {
    uint8_t *codes = reinterpret_cast<uint8_t *>(ws);
    float *scales = reinterpret_cast<float *>(ws + linear_codes_bytes(T, K));
    moe::launch_to_fp8(static_cast<const uint16_t *>(x), x_stride, x_dtype, T, K, codes, scales,
                       s);
    MOE_HIP(hipGetLastError());
    a.x = codes;
    a.x_stride = K;
    a.xs = scales;
    x_dtype = MOE_DTYPE_E4M3;
  }
  a.w = w;
  a.ws = w_scales;
  a.bias = static_cast<const uint16_t *>(bias);
  a.y = static_cast<uint16_t *>(y);
  a.T = T;
  a.K = K;
  a.N = N;
  moe::launch_linear(a, x_dtype, out_dtype, s);
  MOE_HIP(hipGetLastError());
  return MOE_OK;
}

int moe_rope_cache(const moe_kv_view *kv, const void *q, int64_t q_token, int64_t q_head,
                   const void *k, int64_t k_token, int64_t k_head, const void *v,
                   int64_t v_token, int64_t v_head, int32_t T, int32_t heads,
                   const double *freqs, int32_t rot, int32_t interleaved, float mscale,
                   const void *q_weight, const void *k_weight, float eps, void *q_out,
                   void *stream) {
  moe::RopeArgs a;
  const int rc = make_kv_args(kv, T, &a.kv);
  if (rc) return rc;
  if (heads <= 0) return fail(MOE_ERR_INVALID, "heads=%d must be positive", heads);
  if (rot < 0 || rot % 2 || rot > kv->head_dim)
    return fail(MOE_ERR_INVALID, "rot=%d must be even, in [0, head_dim=%d]", rot, kv->head_dim);
  if (!(eps >= 0.f)) return fail(MOE_ERR_INVALID, "eps=%g must not be negative", eps);
  if (T == 0) return MOE_OK;
  if (!q || !k || !v || !q_out || (rot > 0 && !freqs))
    return fail(MOE_ERR_INVALID, "NULL q/k/v/q_out/freqs");
  a.q = static_cast<const uint16_t *>(q);
  a.k = static_cast<const uint16_t *>(k);
  a.v = static_cast<const uint16_t *>(v);
  a.q_st = q_token;
  a.q_sh = q_head;
  a.k_st = k_token;
  a.k_sh = k_head;
  a.v_st = v_token;
  a.v_sh = v_head;
  a.freqs = freqs;
  a.qw = static_cast<const uint16_t *>(q_weight);
  a.kw = static_cast<const uint16_t *>(k_weight);
  a.out = static_cast<uint16_t *>(q_out);
  a.heads = heads;
  a.rot = rot;
  a.mscale = mscale;
  a.eps = eps;
  (void)hipGetLastError();
  moe::launch_rope(a, kv->dtype, interleaved != 0, static_cast<hipStream_t>(stream));
  MOE_HIP(hipGetLastError());
  return MOE_OK;
}

size_t moe_attn_paged_workspace(const moe_kv_view *kv, int32_t T, int32_t heads,
                                int32_t window) {
  moe::KvArgs a;
  if (T <= 0 || heads <= 0 || window < 0 || make_kv_args(kv, T, &a) || heads % a.heads) return 0;
  return moe::attn_workspace(a, heads, window);
}

int moe_attn_paged(const moe_kv_view *kv, const void *q, int64_t q_token, int64_t q_head,
                   int32_t T, int32_t heads, float scale, int32_t window, const float *sinks,
                   void *out, void *workspace, size_t workspace_bytes, void *stream) {
  moe::AttnArgs a;
  const int rc = make_kv_args(kv, T, &a.kv);
  if (rc) return rc;
  if (heads <= 0 || heads % kv->kv_heads)
    return fail(MOE_ERR_INVALID, "heads=%d must be a positive multiple of kv_heads=%d", heads,
                kv->kv_heads);
  if (!moe::attn_supported(kv->head_dim, heads, kv->kv_heads))
    return fail(MOE_ERR_UNSUPPORTED,
                "no attention kernel compiled for head_dim=%d with %d heads per key head",
                kv->head_dim, heads / kv->kv_heads);
  if (window < 0) return fail(MOE_ERR_INVALID, "window=%d is negative", window);
  if (!(scale >= 0.f && scale <= 1e30f))
    return fail(MOE_ERR_INVALID, "scale=%g outside [0, 1e30]", scale);
  if (T == 0) return MOE_OK;
  if (!moe::attn_fits(a.kv, heads, window))
    return fail(MOE_ERR_UNSUPPORTED, "T=%d rows of %d heads pass one launch", T, heads);
  if (!q || !out) return fail(MOE_ERR_INVALID, "NULL q/out");
  if (!aligned(q, 16) || q_token % 8 || q_head % 8 || !aligned(kv->k, 16) ||
      !aligned(kv->v, 16) || !aligned(out, 16))
    return fail(MOE_ERR_INVALID, "q's rows, the pages and out must be 16-byte aligned");
  const size_t need = moe::attn_workspace(a.kv, heads, window);
  if (need && (!workspace || !aligned(workspace, 256)))
    return fail(MOE_ERR_INVALID, "workspace NULL or not 256-byte aligned");
  if (workspace_bytes < need)
    return fail(MOE_ERR_INVALID, "workspace %zu < %zu bytes", workspace_bytes, need);
  a.q = static_cast<const uint16_t *>(q);
  a.q_st = q_token;
  a.q_sh = q_head;
  a.sinks = sinks;
  a.out = static_cast<uint16_t *>(out);
  a.heads = heads;
  a.window = window;
  a.scale = scale;
  (void)hipGetLastError();
  moe::launch_attn(a, kv->dtype, workspace, static_cast<hipStream_t>(stream));
  MOE_HIP(hipGetLastError());
  return MOE_OK;
}

}  // extern "C"
