// y = (x in e4m3) (w in e4m3)^T with a 32-bit scale per 128 columns of a row of x
// and per 128 x 128 block of w.
#include "layer.h"

namespace moe {

// One thread per output.
template <class T>
__global__ __launch_bounds__(256) void linear_simple_kernel(LinearArgs a) {
  const int n = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
  if (n >= a.N) return;
  const int blocks = (a.K + kFp8Block - 1) / kFp8Block;
  float y = 0.f;
  for (int b = 0; b < blocks; ++b) {
    float acc = 0.f;
    for (int k = b * kFp8Block; k < min(a.K, (b + 1) * kFp8Block); ++k)
      acc = fmaf(__builtin_amdgcn_cvt_f32_fp8(a.x[t * a.x_stride + k], 0),
                 __builtin_amdgcn_cvt_f32_fp8(a.w[(int64_t)n * a.K + k], 0), acc);
    y = fmaf(acc, a.xs[(int64_t)t * blocks + b] * a.ws[(n / kFp8Block) * blocks + b], y);
  }
  if (a.bias) y += T::load(a.bias[n]);
  a.y[(int64_t)t * a.N + n] = (uint16_t)T::store(y);
}

size_t linear_workspace(int, int, int) { return 0; }

void launch_linear(const LinearArgs &a, int out_dtype, hipStream_t s) {
  const dim3 g((a.N + 255) / 256, a.T), b(256);
  if (out_dtype == MOE_DTYPE_BF16) hipLaunchKernelGGL((linear_simple_kernel<Bf16>), g, b, 0, s, a);
  else hipLaunchKernelGGL((linear_simple_kernel<F16>), g, b, 0, s, a);
}

}  // namespace moe
