// Product of 8-bit floats (e4m3) with a scale for each row and 128 columns of the activations and for each 128 x 128 block
// of the weights:  y[m, n] = sum over blocks b of  sx[m, b] sw[n / 128, b] sum_k qx[m, 128 b + k] qw[n, 128 b + k]  + bias[n]
#include "rows.hpp"

namespace mv {
namespace {

__device__ __forceinline__ float from_e4m3(unsigned word, int byte) {
  switch (byte) {
    case 0: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 0);
    case 1: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 1);
    case 2: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 2);
    default: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 3);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void product_kernel(const unsigned *q, const float *qs, const unsigned *w, const float *ws,
                                                      const T *bias, T *y, long rows, int inputs, int outputs) {
  const long at = static_cast<long>(linear_block()) * 256 + threadIdx.x;
  if (at >= rows * outputs) return;
  const long m = at / outputs;
  const int n = static_cast<int>(at % outputs), blocks = inputs / kBlock;
  float sum = 0.f;
  for (int b = 0; b < blocks; ++b) {
    float part = 0.f;
    for (int k = 0; k < kBlock / 4; ++k) {
      const unsigned x = q[m * (inputs / 4) + b * (kBlock / 4) + k], v = w[static_cast<long>(n) * (inputs / 4) + b * (kBlock / 4) + k];
#pragma unroll
      for (int i = 0; i < 4; ++i) part += from_e4m3(x, i) * from_e4m3(v, i);
    }
    sum += part * (qs[m * blocks + b] * ws[static_cast<long>(n / kBlock) * blocks + b]);
  }
  if (bias) sum += load(bias + n);
  y[at] = store_cast<T>(sum);
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" {

size_t mv_block_linear_workspace_bytes(int64_t rows, int inputs, int outputs) { return 0; }

int mv_block_linear(const void *q, const void *q_scales, const void *weight, const void *weight_scales, const void *bias,
                    void *y, int64_t rows, int inputs, int outputs, int dtype, void *workspace, size_t workspace_bytes,
                    void *stream) {
  MV_REQUIRE(dtype == MV_F16 || dtype == MV_BF16, "dtype %d of the output is not float16 or bfloat16", dtype);
  MV_REQUIRE(rows >= 0 && inputs > 0 && outputs >= 0 && inputs % kBlock == 0, "wrong sizes: %ld rows, %d inputs (whole blocks of 128), %d outputs",
             static_cast<long>(rows), inputs, outputs);
  if (rows == 0 || outputs == 0) return MV_OK;
  MV_REQUIRE(q && q_scales && weight && weight_scales && y, "a tensor is missing");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid = linear_grid((rows * outputs + 255) / 256, 256);
  if (dtype == MV_F16)
    product_kernel<__half><<<grid, 256, 0, s>>>(static_cast<const unsigned *>(q), static_cast<const float *>(q_scales),
        static_cast<const unsigned *>(weight), static_cast<const float *>(weight_scales), static_cast<const __half *>(bias),
        static_cast<__half *>(y), rows, inputs, outputs);
  else
    product_kernel<__hip_bfloat16><<<grid, 256, 0, s>>>(static_cast<const unsigned *>(q), static_cast<const float *>(q_scales),
        static_cast<const unsigned *>(weight), static_cast<const float *>(weight_scales), static_cast<const __hip_bfloat16 *>(bias),
        static_cast<__hip_bfloat16 *>(y), rows, inputs, outputs);
  return check_launch("block_linear");
}

}  // extern "C"
