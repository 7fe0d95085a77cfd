// y = x w^T for block-scaled e4m3 matrices:
//   y[m, n] = sum_b xs[m, b] * ws[n / 128, b] * sum_{k in block b} xq[m, k] wq[n, k]  (+ bias[n])
// Products and sums in 32 bits, rounded once to the output's type.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "fp8.cuh"

namespace ms {

__device__ __forceinline__ float e4m3_value(uint8_t c) {
  __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
  return __half2float(__half(h));
}

template <int OUT>
__device__ __forceinline__ void store_out(void* y, long long at, float v) {
  if (OUT == DT_F32) static_cast<float*>(y)[at] = v;
  else if (OUT == DT_F16) static_cast<__half*>(y)[at] = __float2half_rn(v);
  else static_cast<uint16_t*>(y)[at] = f2bf(v);
}

// 64 x 64 outputs per CTA of 16 x 16 threads, 32 features a step
template <int OUT>
__global__ void __launch_bounds__(256) k_linear_fp8(LinearArgs a) {
  __shared__ float sx[64][33], sw[64][33];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, kb = (a.K + FP8_BLOCK - 1) / FP8_BLOCK;
  float acc[4][4] = {};
  for (int b = 0; b < kb; ++b) {
    float part[4][4] = {};
    for (int k0 = b * FP8_BLOCK; k0 < min(a.K, (b + 1) * FP8_BLOCK); k0 += 32) {
      __syncthreads();
      for (int i = threadIdx.x; i < 64 * 32; i += 256) {
        const int r = i >> 5, c = i & 31;
        const bool in = k0 + c < a.K;
        sx[r][c] = in && m0 + r < a.M ? e4m3_value(a.x[(m0 + r) * a.x_stride + k0 + c]) : 0.f;
        sw[r][c] = in && n0 + r < a.N ? e4m3_value(a.w[(n0 + r) * a.w_stride + k0 + c]) : 0.f;
      }
      __syncthreads();
      for (int k = 0; k < 32; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][j] = fmaf(sx[ty + 16 * i][k], sw[tx + 16 * j][k], part[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
        if (m < a.M && n < a.N)
          acc[i][j] = fmaf(a.xs[m * a.xs_stride + b] * a.ws[(long long)(n / FP8_BLOCK) * kb + b], part[i][j], acc[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < a.M && n < a.N) store_out<OUT>(a.y, m * a.y_stride + n, acc[i][j] + (a.bias ? a.bias[n] : 0.f));
    }
}

cudaError_t launch_linear_fp8(const LinearArgs& a, int out_dtype, int sms, cudaStream_t s) {
  (void)sms;
  const dim3 grid((a.N + 63) / 64, (a.M + 63) / 64);
  if (out_dtype == DT_BF16) k_linear_fp8<DT_BF16><<<grid, 256, 0, s>>>(a);
  else if (out_dtype == DT_F16) k_linear_fp8<DT_F16><<<grid, 256, 0, s>>>(a);
  else k_linear_fp8<DT_F32><<<grid, 256, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace ms
