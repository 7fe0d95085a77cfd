// Residual add + RMSNorm + e4m3 codes with a scale per 128 features, one
// pass over the rows.
//
//   h = round(x + res)                      (x's type; h = x without res)
//   y = (h * (1 / sqrt(mean(h^2) + eps))) * w          (h without w)
//   per 128 features: s = group_scale(max|y|), q = e4m3(y / s)
//
// The squares are summed in 64 bits and the factor is rounded to 32 once, so
// it does not depend on the order of the sum: a code or a scale next to a
// border is the same whatever the launch shape. Everything after it is one
// 32-bit rounding per product.
//
// Bound by memory: x, res, h and the codes once each. A row stays in
// registers between the sum and the codes. Eight consecutive features per
// thread: 16 lanes make a group, its maximum is four shuffles.
#include <cuda_fp16.h>

#include "fp8.cuh"

namespace ms {

template <int DT> struct Elem;
template <> struct Elem<DT_BF16> { using T = uint16_t; };
template <> struct Elem<DT_F16> { using T = uint16_t; };
template <> struct Elem<DT_F32> { using T = float; };

template <int DT>
__device__ __forceinline__ float elem_load(const typename Elem<DT>::T* p) {
  if constexpr (DT == DT_F32) return *p;
  else if constexpr (DT == DT_F16) return __half2float(__ushort_as_half(*p));
  else return bf2f(*p);
}
// v rounded to the type, as a float
template <int DT>
__device__ __forceinline__ float elem_round(float v) {
  if constexpr (DT == DT_F32) return v;
  else if constexpr (DT == DT_F16) return __half2float(__float2half_rn(v));
  else return bfr(v);
}
template <int DT>
__device__ __forceinline__ void elem_store(typename Elem<DT>::T* p, float v) {
  if constexpr (DT == DT_F32) *p = v;
  else if constexpr (DT == DT_F16) *p = __half_as_ushort(__float2half_rn(v));
  else *p = f2bf(v);
}

// Row values of chunk c (8 features from 8c); features past d read as 0.
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T* row, int c, int d, float* v) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 8 * c + i < d ? elem_load<DT>(row + 8 * c + i) : 0.f;
}

template <int DT>
__global__ void __launch_bounds__(256) k_norm_fp8(NormArgs a) {
  using E = typename Elem<DT>::T;
  __shared__ double red[8];
  const int d = a.d, chunks = (d + 7) / 8, groups = (d + FP8_BLOCK - 1) / FP8_BLOCK;
  for (int t = blockIdx.x; t < a.T; t += gridDim.x) {
    const E* x = static_cast<const E*>(a.x) + t * a.x_stride;
    const E* r = a.res ? static_cast<const E*>(a.res) + t * a.res_stride : nullptr;
    auto row8 = [&](int c, float* v) {
      load8<DT>(x, c, d, v);
      if (r) {
        float u[8];
        load8<DT>(r, c, d, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = elem_round<DT>(__fadd_rn(v[i], u[i]));
      }
    };
    float f = 1.f;
    if (a.w) {
      double ss = 0.0;
      for (int c = threadIdx.x; c < chunks; c += 256) {
        float v[8];
        row8(c, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fma((double)v[i], (double)v[i], ss);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(MS_FULL, ss, o);
      __syncthreads();
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
      __syncthreads();
      ss = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += red[i];
      f = (float)(1.0 / sqrt(ss / (double)d + a.eps));
    }
    // every lane of a group's 16 takes part in its maximum
    for (int c = threadIdx.x; c < groups * 16; c += 256) {
      float v[8];
      row8(c, v);
      if (a.h)
        for (int i = 0; i < 8 && 8 * c + i < d; ++i)
          elem_store<DT>(static_cast<E*>(a.h) + t * a.h_stride + 8 * c + i, v[i]);
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (a.w && 8 * c + i < d)
          v[i] = __fmul_rn(__fmul_rn(v[i], f), elem_load<DT>(static_cast<const E*>(a.w) + 8 * c + i));
        m = max_nan(m, fabsf(v[i]));
      }
      if (a.y)
        for (int i = 0; i < 8 && 8 * c + i < d; ++i)
          elem_store<DT>(static_cast<E*>(a.y) + t * a.y_stride + 8 * c + i, v[i]);
      const unsigned lanes = 0xffffu << (threadIdx.x & 16);
#pragma unroll
      for (int o = 8; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(lanes, m, o));
      float inv;
      const float s = group_scale(m, &inv);
      if ((threadIdx.x & 15) == 0) a.s[(long long)t * groups + c / 16] = s;
      for (int i = 0; i < 8 && 8 * c + i < d; ++i)
        a.q[t * a.q_stride + 8 * c + i] = (uint8_t)e4m3x2(v[i] * inv, 0.f);
    }
  }
}

cudaError_t launch_norm_fp8(const NormArgs& a, int dtype, int sms, cudaStream_t s) {
  const int grid = a.T < sms * 8 ? a.T : sms * 8;
  if (dtype == DT_BF16) k_norm_fp8<DT_BF16><<<grid, 256, 0, s>>>(a);
  else if (dtype == DT_F16) k_norm_fp8<DT_F16><<<grid, 256, 0, s>>>(a);
  else k_norm_fp8<DT_F32><<<grid, 256, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace ms
