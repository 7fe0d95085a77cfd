// The block-scaled e4m3 format of the fp8 operators.
//
// A matrix is e4m3 codes (OCP FP8, finite, no infinities) and fp32 scales,
// value = code * scale. Activations carry one scale per row and 128
// consecutive features (the last group of a row may be shorter), weights one
// per 128 x 128 block. The quantiser's scales are powers of two, so dividing
// by one is exact and a code depends on the value alone; the products take
// any fp32 scales whose products stay in the normal range of 32 bits.
#pragma once
#include "ms_common.cuh"

namespace ms {

constexpr int FP8_BLOCK = 128;
constexpr int DT_BF16 = 0, DT_F16 = 1, DT_F32 = 2;

// max that keeps a NaN (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The scale of a group whose largest magnitude is a, and its reciprocal:
// s the smallest power of two with max(a, 2^-100) <= 448 s. 448 = 1.75 * 2^8,
// so with a = 1.m * 2^k it is 2^(k-8) for 1.m <= 1.75 and 2^(k-7) above.
// Both are NaN when a is an infinity or a NaN, which makes every code of the
// group NaN.
__device__ __forceinline__ float group_scale(float a, float* inv) {
  const uint32_t b = __float_as_uint(max_nan(a, 7.88860905e-31f));   // 2^-100
  // the carry out of the fraction is the step from 1.75 to the next exponent
  const uint32_t e = (b + 0x1fffffu) & 0xff800000u;
  const bool bad = b >= 0x7f800000u;
  *inv = __uint_as_float(bad ? 0x7fc00000u : (262u << 23) - e);
  return __uint_as_float(bad ? 0x7fc00000u : e - (8u << 23));
}

// two floats -> two e4m3 codes (lo in the low byte), nearest even; NaN -> 0x7f
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

struct NormArgs {
  const void* x;          // [T, d] rows of x_stride elements
  const void* res;        // or null
  const void* w;          // [d], or null: quantise x as it is
  void* h;                // x + res, or null
  void* y;                // the normalised rows before quantisation, or null
  uint8_t* q;             // [T, d] codes, rows of q_stride bytes
  float* s;               // [T, ceil(d / 128)]
  long long x_stride, res_stride, h_stride, y_stride, q_stride;
  int T, d;
  double eps;
};
cudaError_t launch_norm_fp8(const NormArgs& a, int dtype, int sms, cudaStream_t s);

struct LinearArgs {
  const uint8_t* x;       // [M, K] codes, rows of x_stride bytes
  const float* xs;        // [M, ceil(K / 128)], rows of xs_stride
  const uint8_t* w;       // [N, K] codes, rows of w_stride bytes
  const float* ws;        // [ceil(N / 128), ceil(K / 128)]
  const float* bias;      // [N] or null
  void* y;                // [M, N], rows of y_stride elements
  long long x_stride, xs_stride, w_stride, y_stride;
  int M, N, K;
};
cudaError_t launch_linear_fp8(const LinearArgs& a, int out_dtype, int sms, cudaStream_t s);
// Address, on the current device, of the status word of the products' kernels.
cudaError_t linear_fp8_status(int** at);

struct Fp8Matrix {        // [E][n][k] codes
  const uint8_t* q;
  const float* s;         // [E][ceil(n / 128)][ceil(k / 128)]
  const float* bias;      // [E][n] or null
};
struct MoeFp8Args {
  const uint16_t* x;      // bf16 [T, d]
  const uint16_t* router; // bf16 [E, d]
  const float* router_bias;   // [E] or null
  Fp8Matrix gate, up, down;
  const uint16_t* res;    // bf16 [T, d] or null
  uint16_t* y;            // bf16 [T, d]
  uint8_t* ws;            // workspace of moe_fp8_workspace() bytes
  int model, T, d, f, E, k, norm_topk;
};
size_t moe_fp8_workspace(int T, int d, int f, int E, int k);
cudaError_t launch_moe_fp8(const MoeFp8Args& a, int sms, cudaStream_t s);
// Self-test of the layer's waits, for more than MOE_FP8_ROUTED_HERE tokens (up
// to that many are routed by every CTA for itself, without a wait): no token
// is ever routed. y and the experts are not touched.
constexpr int MOE_FP8_ROUTED_HERE = 12;
cudaError_t launch_moe_fp8_lost(const MoeFp8Args& a, int sms, cudaStream_t s);
// Address, on the current device, of the status word of the layer's kernels.
cudaError_t moe_fp8_status(int** at);

}  // namespace ms
