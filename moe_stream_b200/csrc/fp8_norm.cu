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
// Bound by memory: x, res, h and the codes once each. A CTA owns a row at a
// time and keeps it in registers between the sum and the codes, the weight
// too, from row to row. Eight consecutive features per thread and chunk: 16
// lanes make a group, its maximum is four shuffles.
#include <algorithm>

#include <cuda_fp16.h>

#include "fp8.cuh"

namespace ms {

template <int DT> struct Elem { using T = uint16_t; };
template <> struct Elem<DT_F32> { using T = float; };

template <int DT>
__device__ __forceinline__ float elem_load(const typename Elem<DT>::T* p) {
  if constexpr (DT == DT_F32) return *p;
  else if constexpr (DT == DT_F16) return __half2float(__ushort_as_half(*p));
  else return bf2f(*p);
}
template <int DT>
__device__ __forceinline__ uint16_t elem_bits(float v) {
  if constexpr (DT == DT_F16) return __half_as_ushort(__float2half_rn(v));
  else return f2bf(v);
}

// Eight features as they lie in memory: half the registers of their values
// for the 16-bit types.
template <int DT> struct Raw { uint32_t u[4]; };
template <> struct Raw<DT_F32> { uint32_t u[8]; };

template <int DT>
__device__ __forceinline__ void unpack(const Raw<DT>& r, float* v) {
#pragma unroll
  for (int i = 0; i < (DT == DT_F32 ? 8 : 4); ++i) {
    if constexpr (DT == DT_F32) {
      v[i] = __uint_as_float(r.u[i]);
    } else if constexpr (DT == DT_F16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.u[i]));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    } else {
      v[2 * i] = __uint_as_float(r.u[i] << 16), v[2 * i + 1] = __uint_as_float(r.u[i] & 0xffff0000u);
    }
  }
}
// rounded to the type
template <int DT>
__device__ __forceinline__ Raw<DT> pack(const float* v) {
  Raw<DT> r;
#pragma unroll
  for (int i = 0; i < (DT == DT_F32 ? 8 : 4); ++i) {
    if constexpr (DT == DT_F32) r.u[i] = __float_as_uint(v[i]);
    else r.u[i] = elem_bits<DT>(v[2 * i]) | (uint32_t)elem_bits<DT>(v[2 * i + 1]) << 16;
  }
  return r;
}
// Features 8c to 8c + 7 of a row; those past d are 0. VEC: whole chunks, rows
// on 16-byte boundaries.
template <int DT, bool VEC>
__device__ __forceinline__ Raw<DT> load8(const typename Elem<DT>::T* row, int c, int d) {
  Raw<DT> r;
  if constexpr (VEC) {
    const uint4* p = reinterpret_cast<const uint4*>(row) + (DT == DT_F32 ? 2 : 1) * c;
#pragma unroll
    for (int i = 0; i < (DT == DT_F32 ? 2 : 1); ++i) {
      const uint4 a = p[i];
      r.u[4 * i] = a.x, r.u[4 * i + 1] = a.y, r.u[4 * i + 2] = a.z, r.u[4 * i + 3] = a.w;
    }
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 8 * c + i < d ? elem_load<DT>(row + 8 * c + i) : 0.f;
    r = pack<DT>(v);
  }
  return r;
}
template <int DT, bool VEC>
__device__ __forceinline__ void store8(typename Elem<DT>::T* row, int c, int d, const Raw<DT>& r) {
  if constexpr (VEC) {
    uint4* p = reinterpret_cast<uint4*>(row) + (DT == DT_F32 ? 2 : 1) * c;
#pragma unroll
    for (int i = 0; i < (DT == DT_F32 ? 2 : 1); ++i)
      p[i] = make_uint4(r.u[4 * i], r.u[4 * i + 1], r.u[4 * i + 2], r.u[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (8 * c + i < d) {
        if constexpr (DT == DT_F32) row[8 * c + i] = __uint_as_float(r.u[i]);
        else row[8 * c + i] = (uint16_t)(r.u[i / 2] >> (16 * (i & 1)));
      }
  }
}

// 1 / sqrt(m), rounded once to 32 bits: two Newton steps in 64 from the 32-bit
// estimate (relative error below 1e-13, far below half a step of the result),
// a few instructions where the 64-bit root and quotient take many.
__device__ __forceinline__ float rms_factor(double m) {
  if (!(m > 1e-37 && m < 1e37)) return (float)(1.0 / sqrt(m));
  double y = (double)rsqrtf((float)m);
#pragma unroll
  for (int i = 0; i < 2; ++i) y = fma(y * 0.5, fma(-m * y, y, 1.0), y);
  return (float)y;
}

// NC chunks per thread; chunk i of a thread is threadIdx.x + i * blockDim.x,
// so the 16 lanes of a group are neighbours.
template <int DT, int NC, bool NORM, bool VEC>
__global__ void __launch_bounds__(512) k_norm_fp8(NormArgs a) {
  using E = typename Elem<DT>::T;
  __shared__ double red[2][16];
  const int d = a.d, chunks = (d + 7) / 8, groups = (d + FP8_BLOCK - 1) / FP8_BLOCK;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Raw<DT> w[NORM ? NC : 1];
  if constexpr (NORM)
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      w[i] = {};
      if (c < chunks) w[i] = load8<DT, VEC>(static_cast<const E*>(a.w), c, d);
    }
  int turn = 0;
  for (int t = blockIdx.x; t < a.T; t += gridDim.x, turn ^= 1) {
    const E* x = static_cast<const E*>(a.x) + t * a.x_stride;
    Raw<DT> h[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      h[i] = {};
      if (c < chunks) h[i] = load8<DT, VEC>(x, c, d);
    }
    float f = 1.f;
    if constexpr (NORM) {
      if (a.res) {
        const E* r = static_cast<const E*>(a.res) + t * a.res_stride;
        Raw<DT> u[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const int c = threadIdx.x + i * blockDim.x;
          if (c < chunks) u[i] = load8<DT, VEC>(r, c, d);
        }
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const int c = threadIdx.x + i * blockDim.x;
          if (c < chunks) {
            float p[8], q[8];
            unpack<DT>(h[i], p);
            unpack<DT>(u[i], q);
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = __fadd_rn(p[j], q[j]);
            h[i] = pack<DT>(p);
            store8<DT, VEC>(static_cast<E*>(a.h) + t * a.h_stride, c, d, h[i]);
          }
        }
      }
      double ss = 0.0;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        float v[8];
        unpack<DT>(h[i], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fma((double)v[j], (double)v[j], ss);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(MS_FULL, ss, o);
      if (warps > 1) {                      // two sets of sums: one barrier a row
        if (lane == 0) red[turn][warp] = ss;
        __syncthreads();
        ss = 0.0;
        for (int i = 0; i < warps; ++i) ss += red[turn][i];
      }
      f = rms_factor(ss / (double)d + a.eps);
    }
    uint8_t* q = a.q + t * a.q_stride;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      float v[8], m = 0.f;
      unpack<DT>(h[i], v);
      if constexpr (NORM) {
        float g[8];
        unpack<DT>(w[i], g);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(__fmul_rn(v[j], f), g[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (VEC || 8 * c + j < d) m = max_nan(m, fabsf(v[j]));      // past d: 0 times an infinite factor
      if (NORM && a.y && c < chunks) store8<DT, VEC>(static_cast<E*>(a.y) + t * a.y_stride, c, d, pack<DT>(v));
      if (VEC && c >= chunks) m = 0.f;
#pragma unroll
      for (int o = 8; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(MS_FULL, m, o));
      float inv;
      const float s = group_scale(m, &inv);
      if ((threadIdx.x & 15) == 0 && c / 16 < groups) a.s[(long long)t * groups + c / 16] = s;
      if (c < chunks) {
        if constexpr (VEC) {
          uint32_t b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = e4m3x2(v[2 * j] * inv, v[2 * j + 1] * inv);
          reinterpret_cast<uint2*>(q)[c] = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (8 * c + j < d) q[8 * c + j] = (uint8_t)e4m3x2(v[j] * inv, 0.f);
        }
      }
    }
  }
}

template <int DT, int NC, bool NORM, bool VEC>
static cudaError_t launch_nc(const NormArgs& a, int threads, int grid, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_norm_fp8<DT, NC, NORM, VEC>, a);
}

template <int DT, bool NORM, bool VEC>
static cudaError_t launch_vec(const NormArgs& a, int sms, cudaStream_t s) {
  const int chunks = (a.d + 7) / 8, whole = (chunks + 31) / 32 * 32;
  // Rows enough to fill the GPU: three chunks a thread, so that a row's
  // barriers and its ragged end cost little; few rows: as many threads as
  // there are chunks.
  const bool many = a.T >= sms * 4;
  int nc = many ? 3 : 1;
  while ((whole + nc - 1) / nc > 512) ++nc;
  const int threads = std::max(32, ((chunks + nc - 1) / nc + 31) / 32 * 32);
  const int per_sm = std::max(1, 2048 / threads);
  const int grid = (int)std::min<long long>(a.T, (long long)sms * per_sm);
  if (nc == 1) return launch_nc<DT, 1, NORM, VEC>(a, threads, grid, s);
  if (nc == 2) return launch_nc<DT, 2, NORM, VEC>(a, threads, grid, s);
  if (nc == 3) return launch_nc<DT, 3, NORM, VEC>(a, threads, grid, s);
  return launch_nc<DT, 4, NORM, VEC>(a, threads, grid, s);      // 16384 features / 8 / 512
}

template <int DT>
static cudaError_t launch_dt(const NormArgs& a, int sms, cudaStream_t s) {
  constexpr int PER = DT == DT_F32 ? 4 : 8;      // elements of 16 bytes
  auto off = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
  const bool vec = a.d % 8 == 0 && !off(a.x) && !off(a.res) && !off(a.w) && !off(a.h) && !off(a.y) && !off(a.q) &&
                   a.x_stride % PER == 0 && (!a.res || a.res_stride % PER == 0) && (!a.h || a.h_stride % PER == 0) &&
                   (!a.y || a.y_stride % PER == 0) && a.q_stride % 8 == 0;
  if (a.w) return vec ? launch_vec<DT, true, true>(a, sms, s) : launch_vec<DT, true, false>(a, sms, s);
  return vec ? launch_vec<DT, false, true>(a, sms, s) : launch_vec<DT, false, false>(a, sms, s);
}

cudaError_t launch_norm_fp8(const NormArgs& a, int dtype, int sms, cudaStream_t s) {
  if (dtype == DT_BF16) return launch_dt<DT_BF16>(a, sms, s);
  if (dtype == DT_F16) return launch_dt<DT_F16>(a, sms, s);
  return launch_dt<DT_F32>(a, sms, s);
}

}  // namespace ms
