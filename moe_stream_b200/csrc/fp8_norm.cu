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
    if constexpr (DT == DT_F32) {
      r.u[i] = __float_as_uint(v[i]);
    } else if constexpr (DT == DT_F16) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      r.u[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      r.u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
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

// The sum of eight squares, in 64 bits.
__device__ __forceinline__ double squares(const float* v) {
  double ss[2] = {0.0, 0.0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double x = (double)v[i];
    ss[i & 1] = fma(x, x, ss[i & 1]);
  }
  return ss[0] + ss[1];
}
// largest of |v|, NaN where one is
__device__ __forceinline__ float max8_nan(const float* v) {
  float m = fabsf(v[0]);
  asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(v[1])), "f"(fabsf(v[2])));
  asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(v[3])), "f"(fabsf(v[4])));
  asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(v[5])), "f"(fabsf(v[6])));
  return max_nan(m, fabsf(v[7]));
}
__device__ __forceinline__ void mul2(float& a, float& b, float x, float y) {
  uint64_t p, q;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  asm("mov.b64 %0, {%1, %2};" : "=l"(q) : "f"(x), "f"(y));
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(p) : "l"(q));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}

// 1 / sqrt(m), rounded once to 32 bits: two Newton steps in 64 from the 32-bit
// estimate (relative error below 1e-13, far below half a step of the result),
// a few instructions where the 64-bit root and quotient take many. Where the
// factor of a row of very small or very large values is no normal 32-bit number,
// *pre, a power of two that the values are multiplied with first, takes part of
// it (a row of zeros may leave more, where any finite factor does).
__device__ __forceinline__ float rms_factor(double m, float* pre) {
  *pre = 1.f;
  if (!(m > 1e-37 && m < 1e37)) {
    double r = 1.0 / sqrt(m);
    if (r < 1e-37) *pre = 0x1p-64f, r *= 0x1p64;
    if (r > 1e37) *pre = 0x1p64f, r *= 0x1p-64;
    if (m > 0.0) r = fmin(r, 1e38);
    return (float)r;
  }
  double y = (double)rsqrtf((float)m);
#pragma unroll
  for (int i = 0; i < 2; ++i) y = fma(y * 0.5, fma(-m * y, y, 1.0), y);
  return (float)y;
}

// A CTA of TPR threads (0: of any number) per row, NC chunks each: chunk i of
// a thread is threadIdx.x + i * TPR, so the 16 lanes of a group are
// neighbours, all but the last chunk are whole, and their places are
// immediates. PIPE: the next row's loads are in flight while this one is
// reduced.
template <int DT, int TPR, int NC, bool NORM, bool VEC>
__global__ void __launch_bounds__(TPR ? TPR : 512) k_norm_fp8(NormArgs a) {
  using E = typename Elem<DT>::T;
  constexpr bool PIPE = NORM && TPR > 0;
  __shared__ double red[2][16];
  const int tpr = TPR ? TPR : blockDim.x;
  const int d = a.d, chunks = (d + 7) / 8, groups = (d + FP8_BLOCK - 1) / FP8_BLOCK;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = tpr >> 5;
  const bool last = (int)threadIdx.x + (NC - 1) * tpr < chunks;      // the last chunk is this thread's
  const double inv_d = 1.0 / (double)d;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Raw<DT> w[PIPE ? NC : 1];
  if constexpr (PIPE)
#pragma unroll
    for (int i = 0; i < NC; ++i)
      w[i] = i + 1 < NC || last ? load8<DT, VEC>(static_cast<const E*>(a.w), threadIdx.x + i * tpr, d) : Raw<DT>{};
  Raw<DT> nx[NC], nr[NORM ? NC : 1];
  auto fetch = [&](int t) {
    const E* x = static_cast<const E*>(a.x) + t * a.x_stride;
#pragma unroll
    for (int i = 0; i < NC; ++i)
      nx[i] = i + 1 < NC || last ? load8<DT, VEC>(x, threadIdx.x + i * tpr, d) : Raw<DT>{};
    if constexpr (NORM)
      if (a.res) {
        const E* r = static_cast<const E*>(a.res) + t * a.res_stride;
#pragma unroll
        for (int i = 0; i < NC; ++i)
          nr[i] = i + 1 < NC || last ? load8<DT, VEC>(r, threadIdx.x + i * tpr, d) : Raw<DT>{};
      }
  };
  if (PIPE && blockIdx.x < a.T) fetch(blockIdx.x);
  int turn = 0;
  for (int t = blockIdx.x; t < a.T; t += gridDim.x, turn ^= 1) {
    if (!PIPE) fetch(t);
    Raw<DT> h[NC];
    double ss = 0.0;
    float f = 1.f, pre = 1.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) h[i] = nx[i];
    if constexpr (NORM) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        float v[8];
        unpack<DT>(h[i], v);
        if (a.res) {
          float u[8];
          unpack<DT>(nr[i], u);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = __fadd_rn(v[j], u[j]);
          h[i] = pack<DT>(v);
          unpack<DT>(h[i], v);
        }
        ss += squares(v);
      }
      if (PIPE && t + (int)gridDim.x < a.T) fetch(t + gridDim.x);    // h may be x or res: another row
      if (a.h) {
        E* o = static_cast<E*>(a.h) + t * a.h_stride;
#pragma unroll
        for (int i = 0; i < NC; ++i)
          if (i + 1 < NC || last) store8<DT, VEC>(o, threadIdx.x + i * tpr, d, h[i]);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(MS_FULL, ss, o);
      if (warps > 1) {                      // two sets of sums: one barrier a row
        if (lane == 0) red[turn][warp] = ss;
        __syncthreads();
        ss = 0.0;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < warps) ss += red[turn][i];
      }
      f = rms_factor(fma(ss, inv_d, a.eps), &pre);
    }
    uint8_t* q = a.q + t * a.q_stride;
    float* s_row = a.s + (long long)t * groups + (threadIdx.x >> 4);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = threadIdx.x + i * tpr;
      const bool mine = i + 1 < NC || last;
      float v[8], m = 0.f;
      unpack<DT>(h[i], v);
      if constexpr (NORM) {
        float g[8] = {};
        if constexpr (PIPE) unpack<DT>(w[i], g);
        else if (mine) unpack<DT>(load8<DT, VEC>(static_cast<const E*>(a.w), c, d), g);
        if (pre != 1.f)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= pre;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          mul2(v[j], v[j + 1], f, f);
          mul2(v[j], v[j + 1], g[j], g[j + 1]);
        }
      }
      // past d: 0 times an infinite factor
      if constexpr (VEC) {
        m = mine ? max8_nan(v) : 0.f;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (8 * c + j < d) m = max_nan(m, fabsf(v[j]));
      }
      if (NORM && a.y && mine) store8<DT, VEC>(static_cast<E*>(a.y) + t * a.y_stride, c, d, pack<DT>(v));
#pragma unroll
      for (int o = 8; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(MS_FULL, m, o));
      float inv;
      const float s = group_scale(m, &inv);
      if ((threadIdx.x & 15) == 0 && mine) s_row[i * (tpr >> 4)] = s;
      if (mine) {
        if constexpr (VEC) {
          uint32_t b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mul2(v[2 * j], v[2 * j + 1], inv, inv);
            b[j] = e4m3x2(v[2 * j], v[2 * j + 1]);
          }
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

template <int DT, int TPR, int NC, bool NORM, bool VEC>
static cudaError_t launch_nc(const NormArgs& a, int threads, int sms, cudaStream_t s) {
  // PIPE: as many CTAs as are resident, so that a row's loads run ahead
  const int per_sm = NORM && TPR ? std::max(1, 512 / threads) : 2048 / threads;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)std::min<long long>(a.T, (long long)per_sm * sms));
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_norm_fp8<DT, TPR, NC, NORM, VEC>, a);
}

template <int DT, int TPR, bool NORM, bool VEC>
static cudaError_t launch_tpr(const NormArgs& a, int threads, int nc, int sms, cudaStream_t s) {
  if (nc == 1) return launch_nc<DT, 0, 1, NORM, VEC>(a, threads, sms, s);
  if (nc == 2) return launch_nc<DT, 0, 2, NORM, VEC>(a, threads, sms, s);
  if (nc == 3) return launch_nc<DT, TPR, 3, NORM, VEC>(a, threads, sms, s);
  return launch_nc<DT, TPR, 4, NORM, VEC>(a, threads, sms, s);       // 16384 features / 8 / 512
}

template <int DT, bool NORM, bool VEC>
static cudaError_t launch_vec(const NormArgs& a, int sms, cudaStream_t s) {
  const int chunks = (a.d + 7) / 8;
  // Rows enough to fill the GPU: three or four chunks a thread, so that a
  // row's barrier costs little (32-bit values, twice the registers: two; 4096
  // x 4096 35.5 us against 38.6 with four); few rows: a thread per chunk.
  if (VEC && a.T >= sms * 4) {
    int threads = 32;
    while (threads < 512 && threads * (DT == DT_F32 ? 2 : 4) < chunks) threads *= 2;
    const int nc = (chunks + threads - 1) / threads;
    if constexpr (DT == DT_F32) {              // below 512 threads: one or two chunks
      if (threads < 512) return launch_tpr<DT, 0, NORM, true>(a, threads, nc, sms, s);
    } else {
      if (threads == 32) return launch_tpr<DT, 32, NORM, true>(a, 32, nc, sms, s);
      if (threads == 64) return launch_tpr<DT, 64, NORM, true>(a, 64, nc, sms, s);
      if (threads == 128) return launch_tpr<DT, 128, NORM, true>(a, 128, nc, sms, s);
      if (threads == 256) return launch_tpr<DT, 256, NORM, true>(a, 256, nc, sms, s);
    }
    return launch_tpr<DT, 512, NORM, true>(a, 512, nc, sms, s);
  }
  const int nc = (chunks + 511) / 512;
  return launch_tpr<DT, 0, NORM, VEC>(a, ((chunks + nc - 1) / nc + 31) / 32 * 32, nc, sms, s);
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
