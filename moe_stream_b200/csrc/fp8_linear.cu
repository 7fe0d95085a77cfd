// y = x w^T for block-scaled e4m3 matrices:
//   y[m, n] = sum_b xs[m, b] * ws[n / 128, b] * sum_{k in block b} xq[m, k] wq[n, k]  (+ bias[n])
// Each block's products go through the tensor cores into a fresh TMEM
// accumulator; the block's scales are applied as it is added, in 32 bits, and
// the sum is rounded once to the output's type.
#include <algorithm>

#include <cudaTypedefs.h>
#include <cuda_fp16.h>

#include "fp8_mma.cuh"

namespace ms {

// first failure of a bounded wait in this file's kernels (ms_fp8_status)
static __device__ int g_linear_status;

template <int OUT>
__device__ __forceinline__ void store_out(void* y, long long at, float v) {
  if (OUT == DT_F32) static_cast<float*>(y)[at] = v;
  else if (OUT == DT_F16) static_cast<__half*>(y)[at] = __float2half_rn(v);
  else static_cast<uint16_t*>(y)[at] = f2bf(v);
}

// ------------------------------------------------------------------ few rows
// The weight is the MMA's A operand (128 of its rows are the TMEM lanes) and
// up to NT rows of x are the columns, so a single token costs no more tensor
// work than sixteen and the weight is read once, as it lies. The blocks of K
// are split over a cluster of CTAs, because few rows leave few tiles; the
// cluster joins its sums through shared memory in rank order, so the result
// does not depend on timing.
//
// Warps 0-3 take finished blocks out of TMEM (one lane quarter each), warp 4
// loads, warp 5 issues the MMAs. TMEM: 256 columns, cut into blocks' buffers.
// Shared memory is between 76 and 113 KB: at most two CTAs on an SM, so their
// TMEM always fits and an allocation never waits for a CTA that itself waits
// for its cluster.
constexpr int FEW_THREADS = 192, FEW_TMEM = 256, FEW_CHUNK = 16;
template <int NT> struct Few {
  static constexpr int STAGES = NT <= 16 ? 5 : NT <= 64 ? 4 : 3;
  static constexpr int STAGE = FP8_W_TILE + NT * 128;
  static constexpr int BUFS = NT <= 32 ? 8 : FEW_TMEM / NT;
  static constexpr int OFF_S = STAGES * STAGE;                      // scales [FEW_CHUNK][NT]
  static constexpr int OFF_BAR = OFF_S + FEW_CHUNK * NT * 4;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;
  static_assert(SMEM > 77824 && SMEM <= 115712, "one or two CTAs on an SM");
  static_assert(NT * 128 * 4 <= OFF_S, "the sums fit over the stages");
  static_assert(BUFS * NT <= FEW_TMEM && STAGE % 1024 == 0, "TMEM columns, tile alignment");
};

template <int NT, int OUT>
__global__ void __launch_bounds__(FEW_THREADS)
    k_linear_few(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, LinearArgs a) {
  using C = Few<NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_scale = reinterpret_cast<float*>(smem + C::OFF_S);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* full = bars;                     // [STAGES] tiles landed
  uint64_t* empty = full + C::STAGES;        // [STAGES] MMAs have read them
  uint64_t* d_full = empty + C::STAGES;      // [BUFS]   a block's product complete
  uint64_t* d_empty = d_full + C::BUFS;      // [BUFS]   taken out
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(d_empty + C::BUFS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = gridDim.x, rank = blockIdx.x;
  const int n0 = blockIdx.y * 128, m0 = blockIdx.z * NT;
  const int kb = (a.K + 127) / 128;
  const int b0 = (int)((long long)kb * rank / split), b1 = (int)((long long)kb * (rank + 1) / split);

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < C::BUFS; ++i) mbar_init(&d_full[i], 1), mbar_init(&d_empty[i], 4);
    fence_barrier_init();
  }
  if (warp == 4 && lane == 0) {
    tma_map_prefetch(&tmW);
    tma_map_prefetch(&tmX);
  }
  if (warp == 5) tmem_get(tmem_at, FEW_TMEM);
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_at;

  float acc[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n] = 0.f;

  if (warp == 4) {
    if (lane == 0) {
      for (int b = b0; b < min(b1, b0 + C::STAGES); ++b) tma_prefetch_2d(&tmW, b * 128, n0);
      grid_wait();
      for (int b = b0, i = 0; b < b1; ++b, ++i) {
        const int s = i % C::STAGES;
        if (i >= C::STAGES && !mbar_wait(&empty[s], ((i / C::STAGES) - 1) & 1, &g_linear_status)) {
          for (int j = i - C::STAGES; j < i; ++j)      // copies in flight land before the CTA ends
            mbar_wait(&full[j % C::STAGES], (j / C::STAGES) & 1, &g_linear_status);
          break;
        }
        mbar_expect_tx(&full[s], C::STAGE);
        tma_tile_2d(smem + s * C::STAGE, &tmW, b * 128, n0, &full[s]);
        tma_tile_2d(smem + s * C::STAGE + FP8_W_TILE, &tmX, b * 128, m0, &full[s]);
      }
    }
  } else if (warp == 5) {
    grid_wait();
    grid_release();
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3(128, NT);
      for (int b = b0, i = 0; b < b1; ++b, ++i) {
        const int s = i % C::STAGES, u = i % C::BUFS;
        if (!mbar_wait(&full[s], (i / C::STAGES) & 1, &g_linear_status)) break;
        if (i >= C::BUFS && !mbar_wait(&d_empty[u], ((i / C::BUFS) - 1) & 1, &g_linear_status)) break;
        tc_after();
        const uint64_t ad = k128_desc(smem + s * C::STAGE), bd = k128_desc(smem + s * C::STAGE + FP8_W_TILE);
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_e4m3(tmem + u * NT, ad + 2 * j, bd + 2 * j, idesc, j != 0);
        mma_done(&empty[s]);
        mma_done(&d_full[u]);
      }
    }
  } else {
    grid_wait();
    const float* ws = a.ws + (long long)blockIdx.y * kb;
    bool ok = true;
    for (int c0 = b0; c0 < b1 && ok; c0 += FEW_CHUNK) {
      const int nc = min(FEW_CHUNK, b1 - c0);
      named_bar(1, 128);                     // the chunk before has been used
      for (int i = threadIdx.x; i < nc * NT; i += 128) {
        const int n = i / nc, c = i - n * nc;
        s_scale[c * NT + n] = m0 + n < a.M ? a.xs[(m0 + n) * a.xs_stride + c0 + c] * ws[c0 + c] : 0.f;
      }
      named_bar(1, 128);
      for (int c = 0; c < nc; ++c) {
        const int i = c0 - b0 + c, u = i % C::BUFS;
        if (!mbar_wait(&d_full[u], (i / C::BUFS) & 1, &g_linear_status)) {
          ok = false;
          break;
        }
        tc_after();
        const uint32_t t = tmem + ((uint32_t)(warp * 32) << 16) + u * NT;
#pragma unroll
        for (int n = 0; n < NT; n += 16) {
          uint32_t v[16];
          tmem_load16(t + n, v);
          tmem_wait16(v);
          const float4* f4 = reinterpret_cast<const float4*>(s_scale + c * NT + n);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 f = f4[j];
            acc[n + 4 * j] = fmaf(__uint_as_float(v[4 * j]), f.x, acc[n + 4 * j]);
            acc[n + 4 * j + 1] = fmaf(__uint_as_float(v[4 * j + 1]), f.y, acc[n + 4 * j + 1]);
            acc[n + 4 * j + 2] = fmaf(__uint_as_float(v[4 * j + 2]), f.z, acc[n + 4 * j + 2]);
            acc[n + 4 * j + 3] = fmaf(__uint_as_float(v[4 * j + 3]), f.w, acc[n + 4 * j + 3]);
          }
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive1(&d_empty[u]);
      }
    }
  }

  // every MMA of this CTA has been waited for by its warps 0-3, so the stages
  // are free; the cluster's sums meet there, [column][lane]
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);
  if (split > 1) {
    if (warp < 4)
#pragma unroll
      for (int n = 0; n < NT; ++n) part[n * 128 + threadIdx.x] = acc[n];
    cluster_sync();
  }
  if (warp < 4 && n0 + (int)threadIdx.x < a.N) {
    const int n = n0 + threadIdx.x;
    const float bias = a.bias ? a.bias[n] : 0.f;
    if (split > 1) {
      uint32_t peer[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) peer[r] = r < split ? cluster_map(part, r) : 0;
      for (int c = rank; c < NT && m0 + c < a.M; c += split) {
        float v = 0.f;
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < split) v += ld_cluster_f32(peer[r] + (c * 128 + threadIdx.x) * 4);
        store_out<OUT>(a.y, (m0 + c) * a.y_stride + n, v + bias);
      }
    } else {
#pragma unroll
      for (int c = 0; c < NT; ++c)
        if (m0 + c < a.M) store_out<OUT>(a.y, (m0 + c) * a.y_stride + n, acc[c] + bias);
    }
  }
  if (split > 1) cluster_sync();             // a peer's sums stay until all have read them
  if (warp == 5) tmem_free(tmem, FEW_TMEM);
}

// ------------------------------------------------------------------ launches
int encode_fp8_map(CUtensorMap* m, const void* base, long long k, long long rows, long long stride, int box_rows,
                   int mats, long long mat_stride) {
  static const auto fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  if (!fn) return -1;
  const cuuint64_t dims[3] = {(cuuint64_t)k, (cuuint64_t)rows, (cuuint64_t)mats};
  const cuuint64_t strides[2] = {(cuuint64_t)stride, (cuuint64_t)mat_stride};
  const cuuint32_t box[3] = {128, (cuuint32_t)box_rows, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, mats > 0 ? 3 : 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? 0
             : -2;
}

template <int NT, int OUT>
static cudaError_t launch_few(const LinearArgs& a, int sms, cudaStream_t s) {
  const int tiles = (a.N + 127) / 128, cols = (a.M + NT - 1) / NT, kb = (a.K + 127) / 128;
  const int split = std::max(1, std::min({8, kb, (sms + tiles * cols - 1) / (tiles * cols)}));
  CUtensorMap tw, tx;
  if (encode_fp8_map(&tw, a.w, a.K, a.N, a.w_stride, 128, 0, 0) ||
      encode_fp8_map(&tx, a.x, a.K, a.M, a.x_stride, NT, 0, 0))
    return cudaErrorInvalidValue;
  auto kern = k_linear_few<NT, OUT>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<NT>::SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(split, tiles, cols);
  cfg.blockDim = dim3(FEW_THREADS);
  cfg.dynamicSmemBytes = Few<NT>::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = split, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, tw, tx, a);
}

template <int OUT>
static cudaError_t launch_out(const LinearArgs& a, int sms, cudaStream_t s) {
  if (a.M <= 16) return launch_few<16, OUT>(a, sms, s);
  if (a.M <= 32) return launch_few<32, OUT>(a, sms, s);
  if (a.M <= 64) return launch_few<64, OUT>(a, sms, s);
  return launch_few<128, OUT>(a, sms, s);
}

cudaError_t launch_linear_fp8(const LinearArgs& a, int out_dtype, int sms, cudaStream_t s) {
  if (out_dtype == DT_BF16) return launch_out<DT_BF16>(a, sms, s);
  if (out_dtype == DT_F16) return launch_out<DT_F16>(a, sms, s);
  return launch_out<DT_F32>(a, sms, s);
}

cudaError_t linear_fp8_status(int** at) { return cudaGetSymbolAddress(reinterpret_cast<void**>(at), g_linear_status); }

}  // namespace ms
