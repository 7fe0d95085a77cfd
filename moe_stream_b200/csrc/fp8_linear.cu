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
  static constexpr int STAGES = NT <= 16 ? 5 : 4;
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
  const int split = cluster_size(), rank = cluster_rank(), tile = cluster_id();
  const int n0 = tile * 128, m0 = blockIdx.y * NT;
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
    if (elect_one())
      for (int b = b0; b < min(b1, b0 + C::STAGES); ++b) tma_prefetch_2d(&tmW, b * 128, n0);
    __syncwarp();
    grid_wait();
    for (int b = b0, i = 0; b < b1; ++b, ++i) {
      const int s = i % C::STAGES;
      if (i >= C::STAGES && !mbar_wait_step(&empty[s], ((i / C::STAGES) - 1) & 1, &g_linear_status)) {
        for (int j = i - C::STAGES; j < i; ++j)      // copies in flight land before the CTA ends
          mbar_wait(&full[j % C::STAGES], (j / C::STAGES) & 1, &g_linear_status);
        break;
      }
      if (elect_one()) {
        mbar_expect_tx(&full[s], C::STAGE);
        tma_tile_2d(smem + s * C::STAGE, &tmW, b * 128, n0, &full[s]);
        tma_tile_2d(smem + s * C::STAGE + FP8_W_TILE, &tmX, b * 128, m0, &full[s]);
      }
      __syncwarp();
    }
  } else if (warp == 5) {
    grid_wait();
    grid_release();
    constexpr uint32_t idesc = idesc_e4m3(128, NT);
    for (int b = b0, i = 0; b < b1; ++b, ++i) {
      const int s = i % C::STAGES, u = i % C::BUFS;
      if (!mbar_wait_step(&full[s], (i / C::STAGES) & 1, &g_linear_status)) break;
      if (i >= C::BUFS && !mbar_wait_step(&d_empty[u], ((i / C::BUFS) - 1) & 1, &g_linear_status)) break;
      tc_after();
      if (elect_one()) {
        const uint64_t ad = k128_desc(smem + s * C::STAGE), bd = k128_desc(smem + s * C::STAGE + FP8_W_TILE);
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_e4m3(tmem + u * NT, ad + 2 * j, bd + 2 * j, idesc, j != 0);
        // no report that nobody waits for: it might come after the CTA's end
        if (b + C::STAGES < b1) mma_done(&empty[s]);
        mma_done(&d_full[u]);
      }
      __syncwarp();
    }
  } else {
    grid_wait();
    const float* ws = a.ws + (long long)tile * kb;
    bool ok = true;
    // after a wait that ran out the warp goes on to the barriers, without the
    // products: others may be waiting there
    for (int c0 = b0; c0 < b1; c0 += FEW_CHUNK) {
      const int nc = min(FEW_CHUNK, b1 - c0);
      named_bar(1, 128);                     // the chunk before has been used
      for (int i = threadIdx.x; i < nc * NT; i += 128) {
        const int n = i / nc, c = i - n * nc;
        s_scale[c * NT + n] = m0 + n < a.M ? a.xs[(m0 + n) * a.xs_stride + c0 + c] * ws[c0 + c] : 0.f;
      }
      named_bar(1, 128);
      for (int c = 0; c < nc; ++c) {
        const int i = c0 - b0 + c, u = i % C::BUFS;
        ok = ok && mbar_wait_step(&d_full[u], (i / C::BUFS) & 1, &g_linear_status);
        if (!ok) break;
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
      const int cols = min(NT, a.M - m0);
      for (int c0 = rank; c0 < cols; c0 += 4 * split) {      // four columns' reads in flight
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < split)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              v[j] += ld_cluster_f32(peer[r] + (min(c0 + j * split, cols - 1) * 128 + threadIdx.x) * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c0 + j * split < cols) store_out<OUT>(a.y, (m0 + c0 + j * split) * a.y_stride + n, v[j] + bias);
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

// ----------------------------------------------------------------- many rows
// Rows of x are the MMA's A operand, so a thread that takes a block out of
// TMEM owns one row and its columns share a scale product. Pairs of CTAs
// compute 256 x 256 outputs (each CTA loads 128 rows of x and 128 of w per
// block, half of what a CTA by itself would need for the same tensor work),
// persistent over the tiles, columns fastest so that the rows of x in flight
// are few.
//
// Every block leaves TMEM, so taking one out has to be as fast as the 512
// cycles of its product: a thread loads 32 columns while it scales the 32
// before (packed products), across blocks too, and gives the buffer back
// before the last of them. That takes 232 registers a thread, given by the
// warps that need none. Two products of 256 x 256 fill TMEM (four of 256 x 128
// were slower, 266 against 260 us for 16384 x 5120 x 2880: twice the barriers).
// A block then takes 0.48 us however few the tiles are, most of it the trip
// between the CTAs of a pair and back. So a single CTA (PAIR false) computes
// 128 x 128 outputs, with four buffers and barriers of its own, where its
// tiles are few (0.39 us); it loads twice the bytes for the same tensor work.
//
// Warps 0-7 take products out of TMEM and write the outputs (lane quarter
// warp % 4, column half warp / 4), warp 8 loads, warp 9 (of the even CTA)
// issues the MMAs, 10 and 11 bring the scales into shared memory eight blocks
// at a time (read one block ahead, their latency was the length of a step:
// 395 us for 16384 x 5120 x 2880). The outputs go through a
// swizzled 4 KB tile of the warp and a tensor store, so that whole lines are
// written; outputs that a tensor map cannot describe are stored one by one.
constexpr int ROWS_THREADS = 384, ROWS_STAGE = 2 * FP8_W_TILE;
constexpr int ROWS_CHUNK = 8;                 // blocks whose scales are staged together
template <bool PAIR> struct Rows {
  static constexpr int STAGES = PAIR ? 4 : 5, BUFS = PAIR ? 2 : 4;
  static constexpr int OUTS = PAIR ? 2 : 1;                          // output tiles per warp
  static constexpr int OFF_OUT = STAGES * ROWS_STAGE;
  static constexpr int OFF_S = OFF_OUT + 8 * OUTS * 4096;            // [2][CHUNK][128] of x
  static constexpr int OFF_SW = OFF_S + 2 * ROWS_CHUNK * 512;        // [2][CHUNK][2] of w
  static constexpr int OFF_B = OFF_SW + 2 * ROWS_CHUNK * 8;          // [4][256] bias of a tile
  static constexpr int OFF_BAR = OFF_B + 4 * 1024;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;
  static_assert(SMEM <= 232448 && SMEM > 232448 - 77824, "alone on its SM");
};

template <int OUT>
__device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
  if (OUT == DT_F16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int OUT, bool PAIR>
__global__ void __launch_bounds__(ROWS_THREADS, 1)
    k_linear_rows(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                  const __grid_constant__ CUtensorMap tmY, int y_map, LinearArgs a) {
  constexpr int CTAS = PAIR ? 2 : 1, TM = 128 * CTAS, TN = 128 * CTAS, COLS = TN / 2;
  using C = Rows<PAIR>;
  constexpr int BUFS = C::BUFS, STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* full = bars;                     // [STAGES] both CTAs' tiles landed (even CTA's)
  uint64_t* empty = full + STAGES;      // [STAGES] MMAs have read them
  uint64_t* d_full = empty + STAGES;    // [BUFS] a product complete
  uint64_t* d_empty = d_full + BUFS;    // [BUFS] taken out by both CTAs (even CTA's)
  uint64_t* s_full = d_empty + BUFS;    // [2] a chunk's scales staged
  uint64_t* s_empty = s_full + 2;            // [2] used
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(s_empty + 2);
  float* s_x = reinterpret_cast<float*>(smem + C::OFF_S);
  float* s_w = reinterpret_cast<float*>(smem + C::OFF_SW);
  float* s_b = reinterpret_cast<float*>(smem + C::OFF_B);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = PAIR ? blockIdx.x & 1 : 0;
  const int kb = (a.K + 127) / 128, nt = (a.N + TN - 1) / TN;
  const int tiles = nt * ((a.M + TM - 1) / TM), first = blockIdx.x / CTAS, step = gridDim.x / CTAS;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < BUFS; ++i) mbar_init(&d_full[i], 1), mbar_init(&d_empty[i], 8 * CTAS);
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 2), mbar_init(&s_empty[i], 8);
    fence_barrier_init();
  }
  if (warp == 8 && lane == 0) {
    tma_map_prefetch(&tmW);
    tma_map_prefetch(&tmX);
  }
  if (warp == 9) {
    if (PAIR) tmem_get2(tmem_at, 512);
    else tmem_get(tmem_at, 512);
  }
  tc_before();
  if (PAIR) cluster_sync();
  else __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_at;
  grid_wait();
  grid_release();

  if (warp >= 8) {
    if (PAIR) regs_down<40>();
    if (warp == 8) {
      const uint32_t full_even = PAIR ? cluster_map(full, 0) : 0;
      bool ok = true;
      int i = 0;
      for (int t = first; t < tiles && ok; t += step) {
        const int m0 = t / nt * TM + rank * 128, n0 = t % nt * TN + rank * 128;
        for (int b = 0; b < kb; ++b, ++i) {
          const int s = i % STAGES;
          if (i >= STAGES && !mbar_wait_step(&empty[s], ((i / STAGES) - 1) & 1, &g_linear_status)) {
            for (int j = i - STAGES; j < i && rank == 0; ++j)
              mbar_wait(&full[j % STAGES], (j / STAGES) & 1, &g_linear_status);
            ok = false;
            break;
          }
          if (elect_one()) {
            if (rank == 0) mbar_expect_tx(&full[s], CTAS * ROWS_STAGE);
            uint8_t* at = smem + s * ROWS_STAGE;
            if (PAIR) {
              tma_tile_pair(at, &tmX, b * 128, m0, full_even + 8 * s);
              tma_tile_pair(at + FP8_W_TILE, &tmW, b * 128, n0, full_even + 8 * s);
            } else {
              tma_tile_2d(at, &tmX, b * 128, m0, &full[s]);
              tma_tile_2d(at + FP8_W_TILE, &tmW, b * 128, n0, &full[s]);
            }
          }
          __syncwarp();
        }
      }
      if (ok) mbar_wait_ring<STAGES>(empty, i, &g_linear_status);
    } else if (warp == 9 && rank == 0) {
      constexpr uint32_t idesc = idesc_e4m3(TM, TN);
      bool ok = true;
      int i = 0;
      for (int t = first; t < tiles && ok; t += step)
        for (int b = 0; b < kb; ++b, ++i) {
          const int s = i % STAGES, u = i % BUFS;
          if (!mbar_wait_step(&full[s], (i / STAGES) & 1, &g_linear_status) ||
              (i >= BUFS && !mbar_wait_step(&d_empty[u], ((i / BUFS) - 1) & 1, &g_linear_status))) {
            ok = false;
            break;
          }
          tc_after();
          if (elect_one()) {
            const uint64_t ad = k128_desc(smem + s * ROWS_STAGE), bd = k128_desc(smem + s * ROWS_STAGE + FP8_W_TILE);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (PAIR) mma_e4m3_pair(tmem + u * TN, ad + 2 * j, bd + 2 * j, idesc, j != 0);
              else mma_e4m3(tmem + u * TN, ad + 2 * j, bd + 2 * j, idesc, j != 0);
            }
            if (PAIR) {
              mma_done_pair(&d_full[u]);
              mma_done_pair(&empty[s]);
            } else {
              mma_done(&d_full[u]);
              mma_done(&empty[s]);
            }
          }
          __syncwarp();
        }
    } else if (warp >= 10) {
      const int r = (warp - 10) * 32 + lane;
      bool ok = true;
      int q = 0, tb = 0;
      for (int t = first; t < tiles && ok; t += step, tb = (tb + 1) & 3) {
        const int m0 = t / nt * TM + rank * 128, n0 = t % nt * TN;
        const float* x0 = a.xs + (long long)min(m0 + r, a.M - 1) * a.xs_stride;
        const float* x1 = a.xs + (long long)min(m0 + r + 64, a.M - 1) * a.xs_stride;
        // the right half's scales, where the tile has one
        const float* w = a.ws + (long long)(n0 / 128 + (PAIR && (lane & 1) && n0 + 128 < a.N ? 1 : 0)) * kb;
        for (int b0 = 0; b0 < kb; b0 += ROWS_CHUNK, ++q) {
          float v0[ROWS_CHUNK], v1[ROWS_CHUNK];
#pragma unroll
          for (int j = 0; j < ROWS_CHUNK; ++j) {
            const int b = min(b0 + j, kb - 1);
            v0[j] = __ldg(x0 + b), v1[j] = __ldg(x1 + b);
          }
          const float vw = __ldg(w + min(b0 + ((lane >> 1) & (ROWS_CHUNK - 1)), kb - 1));
          const int u = q & 1;
          if (q >= 2 && !mbar_wait_step(&s_empty[u], ((q >> 1) - 1) & 1, &g_linear_status)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int j = 0; j < ROWS_CHUNK; ++j) {
            s_x[(u * ROWS_CHUNK + j) * 128 + r] = v0[j];
            s_x[(u * ROWS_CHUNK + j) * 128 + r + 64] = v1[j];
          }
          if (warp == 10 && lane < 2 * ROWS_CHUNK) s_w[u * 2 * ROWS_CHUNK + lane] = vw;
          // a tile's bias lies there until its outputs are written: by then this
          // warp is at most three tiles further
          if (b0 == 0 && a.bias)
            for (int n = r; n < TN; n += 64) s_b[tb * 256 + n] = n0 + n < a.N ? __ldg(a.bias + n0 + n) : 0.f;
          __syncwarp();
          if (lane == 0) mbar_arrive1(&s_full[u]);
        }
      }
    }
  } else {
    if (PAIR) regs_up<232>();
    const uint32_t d_empty_even = PAIR ? cluster_map(d_empty, 0) : 0;
    const int quarter = warp & 3, half = warp >> 2;
    uint8_t* outs = smem + C::OFF_OUT + warp * (C::OUTS * 4096);
    int i = 0, q = 0, tb = 0, ob = 0;
    bool ok = true;
    const uint32_t d0 = tmem + ((uint32_t)(quarter * 32) << 16) + half * COLS;
    for (int t = first; t < tiles; t += step, tb = (tb + 1) & 3) {
      const int m = t / nt * TM + rank * 128 + quarter * 32 + lane, n0 = t % nt * TN + half * COLS;
      float acc[COLS];
#pragma unroll
      for (int n = 0; n < COLS; ++n) acc[n] = 0.f;
      uint32_t v[2][32];
      ok = mbar_wait_step(&d_full[i % BUFS], (i / BUFS) & 1, &g_linear_status);
      if (!ok) break;
      tc_after();
      tmem_load32(d0 + i % BUFS * TN, v[0]);
      for (int b = 0; b < kb; ++b, ++i) {
        const int sb = b % ROWS_CHUNK, su = q & 1;
        const bool chunk_end = sb == ROWS_CHUNK - 1 || b == kb - 1;
        if (sb == 0) ok = mbar_wait_step(&s_full[su], (q >> 1) & 1, &g_linear_status);
        if (!ok) break;
        const uint64_t ff =
            twice(s_x[(su * ROWS_CHUNK + sb) * 128 + quarter * 32 + lane] * s_w[(su * ROWS_CHUNK + sb) * 2 + half]);
        const uint32_t d = d0 + i % BUFS * TN;
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
          uint32_t *now = v[c / 32 & 1], *next = v[c / 32 & 1 ^ 1];
          tmem_wait32(now);
          if (c + 32 < COLS) {
            tmem_load32(d + c + 32, next);
          } else {
            tc_before();
            __syncwarp();
            if (lane == 0) {
              if (PAIR) mbar_arrive_cluster(d_empty_even + 8 * (i % BUFS));
              else mbar_arrive1(&d_empty[i % BUFS]);
              if (chunk_end) mbar_arrive1(&s_empty[su]);
            }
            q += chunk_end;
            if (b + 1 < kb) {
              ok = mbar_wait_step(&d_full[(i + 1) % BUFS], ((i + 1) / BUFS) & 1, &g_linear_status);
              tc_after();
              tmem_load32(d0 + (i + 1) % BUFS * TN, next);
            }
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) fma2(acc[c + j], acc[c + j + 1], now[j], now[j + 1], ff);
        }
      }
      if (!ok) break;
#pragma unroll
      for (int h = 0; h < COLS / 64; ++h) {
        const int c0 = n0 + 64 * h;
        if (c0 >= a.N) break;
        float* o64 = acc + 64 * h;
        if (a.bias) {
          const float4* b4 = reinterpret_cast<const float4*>(s_b + tb * 256 + half * COLS + 64 * h);
#pragma unroll
          for (int n = 0; n < 16; ++n) {
            const float4 bias = b4[n];
            o64[4 * n] += bias.x, o64[4 * n + 1] += bias.y, o64[4 * n + 2] += bias.z, o64[4 * n + 3] += bias.w;
          }
        }
        if (y_map) {
          constexpr int PER = OUT == DT_F32 ? 32 : 64;       // columns of a 128-byte tile row
#pragma unroll
          for (int c = 0; c < 64; c += PER) {
            uint4 o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (OUT == DT_F32) {
                o[j] = make_uint4(__float_as_uint(o64[c + 4 * j]), __float_as_uint(o64[c + 4 * j + 1]),
                                  __float_as_uint(o64[c + 4 * j + 2]), __float_as_uint(o64[c + 4 * j + 3]));
              } else {
                o[j] = make_uint4(pack_out<OUT>(o64[8 * j], o64[8 * j + 1]), pack_out<OUT>(o64[8 * j + 2], o64[8 * j + 3]),
                                  pack_out<OUT>(o64[8 * j + 4], o64[8 * j + 5]), pack_out<OUT>(o64[8 * j + 6], o64[8 * j + 7]));
              }
            }
            tma_store_read_wait<C::OUTS - 1>();      // lane 0 sent the tile that lay here
            __syncwarp();
            uint8_t* out = outs + ob;
            if (C::OUTS == 2) ob ^= 4096;
#pragma unroll
            for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(out + lane * 128 + ((j ^ (lane & 7)) << 4)) = o[j];
            fence_async_shared();
            __syncwarp();
            if (lane == 0 && c0 + c < a.N && m < a.M) tma_store_2d(&tmY, out, c0 + c, m);
          }
        } else if (m < a.M) {
#pragma unroll
          for (int n = 0; n < 64; ++n)
            if (c0 + n < a.N) store_out<OUT>(a.y, m * a.y_stride + c0 + n, o64[n]);
        }
      }
    }
    if (lane == 0) tma_store_wait();
  }
  tc_before();
  if (PAIR) cluster_sync();                  // the even CTA's barriers serve both to the end
  else __syncthreads();
  if (warp == 9) {
    if (PAIR) tmem_free2(tmem, 512);
    else tmem_free(tmem, 512);
  }
}

// ------------------------------------------------------------------ launches
static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const auto fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

int encode_fp8_map(CUtensorMap* m, const void* base, long long k, long long rows, long long stride, int box_rows,
                   int mats, long long mat_stride) {
  const auto fn = encode_fn();
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
  // Clusters of 2, 4 and 8 (others fill the GPU unevenly: 23 tiles of K 4096,
  // 4 CTAs a tile 5.7 us, 6 6.1, 7 6.5). Four CTAs a tile pay while all are
  // resident, eight only while each has an SM (23 tiles 6.4 us, 40 tiles of K
  // 2048 9.0 against 5.0; 16 tiles of K 4096 4.7 against 5.2).
  const long long n = (long long)tiles * cols;
  int split = 8 * n <= sms ? 8 : 4 * n <= 2 * sms ? 4 : 2 * n <= 2 * sms ? 2 : 1;
  while (split > kb) split /= 2;
  CUtensorMap tw, tx;
  if (encode_fp8_map(&tw, a.w, a.K, a.N, a.w_stride, 128, 0, 0) ||
      encode_fp8_map(&tx, a.x, a.K, a.M, a.x_stride, NT, 0, 0))
    return cudaErrorInvalidValue;
  auto kern = k_linear_few<NT, OUT>;
  cudaError_t e = allow_shared<k_linear_few<NT, OUT>>(Few<NT>::SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(split * tiles, cols);       // x alone goes beyond 65535
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

// y [M][N] as 32-row tiles of 128 bytes, swizzled; false where a tensor map
// cannot describe it (rows that do not start on 16-byte boundaries)
template <int OUT>
static bool encode_out_map(CUtensorMap* m, const LinearArgs& a) {
  constexpr int SZ = OUT == DT_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a.y) % 16 || a.y_stride * SZ % 16) return false;
  const auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)a.N, (cuuint64_t)a.M};
  const cuuint64_t strides[1] = {(cuuint64_t)a.y_stride * SZ};
  const cuuint32_t box[2] = {128 / SZ, 32};
  const cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType t = OUT == DT_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                : OUT == DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return fn(m, t, 2, a.y, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int OUT, bool PAIR>
static cudaError_t launch_rows(const LinearArgs& a, int sms, cudaStream_t s) {
  constexpr int CTAS = PAIR ? 2 : 1, T = 128 * CTAS;
  const long long tiles = (long long)((a.N + T - 1) / T) * ((a.M + T - 1) / T);
  CUtensorMap tw, tx, ty{};
  if (encode_fp8_map(&tw, a.w, a.K, a.N, a.w_stride, 128, 0, 0) ||
      encode_fp8_map(&tx, a.x, a.K, a.M, a.x_stride, 128, 0, 0))
    return cudaErrorInvalidValue;
  const int y_map = encode_out_map<OUT>(&ty, a);
  auto kern = k_linear_rows<OUT, PAIR>;
  cudaError_t e = allow_shared<k_linear_rows<OUT, PAIR>>(Rows<PAIR>::SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)std::min<long long>(tiles, sms / CTAS) * CTAS);
  cfg.blockDim = dim3(ROWS_THREADS);
  cfg.dynamicSmemBytes = Rows<PAIR>::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTAS, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, tw, tx, ty, y_map, a);
}

template <int OUT>
static cudaError_t launch_out(const LinearArgs& a, int sms, cudaStream_t s) {
  if (a.M <= 16) return launch_few<16, OUT>(a, sms, s);
  if (a.M <= 32) return launch_few<32, OUT>(a, sms, s);
  if (a.M <= 64) return launch_few<64, OUT>(a, sms, s);
  // Beyond 64 rows: the first kernel while its 128 x 64 tiles leave room to
  // cut a long K between CTAs, then single CTAs while their 128 x 128 tiles fit
  // the GPU at once, then pairs (us, in this order: M 128, N 2880, K 4096 12.0,
  // 16.6, 20.1; M 512, N 1024, K 4096 11.8, 16.2, 19.8; M 384, N 5120, K 2880
  // 20.4, 13.6, 16.4; M 512, N 5120, K 2880 35.8, 22.6, 16.7; M 128, N 2880, K
  // 1024 6.6, 6.1, 8.0, K 1536 7.5, 7.9, 9.8, K 512 5.8, 4.5, 6.3). Of 104
  // shapes, N 1024 to 5120, K 512 to 4096, M 96 to 4096, the one chosen is
  // within 6 % of the best but for N 1024, K 1024 (M 96 5.9 against 5.0).
  const long long rows = (a.N + 127) / 128;
  if (a.K > 1024 && 2 * rows * ((a.M + 63) / 64) <= sms) return launch_few<64, OUT>(a, sms, s);
  if (rows * ((a.M + 127) / 128) <= sms) return launch_rows<OUT, false>(a, sms, s);
  return launch_rows<OUT, true>(a, sms, s);
}

cudaError_t launch_linear_fp8(const LinearArgs& a, int out_dtype, int sms, cudaStream_t s) {
  if (out_dtype == DT_BF16) return launch_out<DT_BF16>(a, sms, s);
  if (out_dtype == DT_F16) return launch_out<DT_F16>(a, sms, s);
  return launch_out<DT_F32>(a, sms, s);
}

cudaError_t linear_fp8_status(int** at) { return cudaGetSymbolAddress(reinterpret_cast<void**>(at), g_linear_status); }

}  // namespace ms
