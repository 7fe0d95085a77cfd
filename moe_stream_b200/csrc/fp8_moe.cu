// A whole mixture-of-experts layer over resident e4m3 experts, for a few
// tokens.
//
//   logits = x router^T (+ bias), 32 bits
//   qwen3: softmax over all experts, the k largest (ties to the lower
//   index), renormalised on request; gpt-oss: the k largest logits, softmax
//   of them
//   (xq, xs) = quantise(x); g, u = gate, up products (+ biases)
//   act = silu(g) u, or with g <- min(g, 7), u <- clamp(u, -7, 7):
//         g sigmoid(1.702 g) (u + 1)
//   (hq, hs) = quantise(act); y = sum_j p_j (hq down^T + bias) (+ residual)
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "fp8.cuh"

namespace ms {

namespace {
__device__ __forceinline__ float code_value(uint8_t c) {
  __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
  return __half2float(__half(h));
}

struct Ws {               // workspace layout
  int* inds;              // [T, k]
  float* probs;           // [T, k]
  float* xv;              // [T, d] dequantised
  float* hv;              // [T * k, f] activations, then dequantised
};
__host__ __device__ inline size_t up16(size_t n) { return (n + 15) / 16 * 16; }
__host__ __device__ inline Ws split(uint8_t* w, int T, int d, int k) {
  Ws o;
  o.inds = reinterpret_cast<int*>(w);
  w += up16(4ull * T * k);
  o.probs = reinterpret_cast<float*>(w);
  w += up16(4ull * T * k);
  o.xv = reinterpret_cast<float*>(w);
  w += up16(4ull * T * d);
  o.hv = reinterpret_cast<float*>(w);
  return o;
}

// v[128 of row], by 128 threads: quantised in place
__device__ __forceinline__ float quantised(float v, float* red) {
  float m = fabsf(v);
#pragma unroll
  for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(MS_FULL, m, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = max_nan(max_nan(red[0], red[1]), max_nan(red[2], red[3]));
  float inv;
  const float s = group_scale(m, &inv);
  return code_value((uint8_t)e4m3x2(v * inv, 0.f)) * s;
}
}  // namespace

__global__ void __launch_bounds__(128) k_moe_route(MoeFp8Args a) {
  __shared__ float logit[512], red[4];
  const Ws w = split(a.ws, a.T, a.d, a.k);
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint16_t* x = a.x + (long long)t * a.d;
  for (int e = warp; e < a.E; e += 4) {
    float s = 0.f;
    for (int i = lane; i < a.d; i += 32) s = fmaf(bf2f(x[i]), bf2f(a.router[(long long)e * a.d + i]), s);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(MS_FULL, s, o);
    if (lane == 0) logit[e] = s + (a.router_bias ? a.router_bias[e] : 0.f);
  }
  for (int i0 = 0; i0 < a.d; i0 += 128) {
    const int i = i0 + threadIdx.x;
    const float v = quantised(i < a.d ? bf2f(x[i]) : 0.f, red);
    if (i < a.d) w.xv[(long long)t * a.d + i] = v;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float top = logit[0], all = 0.f, sel = 0.f;
    for (int e = 0; e < a.E; ++e) top = max_nan(top, logit[e]);
    for (int e = 0; e < a.E; ++e) all += expf(logit[e] - top);
    unsigned long long used[8] = {};
    for (int j = 0; j < a.k; ++j) {
      int best = -1;
      for (int e = 0; e < a.E; ++e)
        if (!(used[e >> 6] >> (e & 63) & 1) && (best < 0 || logit[e] > logit[best])) best = e;
      used[best >> 6] |= 1ull << (best & 63);
      w.inds[t * a.k + j] = best;
      const float p = expf(logit[best] - top);
      w.probs[t * a.k + j] = p;
      sel += p;
    }
    const float div = a.model == 1 || a.norm_topk ? sel : all;
    for (int j = 0; j < a.k; ++j) w.probs[t * a.k + j] /= div;
  }
}

__global__ void __launch_bounds__(128) k_moe_up(MoeFp8Args a) {
  __shared__ float red[4];
  const Ws w = split(a.ws, a.T, a.d, a.k);
  const int p = blockIdx.y, e = w.inds[p], n = blockIdx.x * 128 + threadIdx.x;
  const int kb = (a.d + 127) / 128, nb = (a.f + 127) / 128;
  const float* xv = w.xv + (long long)(p / a.k) * a.d;
  float g = 0.f, u = 0.f;
  if (n < a.f) {
    for (int b = 0; b < kb; ++b) {
      float pg = 0.f, pu = 0.f;
      for (int i = b * 128; i < min(a.d, (b + 1) * 128); ++i) {
        pg = fmaf(xv[i], code_value(a.gate.q[((long long)e * a.f + n) * a.d + i]), pg);
        pu = fmaf(xv[i], code_value(a.up.q[((long long)e * a.f + n) * a.d + i]), pu);
      }
      const long long s = ((long long)e * nb + n / 128) * kb + b;
      g = fmaf(pg, a.gate.s[s], g);
      u = fmaf(pu, a.up.s[s], u);
    }
    if (a.gate.bias) g += a.gate.bias[(long long)e * a.f + n];
    if (a.up.bias) u += a.up.bias[(long long)e * a.f + n];
    if (a.model == 1) {
      g = g > 7.f ? 7.f : g;
      u = u > 7.f ? 7.f : u < -7.f ? -7.f : u;
      g = g / (1.f + expf(-1.702f * g)) * (u + 1.f);
    } else {
      g = g / (1.f + expf(-g)) * u;
    }
  }
  g = quantised(g, red);
  if (n < a.f) w.hv[(long long)p * a.f + n] = g;
}

__global__ void __launch_bounds__(128) k_moe_down(MoeFp8Args a) {
  const Ws w = split(a.ws, a.T, a.d, a.k);
  const int t = blockIdx.y, n = blockIdx.x * 128 + threadIdx.x;
  const int kb = (a.f + 127) / 128, nb = (a.d + 127) / 128;
  if (n >= a.d) return;
  float y = 0.f;
  for (int j = 0; j < a.k; ++j) {
    const int p = t * a.k + j, e = w.inds[p];
    const float* hv = w.hv + (long long)p * a.f;
    float o = 0.f;
    for (int b = 0; b < kb; ++b) {
      float po = 0.f;
      for (int i = b * 128; i < min(a.f, (b + 1) * 128); ++i)
        po = fmaf(hv[i], code_value(a.down.q[((long long)e * a.d + n) * a.f + i]), po);
      o = fmaf(po, a.down.s[((long long)e * nb + n / 128) * kb + b], o);
    }
    if (a.down.bias) o += a.down.bias[(long long)e * a.d + n];
    y = fmaf(w.probs[p], o, y);
  }
  if (a.res) y += bf2f(a.res[(long long)t * a.d + n]);
  a.y[(long long)t * a.d + n] = f2bf(y);
}

size_t moe_fp8_workspace(int T, int d, int f, int E, int k) {
  (void)E;
  return 2 * up16(4ull * T * k) + up16(4ull * T * d) + up16(4ull * T * k * f);
}

cudaError_t launch_moe_fp8(const MoeFp8Args& a, int sms, cudaStream_t s) {
  (void)sms;
  k_moe_route<<<a.T, 128, 0, s>>>(a);
  k_moe_up<<<dim3((a.f + 127) / 128, a.T * a.k), 128, 0, s>>>(a);
  k_moe_down<<<dim3((a.d + 127) / 128, a.T), 128, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace ms
