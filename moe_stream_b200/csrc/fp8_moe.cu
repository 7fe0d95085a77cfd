// A whole mixture-of-experts layer over resident e4m3 experts, for a few
// tokens, in two kernels.
//
//   logits = x router^T (+ bias), 32 bits
//   qwen3: softmax over all experts, the k largest (ties to the lower
//   index), renormalised on request; gpt-oss: the k largest logits, softmax
//   of them
//   (xq, xs) = quantise(x); g, u = gate, up products (+ biases)
//   act = silu(g) u, or with g <- min(g, 7), u <- clamp(u, -7, 7):
//         g sigmoid(1.702 g) (u + 1)
//   (hq, hs) = quantise(act); y = sum_j p_j (hq down^T + bias) (+ residual)
//
// Bound by memory: every routed expert's codes once. k_moe_route makes the
// logits and x's codes; k_moe_experts streams the experts. Each of its CTAs
// (one per SM) works out the routing for itself, which is less than a trip
// through memory, then takes tasks off one counter:
//
//   up       128 features of d_ff of one expert, gate and up rows, a range of
//            the blocks of d (all of them where there are tiles enough; else
//            the sums meet in the workspace, at the CTA that brings a tile's
//            last one); then the activation, the quantised 128 features (they
//            are one block of the down product) and the tile's flag
//   down     128 features of d of one expert, a range of the blocks of f, each
//            of which it may load once its flag is up
//   combine  128 features of four tokens: the weighted sum over experts
//
// Tasks are numbered in this order and a task waits only for lower numbers,
// which running CTAs hold, so the kernel ends however few of its CTAs run at a
// time (another call may hold the other SMs). Sums are added in a fixed order:
// results do not depend on timing.
//
// Products run on the tensor cores with the weight as operand A (128 rows, the
// TMEM lanes) and all the tokens (up) or the expert's rows (down) as up to 64
// columns, so no weight passes through registers. One pipeline serves both: a
// step is one 128 x 128 weight tile times one activation tile.
// Warps 0-3 take products out of TMEM and do the rest of a task, warp 4 loads
// weights and takes tasks, warp 5 issues MMAs, warp 6 loads activations and
// warp 7 the scales; these two wait for the flags, so that weights are in
// flight meanwhile.
#include <algorithm>

#include <cuda_fp16.h>

#include "fp8_mma.cuh"

namespace ms {

// first failure of a bounded wait in this file's kernels (ms_fp8_status)
static __device__ int g_moe_status;

namespace {

constexpr int MOE_FAC = 16;            // blocks of a task at most
constexpr int MOE_SPLIT = 8;           // ranges of a tile's blocks at most
constexpr int COMBINE_T = 4;           // tokens of a combine task, one per warp

__host__ __device__ inline int blocks128(int n) { return (n + 127) / 128; }
inline long long up16(long long n) { return (n + 15) / 16 * 16; }

// Ranges that a tile's blocks may be cut into: enough for a task's scales to
// fit and for few tiles to fill the GPU, while the sums in the workspace stay
// below 64 MB a matrix.
inline int split_cap(long long pairs, int n, int kb) {
  const long long fit = (64ll << 20) / (pairs * n * 4);
  const int least = (kb + MOE_FAC - 1) / MOE_FAC;
  return std::max(least, (int)std::min<long long>(std::max<long long>(fit, 2), MOE_SPLIT));
}

}  // namespace

struct MoeWs {            // workspace layout
  float* logits;          // [T, E]
  uint8_t* xq;            // [T, d]
  float* xs;              // [T, blocks of d]
  uint8_t* hq;            // [P, f]  rows by expert, then token
  float* hs;              // [P, blocks of f]
  float* up_part;         // [S1][2][P][f]
  float* dn_part;         // [S2][P][d]
  unsigned* next;         // next task; this and the following are zeroed by k_moe_route
  unsigned* brought;      // [up tile] ranges brought
  unsigned* flag;         // [up tile] its block is quantised
  unsigned* dn_done;      // [tile of d] down tasks done
  int counters;           // words from next on
  int cap1, cap2;         // split_cap of the up and down tiles
};

static long long layout_ws(uint8_t* w, int T, int d, int f, int E, int k, MoeWs* o) {
  const long long P = (long long)T * k;
  const int tiles = (int)std::min<long long>(P, E) * blocks128(f);
  uint8_t* const w0 = w;
  o->cap1 = split_cap(2 * P, f, blocks128(d)), o->cap2 = split_cap(P, d, blocks128(f));
  o->xq = w, w += up16((long long)T * d);
  o->hq = w, w += up16(P * f);
  o->logits = reinterpret_cast<float*>(w), w += up16(4ll * T * E);
  o->xs = reinterpret_cast<float*>(w), w += up16(4ll * T * blocks128(d));
  o->hs = reinterpret_cast<float*>(w), w += up16(4 * P * blocks128(f));
  o->up_part = reinterpret_cast<float*>(w), w += 8ll * o->cap1 * P * f;
  o->dn_part = reinterpret_cast<float*>(w), w += 4ll * o->cap2 * P * d;
  o->next = reinterpret_cast<unsigned*>(w);
  o->brought = o->next + 1, o->flag = o->brought + tiles, o->dn_done = o->flag + tiles;
  o->counters = 1 + 2 * tiles + blocks128(d);
  w += up16(4ll * o->counters);
  return w - w0;
}

// --------------------------------------------------------------------- route
// A warp per expert and TG tokens; the CTAs after the experts' quantise x, a
// warp per token, and zero the counters.
template <int TG>
__global__ void __launch_bounds__(256) k_moe_route(MoeFp8Args a, MoeWs w) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = a.d / 8, ex = (a.E + 7) / 8;
  grid_wait();
  grid_release();
  if ((int)blockIdx.x < ex) {
    const int e = blockIdx.x * 8 + warp, t0 = blockIdx.y * TG;
    if (e >= a.E) return;
    const uint4* wr = reinterpret_cast<const uint4*>(a.router + (long long)e * a.d);
    float acc[TG];
#pragma unroll
    for (int t = 0; t < TG; ++t) acc[t] = 0.f;
#pragma unroll(TG == 1 ? 8 : 2)
    for (int c = lane; c < chunks; c += 32) {
      const uint4 v = __ldg(wr + c);
      const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int t = 0; t < TG; ++t) {
        const uint4 u = *(reinterpret_cast<const uint4*>(a.x + (long long)min(t0 + t, a.T - 1) * a.d) + c);
        const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[t] = fmaf(__uint_as_float(vw[i] << 16), __uint_as_float(uw[i] << 16), acc[t]);
          acc[t] = fmaf(__uint_as_float(vw[i] & 0xffff0000u), __uint_as_float(uw[i] & 0xffff0000u), acc[t]);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < TG; ++t) {
#pragma unroll
      for (int o = 16; o; o >>= 1) acc[t] += __shfl_xor_sync(MS_FULL, acc[t], o);
      if (lane == 0 && t0 + t < a.T)
        w.logits[(t0 + t) * a.E + e] = acc[t] + (a.router_bias ? a.router_bias[e] : 0.f);
    }
    return;
  }
  const int q = blockIdx.x - ex, nq = gridDim.x - ex;          // q-th of the quantising CTAs of this row
  if (blockIdx.y == 0 && q == 0)
    for (int i = threadIdx.x; i < w.counters; i += 256) w.next[i] = 0;
  const int groups = blocks128(a.d);
  // a half-warp per group of 128 features
  for (int i = (blockIdx.y * nq + q) * 16 + warp * 2 + (lane >> 4); i < a.T * groups; i += gridDim.y * nq * 16) {
    const int t = i / groups, c = (i - t * groups) * 16 + (lane & 15);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (c < chunks) v = *(reinterpret_cast<const uint4*>(a.x + (long long)t * a.d) + c);
    const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      m = max_nan(m, max_nan(fabsf(__uint_as_float(vw[j] << 16)), fabsf(__uint_as_float(vw[j] & 0xffff0000u))));
    const unsigned lanes = 0xffffu << (lane & 16);
#pragma unroll
    for (int o = 8; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(lanes, m, o));
    float inv;
    const float s = group_scale(m, &inv);
    if ((lane & 15) == 0) w.xs[i] = s;
    uint32_t r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      r[j] = e4m3x2(__uint_as_float(vw[j] << 16) * inv, __uint_as_float(vw[j] & 0xffff0000u) * inv);
    if (c < chunks)
      *(reinterpret_cast<uint2*>(w.xq + (long long)t * a.d) + c) = make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
  }
}

// ------------------------------------------------------------------- experts
template <int NT> struct Moe {
  static constexpr int STAGE = FP8_W_TILE + NT * 128;
  static constexpr int STAGES = NT <= 16 ? 10 : NT <= 32 ? 9 : 7;
  static constexpr int BUFS = 8;
  static constexpr int OFF_FAC = STAGES * STAGE;                     // [2][FAC][2][NT] scale products
  static constexpr int OFF_PROB = OFF_FAC + 2 * MOE_FAC * 2 * NT * 4;   // [NT][32]
  static constexpr int OFF_IND = OFF_PROB + NT * 32 * 4;             // [NT][32] bytes
  static constexpr int OFF_MASK = OFF_IND + NT * 32;                 // [256] tokens of an expert, 64 bits
  static constexpr int OFF_START = OFF_MASK + 256 * 8;               // [256] its first row
  static constexpr int OFF_GROUP = OFF_START + 256 * 4;              // [256] experts that are routed to, ascending
  static constexpr int OFF_RED = OFF_GROUP + 256;                    // [NT][4] maxima, then four words
  static constexpr int OFF_TASK = OFF_RED + NT * 16 + 16;            // [4] tasks
  static constexpr int OFF_BAR = OFF_TASK + 4 * 32;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
  static_assert(SMEM <= 232448 && SMEM > 232448 - 77824, "alone on its SM");
  static_assert(STAGE % 1024 == 0 && BUFS * NT <= 512, "tile alignment, TMEM columns");
};

struct __align__(32) Task {
  int kind;               // 0 up, 1 down, 2 combine, 3 none left
  int g, tile, s, b0, b1; // group, feature tile, range and its blocks (combine: s the four tokens)
};

struct Shape {            // what the tasks are
  int G, FT, DT, KB1, KB2, S1, S2, n_up, n_dn, n_co;
  __device__ __forceinline__ Task task(unsigned id) const {
    Task t;
    if (id < (unsigned)n_up) {
      t.kind = 0;
      t.s = id % S1;
      const int v = id / S1;
      t.tile = v % FT, t.g = v / FT;
      t.b0 = KB1 * t.s / S1, t.b1 = KB1 * (t.s + 1) / S1;
    } else if (id < (unsigned)(n_up + n_dn)) {
      t.kind = 1;
      const int i = id - n_up;
      t.s = i % S2;
      const int v = i / S2;
      t.tile = v % DT, t.g = v / DT;
      t.b0 = KB2 * t.s / S2, t.b1 = KB2 * (t.s + 1) / S2;
    } else if (id < (unsigned)(n_up + n_dn + n_co)) {
      const int i = id - n_up - n_dn;
      t.kind = 2, t.g = 0, t.tile = i % DT, t.s = i / DT, t.b0 = t.b1 = 0;
    } else {
      t.kind = 3, t.g = t.tile = t.s = t.b0 = t.b1 = 0;
    }
    return t;
  }
};

// Ranges for n tiles of kb blocks on `ctas` CTAs, by a warp (a number per
// lane): the least (rounds of tasks, half a round for the ragged end) x
// (blocks of a task, half a block for its end and `join` for sums that have to
// meet). In blocks: a Qwen3 up tile's join was about two of its blocks long.
__device__ __forceinline__ int choose_split(int n, int kb, int ctas, int cap, float join) {
  const int s = (threadIdx.x & 31) + 1;
  float rounds = (float)(n * s) / (float)ctas;
  rounds = rounds <= 1.f ? 1.f : rounds + 0.5f;
  const float cost = rounds * ((float)((kb + s - 1) / s) + 0.5f + (s > 1 ? join : 0.f));
  const bool can = s >= (kb + MOE_FAC - 1) / MOE_FAC && s <= cap && s <= kb;
  const unsigned key = can ? __float_as_uint(cost) : 0x7f800000u;
  const unsigned least = __reduce_min_sync(MS_FULL, key);
  return __ffs(__ballot_sync(MS_FULL, key == least));
}

__device__ __forceinline__ unsigned ld_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// counts, after everything that this CTA wrote before its last barrier
__device__ __forceinline__ void red_release(unsigned* p) {
  asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p) : "memory");
}
__device__ __forceinline__ unsigned add_acq_rel(unsigned* p) {
  unsigned v;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(MS_FULL, v, o));
  return v;
}
__device__ __forceinline__ float activate(int model, float g, float u) {
  if (model == 1) {
    g = g > 7.f ? 7.f : g;
    u = u > 7.f ? 7.f : u < -7.f ? -7.f : u;
    return g / (1.f + expf(-1.702f * g)) * (u + 1.f);
  }
  return g / (1.f + expf(-g)) * u;
}
// code of feature f of a row whose four warps' maxima are max4; thread 0 the scale
__device__ __forceinline__ void put_code(const MoeWs& w, int f_all, int f, int tid, int tile, int tiles, long long row,
                                         float h, const float* max4) {
  const float4 m = *reinterpret_cast<const float4*>(max4);
  float inv;
  const float s = group_scale(max_nan(max_nan(m.x, m.y), max_nan(m.z, m.w)), &inv);
  if (f < f_all) w.hq[row * f_all + f] = (uint8_t)e4m3x2(h * inv, 0.f);
  if (tid == 0) w.hs[row * tiles + tile] = s;
}
__device__ __forceinline__ void fence_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }

// Waits until *p >= want, a second at most.
__device__ __forceinline__ bool wait_count(const unsigned* p, unsigned want) {
  if (ld_acquire(p) >= want) return true;
  const unsigned long long t0 = global_ns();
  for (unsigned i = 0; i < MBAR_SPIN_LIMIT; ++i) {
    if (ld_acquire(p) >= want) return true;
    if ((i & 63) == 63 && (global_ns() - t0 > MBAR_WAIT_NS || timed_out(&g_moe_status))) break;
  }
  atomicCAS(&g_moe_status, 0, ST_E_TIMEOUT);
  return false;
}

struct MoeMaps {
  CUtensorMap gate, up, down, x, h, h16;
};

template <int NT>
__global__ void __launch_bounds__(256, 1)
    k_moe_experts(const __grid_constant__ MoeMaps maps, const __grid_constant__ MoeFp8Args a,
                  const __grid_constant__ MoeWs w) {
  using C = Moe<NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_fac = reinterpret_cast<float*>(smem + C::OFF_FAC);
  float* s_prob = reinterpret_cast<float*>(smem + C::OFF_PROB);
  uint8_t* s_ind = smem + C::OFF_IND;
  unsigned long long* s_mask = reinterpret_cast<unsigned long long*>(smem + C::OFF_MASK);
  int* s_start = reinterpret_cast<int*>(smem + C::OFF_START);
  uint8_t* s_group = smem + C::OFF_GROUP;
  float* s_red = reinterpret_cast<float*>(smem + C::OFF_RED);
  volatile int* s_word = reinterpret_cast<volatile int*>(s_red + NT * 4); // last, groups, S1, S2
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);        // [STAGES] both tiles landed
  uint64_t* empty = full + C::STAGES;                                     // [STAGES] read by the MMAs
  uint64_t* d_full = empty + C::STAGES;                                   // [BUFS] a product complete
  uint64_t* d_empty = d_full + C::BUFS;                                   // [BUFS] taken out
  uint64_t* f_full = d_empty + C::BUFS;                                   // [2] a task's scales there
  uint64_t* f_empty = f_full + 2;                                         // [2] used
  uint64_t* t_full = f_empty + 2;                                         // [4] a task taken
  uint64_t* t_empty = t_full + 4;                                         // [4] done by all roles
  Task* s_task = reinterpret_cast<Task*>(smem + C::OFF_TASK);             // [4]
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(t_empty + 4);
  int* const status = &g_moe_status;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int P = a.T * a.k;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) mbar_init(&full[i], 2), mbar_init(&empty[i], 1);
    for (int i = 0; i < C::BUFS; ++i) mbar_init(&d_full[i], 1), mbar_init(&d_empty[i], 4);
    for (int i = 0; i < 2; ++i) mbar_init(&f_full[i], 1), mbar_init(&f_empty[i], 4);
    for (int i = 0; i < 4; ++i) mbar_init(&t_full[i], 1), mbar_init(&t_empty[i], 7);
    fence_barrier_init();
  }
  for (int e = threadIdx.x; e < 256; e += 256) s_mask[e] = 0;
  if (warp == 5) tmem_get(tmem_at, 512);
  if (warp == 4 && lane < 6) tma_map_prefetch(reinterpret_cast<const CUtensorMap*>(&maps) + lane);
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_at;
  grid_wait();

  unsigned first_task = 0;
  if (warp == 4 && lane == 0) first_task = atomicAdd(w.next, 1u);    // back by the time it can be read

  // ---- the routing, a warp per token
  for (int t = warp; t < a.T; t += 8) {
    uint32_t key[8];                        // ordered like the logits; a NaN is below all
    float v[8];
    bool nan = false;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = lane + 32 * i;
      v[i] = e < a.E ? __ldcg(w.logits + t * a.E + e) + 0.f : 0.f;       // -0 is 0
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = __float_as_uint(v[i]);
      nan |= v[i] != v[i];
      key[i] = lane + 32 * i < a.E ? (v[i] != v[i] ? 1u : b ^ ((uint32_t)((int)b >> 31) | 0x80000000u)) : 0u;
      top = max(top, key[i]);
    }
    top = __reduce_max_sync(MS_FULL, top);
    const uint32_t top_bits = top & 0x80000000u ? top ^ 0x80000000u : ~top;
    const float m = __any_sync(MS_FULL, nan) ? __uint_as_float(0x7fc00000u) : __uint_as_float(top_bits);
    uint32_t mine_key = 0;                  // lane j: the j-th choice
    int mine = 0;
    float all = 0.f;
    if (a.model == 0 && !a.norm_topk) {
#pragma unroll
      for (int i = 0; i < 8; ++i) all += lane + 32 * i < a.E ? expf(v[i] - m) : 0.f;
#pragma unroll
      for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(MS_FULL, all, o);
    }
    for (int j = 0; j < a.k; ++j) {
      const uint32_t b0 = max(max(key[0], key[1]), max(key[2], key[3]));
      const uint32_t b1 = max(max(key[4], key[5]), max(key[6], key[7]));
      const uint32_t best = __reduce_max_sync(MS_FULL, max(b0, b1));
      int e = 1 << 20;
#pragma unroll
      for (int i = 7; i >= 0; --i)
        if (key[i] == best) e = lane + 32 * i;
      const int first = __reduce_min_sync(MS_FULL, e);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (lane + 32 * i == first) key[i] = 0;
      if (lane == j) mine = first, mine_key = best;
    }
    const float l = __uint_as_float(mine_key & 0x80000000u ? mine_key ^ 0x80000000u : ~mine_key);
    float p = lane < a.k ? expf(l - m) : 0.f, sel = p;
#pragma unroll
    for (int o = 16; o; o >>= 1) sel += __shfl_xor_sync(MS_FULL, sel, o);
    if (lane < a.k) {
      s_prob[t * 32 + lane] = p / (a.model == 1 || a.norm_topk ? sel : all);
      s_ind[t * 32 + lane] = (uint8_t)mine;
      atomicOr(&s_mask[mine], 1ull << t);
    }
  }
  __syncthreads();
  if (warp == 0) {                          // groups in expert order and their first rows
    int G = 0, row = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
      const int e = e0 + lane, n = e < a.E ? __popcll(s_mask[e]) : 0;
      const unsigned has = __ballot_sync(MS_FULL, n > 0);
      if (!has) continue;
      int at = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(MS_FULL, at, o);
        if (lane >= o) at += u;
      }
      if (n > 0) {
        s_group[G + __popc(has & ((1u << lane) - 1))] = (uint8_t)e;
        s_start[e] = row + at - n;
      }
      G += __popc(has);
      row += __shfl_sync(MS_FULL, at, 31);
    }
    const int s1 = choose_split(G * blocks128(a.f), blocks128(a.d), gridDim.x, w.cap1, 2.f);
    const int s2 = choose_split(G * blocks128(a.d), blocks128(a.f), gridDim.x, w.cap2, 0.5f);
    if (lane == 0) s_word[1] = G, s_word[2] = s1, s_word[3] = s2;
  }
  __syncthreads();
  Shape sh;
  sh.G = s_word[1], sh.S1 = s_word[2], sh.S2 = s_word[3];
  sh.FT = blocks128(a.f), sh.DT = blocks128(a.d), sh.KB1 = sh.DT, sh.KB2 = sh.FT;
  sh.n_up = sh.G * sh.FT * sh.S1, sh.n_dn = sh.G * sh.DT * sh.S2;
  sh.n_co = sh.DT * ((a.T + COMBINE_T - 1) / COMBINE_T);

  if (warp == 4) {
    // ---- tasks and weight tiles
    bool ok = true;
    int i = 0;
    for (int n = 0; ok; ++n) {
      if (n >= 4) ok = mbar_wait_step(&t_empty[n & 3], ((n >> 2) - 1) & 1, status);
      unsigned id = first_task;
      if (n > 0 && lane == 0) id = ok ? atomicAdd(w.next, 1u) : 0xffffffffu;
      id = __shfl_sync(MS_FULL, id, 0);
      const Task t = sh.task(id);
      if (lane == 0) {
        s_task[n & 3] = t;
        mbar_arrive1(&t_full[n & 3]);
      }
      if (t.kind == 3) break;
      if (t.kind == 2) {                     // one at a time, so that other CTAs take the next
        ok = mbar_wait_step(&t_empty[n & 3], (n >> 2) & 1, status);
        continue;
      }
      const int e = s_group[t.g];
      const int per = t.kind == 0 ? 2 : 1;
      for (int b = t.b0; b < t.b1 && ok; ++b)
        for (int h = 0; h < per; ++h, ++i) {
          const int s = i % C::STAGES;
          if (i >= C::STAGES && !mbar_wait_step(&empty[s], ((i / C::STAGES) - 1) & 1, status)) {
            // copies in flight land before the CTA ends
            for (int j = i - C::STAGES; j < i && mbar_wait(&full[j % C::STAGES], (j / C::STAGES) & 1, status);) ++j;
            ok = false;
            break;
          }
          if (elect_one()) {
            mbar_expect_tx(&full[s], FP8_W_TILE);
            tma_tile_3d(smem + s * C::STAGE, t.kind == 1 ? &maps.down : h ? &maps.up : &maps.gate, b * 128,
                        t.tile * 128, e, &full[s]);
          }
          __syncwarp();
        }
    }
  } else if (warp == 5) {
    // ---- MMAs
    bool ok = true;
    int i = 0;
    for (int n = 0; ok; ++n) {
      if (!mbar_wait_step(&t_full[n & 3], (n >> 2) & 1, status)) break;
      const Task t = s_task[n & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive1(&t_empty[n & 3]);
      if (t.kind == 3) break;
      if (t.kind == 2) continue;
      const bool few = NT > 16 && t.kind == 1 && __popcll(s_mask[s_group[t.g]]) <= 16;
      const uint32_t idesc = few ? idesc_e4m3(128, 16) : idesc_e4m3(128, NT);
      const int steps = (t.b1 - t.b0) * (t.kind == 0 ? 2 : 1);
      for (int j = 0; j < steps; ++j, ++i) {
        const int s = i % C::STAGES, u = i % C::BUFS;
        if (!mbar_wait_step(&full[s], (i / C::STAGES) & 1, status) ||
            (i >= C::BUFS && !mbar_wait_step(&d_empty[u], ((i / C::BUFS) - 1) & 1, status))) {
          ok = false;
          break;
        }
        tc_after();
        if (elect_one()) {
          const uint64_t ad = k128_desc(smem + s * C::STAGE), bd = k128_desc(smem + s * C::STAGE + FP8_W_TILE);
#pragma unroll
          for (int q = 0; q < 4; ++q) mma_e4m3(tmem + u * NT, ad + 2 * q, bd + 2 * q, idesc, q != 0);
          mma_done(&empty[s]);
          mma_done(&d_full[u]);
        }
        __syncwarp();
      }
    }
  } else if (warp == 6) {
    // ---- activation tiles
    bool ok = true;
    int i = 0;
    for (int n = 0; ok; ++n) {
      if (!mbar_wait_step(&t_full[n & 3], (n >> 2) & 1, status)) break;
      const Task t = s_task[n & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive1(&t_empty[n & 3]);
      if (t.kind == 3) break;
      if (t.kind == 2) continue;
      const int e = s_group[t.g], rows = __popcll(s_mask[e]), start = s_start[e], nb = t.b1 - t.b0;
      if (t.kind == 1) {
        for (int b = t.b0 + lane; b < t.b1; b += 32) wait_count(w.flag + t.g * sh.FT + b, 1);
        __syncwarp();
        fence_async_all();
      }
      const bool few = NT > 16 && t.kind == 1 && rows <= 16;
      const int steps = nb * (t.kind == 0 ? 2 : 1);
      for (int j = 0; j < steps; ++j, ++i) {
        const int s = i % C::STAGES;
        if (i >= C::STAGES && !mbar_wait_step(&empty[s], ((i / C::STAGES) - 1) & 1, status)) {
          ok = false;
          break;
        }
        const int b = t.b0 + (t.kind == 0 ? j >> 1 : j);
        if (elect_one()) {
          mbar_expect_tx(&full[s], few ? 16 * 128 : NT * 128);
          tma_tile_2d(smem + s * C::STAGE + FP8_W_TILE, t.kind == 0 ? &maps.x : few ? &maps.h16 : &maps.h, b * 128,
                      t.kind == 0 ? 0 : start, &full[s]);
        }
        __syncwarp();
      }
    }
  } else if (warp == 7) {
    // ---- products of the activations' and the weights' scales, a task ahead
    bool ok = true;
    int c = 0;
    for (int n = 0; ok; ++n) {
      if (!mbar_wait_step(&t_full[n & 3], (n >> 2) & 1, status)) break;
      const Task t = s_task[n & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive1(&t_empty[n & 3]);
      if (t.kind == 3) break;
      if (t.kind == 2) continue;
      const int e = s_group[t.g], rows = __popcll(s_mask[e]), start = s_start[e], nb = t.b1 - t.b0;
      // a lane keeps to one block (16 of them, two columns at a time)
      const int b = t.b0 + min(lane & 15, nb - 1), wb = lane & 15, r0 = lane >> 4;
      const int u = c & 1;
      float* fac = s_fac + u * (MOE_FAC * 2 * NT) + wb * 2 * NT;
      if (t.kind == 0) {
        const long long at = ((long long)e * sh.FT + t.tile) * sh.KB1 + b;
        const float wg = __ldg(a.gate.s + at), wu = __ldg(a.up.s + at);
        if (c >= 2) ok = mbar_wait_step(&f_empty[u], ((c >> 1) - 1) & 1, status);
#pragma unroll 8
        for (int r = r0; r < a.T; r += 2) {
          const float x = __ldcg(w.xs + r * sh.KB1 + b);
          if (wb < nb) fac[r] = x * wg, fac[NT + r] = x * wu;
        }
      } else {
        const float wd = __ldg(a.down.s + ((long long)e * sh.DT + t.tile) * sh.KB2 + b);
        wait_count(w.flag + t.g * sh.FT + b, 1);
        __syncwarp();
        if (c >= 2) ok = mbar_wait_step(&f_empty[u], ((c >> 1) - 1) & 1, status);
#pragma unroll 8
        for (int r = r0; r < rows; r += 2) {
          const float x = __ldcg(w.hs + (long long)(start + r) * sh.KB2 + b);
          if (wb < nb) fac[r] = x * wd;
        }
      }
      ++c;
      __syncwarp();
      if (lane == 0) mbar_arrive1(&f_full[u]);
    }
  } else if (warp < 4) {
    // ---- products out of TMEM, and what follows them
    bool ok = true;
    int i = 0, c = 0;
    const int tid = threadIdx.x;
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    float acc[2][NT];
    for (int n = 0; ok; ++n) {
      if (!mbar_wait_step(&t_full[n & 3], (n >> 2) & 1, status)) break;
      const Task t = s_task[n & 3];
      __syncwarp();
      if (t.kind != 2 && lane == 0) mbar_arrive1(&t_empty[n & 3]);
      if (t.kind == 3) break;
      if (t.kind == 2) {
        // y of four tokens, one per warp: rows in the order of the token's
        // choices, ranges in order
        if (tid == 0) wait_count(w.dn_done + t.tile, (unsigned)(sh.G * sh.S2));
        named_bar(1, 128);
        const int f = t.tile * 128 + lane * 4, tok = t.s * COMBINE_T + warp;
        if (f < a.d && tok < a.T) {
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          const unsigned long long below = (1ull << tok) - 1;
          for (int j0 = 0; j0 < a.k; j0 += 8) {
            float4 o[8];
            const float* part[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int e = s_ind[tok * 32 + min(j0 + j, a.k - 1)];
              part[j] = w.dn_part + (long long)(s_start[e] + __popcll(s_mask[e] & below)) * a.d + f;
              o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            for (int s = 0; s < sh.S2; ++s) {
              float4 u[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) u[j] = __ldcg(reinterpret_cast<const float4*>(part[j] + s * (long long)P * a.d));
#pragma unroll
              for (int j = 0; j < 8; ++j) o[j].x += u[j].x, o[j].y += u[j].y, o[j].z += u[j].z, o[j].w += u[j].w;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (j0 + j < a.k) {
                const float p = s_prob[tok * 32 + j0 + j];
                if (a.down.bias) {
                  const float* b = a.down.bias + (long long)s_ind[tok * 32 + j0 + j] * a.d + f;
                  o[j].x += __ldg(b), o[j].y += __ldg(b + 1), o[j].z += __ldg(b + 2), o[j].w += __ldg(b + 3);
                }
                y.x = fmaf(p, o[j].x, y.x), y.y = fmaf(p, o[j].y, y.y);
                y.z = fmaf(p, o[j].z, y.z), y.w = fmaf(p, o[j].w, y.w);
              }
          }
          const long long at = (long long)tok * a.d + f;
          if (a.res) {
            const uint2 r = *reinterpret_cast<const uint2*>(a.res + at);
            y.x += __uint_as_float(r.x << 16), y.y += __uint_as_float(r.x & 0xffff0000u);
            y.z += __uint_as_float(r.y << 16), y.w += __uint_as_float(r.y & 0xffff0000u);
          }
          *reinterpret_cast<uint2*>(a.y + at) =
              make_uint2((uint32_t)f2bf(y.x) | (uint32_t)f2bf(y.y) << 16, (uint32_t)f2bf(y.z) | (uint32_t)f2bf(y.w) << 16);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive1(&t_empty[n & 3]);
        continue;
      }
      const int e = s_group[t.g], start = s_start[e];
      const unsigned long long mask = s_mask[e];
      const int rows = __popcll(mask);
      const int cols = t.kind == 0 ? a.T : rows;
      const float* fac = s_fac + (c & 1) * (MOE_FAC * 2 * NT);
      ok = mbar_wait_step(&f_full[c & 1], (c >> 1) & 1, status);
#pragma unroll
      for (int m = 0; m < NT; ++m) acc[0][m] = acc[1][m] = 0.f;
      auto take = [&](float* sum, const float* f) {
        const int u = i % C::BUFS;
        if (!mbar_wait_step(&d_full[u], (i / C::BUFS) & 1, status)) return false;
        tc_after();
#pragma unroll
        for (int m = 0; m < NT; m += 16) {
          if (m >= cols) break;
          uint32_t v[16];
          tmem_load16(lanes + u * NT + m, v);
          tmem_wait16(v);
          const float4* f4 = reinterpret_cast<const float4*>(f + m);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4 x = f4[q];
            sum[m + 4 * q] = fmaf(__uint_as_float(v[4 * q]), x.x, sum[m + 4 * q]);
            sum[m + 4 * q + 1] = fmaf(__uint_as_float(v[4 * q + 1]), x.y, sum[m + 4 * q + 1]);
            sum[m + 4 * q + 2] = fmaf(__uint_as_float(v[4 * q + 2]), x.z, sum[m + 4 * q + 2]);
            sum[m + 4 * q + 3] = fmaf(__uint_as_float(v[4 * q + 3]), x.w, sum[m + 4 * q + 3]);
          }
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive1(&d_empty[u]);
        ++i;
        return true;
      };
      for (int b = t.b0; b < t.b1 && ok; ++b) {
        const float* f = fac + (b - t.b0) * 2 * NT;
        ok = take(acc[0], f);
        if (t.kind == 0 && ok) ok = take(acc[1], f + NT);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive1(&f_empty[c & 1]);
      ++c;
      if (!ok) break;
      const int f = t.tile * 128 + tid;
      if (t.kind == 1) {
        float* part = w.dn_part + (t.s * (long long)P + start) * a.d + f;
        if (f < a.d)
#pragma unroll
          for (int m = 0; m < NT; ++m)
            if (m < rows) __stcg(part + (long long)m * a.d, acc[0][m]);
        named_bar(1, 128);
        if (tid == 0) red_release(w.dn_done + t.tile);
        continue;
      }
      const int tile = t.g * sh.FT + t.tile;
      const float bg = a.gate.bias && f < a.f ? __ldg(a.gate.bias + (long long)e * a.f + f) : 0.f;
      const float bu = a.up.bias && f < a.f ? __ldg(a.up.bias + (long long)e * a.f + f) : 0.f;
      if (sh.S1 > 1) {
        if (f < a.f) {
          float* pg = w.up_part + (t.s * 2ll * P + start) * a.f + f;
          float* pu = pg + (long long)P * a.f;
          long long at = 0;
#pragma unroll
          for (int m = 0; m < NT; ++m)
            if (mask >> m & 1) {
              __stcg(pg + at, acc[0][m]);
              __stcg(pu + at, acc[1][m]);
              at += a.f;
            }
        }
        named_bar(1, 128);
        if (tid == 0) s_word[0] = add_acq_rel(w.brought + tile) == (unsigned)(sh.S1 - 1);
        named_bar(1, 128);
        const bool last = s_word[0];
        named_bar(1, 128);                   // all have read the word
        if (!last) continue;
        for (int r0 = 0; r0 < rows; r0 += 4) {
          float g[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
          if (f < a.f)
#pragma unroll 3
            for (int s = 0; s < sh.S1; ++s)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float* at = w.up_part + (s * 2ll * P + start + min(r0 + r, rows - 1)) * a.f + f;
                g[r] += __ldcg(at), u[r] += __ldcg(at + (long long)P * a.f);
              }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            g[r] = f < a.f ? activate(a.model, g[r] + bg, u[r] + bu) : 0.f;
            u[r] = warp_max(fabsf(g[r]));
          }
          if (lane == 0)
#pragma unroll
            for (int r = 0; r < 4; ++r) s_red[r * 4 + warp] = u[r];
          named_bar(1, 128);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r0 + r < rows) put_code(w, a.f, f, tid, t.tile, sh.KB2, start + r0 + r, g[r], s_red + r * 4);
          named_bar(1, 128);                 // the maxima have been read
        }
      } else {
        // a row's activations stay in the registers of its column
#pragma unroll
        for (int m = 0; m < NT; ++m)
          if (mask >> m & 1) {
            acc[0][m] = f < a.f ? activate(a.model, acc[0][m] + bg, acc[1][m] + bu) : 0.f;
            const float top = warp_max(fabsf(acc[0][m]));
            if (lane == 0) s_red[m * 4 + warp] = top;
          }
        named_bar(1, 128);
        int row = start;
#pragma unroll
        for (int m = 0; m < NT; ++m)
          if (mask >> m & 1) put_code(w, a.f, f, tid, t.tile, sh.KB2, row++, acc[0][m], s_red + m * 4);
      }
      fence_async_all();                     // the codes are read by tensor copies
      named_bar(1, 128);
      if (tid == 0) red_release(w.flag + tile);
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 5) tmem_free(tmem, 512);
}

// ------------------------------------------------------------------ launches
size_t moe_fp8_workspace(int T, int d, int f, int E, int k) {
  MoeWs w;
  return (size_t)layout_ws(nullptr, T, d, f, E, k, &w);
}

template <int NT>
static cudaError_t launch_experts(const MoeFp8Args& a, const MoeWs& w, int sms, cudaStream_t s) {
  const long long P = (long long)a.T * a.k, ew = (long long)a.d * a.f;
  MoeMaps m;
  if (encode_fp8_map(&m.gate, a.gate.q, a.d, a.f, a.d, 128, a.E, ew) ||
      encode_fp8_map(&m.up, a.up.q, a.d, a.f, a.d, 128, a.E, ew) ||
      encode_fp8_map(&m.down, a.down.q, a.f, a.d, a.f, 128, a.E, ew) ||
      encode_fp8_map(&m.x, w.xq, a.d, a.T, a.d, NT, 0, 0) || encode_fp8_map(&m.h, w.hq, a.f, P, a.f, NT, 0, 0) ||
      encode_fp8_map(&m.h16, w.hq, a.f, P, a.f, 16, 0, 0))
    return cudaErrorInvalidValue;
  auto kern = k_moe_experts<NT>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Moe<NT>::SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(sms);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = Moe<NT>::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, m, a, w);
}

template <int TG>
static cudaError_t launch_route(const MoeFp8Args& a, const MoeWs& w, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  const int rows = (a.T + TG - 1) / TG;
  // a quantising CTA per 16 groups of its share of the tokens
  cfg.gridDim = dim3((a.E + 7) / 8 + std::max(1, (TG * blocks128(a.d) + 15) / 16), rows);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_moe_route<TG>, a, w);
}

cudaError_t launch_moe_fp8(const MoeFp8Args& a, int sms, cudaStream_t s) {
  MoeWs w;
  layout_ws(a.ws, a.T, a.d, a.f, a.E, a.k, &w);
  cudaError_t e = a.T == 1 ? launch_route<1>(a, w, s) : a.T <= 16 ? launch_route<4>(a, w, s) : launch_route<8>(a, w, s);
  if (e != cudaSuccess) return e;
  if (a.T <= 16) return launch_experts<16>(a, w, sms, s);
  if (a.T <= 32) return launch_experts<32>(a, w, sms, s);
  return launch_experts<64>(a, w, sms, s);
}

cudaError_t moe_fp8_status(int** at) { return cudaGetSymbolAddress(reinterpret_cast<void**>(at), g_moe_status); }

}  // namespace ms
