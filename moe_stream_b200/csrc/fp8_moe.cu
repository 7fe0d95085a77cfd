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
// (one per SM) works out the routing of up to twelve tokens for itself, a warp
// per token, which is less than a trip through memory; more tokens are shared
// out. Then it takes tasks off one counter:
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
// TMEM lanes) and the expert's rows as columns, sixteen or up to 64 of them, so
// no weight passes through registers; an up task gathers its tokens' codes. One
// pipeline serves both: a step is two 128 x 128 weight tiles, an up task's gate
// and up tile of one block or a down task's tiles of two blocks (of one, where
// the expert has more than 16 rows).
//
// A single token (ONE) hands its sums and codes on as 8-byte words of a value
// and a mark, which k_moe_route has cleared: the reader polls the word itself.
// Handing on by a flag costs two trips more, a fence before the flag and a
// load after it, and one token's layer is a chain of such trips (a Qwen3 token
// 26.2 us by flags, 21.2 by words).
//
// Warps 0-3 and 8-11 take products out of TMEM and do the rest of a task, two
// groups with a task each, so that one's end overlaps the other's products;
// warp 4 loads weights and takes tasks, warp 5 issues MMAs, warp 6 loads
// activations and warp 7 the scales; these two wait for the flags, so that
// weights are in flight meanwhile.
#include <algorithm>

#include <cuda_fp16.h>

#include "fp8_mma.cuh"

namespace ms {

// first failure of a bounded wait in this file's kernels (ms_fp8_status). For
// reporting alone: what a call does after a wait that ran out goes by the word
// in its own workspace, so it does not outlive the call or reach another.
static __device__ int g_moe_status;

namespace {

constexpr int MOE_FAC = 16;            // blocks of a task at most
constexpr int MOE_SPLIT = 8;           // ranges of a tile's blocks at most
constexpr int COMBINE_T = 4;           // tokens of a combine task, one per warp
constexpr int MOE_THREADS = 384, MOE_ROWS = 8;    // MOE_ROWS: rows of activations passed on at a time
static_assert(MOE_THREADS / 32 == MOE_FP8_ROUTED_HERE, "a warp per token");

__host__ __device__ inline int blocks128(int n) { return (n + 127) / 128; }
inline long long up16(long long n) { return (n + 15) / 16 * 16; }

// Ranges that a tile's blocks may be cut into at most: as many as a task's
// scales need to fit (a range of 16 blocks), two in any case, and up to eight,
// so that few tiles fill the GPU, while the sums in the workspace stay below 64
// MB a matrix. The first two go before the 64 MB: 64 tokens of 32 choices with
// d and f 16384 take 2 GB for gate and up and 1 GB for down.
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
  int* inds;              // [T, k] choices, largest first (more than four tokens)
  float* probs;           // [T, k]
  unsigned* next;         // next task; this and the following are zeroed by k_moe_route
  unsigned* rt_next;      // next token to route
  unsigned* routed;       // tokens routed
  int* failed;            // ST_E_TIMEOUT once a wait of this call has run out
  unsigned* brought;      // [up tile] ranges brought
  unsigned* flag;         // [up tile] its block is quantised
  unsigned* dn_done;      // [tile of d] warps that are done with down tasks
  unsigned* up_done;      // up tiles whose flag is up
  int counters;           // words from next on
  int cap1, cap2;         // split_cap of the up and down tiles
  // one token: words of a value and a mark, zeroed by k_moe_route
  unsigned long long* up_w;   // [S1 - 1][2][k][f]
  unsigned long long* h_w;    // [k][f / 4] four codes each
  unsigned long long* hs_w;   // [k][blocks of f]
  unsigned long long* dn_w;   // [S2][k][d]
  long long words;        // of all of them
  int S1, S2;             // ranges of its tiles
};

// Ranges for n tiles of kb blocks on `ctas` CTAs are the number with the least
// (rounds of tasks, half a round for the ragged end) x (blocks of a task, half
// a block for its end and `join` for sums that have to meet). In blocks: a
// Qwen3 up tile's join was about two of its blocks long.
__host__ __device__ inline float split_cost(int s, int n, int kb, int ctas, float join) {
  float rounds = (float)(n * s) / (float)ctas;
  rounds = rounds <= 1.f ? 1.f : rounds + 0.5f;
  return rounds * ((float)((kb + s - 1) / s) + 0.5f + (s > 1 ? join : 0.f));
}
static int best_split(int n, int kb, int ctas, int cap, float join) {
  int best = (kb + MOE_FAC - 1) / MOE_FAC;
  for (int s = best + 1; s <= cap && s <= kb; ++s)
    if (split_cost(s, n, kb, ctas, join) < split_cost(best, n, kb, ctas, join)) best = s;
  return best;
}

static long long layout_ws(uint8_t* w, int T, int d, int f, int E, int k, int ctas, MoeWs* o) {
  const long long P = (long long)T * k;
  const int tiles = (int)std::min<long long>(P, E) * blocks128(f);
  uint8_t* const base = w;
  *o = MoeWs{};
  o->cap1 = split_cap(2 * P, f, blocks128(d)), o->cap2 = split_cap(P, d, blocks128(f));
  o->xq = w, w += up16((long long)T * d);
  o->hq = w, w += up16(P * f);
  o->logits = reinterpret_cast<float*>(w), w += up16(4ll * T * E);
  o->xs = reinterpret_cast<float*>(w), w += up16(4ll * T * blocks128(d));
  o->hs = reinterpret_cast<float*>(w), w += up16(4 * P * blocks128(f));
  o->up_part = o->dn_part = nullptr;
  if (T == 1) {
    const int FT = blocks128(f), DT = blocks128(d);
    o->S1 = best_split(k * FT, DT, ctas, MOE_SPLIT, 1.f), o->S2 = best_split(k * DT, FT, ctas, MOE_SPLIT, 0.5f);
    const auto w0 = reinterpret_cast<unsigned long long*>(w);
    o->h_w = w0, o->hs_w = o->h_w + (long long)k * f / 4;
    o->dn_w = o->hs_w + (k * FT + 1) / 2 * 2, o->up_w = o->dn_w + (long long)o->S2 * k * d;
    o->words = o->up_w + (o->S1 - 1) * 2ll * k * f - w0;
    // room for any number of CTAs
    w += 8 * ((long long)k * f / 4 + k * FT + 1 + (long long)MOE_SPLIT * k * d + (MOE_SPLIT - 1) * 2ll * k * f);
    w += (16 - (w - base) % 16) % 16;
  } else {
    o->up_part = reinterpret_cast<float*>(w), w += 8ll * o->cap1 * P * f;
    o->dn_part = reinterpret_cast<float*>(w), w += 4ll * o->cap2 * P * d;
  }
  o->inds = reinterpret_cast<int*>(w), w += up16(4 * P);
  o->probs = reinterpret_cast<float*>(w), w += up16(4 * P);
  o->next = reinterpret_cast<unsigned*>(w), o->rt_next = o->next + 1, o->routed = o->next + 2;
  o->failed = reinterpret_cast<int*>(o->next + 3);
  o->brought = o->next + 4, o->flag = o->brought + tiles, o->dn_done = o->flag + tiles;
  o->up_done = o->dn_done + blocks128(d);
  o->counters = 5 + 2 * tiles + blocks128(d);
  w += up16(4ll * o->counters);
  return w - base;
}

// --------------------------------------------------------------------- route
// Four warps per expert and TG tokens, two experts a CTA, so that all loads of
// a warp are in flight at once; the CTAs after the experts' quantise x and
// clear the counters.
template <int TG>
__global__ void __launch_bounds__(256) k_moe_route(MoeFp8Args a, MoeWs w) {
  __shared__ float part[8][TG];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = a.d / 8, ex = (a.E + 1) / 2;
  const int e = min((int)blockIdx.x * 2 + (warp >> 2), a.E - 1), c0 = (warp & 3) * 32 + lane;
  const uint4* wr = reinterpret_cast<const uint4*>(a.router + (long long)e * a.d);
  if ((int)blockIdx.x < ex)                  // into L2 alone: it may run ahead of what wrote it
    for (int c = c0; c < chunks; c += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(wr + c));
  grid_wait();
  grid_release();
  if ((int)blockIdx.x < ex) {
    const int t0 = blockIdx.y * TG;
    float acc[TG];
#pragma unroll
    for (int t = 0; t < TG; ++t) acc[t] = 0.f;
#pragma unroll(TG == 1 ? 4 : TG == 4 ? 3 : 2)
    for (int c = c0; c < chunks; c += 128) {
      const uint4 v = wr[c];
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
    for (int o = 16; o; o >>= 1)
#pragma unroll
      for (int t = 0; t < TG; ++t) acc[t] += __shfl_xor_sync(MS_FULL, acc[t], o);
    if (lane == 0)
#pragma unroll
      for (int t = 0; t < TG; ++t) part[warp][t] = acc[t];
    __syncthreads();
    const int q = threadIdx.x / TG, t = threadIdx.x % TG, eo = blockIdx.x * 2 + q;
    if (q < 2 && eo < a.E && t0 + t < a.T)
      w.logits[(t0 + t) * a.E + eo] = ((part[4 * q][t] + part[4 * q + 1][t]) + (part[4 * q + 2][t] + part[4 * q + 3][t])) +
                                      (a.router_bias ? a.router_bias[eo] : 0.f);
    return;
  }
  const int q = blockIdx.x - ex, nq = gridDim.x - ex;          // q-th of the quantising CTAs of this row
  if (blockIdx.y == 0 && q == 0)
    for (int i = threadIdx.x; i < w.counters; i += 256) w.next[i] = 0;
  if (TG == 1)
    for (long long i = q * 256 + threadIdx.x; i < w.words / 2; i += nq * 256)
      reinterpret_cast<uint4*>(w.h_w)[i] = make_uint4(0, 0, 0, 0);
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
  static constexpr int ACT = NT <= 32 ? 4096 : NT * 128;             // activation tiles of a step
  static constexpr int STAGE = 2 * FP8_W_TILE + ACT;
  static constexpr int STAGES = NT <= 32 ? 5 : 4;
  static constexpr int BUFS = NT <= 32 ? 4 : 2;                      // of each group
  static constexpr int OFF_FAC = STAGES * STAGE;                     // [2][FAC][2][NT] scale products
  static constexpr int OFF_ROWS = OFF_FAC + 2 * MOE_FAC * 2 * NT * 4;   // [2][2][ROWS][128] gate and up sums
  static constexpr int OFF_PROB = OFF_ROWS + 2 * 2 * MOE_ROWS * 512; // [NT][32]
  static constexpr int OFF_ROW = OFF_PROB + NT * 32 * 4;             // [NT][32] 16-bit: rows of the choices
  static constexpr int OFF_TOK = OFF_ROW + NT * 64;                  // [T * k] bytes: tokens of the rows
  static constexpr int OFF_MASK = OFF_TOK + NT * 32;                 // [256] tokens of an expert, 64 bits
  static constexpr int OFF_START = OFF_MASK + 256 * 8;               // [256] its first row
  static constexpr int OFF_GROUP = OFF_START + 256 * 4;              // [256] experts that are routed to, ascending
  static constexpr int OFF_TASK = OFF_GROUP + 256;                   // [4] tasks
  static constexpr int OFF_WORD = OFF_TASK + 4 * 32;                 // a few words
  static constexpr int OFF_BAR = OFF_WORD + 64;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
  static_assert(SMEM <= 232448 && SMEM > 232448 - 77824, "alone on its SM");
  static_assert(STAGE % 1024 == 0 && 2 * BUFS * 2 * NT <= 512, "tile alignment, TMEM columns");
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

// The best number of ranges, by a warp (a number per lane).
__device__ __forceinline__ int choose_split(int n, int kb, int ctas, int cap, float join) {
  const int s = (threadIdx.x & 31) + 1;
  const bool can = s >= (kb + MOE_FAC - 1) / MOE_FAC && s <= cap && s <= kb;
  const unsigned key = can ? __float_as_uint(split_cost(s, n, kb, ctas, join)) : 0x7f800000u;
  const unsigned least = __reduce_min_sync(MS_FULL, key);
  return __ffs(__ballot_sync(MS_FULL, key == least));
}

// Records that a wait of the call whose word `failed` is ran out.
__device__ __forceinline__ void wait_ran_out(int* failed) {
  atomicExch(failed, ST_E_TIMEOUT);
  atomicCAS(&g_moe_status, 0, ST_E_TIMEOUT);
}
__device__ __forceinline__ bool wait_step(uint64_t* bar, unsigned phase, int* failed) {
  if (mbar_wait_step(bar, phase, nullptr)) return true;
  wait_ran_out(failed);
  return false;
}

// A value and its mark in one word, written and read whole.
__device__ __forceinline__ void put_word(unsigned long long* p, uint32_t v) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(1ull << 32 | v) : "memory");
}
__device__ __forceinline__ unsigned long long get_word(const unsigned long long* p) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
// Four words from each of four places, once all are written; a second at most.
__device__ __forceinline__ void wait_quads(const unsigned long long* const* p, uint32_t (*v)[4], int* failed) {
  unsigned long long t0 = 0;
  for (unsigned i = 0;; ++i) {
    unsigned have = 0;
    unsigned long long x[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) x[j][q] = get_word(p[j] + q);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[j][q] = (uint32_t)x[j][q], have += (unsigned)(x[j][q] >> 32);
    if (have == 16) return;
    if ((i & 63) == 63) {
      const unsigned long long now = global_ns();
      if (!t0) t0 = now;
      if (now - t0 > MBAR_WAIT_NS || timed_out(failed)) break;
    }
  }
  wait_ran_out(failed);
}
// v[q] = the value of word p[q * stride] for q < n, as wait_quads.
template <int N>
__device__ __forceinline__ void wait_words(const unsigned long long* p, long long stride, int n, uint32_t* v,
                                           int* failed) {
  unsigned long long t0 = 0;
  unsigned have = 0;
  for (unsigned i = 0;; ++i) {
    unsigned long long x[N];
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (q < n) x[q] = get_word(p + q * stride);
    have = 0;
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (q < n) v[q] = (uint32_t)x[q], have += (unsigned)(x[q] >> 32);
    if (have == (unsigned)n) return;
    if ((i & 63) == 63) {
      const unsigned long long now = global_ns();
      if (!t0) t0 = now;
      if (now - t0 > MBAR_WAIT_NS || timed_out(failed)) break;
    }
  }
  wait_ran_out(failed);
}

__device__ __forceinline__ unsigned ld_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void fence_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }
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
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(MS_FULL, v, o);
  return v;
}
// a key that orders like the float; a NaN is below all, 0 below every key
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return v != v ? 1u : b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// both models' activation: silu(g) u with alpha 1, beta 0, limit infinity;
// gpt-oss alpha 1.702, beta 1, limit 7
struct Act {
  float alpha, beta, limit;
  __device__ __forceinline__ float operator()(float g, float u) const {
    g = g > limit ? limit : g;
    u = u > limit ? limit : u < -limit ? -limit : u;
    return __fdividef(g, 1.f + expf(-alpha * g)) * (u + beta);
  }
};

// Waits until *p >= want, a second at most.
__device__ __forceinline__ bool wait_count(const unsigned* p, unsigned want, int* failed) {
  if (ld_acquire(p) >= want) return true;
  const unsigned long long t0 = global_ns();
  for (unsigned i = 0; i < MBAR_SPIN_LIMIT; ++i) {
    if (ld_acquire(p) >= want) return true;
    if ((i & 63) == 63 && (global_ns() - t0 > MBAR_WAIT_NS || timed_out(failed))) break;
  }
  wait_ran_out(failed);
  return false;
}

// The flags of blocks b0 to b1 of a group, by a warp; `all` once every tile's
// flag is up, from when on there is nothing to wait for.
__device__ __forceinline__ void wait_flags(const unsigned* flag, int b0, int b1, const unsigned* up_done, unsigned tiles,
                                           bool* all, int* failed) {
  if (*all) return;
  const int lane = threadIdx.x & 31;
  const unsigned v = ld_acquire(lane == 31 ? up_done : flag + min(b0 + lane, b1 - 1));
  *all = __shfl_sync(MS_FULL, v, 31) == tiles;
  if (!*all && lane < 31 && v == 0) wait_count(flag + min(b0 + lane, b1 - 1), 1, failed);
  __syncwarp();
  fence_async_all();
}

// A token's experts: lane j holds the j-th choice and its key.
struct Choice {
  int expert;
  uint32_t key;
  float top, all;           // largest logit (NaN where one is); sum over all experts, if it is asked for
};
// The largest logit one after another. The code runs once, cold, so it is
// kept short.
__device__ __forceinline__ Choice choose(const float* logits, const MoeFp8Args& a, int lane) {
  uint32_t key[8];
  float v[8];
  bool nan = false;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = lane + 32 * i;
    v[i] = e < a.E ? __ldcg(logits + e) + 0.f : 0.f;      // -0 is 0
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    nan |= v[i] != v[i];
    key[i] = lane + 32 * i < a.E ? order_key(v[i]) : 0u;
    top = max(top, key[i]);
  }
  Choice c{0, 0u, 0.f, 0.f};
  const float m = key_value(__reduce_max_sync(MS_FULL, top));
  c.top = __any_sync(MS_FULL, nan) ? __uint_as_float(0x7fc00000u) : m;
  if (a.model == 0 && !a.norm_topk) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c.all += lane + 32 * i < a.E ? expf(v[i] - c.top) : 0.f;
    c.all = warp_sum(c.all);
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
    if (lane == j) c.expert = first, c.key = best;
  }
  return c;
}
// lane j: the j-th choice's share
__device__ __forceinline__ float share(const Choice& c, const MoeFp8Args& a, int lane) {
  const float p = lane < a.k ? expf(key_value(c.key) - c.top) : 0.f;
  const float sel = warp_sum(p);
  return p / (a.model == 1 || a.norm_topk ? sel : c.all);
}

struct MoeMaps {
  CUtensorMap gate, up, down, x, h;
};

template <int NT, bool ONE>
__global__ void __launch_bounds__(MOE_THREADS, 1)
    k_moe_experts(const __grid_constant__ MoeMaps maps, const __grid_constant__ MoeFp8Args a,
                  const __grid_constant__ MoeWs w) {
  using C = Moe<NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_fac = reinterpret_cast<float*>(smem + C::OFF_FAC);
  float* s_prob = reinterpret_cast<float*>(smem + C::OFF_PROB);
  uint16_t* s_row = reinterpret_cast<uint16_t*>(smem + C::OFF_ROW);
  uint8_t* s_tok = smem + C::OFF_TOK;
  unsigned long long* s_mask = reinterpret_cast<unsigned long long*>(smem + C::OFF_MASK);
  int* s_start = reinterpret_cast<int*>(smem + C::OFF_START);
  uint8_t* s_group = smem + C::OFF_GROUP;
  volatile int* s_word = reinterpret_cast<volatile int*>(smem + C::OFF_WORD);   // last [2][2], S1, S2; [8] sums
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);        // [STAGES] both tiles landed
  uint64_t* empty = full + C::STAGES;                                     // [STAGES] read by the MMAs
  uint64_t* d_full = empty + C::STAGES;                                   // [2][BUFS] a group's product complete
  uint64_t* d_empty = d_full + 2 * C::BUFS;                               // [2][BUFS] taken out
  uint64_t* f_full = d_empty + 2 * C::BUFS;                                   // [2] a task's scales there
  uint64_t* f_empty = f_full + 2;                                         // [2] used
  uint64_t* t_full = f_empty + 2;                                         // [4] a task taken
  uint64_t* t_empty = t_full + 4;                                         // [4] done by all roles
  Task* s_task = reinterpret_cast<Task*>(smem + C::OFF_TASK);             // [4]
  uint64_t* g_bar = t_empty + 4;                                          // [2] a group's warps meet
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(g_bar + 2);
  int* const failed = w.failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int P = a.T * a.k;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) mbar_init(&full[i], 2), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2 * C::BUFS; ++i) mbar_init(&d_full[i], 1), mbar_init(&d_empty[i], 4);
    for (int i = 0; i < 2; ++i) mbar_init(&f_full[i], 1), mbar_init(&f_empty[i], 4), mbar_init(&g_bar[i], 4);
    for (int i = 0; i < 4; ++i) mbar_init(&t_full[i], 1), mbar_init(&t_empty[i], 11);
    fence_barrier_init();
  }
  if (threadIdx.x < 256) s_mask[threadIdx.x] = 0;
  if (warp == 5) tmem_get(tmem_at, 512);
  if (warp == 4 && lane < 5) tma_map_prefetch(reinterpret_cast<const CUtensorMap*>(&maps) + lane);
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_at;
  grid_wait();

  unsigned first_task = 0;
  if (warp == 4 && lane == 0) first_task = atomicAdd(w.next, 1u);    // back by the time it can be read

  // ---- the routing, a warp per token
  const bool shared_out = !ONE && a.T > MOE_THREADS / 32;
  int G = a.k;
  if constexpr (ONE) {
    Choice c;
    if (warp == 0) {
      c = choose(w.logits, a, lane);
      int rank = 0;                         // rows lie in the order of their experts
      for (int j = 0; j < a.k; ++j) rank += __shfl_sync(MS_FULL, c.expert, j) < c.expert;
      if (lane < a.k) {
        s_group[rank] = (uint8_t)c.expert;
        s_start[c.expert] = rank;
        s_mask[c.expert] = 1;
        s_row[lane] = (uint16_t)rank;
        s_tok[rank] = 0;
      }
    }
    __syncthreads();
    if (warp == 0) {                        // read by this warp alone, at the end
      const float p = share(c, a, lane);
      if (lane < a.k) s_prob[lane] = p;
    }
  } else if (!shared_out || warp == 0) {
    for (int t = warp;; t = a.T) {
      if (shared_out) {
        if (lane == 0) t = (int)atomicAdd(w.rt_next, 1u);
        t = __shfl_sync(MS_FULL, t, 0);
      }
      if (t >= a.T) break;
      const Choice c = choose(w.logits + t * a.E, a, lane);
      const float p = share(c, a, lane);
      if (lane < a.k) {
        if (shared_out) {
          __stcg(w.probs + t * a.k + lane, p);
          __stcg(w.inds + t * a.k + lane, c.expert);
        } else {
          s_prob[t * 32 + lane] = p;
          s_row[t * 32 + lane] = (uint16_t)c.expert;
          atomicOr(&s_mask[c.expert], 1ull << t);
        }
      }
      __syncwarp();
      if (shared_out && lane == 0) red_release(w.routed);
      if (!shared_out) break;
    }
  }
  bool lost = false;                        // the routing never came: this CTA takes no tasks
  if (shared_out) {
    if (threadIdx.x == 0) s_word[0] = wait_count(w.routed, (unsigned)a.T, failed);
    __syncthreads();
    lost = !s_word[0];
    for (int q = threadIdx.x; q < P && !lost; q += MOE_THREADS) {
      const int t = q / a.k, at = t * 32 + q - t * a.k, e = __ldcg(w.inds + q);
      s_prob[at] = __ldcg(w.probs + q);
      s_row[at] = (uint16_t)e;
      atomicOr(&s_mask[e], 1ull << t);
    }
  }
  if constexpr (!ONE) {
    __syncthreads();
    // groups: the experts that have rows, ascending; their rows follow each other
    const int mine_n = threadIdx.x < 256 ? __popcll(s_mask[threadIdx.x]) : 0;
    G = __syncthreads_count(mine_n > 0);
    if (warp < 8) {                           // rows in the low half, groups in the high; sums of the warps before
      int at = mine_n + (mine_n ? 1 << 16 : 0);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(MS_FULL, at, o);
        if (lane >= o) at += u;
      }
      if (lane == 31) s_word[8 + warp] = at;
      named_bar(1, 256);
      for (int q = 0; q < warp; ++q) at += s_word[8 + q];
      if (mine_n) {
        s_group[(at >> 16) - 1] = (uint8_t)threadIdx.x;
        s_start[threadIdx.x] = (at & 0xffff) - mine_n;
      }
    } else if (warp < 10) {
      const int nf = blocks128(a.f), nd = blocks128(a.d);
      const int split = warp == 8 ? choose_split(G * nf, nd, gridDim.x, w.cap1, 2.f)
                                  : choose_split(G * nd, nf, gridDim.x, w.cap2, 0.5f);
      if (lane == 0) s_word[warp - 4] = split;
    }
    __syncthreads();
    for (int q = threadIdx.x; q < P && !lost; q += MOE_THREADS) {     // a choice's row, a row's token
      const int t = q / a.k, at = t * 32 + q - t * a.k, e = s_row[at];
      const int row = s_start[e] + __popcll(s_mask[e] & ((1ull << t) - 1));
      s_row[at] = (uint16_t)row;
      s_tok[row] = (uint8_t)t;
    }
    __syncthreads();
  }
  Shape sh;
  sh.G = G, sh.S1 = ONE ? w.S1 : s_word[4], sh.S2 = ONE ? w.S2 : s_word[5];
  sh.FT = blocks128(a.f), sh.DT = blocks128(a.d), sh.KB1 = sh.DT, sh.KB2 = sh.FT;
  sh.n_up = sh.G * sh.FT * sh.S1, sh.n_dn = sh.G * sh.DT * sh.S2;
  sh.n_co = lost ? 0 : sh.DT * ((a.T + COMBINE_T - 1) / COMBINE_T);

  // blocks of a down step
  auto down_per = [&](int g) { return __popcll(s_mask[s_group[g]]) <= 16 ? 2 : 1; };

  if (NT == 64 && warp >= 4 && warp < 8) regs_down<40>();
  if (warp == 4) {
    // ---- tasks and weight tiles
    const uint64_t once = l2_evict_first();
    bool ok = true;
    int i = 0, n = 0;
    auto take = [&](unsigned id) {           // the n-th task, published to the other warps
      if (n >= 4 && !wait_step(&t_empty[n & 3], ((n >> 2) - 1) & 1, failed)) ok = false;
      const Task t = sh.task(ok ? id : 0xffffffffu);      // after a failure the other warps end
      if (lane == 0) {
        s_task[n & 3] = t;
        mbar_arrive1(&t_full[n & 3]);
      }
      ++n;
      return t;
    };
    auto ticket = [&] {
      unsigned id = 0;
      if (lane == 0) id = atomicAdd(w.next, 1u);
      return __shfl_sync(MS_FULL, id, 0);
    };
    Task t = take(__shfl_sync(MS_FULL, first_task, 0));
    while (t.kind != 3) {
      if (t.kind == 2) {                     // one at a time, so that other CTAs take the next
        if (!wait_step(&t_empty[(n - 1) & 3], ((n - 1) >> 2) & 1, failed)) ok = false;
        t = take(ticket());
        continue;
      }
      // the next task is known before this one's tiles are out: its scales and
      // activations are fetched meanwhile
      const Task next = take(ticket());
      const int e = s_group[t.g], per = t.kind == 0 ? 1 : down_per(t.g);
      for (int b = t.b0; b < t.b1 && ok; b += per, ++i) {
        const int s = i % C::STAGES;
        if (i >= C::STAGES && !wait_step(&empty[s], ((i / C::STAGES) - 1) & 1, failed)) {
          // copies in flight land before the CTA ends
          for (int j = i - C::STAGES; j < i && mbar_wait(&full[j % C::STAGES], (j / C::STAGES) & 1, nullptr);) ++j;
          ok = false;
          break;
        }
        if (elect_one()) {
          uint8_t* at = smem + s * C::STAGE;
          const int tiles = t.kind == 0 ? 2 : min(per, t.b1 - b);
          mbar_expect_tx(&full[s], tiles * FP8_W_TILE);
          if (t.kind == 0) {
            tma_tile_3d_once(at, &maps.gate, b * 128, t.tile * 128, e, &full[s], once);
            tma_tile_3d_once(at + FP8_W_TILE, &maps.up, b * 128, t.tile * 128, e, &full[s], once);
          } else {
            for (int h = 0; h < tiles; ++h)
              tma_tile_3d_once(at + h * FP8_W_TILE, &maps.down, (b + h) * 128, t.tile * 128, e, &full[s], once);
          }
        }
        __syncwarp();
      }
      if (!ok) {
        if (next.kind != 3) take(0);
        break;
      }
      t = next;
    }
    if (ok) mbar_wait_ring<C::STAGES>(empty, i, nullptr);
  } else if (warp == 5) {
    // ---- MMAs. Each group has buffers of its own and meets every phase of
    // their barriers in turn: a wait for a parity does not tell a phase from
    // the one two before it.
    bool ok = true;
    int i = 0, c = 0, j0 = 0, j1 = 0;        // steps; compute tasks; steps of each group
    for (int n = 0; ok; ++n) {
      if (!wait_step(&t_full[n & 3], (n >> 2) & 1, failed)) break;
      const Task t = s_task[n & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive1(&t_empty[n & 3]);
      if (t.kind == 3) break;
      if (t.kind == 2) continue;
      const int per = t.kind == 0 ? 1 : down_per(t.g);
      const uint32_t idesc = idesc_e4m3(128, (__popcll(s_mask[s_group[t.g]]) + 15) & ~15);
      const int grp = c++ & 1;
      for (int b = t.b0; b < t.b1; b += per, ++i) {
        const int j = grp ? j1++ : j0++;
        const int s = i % C::STAGES, u = grp * C::BUFS + j % C::BUFS;
        if (!wait_step(&full[s], (i / C::STAGES) & 1, failed) ||
            (j >= C::BUFS && !wait_step(&d_empty[u], ((j / C::BUFS) - 1) & 1, failed))) {
          ok = false;
          break;
        }
        tc_after();
        if (elect_one()) {
          const uint8_t* at = smem + s * C::STAGE;
          const uint64_t ad = k128_desc(at), bd = k128_desc(at + 2 * FP8_W_TILE);
          const int tiles = t.kind == 0 ? 2 : min(per, t.b1 - b);
          const int next_b = t.kind == 0 ? 0 : 2048 / 16;
          for (int h = 0; h < tiles; ++h)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              mma_e4m3(tmem + (2 * u + h) * NT, ad + h * (FP8_W_TILE / 16) + 2 * q, bd + h * next_b + 2 * q, idesc, q != 0);
          mma_done(&d_full[u]);
          mma_done(&empty[s]);
        }
        __syncwarp();
      }
    }
  } else if (warp == 6) {
    // ---- activation tiles
    bool ok = true, all_up = false;
    int i = 0;
    for (int n = 0; ok; ++n) {
      if (!wait_step(&t_full[n & 3], (n >> 2) & 1, failed)) break;
      const Task t = s_task[n & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive1(&t_empty[n & 3]);
      if (t.kind == 3) break;
      if (t.kind == 2) continue;
      const int e = s_group[t.g], start = s_start[e], rows = __popcll(s_mask[e]);
      const int per = t.kind == 0 ? 1 : down_per(t.g);
      if constexpr (ONE)
        if (t.kind == 1) {
          // the row's codes, word by word, into the first row of the tiles
          const int n4 = a.f / 4;
          uint32_t v[MOE_FAC];
#pragma unroll
          for (int q = 0; q < MOE_FAC; ++q) v[q] = 0;
          // a lane's last block may lie beyond f
          const int at0 = t.b0 * 32 + lane, nb = t.b1 - t.b0 - (at0 + (t.b1 - t.b0 - 1) * 32 >= n4);
          wait_words<MOE_FAC>(w.h_w + (long long)start * n4 + at0, 32, nb, v, failed);
#pragma unroll
          for (int q = 0; q < MOE_FAC; q += 2) {
            if (t.b0 + q >= t.b1) break;
            const int s = i % C::STAGES;
            if (i >= C::STAGES && !wait_step(&empty[s], ((i / C::STAGES) - 1) & 1, failed)) {
              ok = false;
              break;
            }
            uint8_t* at = smem + s * C::STAGE + 2 * FP8_W_TILE + 4 * lane;
            *reinterpret_cast<uint32_t*>(at) = q < nb ? v[q] : 0;
            *reinterpret_cast<uint32_t*>(at + 2048) = q + 1 < nb ? v[q + 1] : 0;
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive1(&full[s]);
            ++i;
          }
          continue;
        }
      int tok[4];                            // up: the tokens of rows 4 lane to 4 lane + 3, none beyond the last
      if (t.kind == 1) {
        wait_flags(w.flag + t.g * sh.FT, t.b0, t.b1, w.up_done, sh.G * sh.FT, &all_up, failed);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) tok[q] = 4 * lane + q < rows ? s_tok[start + 4 * lane + q] : a.T;
      }
      for (int b = t.b0; b < t.b1; b += per, ++i) {
        const int s = i % C::STAGES;
        if (i >= C::STAGES && !wait_step(&empty[s], ((i / C::STAGES) - 1) & 1, failed)) {
          ok = false;
          break;
        }
        uint8_t* at = smem + s * C::STAGE + 2 * FP8_W_TILE;
        if (t.kind == 0) {
          if (elect_one()) mbar_expect_tx(&full[s], (rows + 3) / 4 * 512);
          __syncwarp();
          if (4 * lane < rows) tma_gather4(at + lane * 512, &maps.x, b * 128, tok[0], tok[1], tok[2], tok[3], &full[s]);
        } else if (elect_one()) {
          const int tiles = min(per, t.b1 - b), boxes = (rows + 15) / 16;
          mbar_expect_tx(&full[s], tiles * boxes * 2048);
          for (int h = 0; h < tiles; ++h)
            for (int q = 0; q < boxes; ++q)
              tma_tile_2d(at + (h + q) * 2048, &maps.h, (b + h) * 128, start + 16 * q, &full[s]);
        }
        __syncwarp();
      }
    }
  } else if (warp == 7) {
    // ---- products of the activations' and the weights' scales, a task ahead
    bool ok = true, all_up = false;
    int c = 0;
    for (int n = 0; ok; ++n) {
      if (!wait_step(&t_full[n & 3], (n >> 2) & 1, failed)) break;
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
        if (c >= 2) ok = wait_step(&f_empty[u], ((c >> 1) - 1) & 1, failed);
#pragma unroll 8
        for (int r = r0; r < rows; r += 2) {
          const float x = __ldcg(w.xs + s_tok[start + r] * sh.KB1 + b);
          if (wb < nb) fac[r] = x * wg, fac[NT + r] = x * wu;
        }
      } else {
        const float wd = __ldg(a.down.s + ((long long)e * sh.DT + t.tile) * sh.KB2 + b);
        if constexpr (ONE) {
          uint32_t x;
          wait_words<1>(w.hs_w + (long long)start * sh.KB2 + b, 0, 1, &x, failed);
          __syncwarp();
          if (c >= 2) ok = wait_step(&f_empty[u], ((c >> 1) - 1) & 1, failed);
          if (lane < nb) fac[0] = __uint_as_float(x) * wd;
          ++c;
          __syncwarp();
          if (lane == 0) mbar_arrive1(&f_full[u]);
          continue;
        }
        wait_flags(w.flag + t.g * sh.FT, t.b0, t.b1, w.up_done, sh.G * sh.FT, &all_up, failed);
        if (c >= 2) ok = wait_step(&f_empty[u], ((c >> 1) - 1) & 1, failed);
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
  } else {
    // ---- products out of TMEM, and what follows them
    if (NT == 64) regs_up<232>();
    const int grp = warp >> 3, tid = threadIdx.x & 127;
    bool ok = true;
    int i = 0, c = 0, met = 0, joins = 0;    // steps of this group; compute tasks
    // A down task is reported a task later: by then its sums have long been
    // written and the fence does not hold the warp up (about 2000 cycles a task
    // otherwise). A task waits for no report but a combine task, before which
    // all are sent.
    unsigned* report = nullptr;
    auto send = [&] {
      if (!ONE && report && lane == 0) red_release(report);
      report = nullptr;
    };
    // the group's warps meet (a wait with a limit, unlike bar.sync)
    auto meet = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive1(&g_bar[grp]);
      if (!wait_step(&g_bar[grp], met & 1, failed)) ok = false;
      ++met;
    };
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    float* s_rows = reinterpret_cast<float*>(smem + C::OFF_ROWS) + grp * (2 * MOE_ROWS * 128);
    float acc[2][NT];
    for (int n = 0; ok; ++n) {
      if (!wait_step(&t_full[n & 3], (n >> 2) & 1, failed)) break;
      const Task t = s_task[n & 3];
      __syncwarp();
      const bool combine = t.kind == 2 && grp == 0;
      if (!combine && lane == 0) mbar_arrive1(&t_empty[n & 3]);
      if (t.kind > 1) send();
      if (t.kind == 3) break;
      if (t.kind == 2) {
        if (!combine) continue;
        // y of four tokens, one per warp: rows in the order of the token's
        // choices, ranges in order
        if (!ONE) {
          if (tid == 0) wait_count(w.dn_done + t.tile, (unsigned)(sh.G * sh.S2 * 4), failed);
          meet();
        }
        const int f = t.tile * 128 + lane * 4, tok = t.s * COMBINE_T + warp;
        if (f < a.d && tok < a.T) {
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          const float* const p0 = w.dn_part + f;
          for (int j0 = 0; j0 < a.k; j0 += 8) {
            float4 o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int s = 0; s < sh.S2; ++s) {
              const int r0 = s * P;
              if constexpr (ONE) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {       // four choices' words in flight
                  const unsigned long long* p[4];
                  uint32_t v[4][4];
#pragma unroll
                  for (int j = 0; j < 4; ++j)
                    p[j] = w.dn_w + (long long)(r0 + s_row[min(j0 + 4 * h + j, a.k - 1)]) * a.d + f;
                  wait_quads(p, v, failed);
#pragma unroll
                  for (int j = 0; j < 4; ++j) {
                    o[4 * h + j].x += __uint_as_float(v[j][0]), o[4 * h + j].y += __uint_as_float(v[j][1]);
                    o[4 * h + j].z += __uint_as_float(v[j][2]), o[4 * h + j].w += __uint_as_float(v[j][3]);
                  }
                }
              } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const int row = r0 + s_row[tok * 32 + min(j0 + j, a.k - 1)];
                  const float4 u = __ldcg(reinterpret_cast<const float4*>(p0 + (long long)row * a.d));
                  o[j].x += u.x, o[j].y += u.y, o[j].z += u.z, o[j].w += u.w;
                }
              }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float p = j0 + j < a.k ? s_prob[tok * 32 + j0 + j] : 0.f;
              if (j0 + j < a.k) {
                y.x = fmaf(p, o[j].x, y.x), y.y = fmaf(p, o[j].y, y.y);
                y.z = fmaf(p, o[j].z, y.z), y.w = fmaf(p, o[j].w, y.w);
              }
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
      const int per = t.kind == 0 ? 1 : down_per(t.g);
      if ((c & 1) != grp) {                  // the other group's
        ++c;
        continue;
      }
      const int e = s_group[t.g], start = s_start[e];
      const int rows = __popcll(s_mask[e]);
      const float* fac = s_fac + grp * (MOE_FAC * 2 * NT);
      ok = wait_step(&f_full[grp], (c >> 1) & 1, failed);
#pragma unroll
      for (int m = 0; m < NT; ++m) acc[0][m] = acc[1][m] = 0.f;
      auto take = [&](float* sum, uint32_t at, const float* f) {
        if constexpr (ONE) {
          sum[0] = fmaf(tmem_read1(at), f[0], sum[0]);
        } else {
#pragma unroll
          for (int m = 0; m < NT; m += 16) {
            if (m >= rows) break;
            uint32_t v[16];
            tmem_load16(at + m, v);
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
        }
      };
      for (int b = t.b0; b < t.b1; b += per, ++i) {
        const int u = grp * C::BUFS + i % C::BUFS;
        if (!ok || !wait_step(&d_full[u], (i / C::BUFS) & 1, failed)) {
          ok = false;
          break;
        }
        tc_after();
        const float* f = fac + (b - t.b0) * 2 * NT;
        const uint32_t at = lanes + 2 * u * NT;
        take(acc[0], at, f);
        if (t.kind == 0) take(acc[1], at + NT, f + NT);
        else if (per == 2 && b + 1 < t.b1) take(acc[0], at + NT, f + 2 * NT);
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive1(&d_empty[u]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive1(&f_empty[grp]);
      ++c;
      if (!ok) break;
      const int f = t.tile * 128 + tid;
      if (t.kind == 1) {
        float* part = w.dn_part + (t.s * (long long)P + start) * a.d + f;
        const float bias = t.s == 0 && a.down.bias && f < a.d ? __ldg(a.down.bias + (long long)e * a.d + f) : 0.f;
        if constexpr (ONE) {
          if (f < a.d) put_word(w.dn_w + (long long)(t.s * P + start) * a.d + f, __float_as_uint(acc[0][0] + bias));
          continue;
        }
        send();
        if (f < a.d)
#pragma unroll
          for (int m = 0; m < NT; m += 8) {
            if (m >= rows) break;
#pragma unroll
            for (int q = 0; q < 8; ++q)
              if (m + q < rows) __stcg(part + (long long)(m + q) * a.d, acc[0][m + q] + bias);
          }
        __syncwarp();
        report = w.dn_done + t.tile;
        continue;
      }
      const int tile = t.g * sh.FT + t.tile;
      if constexpr (ONE) {
        // the last range's CTA adds the others' sums to its own
        if (f < a.f) {
          unsigned long long* word = w.up_w + (long long)start * a.f + f;
          const long long stride = (long long)a.k * a.f;
          if (t.s < sh.S1 - 1) {
            put_word(word + 2 * t.s * stride, __float_as_uint(acc[0][0]));
            put_word(word + (2 * t.s + 1) * stride, __float_as_uint(acc[1][0]));
          } else if (sh.S1 > 1) {
            uint32_t v[2 * (MOE_SPLIT - 1)];
            wait_words<2 * (MOE_SPLIT - 1)>(word, stride, 2 * (sh.S1 - 1), v, failed);
            float g = 0.f, u = 0.f;
#pragma unroll
            for (int q = 0; q < MOE_SPLIT - 1; ++q)
              if (q < sh.S1 - 1) g += __uint_as_float(v[2 * q]), u += __uint_as_float(v[2 * q + 1]);
            acc[0][0] += g, acc[1][0] += u;
          }
        }
        if (t.s < sh.S1 - 1) continue;
      } else if (sh.S1 > 1) {
        if (f < a.f) {
          float* pg = w.up_part + (t.s * 2ll * P + start) * a.f + f;
          float* pu = pg + (long long)P * a.f;
#pragma unroll
          for (int m = 0; m < NT; ++m)
            if (m < rows) {
              __stcg(pg + (long long)m * a.f, acc[0][m]);
              __stcg(pu + (long long)m * a.f, acc[1][m]);
            }
        }
        meet();
        volatile int* last = s_word + 2 * grp + (joins++ & 1);
        if (tid == 0) *last = add_acq_rel(w.brought + tile) == (unsigned)(sh.S1 - 1);
        meet();
        if (!*last) continue;
      }
      // a warp per row: four features a lane
      const Act act = a.model == 1 ? Act{1.702f, 1.f, 7.f} : Act{1.f, 0.f, __uint_as_float(0x7f800000u)};
      const int f4 = t.tile * 128 + lane * 4;
      const bool in = f4 < a.f;
      float bg[4] = {0.f, 0.f, 0.f, 0.f}, bu[4] = {0.f, 0.f, 0.f, 0.f};
      if (in)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (a.gate.bias) bg[q] = __ldg(a.gate.bias + (long long)e * a.f + f4 + q);
          if (a.up.bias) bu[q] = __ldg(a.up.bias + (long long)e * a.f + f4 + q);
        }
      for (int r0 = 0; r0 < rows; r0 += MOE_ROWS) {
        if (ONE || sh.S1 == 1) {             // this tile's sums are in the registers of their columns
#pragma unroll
          for (int m = 0; m < NT; m += MOE_ROWS)
            if (m == r0) {
#pragma unroll
              for (int q = 0; q < MOE_ROWS; ++q) {
                s_rows[q * 128 + tid] = acc[0][m + q];
                s_rows[(MOE_ROWS + q) * 128 + tid] = acc[1][m + q];
              }
            }
          meet();
        }
        for (int r = r0 + (warp & 3); r < min(rows, r0 + MOE_ROWS); r += 4) {
          float4 g = make_float4(0.f, 0.f, 0.f, 0.f), u = g;
          if (ONE || sh.S1 == 1) {
            g = *reinterpret_cast<const float4*>(s_rows + (r - r0) * 128 + lane * 4);
            u = *reinterpret_cast<const float4*>(s_rows + (MOE_ROWS + r - r0) * 128 + lane * 4);
          } else if (in) {
            const float* at = w.up_part + (long long)(start + r) * a.f + f4;
#pragma unroll 4
            for (int s = 0; s < sh.S1; ++s) {
              const float4 x = __ldcg(reinterpret_cast<const float4*>(at + s * 2ll * P * a.f));
              const float4 y = __ldcg(reinterpret_cast<const float4*>(at + (s * 2ll + 1) * P * a.f));
              g.x += x.x, g.y += x.y, g.z += x.z, g.w += x.w;
              u.x += y.x, u.y += y.y, u.z += y.z, u.w += y.w;
            }
          }
          const float h0 = in ? act(g.x + bg[0], u.x + bu[0]) : 0.f;
          const float h1 = in ? act(g.y + bg[1], u.y + bu[1]) : 0.f;
          const float h2 = in ? act(g.z + bg[2], u.z + bu[2]) : 0.f;
          const float h3 = in ? act(g.w + bg[3], u.w + bu[3]) : 0.f;
          float inv;
          const float s = group_scale(
              warp_max(max_nan(max_nan(fabsf(h0), fabsf(h1)), max_nan(fabsf(h2), fabsf(h3)))), &inv);
          const uint32_t codes = e4m3x2(h0 * inv, h1 * inv) | e4m3x2(h2 * inv, h3 * inv) << 16;
          if constexpr (ONE) {
            if (in) put_word(w.h_w + ((long long)(start + r) * a.f + f4) / 4, codes);
            if (lane == 0) put_word(w.hs_w + (long long)(start + r) * sh.KB2 + t.tile, __float_as_uint(s));
            continue;
          }
          if (in) *reinterpret_cast<uint32_t*>(w.hq + (long long)(start + r) * a.f + f4) = codes;
          if (lane == 0) w.hs[(long long)(start + r) * sh.KB2 + t.tile] = s;
        }
        if (ONE || sh.S1 == 1) meet();       // the rows have been read
      }
      if (ONE) continue;
      fence_async_all();                     // the codes are read by tensor copies
      meet();
      if (tid == 0) {
        red_release(w.flag + tile);
        red_release(w.up_done);
      }
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 5) tmem_free(tmem, 512);
}

// ------------------------------------------------------------------ launches
size_t moe_fp8_workspace(int T, int d, int f, int E, int k) {
  MoeWs w;
  return (size_t)layout_ws(nullptr, T, d, f, E, k, 148, &w);
}

template <int NT, bool ONE>
static cudaError_t launch_experts(const MoeFp8Args& a, const MoeWs& w, int sms, cudaStream_t s) {
  const long long P = (long long)a.T * a.k, ew = (long long)a.d * a.f;
  MoeMaps m;
  if (encode_fp8_map(&m.gate, a.gate.q, a.d, a.f, a.d, 128, a.E, ew) ||
      encode_fp8_map(&m.up, a.up.q, a.d, a.f, a.d, 128, a.E, ew) ||
      encode_fp8_map(&m.down, a.down.q, a.f, a.d, a.f, 128, a.E, ew) ||
      encode_fp8_map(&m.x, w.xq, a.d, a.T, a.d, 1, 0, 0) || encode_fp8_map(&m.h, w.hq, a.f, P, a.f, 16, 0, 0))
    return cudaErrorInvalidValue;
  auto kern = k_moe_experts<NT, ONE>;
  cudaError_t e = allow_shared<k_moe_experts<NT, ONE>>(Moe<NT>::SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(sms);
  cfg.blockDim = dim3(MOE_THREADS);
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
  // a quantising CTA per 16 groups of its share of the tokens, or per 16 KB to clear
  const int clear = TG == 1 ? (int)std::min<long long>(64, (w.words + 2047) / 2048) : 1;
  cfg.gridDim = dim3((a.E + 1) / 2 + std::max(clear, (TG * blocks128(a.d) + 15) / 16), rows);
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
  layout_ws(a.ws, a.T, a.d, a.f, a.E, a.k, sms, &w);
  cudaError_t e = a.T == 1 ? launch_route<1>(a, w, s) : a.T <= 16 ? launch_route<4>(a, w, s) : launch_route<8>(a, w, s);
  if (e != cudaSuccess) return e;
  if (a.T == 1) return launch_experts<16, true>(a, w, sms, s);
  if (a.T <= 16) return launch_experts<16, false>(a, w, sms, s);
  if (a.T <= 32) return launch_experts<32, false>(a, w, sms, s);
  return launch_experts<64, false>(a, w, sms, s);
}

// The experts' kernel over a workspace in which no token is ever routed: every
// CTA's wait for the routing runs out after its second.
cudaError_t launch_moe_fp8_lost(const MoeFp8Args& a, int sms, cudaStream_t s) {
  MoeWs w;
  layout_ws(a.ws, a.T, a.d, a.f, a.E, a.k, sms, &w);
  cudaError_t e = cudaMemsetAsync(w.next, 0, 4ll * w.counters, s);
  if (e == cudaSuccess) e = cudaMemsetAsync(w.rt_next, 0x7f, 4, s);     // beyond the last token
  if (e != cudaSuccess) return e;
  return a.T <= 16   ? launch_experts<16, false>(a, w, sms, s)
         : a.T <= 32 ? launch_experts<32, false>(a, w, sms, s)
                     : launch_experts<64, false>(a, w, sms, s);
}

cudaError_t moe_fp8_status(int** at) { return cudaGetSymbolAddress(reinterpret_cast<void**>(at), g_moe_status); }

}  // namespace ms
