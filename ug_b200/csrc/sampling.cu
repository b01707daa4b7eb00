// Choice of a token per row of logits from given random numbers: temperature, top-k, top-p, min-p.
//
// With m = max x, token i weighs w_i = exp((x_i - m) / T).  In the order of falling logits, equal ones by index, the first k tokens stay;
// of these the shortest beginning whose weights reach top_p of theirs; of these the ones with w_i >= min_p.  The token is the first one,
// by index, at which the running sum of what stays exceeds u times its total.
//
// A row is held in the shared memory of one cluster of up to 8 CTAs: it is read from memory once.  Every cut is a threshold on the
// logit (and, among equal ones, on the index).  It is found without a sort: a histogram over the distance from the best logit, in
// steps of T / 32, says in which step the cut falls; the tokens up to that step, where they are few, are gathered and ranked against
// one another, and the whole choice is made among them; where they are many only those of that step are ranked; where these are many too
// (equal logits, a flat row), the next histogram divides the step by the logits' bits, until one logit or few tokens are left.
//
// Weights are summed as integers, in units of 2^-44 of the largest one: sums do not depend on their order, so that any number of CTAs and
// any order of atomics gives the same token, and 2^18 tokens fit 63 bits.  A weight is off by half a unit and by 9e-15 of itself, a running sum by
// less than 4e-14 of the total.  A choice between neighbours hangs on sums that differ by one weight: in a flat row of 1e5 a target lies that near a border
// once in 1e8 rows (2 x 1e5 x 4e-14), near enough for 32-bit exponentials (1e-7) to draw another token once in 50.  A token of less than 2^-45 of the best
// one's weight is never drawn.
#include "sampling.cuh"

#include <cuda_bf16.h>

#include <algorithm>

#include "tc_ptx.cuh"

namespace {

using ugb_tc::cluster_sync_all;
using ugb_tc::mapa_u32;
using ugb_tc::smem_u32;
typedef unsigned long long u64;

constexpr int THREADS = 512, WARPS = THREADS / 32, CLUSTER_MAX = 8;
constexpr int STEPS = 1024, RANKED = 256;
constexpr float STEPS_PER_T = 32.0f;                       // 1024 steps reach to exp(-32) < 2^-45: what is beyond weighs nothing
constexpr int POWER_BITS = 9, POWERS = 1 << POWER_BITS;      // as many as threads
constexpr float LOWEST_ABOVE = -3.4028232e38f;             // the second lowest value

struct Params {
  const void *logits;
  const float *temperature, *top_p, *min_p, *u;
  const int *top_k;
  int *tokens;
  float *prob;
  int rows, vocab, chunk, seg;                             // chunk: logits of a CTA; seg: of a thread (odd: no bank conflicts)
  long long ld;
  ugb_status_word *status;
};

__device__ __forceinline__ uint32_t key_of(float x) {      // ascending with the value; -0 counts as 0
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ u64 peer_u64(uint32_t addr, int rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_u32(addr, (uint32_t)rank)) : "memory");
  return v;
}

struct Shared {
  u64 warp_sum[WARPS];
  double power[POWERS];                                    // 2^(i / POWERS)
  u64 hist[STEPS];
  u64 in_step[RANKED], before_step[RANKED];                // tokens by place()
  u64 ranked[RANKED], sorted[RANKED];
  int count[THREADS];
  int n_in, n_before;
  uint32_t key_min, key_max;                               // of the step's tokens
  u64 slot[16];                                            // what the peers read: none is written twice without a cluster barrier behind the reads
  u64 pick[4];
};

// Weights, in units of 2^-44 of the best one's, by Tang's table method for the exponential: with t = 512 (x - best) log2(e) / T = n + f, |f| <= 1/2,
// 2^(t / 512) is a power from the table, shifted, times 2^(f / 512) by its series to f^3 (off by (ln 2 / 1024)^4 / 24 = 8.8e-15 of the value).
struct Weights {
  float best, lowest;
  double best_d, k;
  const double *power;
  __device__ __forceinline__ Weights(float best_, float temperature, const double *power_) : best(best_), best_d(best_), power(power_) {
    const float below = nextafterf(best, -INFINITY);
    // where the next smaller value weighs nothing already, a larger T does not change that, and keeps t within the integers
    const double t = fmax((double)temperature, (best_d - (double)below) / 64.0);
    k = POWERS * 1.4426950408889634 / t;
    lowest = fmaxf(fminf(best - 64.0f * temperature, below), -3.4028234e38f);         // exp(-42) and less from here on, rounding included; -inf too
    per_unit = (float)fmin(STEPS_PER_T / t, 3.0e38);
  }
  float per_unit;                                          // steps of the histogram per unit of the logit
  __device__ __forceinline__ u64 units(float x) const {
    const double d = (double)fmaxf(x, lowest) - best_d;
    const double shifted = fma(d, k, 6755399441055744.0);  // + 1.5 * 2^52: the integer is in the low bits
    const double f = fma(d, k, 6755399441055744.0 - shifted);
    const int n = __double2loint(shifted);
    constexpr double C = 0.69314718055994531 / POWERS;
    double e = fma(f, C * C * C / 6.0, C * C / 2.0);
    e = fma(e, f, C);
    e = fma(e, f, 1.0);
    const double w = power[n & (POWERS - 1)];
    // + 2^8, whose last place is 2^-44
    e = fma(__hiloint2double(__double2hiint(w) + ((n >> POWER_BITS) << 20), __double2loint(w)), e, 256.0);
    return ((u64)(uint32_t)(__double2hiint(e) - 0x40700000) << 32) | (uint32_t)__double2loint(e);
  }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the CTA, to every thread.
__device__ __forceinline__ u64 block_sum(u64 v, Shared &sh) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.warp_sum[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh.warp_sum[threadIdx.x & (WARPS - 1)];
#pragma unroll
  for (int o = WARPS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Order of a token: falling logit, then rising index.  A larger place comes first.
__device__ __forceinline__ u64 place(uint32_t key, int index) { return ((u64)key << 32) | (uint32_t)~(uint32_t)index; }
__device__ __forceinline__ uint32_t key_at(u64 place) { return (uint32_t)(place >> 32); }
__device__ __forceinline__ int index_at(u64 place) { return (int)~(uint32_t)place; }

// The logits of one row that this CTA holds, and where it stands in the cluster.
template <typename T> struct Row {
  const T *x;
  int base, len, rank, size, seg;
  __device__ __forceinline__ float at(int i) const { return (float)x[i]; }
  // f(index in the CTA, logit) for this thread's share, four at a time
  template <typename F> __device__ __forceinline__ void each(F f) const {
    const int from = min(len, (int)threadIdx.x * seg), to = min(len, ((int)threadIdx.x + 1) * seg);
    int i = from;
    for (; i + 4 <= to; i += 4) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = at(i + j);
#pragma unroll
      for (int j = 0; j < 4; ++j) f(i + j, v[j]);
    }
    for (; i < to; ++i) f(i, at(i));
  }
};

// Sum over the cluster of what the CTAs put in; `before`: that of lower ranks.
template <typename T> __device__ __forceinline__ u64 cluster_sum(u64 mine, const Row<T> &r, Shared &sh, int slot, u64 *before) {
  if (threadIdx.x == 0) sh.slot[slot] = mine;
  cluster_sync_all();
  u64 v[CLUSTER_MAX], all = 0, low = 0;
#pragma unroll
  for (int c = 0; c < CLUSTER_MAX; ++c) v[c] = c < r.size ? peer_u64(smem_u32(&sh.slot[slot]), c) : 0;
#pragma unroll
  for (int c = 0; c < CLUSTER_MAX; ++c) {
    if (c < r.rank) low += v[c];
    all += v[c];
  }
  *before = low;
  return all;
}

// The first index, over the whole row, at which the running sum of the weights exceeds `target`; in every CTA.  `mine`: this thread's sum.
template <typename T, typename F>
__device__ int find_index(const Row<T> &r, Shared &sh, u64 target, u64 mine, u64 before, F weigh, int slot, u64 *weight) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 run = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += n;
  }
  __syncthreads();
  if (lane == 31) sh.warp_sum[warp] = run;
  if (threadIdx.x == 0) sh.slot[slot] = sh.slot[slot + 1] = 0;
  __syncthreads();
  u64 low = before;
  for (int w = 0; w < warp; ++w) low += sh.warp_sum[w];
  const uint32_t owner = __ballot_sync(0xffffffffu, low + run - mine <= target && target < low + run);
  if (owner) {                                             // one thread of one CTA: its warp looks through its share together
    const int src = __ffs(owner) - 1, first = (warp * 32 + src) * r.seg, end = min(r.len, first + r.seg);
    u64 sum = __shfl_sync(0xffffffffu, low + run - mine, src);
    for (int i0 = first; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      const u64 w = i < end ? weigh(r.at(i), r.base + i) : 0;
      u64 upto = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 n = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += n;
      }
      const uint32_t over = __ballot_sync(0xffffffffu, sum + upto > target);
      if (over) {
        if (lane == __ffs(over) - 1) {
          sh.slot[slot] = (u64)(r.base + i) + 1;
          sh.slot[slot + 1] = w;
        }
        break;
      }
      sum += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  cluster_sync_all();
  u64 at = 0, w = 0;
  for (int c = 0; c < r.size; ++c) {
    at += peer_u64(smem_u32(&sh.slot[slot]), c);
    w += peer_u64(smem_u32(&sh.slot[slot + 1]), c);
  }
  if (weight) *weight = w;
  return (int)at - 1;
}

// Into which of STEPS steps a token falls, by falling logit; STEPS: beyond all, -1: before all.
struct ByDistance {                                        // from the best logit; rounding keeps the order
  float best, per_unit;
  __device__ __forceinline__ int of(float x) const {
    const float d = (best - x) * per_unit;
    return d < (float)STEPS ? (int)d : STEPS;
  }
  __device__ __forceinline__ bool behind(float x, int step) const { return (best - x) * per_unit >= (float)(step + 1); }
};
struct ByKey {                                             // of the keys min .. max
  uint32_t max;
  int shift;
  float low, high;                                         // their values
  __device__ __forceinline__ int of(float x) const { return x > high ? -1 : x < low ? STEPS : (int)((max - key_of(x)) >> shift); }
  __device__ __forceinline__ bool behind(float x, int step) const { return x < low || (x <= high && (int)((max - key_of(x)) >> shift) > step); }
};

// Adds weigh(logit, index) of the tokens of all steps to the histogram, over the cluster, and finds the step in which the running sum reaches the
// target that `goal` makes of the whole sum.  Returns the step (STEPS: it is not reached); above: the sum before it, within: its own.
template <typename T, typename S, typename F, typename G>
__device__ int find_step(const Row<T> &r, Shared &sh, const S &steps, F weigh, G goal, u64 *above, u64 *within, u64 *whole, u64 *target) {
  for (int i = threadIdx.x; i < STEPS; i += THREADS) sh.hist[i] = 0;
  if (threadIdx.x == 0) {
    sh.n_in = sh.n_before = 0;
    sh.key_min = 0xffffffffu;
    sh.key_max = 0;
  }
  __syncthreads();
  r.each([&](int i, float v) {
    const int at = steps.of(v);
    const u64 w = at < 0 || at >= STEPS ? 0 : weigh(v, r.base + i);
    if (w) {
      uint32_t *h = reinterpret_cast<uint32_t *>(&sh.hist[at]);        // 64 bits in two halves: shared memory adds 32 at a time
      const uint32_t old = atomicAdd(h, (uint32_t)w);
      const uint32_t high = (uint32_t)(w >> 32) + (old + (uint32_t)w < old ? 1u : 0u);
      if (high) atomicAdd(h + 1, high);
    }
  });
  cluster_sync_all();
  constexpr int PER = STEPS / THREADS;
  u64 v[PER], mine = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    u64 c[CLUSTER_MAX];
#pragma unroll
    for (int k = 0; k < CLUSTER_MAX; ++k) c[k] = k < r.size ? peer_u64(smem_u32(&sh.hist[threadIdx.x * PER + j]), k) : 0;
    v[j] = 0;
#pragma unroll
    for (int k = 0; k < CLUSTER_MAX; ++k) v[j] += c[k];
    mine += v[j];
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 run = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += n;
  }
  if (lane == 31) sh.warp_sum[warp] = run;
  if (threadIdx.x == 0) sh.pick[0] = STEPS;
  __syncthreads();
  u64 all = 0, low = run - mine;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) low += sh.warp_sum[w];
    all += sh.warp_sum[w];
  }
  *whole = all;
  const u64 t = goal(all);
  *target = t;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (low < t && t <= low + v[j]) {
      sh.pick[0] = (u64)(threadIdx.x * PER + j);
      sh.pick[1] = low;
      sh.pick[2] = v[j];
    }
    low += v[j];
  }
  __syncthreads();
  *above = sh.pick[1];
  *within = sh.pick[2];
  return (int)sh.pick[0];
}

// Lists the tokens of step `in` and (before) of the steps before it, up to RANKED of each kind, every CTA its own.  n_in, n_before: how many there
// are in the cluster (more than RANKED: that many or more); mine: this thread's tokens of the step; min, max: the keys of the step's.
template <typename T, typename S, typename F>
__device__ void gather(const Row<T> &r, Shared &sh, const S &steps, int in, bool before, F valid, int slot, int *n_in, int *n_before, int *mine, uint32_t *min_key,
                       uint32_t *max_key) {
  float low = INFINITY, high = -INFINITY;
  int count = 0;
  r.each([&](int i, float x) {
    if (steps.behind(x, in) || !valid(x, r.base + i)) return;
    const bool here = steps.of(x) == in;
    if (here) { low = fminf(low, x); high = fmaxf(high, x); ++count; }
    if (!here && !before) return;
    int *n = here ? &sh.n_in : &sh.n_before;
    if (*reinterpret_cast<volatile int *>(n) > RANKED) return;
    const int j = atomicAdd(n, 1);
    if (j < RANKED) (here ? sh.in_step : sh.before_step)[j] = place(key_of(x), r.base + i);
  });
  *mine = count;
  uint32_t lo = count ? key_of(low) : 0xffffffffu, hi = count ? key_of(high) : 0;
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if ((threadIdx.x & 31) == 0) {
    atomicMin(&sh.key_min, lo);
    atomicMax(&sh.key_max, hi);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    sh.slot[slot] = ((u64)(uint32_t)sh.n_before << 32) | (uint32_t)sh.n_in;
    sh.slot[slot + 1] = ((u64)sh.key_max << 32) | sh.key_min;
  }
  cluster_sync_all();
  *n_in = *n_before = 0;
  lo = 0xffffffffu;
  hi = 0;
  for (int c = 0; c < r.size; ++c) {
    const u64 v = peer_u64(smem_u32(&sh.slot[slot]), c), k = peer_u64(smem_u32(&sh.slot[slot + 1]), c);
    *n_in += (int)(uint32_t)v;
    *n_before += (int)(v >> 32);
    lo = min(lo, (uint32_t)k);
    hi = max(hi, (uint32_t)(k >> 32));
  }
  *min_key = lo;
  *max_key = hi;
}

// Copies the peers' lists (both, or those of the step alone) together.  At most RANKED tokens, the caller has seen to that.
template <typename T> __device__ void collect(const Row<T> &r, Shared &sh, int slot, bool both) {
  int at = 0;
  for (int c = 0; c < r.size; ++c) {
    const u64 v = peer_u64(smem_u32(&sh.slot[slot]), c);
    const int n_in = (int)(uint32_t)v, n = n_in + (both ? (int)(v >> 32) : 0);
    if ((int)threadIdx.x < n) sh.ranked[at + threadIdx.x] = peer_u64(smem_u32((int)threadIdx.x < n_in ? &sh.in_step[threadIdx.x] : &sh.before_step[threadIdx.x - n_in]), c);
    at += n;
  }
  __syncthreads();
}

// sh.ranked[0 .. n) -> sh.sorted, the largest first.  THREADS / RANKED threads count what is ahead of a value.
__device__ __forceinline__ void sort_ranked(Shared &sh, int n) {
  const int i = threadIdx.x & (RANKED - 1);
  const u64 me = i < n ? sh.ranked[i] : 0;
  int ahead = 0;
  if (i < n) {
#pragma unroll 4
    for (int j = threadIdx.x / RANKED; j < n; j += THREADS / RANKED) ahead += sh.ranked[j] > me ? 1 : 0;
  }
  sh.count[threadIdx.x] = ahead;
  __syncthreads();
  if ((int)threadIdx.x < n) {
#pragma unroll
    for (int k = 1; k < THREADS / RANKED; ++k) ahead += sh.count[threadIdx.x + k * RANKED];
    sh.sorted[ahead] = me;
  }
  __syncthreads();
}

// Sum of the values of the threads before this one.
__device__ __forceinline__ u64 block_before(u64 v, Shared &sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 run = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += n;
  }
  __syncthreads();
  if (lane == 31) sh.warp_sum[warp] = run;
  __syncthreads();
  u64 low = run - v;
  for (int w = 0; w < warp; ++w) low += sh.warp_sum[w];
  return low;
}

__device__ __forceinline__ float load1(const float *p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16 *p) { return (float)*p; }

// grid (cluster size x rows): one cluster per row.
template <typename T>
__global__ void __launch_bounds__(THREADS)
sample_kernel(Params p, int size) {
  extern __shared__ __align__(16) unsigned char held[];
  T *x = reinterpret_cast<T *>(held);
  __shared__ Shared sh;
  const int row = blockIdx.x / size, me = blockIdx.x % size;
  Row<T> r;
  r.x = x; r.rank = me; r.size = size; r.seg = p.seg;
  r.base = min(p.vocab, me * p.chunk);
  r.len = min(p.vocab - r.base, p.chunk);
  const float temperature = p.temperature ? p.temperature[row] : 1.0f, top_p = p.top_p ? p.top_p[row] : 1.0f, min_p = p.min_p ? p.min_p[row] : 0.0f;
  const float u = p.u[row];
  const int top_k = p.top_k ? p.top_k[row] : 0;
  // negated comparisons: a NaN is refused
  if (!(temperature >= 0.0f && temperature <= 1e20f) || top_k < 0 || !(top_p > 0.0f) || !(min_p >= 0.0f && min_p <= 1.0f) || !(u >= 0.0f && u < 1.0f)) {
    if (me == 0 && threadIdx.x == 0 && atomicCAS(&p.status->code, 0u, (unsigned)UGB_ERR_INVALID) == 0u) p.status->detail = (unsigned)row;
    return;                                                // the whole cluster: the row is left as it was
  }
  const T *g = (const T *)p.logits + (long long)row * p.ld + r.base;
  // NaN becomes -inf, which is no candidate: a maximum ignores it
  float best = -INFINITY;
  constexpr int PER = 16 / (int)sizeof(T);
  if (((uintptr_t)g & 15) == 0) {
    for (int i = threadIdx.x * PER; i + PER <= r.len; i += THREADS * PER) {
      uint4 v = __ldcs(reinterpret_cast<const uint4 *>(g + i));
      uint32_t *w = &v.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          const float f = fmaxf(__uint_as_float(w[j]), -INFINITY);
          w[j] = __float_as_uint(f);
          best = fmaxf(best, f);
        } else {
          const float a = fmaxf(__uint_as_float(w[j] << 16), -INFINITY), b = fmaxf(__uint_as_float(w[j] & 0xffff0000u), -INFINITY);
          w[j] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
          best = fmaxf(best, fmaxf(a, b));
        }
      }
      *reinterpret_cast<uint4 *>(x + i) = v;
    }
    for (int i = r.len / PER * PER + threadIdx.x; i < r.len; i += THREADS) {
      const float f = fmaxf(load1(g + i), -INFINITY);
      x[i] = (T)f;
      best = fmaxf(best, f);
    }
  } else {
    for (int i = threadIdx.x; i < r.len; i += THREADS) {
      const float f = fmaxf(load1(g + i), -INFINITY);
      x[i] = (T)f;
      best = fmaxf(best, f);
    }
  }
  static_assert(POWERS == THREADS, "one power per thread");
  sh.power[threadIdx.x] = exp2(threadIdx.x / (double)POWERS);
  uint32_t top = __reduce_max_sync(0xffffffffu, key_of(best));
  if ((threadIdx.x & 31) == 0) sh.warp_sum[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x < 32) {
    top = __reduce_max_sync(0xffffffffu, threadIdx.x < WARPS ? (uint32_t)sh.warp_sum[threadIdx.x] : 0);
    if (threadIdx.x == 0) sh.slot[0] = top;
  }
  cluster_sync_all();
  top = 0;
#pragma unroll
  for (int c = 0; c < CLUSTER_MAX; ++c)
    if (c < size) top = max(top, (uint32_t)peer_u64(smem_u32(&sh.slot[0]), c));
  best = value_of(top);
  int token = -1;
  float prob = 0.0f;
  if (best == -INFINITY) {                                 // nothing to choose from
  } else if (temperature == 0.0f) {
    u64 mine = 0, before;                                  // the first of the best ones
    r.each([&](int, float v) { mine += v == best ? 1 : 0; });
    cluster_sum(block_sum(mine, sh), r, sh, 11, &before);
    token = find_index(r, sh, 0, mine, before, [&](float v, int) { return (u64)(v == best ? 1 : 0); }, 12, nullptr);
    prob = 1.0f;
  } else {
    if (best == INFINITY || best < LOWEST_ABOVE) {         // infinitely better than the others, or these are -inf: equal ones weigh the same
      r.each([&](int i, float v) { x[i] = (T)(v == best ? 0.0f : -INFINITY); });          // a thread's own share: other threads read it behind barriers
      best = 0.0f;
    }
    const Weights weights(best, temperature, sh.power);
    const u64 low = min_p > 0.0f ? (u64)ceil((double)min_p * 17592186044416.0) : 0;       // 2^44 units
    auto share_of = [&](u64 sum) { return min(sum, max((u64)1, (u64)ceil((double)top_p * (double)sum))); };
    auto drawn = [&](u64 sum) { return min(sum - 1, __umul64hi((u64)((double)u * 18446744073709551616.0), sum)); };
    const bool by_k = top_k > 0 && top_k < p.vocab, by_p = top_p < 1.0f;
    // behind this step everything weighs less than min_p (a step more, for the rounding of both sides)
    const int low_step = min_p > 0.0f ? min(STEPS - 1, (int)(-logf(min_p) * STEPS_PER_T) + 1) : STEPS - 1;
    float cut = -INFINITY;                                 // tokens above it stay, and of those at it the ones up to index `last`
    int last = p.vocab;
    auto stays = [&](float v, int i) { return v > cut || (v == cut && i <= last); };
    // The choice among n ranked tokens, all that can be chosen; sum: what top_p is a share of, unless that is the first top_k.  CTA 0 alone.
    auto finish = [&](int n, bool first_k, u64 sum) {
      sort_ranked(sh, n);
      const u64 e = (int)threadIdx.x < n ? sh.sorted[threadIdx.x] : 0;
      const u64 units = (int)threadIdx.x < n ? weights.units(value_of(key_at(e))) : 0;
      bool in = (int)threadIdx.x < n && (!first_k || (int)threadIdx.x < top_k);
      if (by_p) {
        const u64 w = in ? units : 0;
        if (first_k) sum = block_sum(w, sh);
        const u64 before = block_before(w, sh);            // a barrier: by every thread, whatever `in` is
        in = in && before < share_of(sum);
      }
      in = in && units >= low;
      // what stays is a beginning: its tokens by index, the lowest first
      const int m = __syncthreads_count(in);
      if (in) sh.ranked[threadIdx.x] = ((u64)(uint32_t)~(uint32_t)index_at(e) << 32) | key_at(e);
      __syncthreads();
      sort_ranked(sh, m);
      const u64 f = (int)threadIdx.x < m ? sh.sorted[threadIdx.x] : 0;
      const u64 w = (int)threadIdx.x < m ? weights.units(value_of((uint32_t)f)) : 0;
      const u64 all = block_sum(w, sh), before = block_before(w, sh), target = drawn(all);
      if (before <= target && target < before + w) {
        p.tokens[row] = (int)~(uint32_t)(f >> 32);
        if (p.prob) p.prob[row] = (float)((double)w / (double)all);
      }
    };
    bool done = false;
    // Finds the cut at which the running sum of weigh over the tokens that stay reaches a target, or makes the choice.
    auto narrow = [&](auto weigh, auto goal, bool first_k, int slot) {
      const ByDistance steps{best, weights.per_unit};
      u64 above, within, whole, target;
      int n_in, n_before, own;
      uint32_t key_min, key_max;
      const int step = find_step(r, sh, steps, weigh, goal, &above, &within, &whole, &target);
      const bool beyond = step == STEPS;                   // fewer tokens weigh anything than top_k: all of them stay
      const int in = min(beyond ? STEPS - 1 : step, by_p && first_k ? STEPS - 1 : low_step);   // top_p after top_k needs all the first top_k
      gather(r, sh, steps, in, true, stays, slot, &n_in, &n_before, &own, &key_min, &key_max);
      if (n_in + n_before <= RANKED) {
        if (me == 0) collect(r, sh, slot, true);
        cluster_sync_all();                                // the others leave
        if (me == 0) finish(n_in + n_before, first_k, whole);
        done = true;
        return;
      }
      if (beyond || in < step) return;                     // this cut takes away nothing that the next ones or min_p leave
      for (;;) {
        if (n_in <= RANKED) {
          collect(r, sh, slot, false);
          sort_ranked(sh, n_in);
          const u64 e = (int)threadIdx.x < n_in ? sh.sorted[threadIdx.x] : 0;
          const u64 w = (int)threadIdx.x < n_in ? weigh(value_of(key_at(e)), index_at(e)) : 0, sum = above + block_before(w, sh);
          if (sum < target && target <= sum + w) sh.pick[3] = e;
          __syncthreads();
          cut = value_of(key_at(sh.pick[3]));
          last = index_at(sh.pick[3]);
          break;
        }
        if (key_min == key_max) {                          // equal logits, which weigh the same: by index
          const u64 w = first_k ? 1 : weights.units(value_of(key_min)), ties = (target - above + w - 1) / w;
          const float level = value_of(key_min);
          auto tied = [&](float v, int i) { return (u64)(v == level && stays(v, i) ? 1 : 0); };
          u64 before;
          cluster_sum(block_sum((u64)own, sh), r, sh, slot + 2, &before);
          last = find_index(r, sh, ties - 1, (u64)own, before, tied, slot + 3, nullptr);
          cut = level;
          break;
        }
        const ByKey keys{key_max, max(0, 22 - __clz(key_max - key_min)), value_of(key_min), value_of(key_max)};       // (max - min) >> shift < 1024
        const u64 over = above;
        const int at = find_step(r, sh, keys, weigh, [&](u64) { return target - over; }, &above, &within, &whole, &target);
        above += over;
        target += over;
        gather(r, sh, keys, at, false, stays, slot, &n_in, &n_before, &own, &key_min, &key_max);
      }
      __syncthreads();
    };
    if (by_k) narrow([&](float, int) { return (u64)1; }, [&](u64) { return (u64)top_k; }, true, 1);
    if (!done && by_p) narrow([&](float v, int i) { return stays(v, i) ? weights.units(v) : (u64)0; }, share_of, false, 6);
    if (done) return;
    auto kept = [&](float v, int i) -> u64 {
      const u64 w = weights.units(v);
      return stays(v, i) && w >= low ? w : 0;
    };
    u64 mine = 0, before, w;
    r.each([&](int i, float v) { mine += kept(v, r.base + i); });
    const u64 all = cluster_sum(block_sum(mine, sh), r, sh, 11, &before);
    token = find_index(r, sh, drawn(all), mine, before, kept, 12, &w);
    prob = (float)((double)w / (double)all);
  }
  if (me == 0 && threadIdx.x == 0) {
    p.tokens[row] = token;
    if (p.prob) p.prob[row] = prob;
  }
  cluster_sync_all();                                      // no CTA leaves while a peer may still read its shared memory
}

template <typename T>
int32_t launch(ugb_device *dev, const Params &p, int size) {
  static bool attr_set[64] = {};
  if (!attr_set[dev->ordinal & 63]) {
    UGB_CUDA(dev, cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 161 * 1024));
    attr_set[dev->ordinal & 63] = true;
  }
  const cudaError_t e = ugb_launch_cluster(sample_kernel<T>, dim3((unsigned)(p.rows * size)), dim3(THREADS), (size_t)p.chunk * sizeof(T), dev->stream, false, size, p, size);
  if (e != cudaSuccess) return ugb_fail(dev, UGB_ERR_CUDA, "launch of sample_kernel failed: %s", cudaGetErrorString(e));
  return ugb_after_launch(dev, "sample_kernel");
}

}  // namespace

int32_t ugb_sample_rows(ugb_device *dev, const ugb_sample_args &a) {
  if (a.rows == 0) return UGB_OK;
  Params p;
  p.logits = a.logits; p.temperature = a.temperature; p.top_p = a.top_p; p.min_p = a.min_p; p.u = a.u; p.top_k = a.top_k; p.tokens = a.tokens;
  p.prob = a.prob; p.rows = a.rows; p.vocab = a.vocab; p.ld = a.ld; p.status = dev->status_dev;
  // CTAs of a row: 4 where rows alone do not fill the GPU or are long, so that two and more share an SM; 8 only where 4 cannot hold it, since every exchange
  // in a cluster costs more the larger it is (1 x 32000 in 1 / 2 / 4 / 8 CTAs 20.9 / 16.4 / 15.6 / 19.8 us, 64 x 32000 44.4 / 30.6 / 28.0 / 49.6, 256 x 131072
  // bf16 in 2 / 4 / 8 370 / 284 / 450)
  int size = 1;
  while (size < 4 && ((long long)a.rows * size < 4LL * dev->sm_count || (a.vocab + size - 1) / size > 8192)) size *= 2;
  if ((long long)(a.vocab / size) * (a.bf16 ? 2 : 4) > 160 * 1024) size = CLUSTER_MAX;
  p.chunk = ((a.vocab + size - 1) / size + 15) / 16 * 16;
  p.seg = (p.chunk + THREADS - 1) / THREADS | 1;
  return a.bf16 ? launch<__nv_bfloat16>(dev, p, size) : launch<float>(dev, p, size);
}

extern "C" int32_t ugb_sample(ugb_device *dev, const ugb_slice *logits, const ugb_slice *temperature, const ugb_slice *top_k, const ugb_slice *top_p,
                              const ugb_slice *min_p, const ugb_slice *u, ugb_slice *tokens, ugb_slice *prob, size_t rows, size_t vocab, size_t ld) {
  if (!dev) return UGB_ERR_INVALID;
  UGB_REQUIRE(dev, logits, UGB_ERR_INVALID, "sample: null slice");
  UGB_REQUIRE(dev, logits->dtype == UGB_F32 || logits->dtype == UGB_BF16, UGB_ERR_DTYPE, "sample: logits must be F32 or BF16, got %s", ugb_dtype_name(logits->dtype));
  UGB_REQUIRE(dev, vocab >= 1 && ld >= vocab, UGB_ERR_SHAPE, "sample: %zu logits in rows of %zu", vocab, ld);
  UGB_REQUIRE(dev, vocab <= (size_t)UGB_SAMPLE_VOCAB_MAX && rows <= (1u << 20) && ld <= (1ull << 40), UGB_ERR_UNSUPPORTED, "sample: %zu rows of %zu logits, at most %d of %d", rows, vocab,
              1 << 20, UGB_SAMPLE_VOCAB_MAX);
  UGB_SLICE(dev, logits, logits->dtype, rows ? (rows - 1) * ld + vocab : 0);
  if (temperature) UGB_SLICE(dev, temperature, UGB_F32, rows);
  if (top_k) UGB_SLICE(dev, top_k, UGB_I32, rows);
  if (top_p) UGB_SLICE(dev, top_p, UGB_F32, rows);
  if (min_p) UGB_SLICE(dev, min_p, UGB_F32, rows);
  UGB_SLICE(dev, u, UGB_F32, rows);
  UGB_SLICE(dev, tokens, UGB_I32, rows);
  if (prob) UGB_SLICE(dev, prob, UGB_F32, rows);
  const ugb_span chosen = ugb_used(tokens, rows), share = ugb_used(prob, rows);
  UGB_REQUIRE(dev, !ugb_overlap({chosen, share}, {ugb_used(logits, rows ? (rows - 1) * ld + vocab : 0)}), UGB_ERR_INVALID, "sample: in place");
  // a row reads its own setting before it writes in its place; a shifted one belongs to another row, which may come later
  for (const ugb_slice *x : {temperature, top_k, top_p, min_p, u})
    for (const ugb_span &y : {chosen, share})
      UGB_REQUIRE(dev, !ugb_overlap(y, ugb_used(x, rows)) || y.from == (uintptr_t)x->ptr, UGB_ERR_INVALID, "sample: an output over other rows' settings");
  if (rows == 0) return UGB_OK;
  UGB_CUDA(dev, cudaSetDevice(dev->ordinal));
  ugb_sample_args a;
  a.logits = logits->ptr; a.bf16 = logits->dtype == UGB_BF16;
  a.temperature = temperature ? (const float *)temperature->ptr : nullptr; a.top_k = top_k ? (const int *)top_k->ptr : nullptr;
  a.top_p = top_p ? (const float *)top_p->ptr : nullptr; a.min_p = min_p ? (const float *)min_p->ptr : nullptr;
  a.u = (const float *)u->ptr; a.tokens = (int *)tokens->ptr; a.prob = prob ? (float *)prob->ptr : nullptr;
  a.rows = (int)rows; a.vocab = (int)vocab; a.ld = (long long)ld;
  return ugb_sample_rows(dev, a);
}
