// Choice of a token per row of logits from given random numbers: temperature, top-k, top-p, min-p.
//
// With m = max x, token i weighs w_i = exp((x_i - m) / T).  In the order of falling logits, equal ones by index, the first k tokens stay;
// of these the shortest beginning whose weights reach top_p of theirs; of these the ones with w_i >= min_p.  The token is the first one,
// by index, at which the running sum of what stays exceeds u times its total.
//
// A row is held in the shared memory of one cluster of up to 8 CTAs: it is read from memory once.  Every cut is a threshold on the
// logit (and, among equal ones, on the index), found by radix selection over the logits' bits, 8 at a time, without a sort.
//
// Weights are summed as integers, in units of 2^-44 of the largest one: sums do not depend on their order, so that any number of CTAs and
// any order of atomics gives the same token, and 2^18 tokens fit 63 bits.  A choice between neighbours hangs on sums that differ
// by one weight: 32-bit exponentials (1e-7 of a sum) would draw another token of a flat row of 1e5 once in some hundred rows, 2^-45 each (4e-11) once
// in 1e6 or more.  A token of less than 2^-45 of the best one's weight is never drawn.
#include "sampling.cuh"

#include <cuda_bf16.h>

#include <algorithm>

#include "tc_ptx.cuh"

namespace {

using ugb_tc::cluster_sync_all;
using ugb_tc::mapa_u32;
using ugb_tc::smem_u32;
typedef unsigned long long u64;

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 256, COPIES = 4, CLUSTER_MAX = 8;
constexpr double UNIT = 17592186044416.0;                  // 2^44

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
__device__ __forceinline__ u64 peer_u64(uint32_t addr, int rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_u32(addr, (uint32_t)rank)) : "memory");
  return v;
}

struct Shared {
  u64 warp_sum[WARPS];
  u64 total[2][BINS];                                      // by digit, of this CTA
  uint32_t lo[2][BINS * COPIES], hi[2][BINS * COPIES];
  u64 slot[16];                                            // what the peers read: one slot per exchange, none is written twice
  u64 pick[4];
};

struct Weights {
  float best;
  double inv_t;
  __device__ __forceinline__ double exact(float x) const { return x == best ? 1.0 : exp(((double)x - (double)best) * inv_t); }
  __device__ __forceinline__ u64 units(float x) const { return (u64)__double2ll_rn(exact(x) * UNIT); }
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

// The logits of one row that this cluster holds, and where a CTA stands in it.
struct Row {
  const float *x;
  int base, len, rank, size, seg;
  __device__ __forceinline__ int from() const { return min(len, (int)threadIdx.x * seg); }
  __device__ __forceinline__ int to() const { return min(len, ((int)threadIdx.x + 1) * seg); }
};

// Sum over the cluster of what the CTAs put in; `before`: that of lower ranks.
__device__ __forceinline__ u64 cluster_sum(u64 mine, const Row &r, Shared &sh, int slot, u64 *before = nullptr) {
  if (threadIdx.x == 0) sh.slot[slot] = mine;
  cluster_sync_all();
  u64 all = 0, low = 0;
  for (int c = 0; c < r.size; ++c) {
    const u64 v = peer_u64(smem_u32(&sh.slot[slot]), c);
    if (c < r.rank) low += v;
    all += v;
  }
  if (before) *before = low;
  return all;
}

// The largest key at which the running sum over falling keys reaches `target` (>= 1, at most the whole sum): its key, and the sum above it.
template <typename F>
__device__ void select_key(const Row &r, Shared &sh, u64 target, F weigh, uint32_t *key, u64 *above) {
  uint32_t prefix = 0;
  u64 over = 0;
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass, par = pass & 1;
    __syncthreads();                                       // the same buffers' last readers, two passes ago, passed a cluster barrier since
    for (int i = threadIdx.x; i < BINS * COPIES; i += THREADS) sh.lo[par][i] = sh.hi[par][i] = 0;
    __syncthreads();
    for (int i = r.from(); i < r.to(); ++i) {
      const uint32_t k = key_of(r.x[i]);
      if (pass > 0 && (k >> (shift + 8)) != prefix) continue;
      const u64 w = weigh(r.x[i], k);
      if (w == 0) continue;
      const int at = ((k >> shift) & 255u) * COPIES + (threadIdx.x & (COPIES - 1));
      const uint32_t old = atomicAdd(&sh.lo[par][at], (uint32_t)w);
      const uint32_t high = (uint32_t)(w >> 32) + (old + (uint32_t)w < old ? 1u : 0u);
      if (high) atomicAdd(&sh.hi[par][at], high);
    }
    __syncthreads();
    if (threadIdx.x < BINS) {
      u64 v = 0;
#pragma unroll
      for (int c = 0; c < COPIES; ++c) v += ((u64)sh.hi[par][threadIdx.x * COPIES + c] << 32) + sh.lo[par][threadIdx.x * COPIES + c];
      sh.total[par][threadIdx.x] = v;
    }
    cluster_sync_all();
    // every warp adds up all bins by itself: lane l those of digits 255 - 8 l downwards
    u64 v[8], mine = 0;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = 0;
      for (int c = 0; c < r.size; ++c) v[j] += peer_u64(smem_u32(&sh.total[par][255 - 8 * lane - j]), c);
      mine += v[j];
    }
    u64 run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 n = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += n;
    }
    const int owner = __ffs(__ballot_sync(0xffffffffu, over + run >= target)) - 1;
    u64 sum = over + run - mine;                           // of the digits above this lane's
    int digit = 0;
    bool found = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!found && sum + v[j] >= target) { found = true; digit = 255 - 8 * lane - j; }
      if (!found) sum += v[j];
    }
    over = __shfl_sync(0xffffffffu, sum, owner & 31);
    prefix = (prefix << 8) | (uint32_t)__shfl_sync(0xffffffffu, digit, owner & 31);
  }
  *key = prefix;
  *above = over;
}

// The first index, over the whole row, at which the running sum of the weights exceeds `target`; in every CTA.  `mine`: this thread's sum.
template <typename F>
__device__ int find_index(const Row &r, Shared &sh, u64 target, u64 mine, u64 before, F weigh, int slot, u64 *weight = nullptr) {
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
  if (low + run - mine <= target && target < low + run) {  // one thread of one CTA
    u64 sum = low + run - mine;
    for (int i = r.from(); i < r.to(); ++i) {
      const u64 w = weigh(r.x[i], r.base + i);
      sum += w;
      if (sum > target) {
        sh.slot[slot] = (u64)(r.base + i) + 1;
        sh.slot[slot + 1] = w;
        break;
      }
    }
  }
  __syncthreads();
  cluster_sync_all();
  u64 at = 0, w = 0;
  for (int c = 0; c < r.size; ++c) {
    at += peer_u64(smem_u32(&sh.slot[slot]), c);
    w += peer_u64(smem_u32(&sh.slot[slot + 1]), c);
  }
  if (weight) *weight = w;
  return (int)at - 1;
}

template <typename T> __device__ __forceinline__ float load1(const T *p) { return (float)*p; }

// grid (cluster size x rows): one cluster per row.
template <typename T>
__global__ void __launch_bounds__(THREADS)
sample_kernel(Params p, int size) {
  extern __shared__ __align__(16) float x[];
  __shared__ Shared sh;
  const int row = blockIdx.x / size, rank = blockIdx.x % size;
  Row r;
  r.x = x; r.rank = rank; r.size = size; r.seg = p.seg;
  r.base = min(p.vocab, rank * p.chunk);
  r.len = min(p.vocab - r.base, p.chunk);
  const float temperature = p.temperature ? p.temperature[row] : 1.0f, top_p = p.top_p ? p.top_p[row] : 1.0f, min_p = p.min_p ? p.min_p[row] : 0.0f;
  const float u = p.u[row];
  const int top_k = p.top_k ? p.top_k[row] : 0;
  // negated comparisons: a NaN is refused
  if (!(temperature >= 0.0f) || isinf(temperature) || top_k < 0 || !(top_p > 0.0f) || !(min_p >= 0.0f && min_p <= 1.0f) || !(u >= 0.0f && u < 1.0f)) {
    if (rank == 0 && threadIdx.x == 0 && atomicCAS(&p.status->code, 0u, (unsigned)UGB_ERR_INVALID) == 0u) p.status->detail = (unsigned)row;
    return;                                                // the whole cluster: the row is left as it was
  }
  const T *g = (const T *)p.logits + (long long)row * p.ld + r.base;
  float best = -INFINITY;
  int at = 0x7fffffff;
  auto take = [&](float v, int i) {
    v = v != v ? -INFINITY : v;                            // a NaN is no candidate
    x[i] = v;
    if (v > best || (v == best && i < at)) { best = v; at = i; }
  };
  constexpr int PER = 16 / (int)sizeof(T);
  if (((uintptr_t)g & 15) == 0) {
    for (int i = threadIdx.x * PER; i + PER <= r.len; i += THREADS * PER) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(g + i));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) take(__uint_as_float(w[j]), i + j);
        else {
          take(__uint_as_float(w[j] << 16), i + 2 * j);
          take(__uint_as_float(w[j] & 0xffff0000u), i + 2 * j + 1);
        }
      }
    }
    for (int i = r.len / PER * PER + threadIdx.x; i < r.len; i += THREADS) take(load1(g + i), i);
  } else {
    for (int i = threadIdx.x; i < r.len; i += THREADS) take(load1(g + i), i);
  }
  // the best logit, equal ones by index: the largest (key, ~index)
  u64 top = at == 0x7fffffff ? 0 : ((u64)key_of(best) << 32) | (uint32_t)~(uint32_t)(r.base + at);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) sh.warp_sum[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < WARPS; ++w) top = max(top, sh.warp_sum[w]);
    sh.slot[0] = top;
  }
  cluster_sync_all();
  top = 0;
  for (int c = 0; c < size; ++c) top = max(top, peer_u64(smem_u32(&sh.slot[0]), c));
  const uint32_t top_key = (uint32_t)(top >> 32);
  const int top_index = (int)~(uint32_t)top;
  Weights weights;
  weights.best = __uint_as_float(top_key & 0x80000000u ? top_key & 0x7fffffffu : ~top_key);
  weights.inv_t = 1.0 / (double)temperature;
  int token = top_index;
  float prob = 1.0f;
  if (weights.best == -INFINITY) {                         // nothing to choose from
    token = -1;
    prob = 0.0f;
  } else if (temperature > 0.0f) {
    uint32_t cut = 0;                                      // keys above `cut` stay, and of those at it the ones of index <= `last`
    u64 ties = 0;                                          // how many of those at it, 0: all
    if (top_k > 0 && top_k < p.vocab) {
      u64 above;
      select_key(r, sh, (u64)top_k, [](float, uint32_t) { return (u64)1; }, &cut, &above);
      ties = (u64)top_k - above;
    }
    if (top_p < 1.0f) {
      u64 sum = 0, at_cut = 0;
      for (int i = r.from(); i < r.to(); ++i) {
        const uint32_t k = key_of(x[i]);
        if (k > cut || (ties == 0 && k == cut)) sum += weights.units(x[i]);
      }
      sum = cluster_sum(block_sum(sum, sh), r, sh, 1);
      if (ties) {                                          // equal logits weigh the same
        const float c = __uint_as_float(cut & 0x80000000u ? cut & 0x7fffffffu : ~cut);
        at_cut = weights.units(c);
        sum += ties * at_cut;
      }
      const u64 target = min(sum, max((u64)1, (u64)ceil((double)top_p * (double)sum)));
      u64 above;
      uint32_t k1;
      const uint32_t k0 = cut;
      select_key(r, sh, target, [&](float v, uint32_t k) { return k >= k0 ? weights.units(v) : (u64)0; }, &k1, &above);
      cut = k1;
      const u64 w = weights.units(__uint_as_float(cut & 0x80000000u ? cut & 0x7fffffffu : ~cut));
      ties = (target - above + w - 1) / w;
    }
    int last = p.vocab;
    if (ties) {
      u64 mine = 0, before;
      for (int i = r.from(); i < r.to(); ++i) mine += key_of(x[i]) == cut ? 1 : 0;
      const u64 all = cluster_sum(block_sum(mine, sh), r, sh, 2, &before);
      if (ties < all) last = find_index(r, sh, ties - 1, mine, before, [&](float v, int) { return (u64)(key_of(v) == cut ? 1 : 0); }, 4);
    }
    const double low = (double)min_p;
    auto kept = [&](float v, int i) -> u64 {
      const uint32_t k = key_of(v);
      if (k < cut || (k == cut && i > last)) return 0;
      const double w = weights.exact(v);
      return w >= low ? (u64)__double2ll_rn(w * UNIT) : 0;
    };
    u64 mine = 0, before;
    for (int i = r.from(); i < r.to(); ++i) mine += kept(x[i], r.base + i);
    const u64 all = cluster_sum(block_sum(mine, sh), r, sh, 3, &before);
    const u64 target = min(all - 1, __umul64hi((u64)((double)u * 18446744073709551616.0), all));
    u64 w;
    token = find_index(r, sh, target, mine, before, kept, 6, &w);
    prob = (float)((double)w / (double)all);
  }
  if (rank == 0 && threadIdx.x == 0) {
    p.tokens[row] = token;
    if (p.prob) p.prob[row] = prob;
  }
  cluster_sync_all();                                      // no CTA leaves while a peer may still read its shared memory
}

template <typename T>
int32_t launch(ugb_device *dev, const Params &p, int size) {
  static bool attr_set[64] = {};
  if (!attr_set[dev->ordinal & 63]) {
    UGB_CUDA(dev, cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, UGB_SAMPLE_VOCAB_MAX / CLUSTER_MAX * 4));
    attr_set[dev->ordinal & 63] = true;
  }
  const cudaError_t e = ugb_launch_cluster(sample_kernel<T>, dim3((unsigned)(p.rows * size)), dim3(THREADS), (size_t)p.chunk * 4, dev->stream, false, size, p, size);
  if (e != cudaSuccess) return ugb_fail(dev, UGB_ERR_CUDA, "launch of sample_kernel failed: %s", cudaGetErrorString(e));
  return ugb_after_launch(dev, "sample_kernel");
}

}  // namespace

int32_t ugb_sample_rows(ugb_device *dev, const ugb_sample_args &a) {
  if (a.rows == 0) return UGB_OK;
  Params p;
  p.logits = a.logits; p.temperature = a.temperature; p.top_p = a.top_p; p.min_p = a.min_p; p.u = a.u; p.top_k = a.top_k; p.tokens = a.tokens;
  p.prob = a.prob; p.rows = a.rows; p.vocab = a.vocab; p.ld = a.ld; p.status = dev->status_dev;
  // CTAs of a row: so many that the GPU is full, and that a row leaves room for three CTAs on an SM
  int size = 1;
  while (size < CLUSTER_MAX && ((long long)a.rows * size < dev->sm_count || (a.vocab + size - 1) / size > 16384)) size *= 2;
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
  UGB_REQUIRE(dev, !ugb_overlap(logits, tokens) && !(prob && (ugb_overlap(logits, prob) || ugb_overlap(tokens, prob))), UGB_ERR_INVALID, "sample: in place");
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
