// Attention of new positions over a sliding window and the first positions of a cache, or over the cache and their ancestors in a
// tree (ugb_window_attend, ugb_tree_attend; see masked_attention.cuh).
//
//   masked_attention_tc_kernel        (masked_attention_tc.cu) bf16 heads of up to 128 values
//   masked_attention_generic_kernel   f32, other heads, unaligned buffers: plain FFMA over tiles of 64 keys
//   masked_combine_kernel             joins the slices of the keys that ran as separate CTAs
//
// One pass over the keys with the running maximum and sum of the softmax, in 32 bits, in powers of two.
#include "masked_attention.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

namespace {

using namespace ugb_masked;

constexpr float LOG2E = 1.4426950408889634f;

using Params = ugb_masked_params;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Whether sequence s is to be computed; raises the status word where its position or its tree is invalid.  By a whole block, and the parents are in `up`
// behind it.
template <bool TREE> __device__ __forceinline__ bool check_sequence(const ugb_mask &m, int s, int pos, int *up, ugb_status_word *status) {
  bool bad = pos < 0 || pos > m.t_max - m.t;
  if constexpr (TREE) {
    for (int j = threadIdx.x; j < m.t; j += blockDim.x) {
      const int a = m.parents[(size_t)s * m.t + j];
      up[j] = a;
      bad |= a < -1 || a >= j;
    }
  }
  bad = __syncthreads_or(bad);
  if (pos == -1) return false;
  if (bad && threadIdx.x == 0) raise_invalid(status, s);
  return !bad;
}

// ------------------------------------------------------------- generic ------
// grid (row tiles, key / value heads x sequences, slices), 256 threads as 16 x 16: rows ty * RM + i, keys tx + 16 j, columns 4 tx + 64 c.  The keys
// that the rows see form one list, without the gap between the first ones and the window, cut into tiles of 64.
// Shared memory, all f32: queries [16 RM][dq + 4], keys [64][dq + 4], values [64][dv + 4], probabilities [16 RM][64 + 4].  The products' operands
// come from there four columns at a time (rows apart by an odd multiple of 16 bytes: no bank conflicts).  COPIES: f32 rows that are aligned are copied
// by cp.async, the keys of the next tile behind this one's scores, the values beside them.  A weight of 0 times an infinite value is NaN: a CTA whose sums are not
// finite goes through its keys again and leaves the products of rows with keys that they do not see out, one by one, in tiles with such values.
constexpr int KEYS = 64;
__device__ __forceinline__ void copy16(float *dst, const float *src, bool valid) {      // zeros if not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <typename T, int RM, int NC, bool TREE, bool COPIES>
__global__ void __launch_bounds__(256, NC == 1 ? 3 : 2)
masked_attention_generic_kernel(Params p) {
  constexpr int TR = 16 * RM, PLD = KEYS + 4;
  extern __shared__ __align__(16) float gsm[];
  __shared__ int up[TREE ? UGB_TREE_MAX : 1];
  __shared__ uint32_t bits[TREE ? TR * 4 : 1];             // of a row: which nodes its node sees
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, dq = p.dq, dv = p.dv, kld = dq + 4, vld = dv + 4;
  float *qs = gsm, *ks = qs + TR * kld, *vs = ks + KEYS * kld, *ps = vs + KEYS * vld;
  const int s = blockIdx.y / p.kv_heads, kvh = blockIdx.y % p.kv_heads, row0 = blockIdx.x * TR, n_rows = min(TR, p.rows - row0);
  const int pos = p.mask.pos[s];
  if (!check_sequence<TREE>(p.mask, s, pos, up, p.status)) {
    if (p.splits > 1 && blockIdx.z == 0 && (int)threadIdx.x < n_rows) p.part_ml[(size_t)blockIdx.y * p.rows + row0 + threadIdx.x] = make_float2(NAN, 0.f);
    return;
  }
  if constexpr (TREE) {
    for (int r = threadIdx.x; r < TR; r += 256) {
      uint32_t w[4] = {0, 0, 0, 0};
      if (r < n_rows)
        for (int j = (row0 + r) / p.share; j >= 0; j = up[j]) w[j >> 5] |= 1u << (j & 31);
#pragma unroll
      for (int e = 0; e < 4; ++e) bits[r * 4 + e] = w[e];
    }
  }
  const T *q = (const T *)p.q, *k = (const T *)p.k + ((size_t)s * p.kv_heads + kvh) * p.mask.t_max * dq, *v = (const T *)p.v + ((size_t)s * p.kv_heads + kvh) * p.mask.t_max * dv;
  const int i0 = row0 / p.share, i1 = (row0 + n_rows - 1) / p.share;
  const Span span = span_of<TREE>(p.mask, pos, i0, i1);
  const int n_keys = span.first + span.end - span.from, tiles = (n_keys + KEYS - 1) / KEYS;
  const int per = (tiles + p.splits - 1) / p.splits, first = blockIdx.z * per, last = min(tiles, first + per);
  auto key_of = [&](int at) { return at < span.first ? at : span.from + at - span.first; };      // position of a place in the list
  // rows of 64 places of the list, 16 lanes a row
  auto fetch = [&](const T *src, int d, float *dst, int ld, int tile) {
    for (int r = ty; r < KEYS; r += 16) {
      const int at = tile * KEYS + r;
      const bool valid = at < n_keys;
      const T *x = src + (size_t)(valid ? key_of(at) : 0) * d;
      if constexpr (COPIES) {
        for (int c = 4 * tx; c < d; c += 64) copy16(dst + r * ld + c, x + c, valid);
      } else {
        for (int c = tx; c < d; c += 16) dst[r * ld + c] = valid ? (float)x[c] : 0.f;
      }
    }
    if constexpr (COPIES) copies_commit();
  };
  if (first < last) fetch(k, dq, ks, kld, first);
  for (int r = ty; r < TR; r += 16) {
    const int row = row0 + r;
    const T *x = q + (((size_t)s * p.mask.t + row / p.share) * p.heads + kvh * p.share + row % p.share) * dq;
    for (int c = tx; c < dq; c += 16) qs[r * kld + c] = r < n_rows ? (float)x[c] * p.scale : 0.f;
  }
  float m[RM], l[RM], o[RM][4 * NC];
  int at[RM];                                              // absolute position of a row's query
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    at[i] = pos + (row0 + ty * RM + i) / p.share;
#pragma unroll
    for (int c = 0; c < 4 * NC; ++c) o[i][c] = 0.f;
  }
  auto all_tiles = [&](auto careful) {
    for (int tile = first; tile < last; ++tile) {
      fetch(v, dv, vs, vld, tile);                           // its last readers are behind the barrier at the end of a tile
      if constexpr (COPIES) copies_wait<1>();                // the keys
      __syncthreads();
      float sc[RM][4];
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[i][j] = 0.f;
      for (int c = 0; c < dq; c += 4) {
        float4 a[RM], b[4];
#pragma unroll
        for (int i = 0; i < RM; ++i) a[i] = *reinterpret_cast<const float4 *>(qs + (ty * RM + i) * kld + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4 *>(ks + (tx + 16 * j) * kld + c);
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sc[i][j] = fmaf(a[i].x, b[j].x, sc[i][j]);
            sc[i][j] = fmaf(a[i].y, b[j].y, sc[i][j]);
            sc[i][j] = fmaf(a[i].z, b[j].z, sc[i][j]);
            sc[i][j] = fmaf(a[i].w, b[j].w, sc[i][j]);
          }
      }
      // a tile that every row sees whole, as most are, needs no mask
      const int low = key_of(tile * KEYS), high = key_of(min(tile * KEYS + KEYS, n_keys) - 1);
      const bool whole = tile * KEYS + KEYS <= n_keys && (TREE ? high < pos : high <= pos + i0 && (low > pos + i1 - p.mask.window || high < p.mask.sinks));
      auto sees = [&](int i, int place) {                    // row ty * RM + i, a place in the list
        const int key = key_of(place);
        bool on;
        if constexpr (TREE) {
          const int node = key - pos;
          on = node < 0 || (node < p.mask.t && (bits[(ty * RM + i) * 4 + (node >> 5)] >> (node & 31) & 1u));
        } else {
          on = key <= at[i] && (key > at[i] - p.mask.window || key < p.mask.sinks);
        }
        return on && place < n_keys;
      };
      if (!whole) {
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (!sees(i, tile * KEYS + tx + 16 * j)) sc[i][j] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < RM; ++i) {
        float mx = fmaxf(fmaxf(sc[i][0], sc[i][1]), fmaxf(sc[i][2], sc[i][3]));
#pragma unroll
        for (int e = 8; e > 0; e >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, e));
        const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.f : mn;       // a row may see nothing of this tile
        const float alpha = ex2(m[i] - base);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float w = ex2(sc[i][j] - base);
          sum += w;
          ps[(ty * RM + i) * PLD + tx + 16 * j] = w;
        }
        l[i] = l[i] * alpha + sum;                           // of this thread's keys; added up behind the last tile
        m[i] = mn;
#pragma unroll
        for (int c = 0; c < 4 * NC; ++c) o[i][c] *= alpha;
      }
      if constexpr (COPIES) copies_wait<0>();                // the values
      bool one_by_one = false;
      if constexpr (careful.value) {
        if (!whole)
          for (int r = ty; r < KEYS; r += 16)                // what this thread has copied
            for (int c = COPIES ? 4 * tx : tx; c < dv; c += COPIES ? 64 : 16)
#pragma unroll
              for (int e = 0; e < (COPIES ? 4 : 1); ++e) one_by_one |= !(fabsf(vs[r * vld + c + e]) < INFINITY);
        one_by_one = __syncthreads_or(one_by_one);
      } else {
        __syncthreads();
      }
      if (tile + 1 < last) fetch(k, dq, ks, kld, tile + 1);  // the scores are done with the keys
      if constexpr (careful.value) {
        if (one_by_one)
#pragma unroll 1
          for (int key = 0; key < KEYS; ++key)
#pragma unroll
            for (int i = 0; i < RM; ++i) {
              if (!sees(i, tile * KEYS + key)) continue;
              const float w = ps[(ty * RM + i) * PLD + key];
#pragma unroll
              for (int c = 0; c < 4 * NC; ++c)
                if (4 * tx + 64 * (c / 4) < dv) o[i][c] = fmaf(w, vs[key * vld + 4 * tx + 64 * (c / 4) + c % 4], o[i][c]);
            }
      }
      for (int key = one_by_one ? KEYS : 0; key < KEYS; key += 4) {
        float4 w[RM];
#pragma unroll
        for (int i = 0; i < RM; ++i) w[i] = *reinterpret_cast<const float4 *>(ps + (ty * RM + i) * PLD + key);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            if (4 * tx + 64 * c >= dv) continue;
            const float4 b = *reinterpret_cast<const float4 *>(vs + (key + e) * vld + 4 * tx + 64 * c);
#pragma unroll
            for (int i = 0; i < RM; ++i) {
              const float a = e == 0 ? w[i].x : e == 1 ? w[i].y : e == 2 ? w[i].z : w[i].w;
              o[i][4 * c] = fmaf(a, b.x, o[i][4 * c]);
              o[i][4 * c + 1] = fmaf(a, b.y, o[i][4 * c + 1]);
              o[i][4 * c + 2] = fmaf(a, b.z, o[i][4 * c + 2]);
              o[i][4 * c + 3] = fmaf(a, b.w, o[i][4 * c + 3]);
            }
          }
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
      for (int e = 8; e > 0; e >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], e);
  };
  all_tiles(std::false_type());
  bool finite = true;                                      // of rows whose weights are numbers
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int c = 0; c < 4 * NC; ++c) finite = finite && (fabsf(o[i][c]) < INFINITY || l[i] != l[i]);
  if (__syncthreads_or(!finite)) {
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < 4 * NC; ++c) o[i][c] = 0.f;
    }
    fetch(k, dq, ks, kld, first);
    all_tiles(std::true_type());
  }
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const int r = ty * RM + i, row = row0 + r;
    if (r >= n_rows) continue;
    if (p.splits == 1) {
      const float f = p.out_scale / l[i];                  // at least 1: a row sees itself; 0 where all its scores are -inf, which gives NaN
      T *out = (T *)p.out + (((size_t)s * p.mask.t + row / p.share) * p.heads + kvh * p.share + row % p.share) * dv;
#pragma unroll
      for (int c = 0; c < 4 * NC; ++c)
        if (4 * tx + 64 * (c / 4) < dv) out[4 * tx + 64 * (c / 4) + c % 4] = (T)(o[i][c] * f);
    } else {
      const size_t pair = (size_t)blockIdx.z * gridDim.y + blockIdx.y;
      if (tx == 0) p.part_ml[pair * p.rows + row] = make_float2(m[i], l[i]);
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (4 * tx + 64 * c < dv) p.part_o[(pair * (dv / 4) + tx + 16 * c) * p.rows + row] = make_float4(o[i][4 * c], o[i][4 * c + 1], o[i][4 * c + 2], o[i][4 * c + 3]);
    }
  }
}

// ------------------------------------------------------------- combine ------
// One CTA per 32 rows of a pair and 32 columns: lane = row, warp = 4 columns.  The slices in their order, whatever order they ran in.  A maximum that is
// NaN marks a row that was not computed and is left as it is.
template <typename T>
__global__ void __launch_bounds__(256)
masked_combine_kernel(Params p, int pairs) {
  __shared__ T done[32][32 + 8];
  ugb_pdl_wait();
  const int blocks = (p.rows + 31) / 32, pair = blockIdx.x / blocks, row0 = blockIdx.x % blocks * 32, n_rows = min(32, p.rows - row0);
  const int s = pair / p.kv_heads, kvh = pair % p.kv_heads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = row0 + min(lane, n_rows - 1);
  const int c = min(blockIdx.y * 8 + warp, p.dv / 4 - 1);  // four columns; the last warps repeat one where dv ends
  const size_t n = (size_t)pairs * p.rows, step = (size_t)pairs * (p.dv / 4) * p.rows;
  const float2 *ml = p.part_ml + (size_t)pair * p.rows + row;
  const float4 *o = p.part_o + ((size_t)pair * (p.dv / 4) + c) * p.rows + row;
  float m = -INFINITY, l = 0.f;
  bool left = false;
#pragma unroll 8
  for (int z = 0; z < p.splits; ++z) {
    const float x = ml[z * n].x;
    left |= x != x;
    m = fmaxf(m, x);
  }
  if (__all_sync(0xffffffffu, left)) return;               // rows of one sequence: all of them or none, in every warp
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int z = 0; z < p.splits; ++z) {
    const float2 w = ml[z * n];
    const bool some = w.x != -INFINITY || w.y != 0.f;      // otherwise nothing was seen, or written; a sum of NaN under a maximum that ignores it goes on
    const float4 v = some ? o[z * step] : make_float4(0.f, 0.f, 0.f, 0.f);
    const float f = some ? ex2(w.x - m) : 0.f;
    l = fmaf(f, w.y, l);
    acc.x = fmaf(f, v.x, acc.x); acc.y = fmaf(f, v.y, acc.y); acc.z = fmaf(f, v.z, acc.z); acc.w = fmaf(f, v.w, acc.w);
  }
  const float f = p.out_scale / l;                         // as above
  T *d = &done[lane][4 * warp];
  d[0] = (T)(acc.x * f); d[1] = (T)(acc.y * f); d[2] = (T)(acc.z * f); d[3] = (T)(acc.w * f);
  __syncthreads();
  const int column = blockIdx.y * 32 + lane;
  for (int r = warp; r < n_rows; r += 8) {
    const int i = (row0 + r) / p.share, h = (row0 + r) % p.share;
    if (column < p.dv) ((T *)p.out)[(((size_t)s * p.mask.t + i) * p.heads + kvh * p.share + h) * p.dv + column] = done[r][lane];
  }
}

size_t generic_smem(int dq, int dv, int rows) { return (size_t)((rows + KEYS) * (dq + 4) + KEYS * (dv + 4) + rows * (KEYS + 4)) * 4; }

template <typename T, int RM, int NC, bool TREE, bool COPIES> cudaError_t launch_generic(dim3 grid, size_t smem, cudaStream_t st, const Params &p) {
  static bool attr_set[64] = {};
  int ordinal = 0;
  cudaError_t e = cudaGetDevice(&ordinal);
  if (e != cudaSuccess) return e;
  if (!attr_set[ordinal & 63]) {
    e = cudaFuncSetAttribute(masked_attention_generic_kernel<T, RM, NC, TREE, COPIES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)generic_smem(256, 256, 16 * RM));
    if (e != cudaSuccess) return e;
    attr_set[ordinal & 63] = true;
  }
  masked_attention_generic_kernel<T, RM, NC, TREE, COPIES><<<grid, 256, smem, st>>>(p);
  return cudaSuccess;
}
template <typename T, int RM, bool TREE, bool COPIES> cudaError_t launch_columns(dim3 grid, size_t smem, cudaStream_t st, const Params &p) {
  if (p.dv <= 64) return launch_generic<T, RM, 1, TREE, COPIES>(grid, smem, st, p);
  if (p.dv <= 128) return launch_generic<T, RM, 2, TREE, COPIES>(grid, smem, st, p);
  return launch_generic<T, RM, 4, TREE, COPIES>(grid, smem, st, p);
}
template <typename T, bool COPIES> cudaError_t launch_rows(bool tree, int rm, dim3 grid, size_t smem, cudaStream_t st, const Params &p) {
  if (rm == 1) return tree ? launch_columns<T, 1, true, COPIES>(grid, smem, st, p) : launch_columns<T, 1, false, COPIES>(grid, smem, st, p);
  return tree ? launch_columns<T, 4, true, COPIES>(grid, smem, st, p) : launch_columns<T, 4, false, COPIES>(grid, smem, st, p);
}

// Slices of the keys, for `items` CTAs' worth of work of `tiles` tiles of 64 keys each on `slots`: what is shortest, in tiles, for the CTA that has most to do,
// where an item's start takes `start` tiles, twice that when its sums leave through memory, and joining them half a tile per slice (measured: 24 nodes
// over 2000 positions in 4 / 6 / 8 / 12 slices 22.5 / 20.5 / 18.5 / 20.5 us, 64 nodes of 16 sequences over 8192 in 1 / 2 / 4 168 / 193 / 198 us, f32 in
// 1 / 2 / 3 / 4, a block of 777, 135 / 121 / 118 / 125 us).  No more items than 16 rounds of CTAs: their sums take memory.
int slices(long long items, long long slots, int tiles, int parts, int start) {
  int best = 1;
  double least = 1e30;
  for (int s = 1; s * parts <= UGB_MASKED_SPLITS && (s == 1 || (tiles >= 2 * s && items * s <= 16 * slots)); ++s) {
    const long long rounds = (items * s + slots - 1) / slots;
    const double all = (double)rounds * ((tiles + s - 1) / s + (s > 1 ? 2 * start : start)) + (s > 1 ? 0.25 * s * (1 + parts) : 0.0);
    if (all < least) { least = all; best = s; }
  }
  return best;
}

}  // namespace

int32_t ugb_masked_attention(ugb_device *dev, const ugb_masked_attention_args &a) {
  if (a.b == 0 || a.t == 0) return UGB_OK;
  const bool tree = a.parents != nullptr;
  Params p;
  p.q = a.q; p.k = a.k; p.v = a.v; p.out = a.out;
  p.mask = ugb_mask{a.pos, a.parents, a.t, a.t_max, a.sinks, a.window};
  p.heads = a.heads; p.kv_heads = a.kv_heads; p.share = a.heads / a.kv_heads; p.rows = a.t * p.share; p.dq = a.dq; p.dv = a.dv;
  p.scale = a.scale * LOG2E; p.out_scale = a.out_scale; p.part_o = nullptr; p.part_ml = nullptr; p.status = dev->status_dev;
  const int pairs = a.b * a.kv_heads;
  const bool tc = ugb_masked_tc_takes(dev, a);
  const int rm = p.rows <= 16 ? 1 : 4, row_tiles = (p.rows + 16 * rm - 1) / (16 * rm);
  // CTAs at a time by the launch bounds.  Heads of 128 / 128 and wider fill an SM's shared memory with one CTA, so that their slices are chosen for more
  // than run (f32, 64 nodes of 32 heads on 8 over 2000 positions: 154 us in the slices chosen, 127 in those of a cache of four times the length).
  long long items = (long long)row_tiles * pairs, slots = (a.dv <= 64 ? 3LL : 2LL) * dev->sm_count;
  int parts = 1, positions = 16 * rm / p.share + 1;
  if (tc) ugb_masked_tc_shape(dev, a, &items, &slots, &parts, &positions);
  // the most keys that the rows of an item can see: their positions are on the device, so a tree over a cache that is mostly empty has more slices than its
  // keys need (24 nodes over 2000 positions in a cache of 2032 / 8192 / 32768 20.7 / 22.8 / 24.8 us, 16 x 64 over 8192 in 8256 / 32768 / 65536 162 / 162 / 195)
  const long long reach = tree ? a.t_max : std::min<long long>(a.t_max, (long long)a.window + std::min(positions, a.t) + a.sinks);
  p.splits = slices(items, slots, (int)((reach + 63) / 64), parts, tc ? 6 : 0);
  const int sums = p.splits * parts;
  const size_t n = (size_t)pairs * p.rows;
  void *work = nullptr;
  if (sums > 1) {
    UGB_CUDA(dev, ugb_malloc_async(dev, &work, (size_t)sums * n * (size_t)(a.dv + 2) * 4));
    p.part_o = (float4 *)work;
    p.part_ml = (float2 *)((float *)work + (size_t)sums * n * a.dv);
  }
  int32_t rc;
  if (tc) {
    rc = ugb_masked_tc_launch(dev, a, p);
  } else {
    const size_t smem = generic_smem(a.dq, a.dv, 16 * rm);
    const dim3 grid((unsigned)row_tiles, (unsigned)pairs, (unsigned)p.splits);
    const bool aligned = (((uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0;
    const cudaError_t e = !a.f32 ? launch_rows<__nv_bfloat16, false>(tree, rm, grid, smem, dev->stream, p)
                          : aligned ? launch_rows<float, true>(tree, rm, grid, smem, dev->stream, p) : launch_rows<float, false>(tree, rm, grid, smem, dev->stream, p);
    rc = e != cudaSuccess ? ugb_fail(dev, UGB_ERR_CUDA, "launch of masked_attention_generic_kernel failed: %s", cudaGetErrorString(e))
                          : ugb_after_launch(dev, "masked_attention_generic_kernel");
  }
  if (rc == UGB_OK && sums > 1) {
    p.splits = sums;
    const dim3 rows((unsigned)(pairs * ((p.rows + 31) / 32)), (unsigned)((a.dv + 31) / 32));
    // a dependent launch: its way to the SMs runs beside the last items' end
    const cudaError_t e = a.f32 ? ugb_launch(masked_combine_kernel<float>, rows, dim3(256), 0, dev->stream, true, p, pairs)
                                : ugb_launch(masked_combine_kernel<__nv_bfloat16>, rows, dim3(256), 0, dev->stream, true, p, pairs);
    rc = e != cudaSuccess ? ugb_fail(dev, UGB_ERR_CUDA, "launch of masked_combine_kernel failed: %s", cudaGetErrorString(e)) : ugb_after_launch(dev, "masked_combine_kernel");
  }
  if (work) cudaFreeAsync(work, dev->stream);
  return rc;
}

namespace {

int32_t attend(ugb_device *dev, const char *what, const ugb_slice *q, const ugb_slice *k, const ugb_slice *v, const ugb_slice *pos, const ugb_slice *parents,
               ugb_slice *out, size_t b, size_t t, size_t heads, size_t kv_heads, size_t dq, size_t dv, size_t t_max, size_t sinks, size_t window, float scale,
               float out_scale) {
  UGB_REQUIRE(dev, q && out, UGB_ERR_INVALID, "%s: null slice", what);
  UGB_REQUIRE(dev, q->dtype == out->dtype && (q->dtype == UGB_BF16 || q->dtype == UGB_F32), UGB_ERR_DTYPE, "%s: activations must be BF16 or F32 alike", what);
  UGB_REQUIRE(dev, kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && dq % 8 == 0 && dv % 8 == 0 && dq > 0 && dv > 0 && heads <= 65535 && b <= (1u << 20) &&
                       t_max <= (1u << 30) && t <= t_max && b * kv_heads <= 65535, UGB_ERR_SHAPE, "%s: unsupported shape", what);
  UGB_REQUIRE(dev, dq <= 256 && dv <= 256, UGB_ERR_UNSUPPORTED, "%s: heads of %zu and %zu values, at most 256", what, dq, dv);
  UGB_REQUIRE(dev, b * t * heads <= (1u << 30), UGB_ERR_UNSUPPORTED, "%s: %zu positions of %zu sequences in one call", what, t, b);
  UGB_SLICE(dev, q, q->dtype, b * t * heads * dq);
  UGB_SLICE(dev, out, q->dtype, b * t * heads * dv);
  UGB_SLICE(dev, k, q->dtype, b * kv_heads * t_max * dq);
  UGB_SLICE(dev, v, q->dtype, b * kv_heads * t_max * dv);
  UGB_SLICE(dev, pos, UGB_I32, b);
  if (parents) UGB_SLICE(dev, parents, UGB_I32, b * t);
  UGB_REQUIRE(dev, !ugb_overlap({ugb_used(out, b * t * heads * dv)}, {ugb_used(q, b * t * heads * dq), ugb_used(k, b * kv_heads * t_max * dq),
                                                                       ugb_used(v, b * kv_heads * t_max * dv), ugb_used(pos, b), ugb_used(parents, b * t)}),
              UGB_ERR_INVALID, "%s: in place", what);
  if (b == 0 || t == 0) return UGB_OK;
  UGB_CUDA(dev, cudaSetDevice(dev->ordinal));
  ugb_masked_attention_args a;
  a.f32 = q->dtype == UGB_F32;
  a.q = q->ptr; a.k = k->ptr; a.v = v->ptr; a.out = out->ptr; a.pos = (const int *)pos->ptr; a.parents = parents ? (const int *)parents->ptr : nullptr;
  a.b = (int)b; a.t = (int)t; a.heads = (int)heads; a.kv_heads = (int)kv_heads; a.dq = (int)dq; a.dv = (int)dv; a.t_max = (int)t_max;
  a.sinks = (int)std::min<size_t>(sinks, t_max); a.window = (int)std::min<size_t>(window, t_max); a.scale = scale; a.out_scale = out_scale;
  return ugb_masked_attention(dev, a);
}

}  // namespace

extern "C" int32_t ugb_window_attend(ugb_device *dev, const ugb_slice *q, const ugb_slice *k, const ugb_slice *v, const ugb_slice *pos, ugb_slice *out, size_t b,
                                     size_t t, size_t heads, size_t kv_heads, size_t dq, size_t dv, size_t t_max, size_t sinks, size_t window, float scale,
                                     float out_scale) {
  if (!dev) return UGB_ERR_INVALID;
  UGB_REQUIRE(dev, window >= 1, UGB_ERR_INVALID, "window_attend: a window of no position");
  return attend(dev, "window_attend", q, k, v, pos, nullptr, out, b, t, heads, kv_heads, dq, dv, t_max, sinks, window, scale, out_scale);
}

extern "C" int32_t ugb_tree_attend(ugb_device *dev, const ugb_slice *q, const ugb_slice *k, const ugb_slice *v, const ugb_slice *pos, const ugb_slice *parents,
                                   ugb_slice *out, size_t b, size_t t, size_t heads, size_t kv_heads, size_t dq, size_t dv, size_t t_max, float scale,
                                   float out_scale) {
  if (!dev) return UGB_ERR_INVALID;
  UGB_REQUIRE(dev, parents, UGB_ERR_INVALID, "tree_attend: null slice");
  UGB_REQUIRE(dev, t <= UGB_TREE_MAX, UGB_ERR_UNSUPPORTED, "tree_attend: %zu nodes, at most %d", t, UGB_TREE_MAX);
  return attend(dev, "tree_attend", q, k, v, pos, parents, out, b, t, heads, kv_heads, dq, dv, t_max, 0, t_max, scale, out_scale);
}
