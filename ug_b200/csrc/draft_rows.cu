// Rows of drafted nodes (ugb_tree_inputs, ugb_cache_keep).  A sequence has pos[s] committed positions; its t nodes occupy the cache
// rows behind them in the order in which they are listed, node i at row pos[s] + i, whatever its depth in the tree.
//
//   tree_inputs_kernel   rotation by depth, norm, append: a node's rotary position is pos[s] + (ancestors of it)
//   cache_keep_kernel    rows of the accepted nodes moved up behind the committed ones
//
// Both move bytes: they are bound by HBM for many rows and by one launch and one dependent chain of loads for few.
#include <cuda_bf16.h>

#include "draft_rows.cuh"

namespace {

// 8 consecutive values: one or two 16-byte accesses where VEC says that they are aligned
template <bool VEC> __device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&f)[8]) {
  static_assert(!VEC, "aligned pieces are fetched as they lie");
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)p[i];
}
template <bool VEC> __device__ __forceinline__ void load8(const float *p, float (&f)[8]) {
  if constexpr (VEC) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = p[i];
  }
}
template <bool VEC> __device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&f)[8]) {
  if constexpr (VEC) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&t);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(f[i]);
  }
}
template <bool VEC> __device__ __forceinline__ void store8(float *p, const float (&f)[8]) {
  if constexpr (VEC) {
    *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = f[i];
  }
}

// 8 values as they lie in memory, so that those of several heads can be on their way in few registers
template <typename T> struct Piece { uint4 w[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ void fetch(const T *p, Piece<T> &r) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = reinterpret_cast<const uint4 *>(p)[i];
}
__device__ __forceinline__ void unpack(const Piece<__nv_bfloat16> &r, float (&f)[8]) {
  const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const Piece<float> &r, float (&f)[8]) {
  f[0] = __uint_as_float(r.w[0].x); f[1] = __uint_as_float(r.w[0].y); f[2] = __uint_as_float(r.w[0].z); f[3] = __uint_as_float(r.w[0].w);
  f[4] = __uint_as_float(r.w[1].x); f[5] = __uint_as_float(r.w[1].y); f[6] = __uint_as_float(r.w[1].z); f[7] = __uint_as_float(r.w[1].w);
}

__device__ __forceinline__ void raise(ugb_status_word *status, int detail) {
  if (atomicCAS(&status->code, 0u, (unsigned)UGB_ERR_INVALID) == 0u) status->detail = (unsigned)detail;
}

// ---------------------------------------------------------------- inputs ----
struct InputParams {
  const void *pre;
  const float *cos_, *sin_;
  const int *pos, *parents;
  void *q, *k, *v;
  int t, heads, kv_heads, dim, vdim, rot, interleaved, norm, t_max;
  float eps;
  ugb_status_word *status;
};

// How the partner of a rotated dimension is reached: pairs (2i, 2i + 1), both in a lane's piece; pairs (i, i + rot / 2) whose partners lie together,
// in another piece (read again, from L1); value by value, which also goes for buffers that are not aligned.
enum { INTERLEAVED, HALVES, SCATTERED };

// A CTA takes `per` nodes of a sequence, one after the other through all their heads: groups of LANES lanes take a query or key head each, 8 dimensions a
// lane (dim <= 8 LANES), two heads on their way at a time; the values are copied as they are.
template <typename T, int LANES, int MODE>
__global__ void __launch_bounds__(256, 4)
tree_inputs_kernel(InputParams p, int per) {
  constexpr int GROUPS = 256 / LANES;
  constexpr bool VEC = MODE != SCATTERED;
  __shared__ int up[UGB_TREE_MAX], at_s[UGB_TREE_MAX];
  const int parts = (p.t + per - 1) / per, s = blockIdx.x / parts, first = blockIdx.x % parts * per, count = min(per, p.t - first);
  const int pos = p.pos[s];
  bool bad = false;
  for (int j = threadIdx.x; j < p.t; j += 256) {
    const int a = p.parents[(size_t)s * p.t + j];
    up[j] = a;
    bad |= a < -1 || a >= j;
  }
  bad = __syncthreads_or(bad);
  if (pos == -1) return;                                   // no sequence in this place
  if (bad || pos < 0 || pos > p.t_max - p.t) {             // all nodes of the sequence stay as they are
    if (threadIdx.x == 0) raise(p.status, bad ? s : pos);
    return;
  }
  if ((int)threadIdx.x < count) {
    int at = pos;
    for (int j = up[first + threadIdx.x]; j >= 0; j = up[j]) ++at;
    at_s[threadIdx.x] = at;
  }
  const int half = p.rot / 2, turned = p.heads + p.kv_heads;
  const size_t ld = (size_t)turned * p.dim + (size_t)p.kv_heads * p.vdim, row0 = (size_t)s * p.t + first;
  const T *pre = (const T *)p.pre + row0 * ld;
  {   // values
    constexpr int N = VEC ? 8 : 1;
    const int pieces = p.kv_heads * p.vdim / N, width = p.vdim / N;
    for (int i = threadIdx.x; i < count * pieces; i += 256) {
      const int node = i / pieces, j = i - node * pieces, h = j / width, c = (j - h * width) * N;
      const T *x = pre + node * ld + (size_t)turned * p.dim + (size_t)h * p.vdim + c;
      T *y = (T *)p.v + (((size_t)s * p.kv_heads + h) * p.t_max + pos + first + node) * p.vdim + c;
      if constexpr (VEC) {
        Piece<T> w;
        fetch(x, w);
#pragma unroll
        for (int e = 0; e < (int)sizeof(T) / 2; ++e) reinterpret_cast<uint4 *>(y)[e] = w.w[e];
      } else {
        *y = *x;
      }
    }
  }
  __syncthreads();
  const int group = threadIdx.x / LANES, c0 = (threadIdx.x % LANES) * 8, total = count * turned;
  const bool on_lane = c0 < p.dim, turns = c0 < p.rot, low = c0 < half;
  const int partner = low ? c0 + half : c0 - half, table = MODE == INTERLEAVED ? c0 / 2 : low ? c0 : c0 - half;
  const float inv_dim = 1.0f / (float)p.dim;
  int node = 0, h = group;                                 // of this group's next head
  while (h >= turned) { h -= turned; ++node; }
  for (int w0 = 0; w0 < total; w0 += 2 * GROUPS) {         // all lanes of a warp stay together for the sums
    Piece<T> own[2], other[2];
    int nodes[2], hs[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      nodes[k] = node;
      hs[k] = h;
      const T *x = pre + node * ld + (size_t)h * p.dim;
      if constexpr (VEC)
        if (on_lane && node < count) {
          fetch(x + c0, own[k]);
          if (MODE == HALVES && turns) fetch(x + partner, other[k]);
        }
      h += GROUPS;
      while (h >= turned) { h -= turned; ++node; }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const bool on = on_lane && nodes[k] < count;
      float f[8], o[8], c[8], n[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = 0.f;
      if (on) {
        const int at = at_s[nodes[k]];
        const float *cs = p.cos_ + (size_t)at * half, *sn = p.sin_ + (size_t)at * half;
        const T *x = pre + nodes[k] * ld + (size_t)hs[k] * p.dim;
        if constexpr (VEC) unpack(own[k], f);
        else load8<false>(x + c0, f);
        if constexpr (MODE == SCATTERED) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int d = c0 + e;
            if (d < p.rot) {
              const bool one = p.interleaved ? d % 2 == 0 : d < half;
              const int i = p.interleaved ? d / 2 : one ? d : d - half, other_d = p.interleaved ? d ^ 1 : one ? d + half : d - half;
              const float a = (float)x[d], b = (float)x[other_d];
              f[e] = one ? a * cs[i] - b * sn[i] : a * cs[i] + b * sn[i];
            }
          }
        } else if (turns) {
          if constexpr (MODE == INTERLEAVED) {             // the table's rows start anywhere
#pragma unroll
            for (int e = 0; e < 8; e += 2)
              if (c0 + e < p.rot) {
                c[0] = cs[table + e / 2];
                n[0] = sn[table + e / 2];
                const float a = f[e], b = f[e + 1];
                f[e] = a * c[0] - b * n[0];
                f[e + 1] = b * c[0] + a * n[0];
              }
          } else {
            unpack(other[k], o);
            load8<true>(cs + table, c);
            load8<true>(sn + table, n);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = f[e] * c[e] + (low ? -o[e] : o[e]) * n[e];
          }
        }
      }
      if (p.norm) {                                        // sum of squares over the lanes of the head, in 32 bits
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
#pragma unroll
        for (int d = LANES / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        const float r = rsqrtf(ss * inv_dim + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= r;
      }
      if (!on) continue;
      const bool query = hs[k] < p.heads;
      T *y = query ? (T *)p.q + ((row0 + nodes[k]) * p.heads + hs[k]) * p.dim
                   : (T *)p.k + (((size_t)s * p.kv_heads + (hs[k] - p.heads)) * p.t_max + pos + first + nodes[k]) * p.dim;
      store8<VEC>(y + c0, f);
    }
  }
}

template <typename T, int MODE> void launch_inputs(dim3 grid, cudaStream_t st, const InputParams &p, int per) {
  if (p.dim <= 64) tree_inputs_kernel<T, 8, MODE><<<grid, 256, 0, st>>>(p, per);
  else if (p.dim <= 128) tree_inputs_kernel<T, 16, MODE><<<grid, 256, 0, st>>>(p, per);
  else tree_inputs_kernel<T, 32, MODE><<<grid, 256, 0, st>>>(p, per);
}
template <typename T> void launch_inputs(int mode, dim3 grid, cudaStream_t st, const InputParams &p, int per) {
  if (mode == INTERLEAVED) launch_inputs<T, INTERLEAVED>(grid, st, p, per);
  else if (mode == HALVES) launch_inputs<T, HALVES>(grid, st, p, per);
  else launch_inputs<T, SCATTERED>(grid, st, p, per);
}

// ------------------------------------------------------------------ keep ----
struct KeepParams {
  void *k, *v;
  const int *pos, *path, *count;
  int kv_heads, dq, dv, t_max, most;
  ugb_status_word *status;
};

// One thread per column piece of a head's rows (W: uint4, or a value of 2 or 4 bytes) moves it for all nodes in order.  path is
// ascending and path[i] >= i, so that no row is written before it has been read, in any batch of ascending moves.
template <typename W, int BYTES>
__global__ void __launch_bounds__(128)
cache_keep_kernel(KeepParams p) {
  constexpr int PER = (int)sizeof(W) / BYTES;              // values of a piece
  __shared__ int path[UGB_TREE_MAX];
  const int s = blockIdx.y, pos = p.pos[s], n = p.count[s];
  bool bad = n < 0 || n > p.most || pos < 0 || pos > p.t_max - n;
  if (!bad && (int)threadIdx.x < n) {
    const int *mine = p.path + (size_t)s * p.most;
    const int node = mine[threadIdx.x];
    path[threadIdx.x] = node;
    bad = node < (int)threadIdx.x || node >= p.t_max - pos || (threadIdx.x > 0 && mine[threadIdx.x - 1] >= node);
  }
  bad = __syncthreads_or(bad);
  if (pos == -1) return;                                   // no sequence in this place
  if (bad) {                                               // the sequence stays as it is
    if (threadIdx.x == 0 && blockIdx.x == 0) raise(p.status, s);
    return;
  }
  const int kp = p.dq / PER, vp = p.dv / PER, per_head = kp + vp;
  const int at = blockIdx.x * 128 + threadIdx.x;
  if (at >= p.kv_heads * per_head) return;
  const int head = at / per_head, c = at % per_head;
  const bool key = c < kp;
  const int ld = key ? kp : vp;
  W *base = (W *)(key ? p.k : p.v) + (((size_t)s * p.kv_heads + head) * p.t_max + pos) * ld + (key ? c : c - kp);
  for (int i0 = 0; i0 < n; i0 += 8) {
    W w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + i < n) w[i] = base[(size_t)path[i0 + i] * ld];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + i < n && path[i0 + i] != i0 + i) base[(size_t)(i0 + i) * ld] = w[i];
  }
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int32_t ugb_tree_inputs(ugb_device *dev, const ugb_slice *pre, const ugb_slice *cos_, const ugb_slice *sin_, const ugb_slice *pos,
                                   const ugb_slice *parents, ugb_slice *q, ugb_slice *kcache, ugb_slice *vcache, size_t b, size_t t, size_t heads,
                                   size_t kv_heads, size_t dim, size_t vdim, size_t rot_dims, int32_t interleaved, int32_t qk_norm, float eps,
                                   size_t t_max) {
  if (!dev) return UGB_ERR_INVALID;
  UGB_REQUIRE(dev, pre && q, UGB_ERR_INVALID, "tree_inputs: null slice");
  UGB_REQUIRE(dev, pre->dtype == q->dtype && (q->dtype == UGB_BF16 || q->dtype == UGB_F32), UGB_ERR_DTYPE,
              "tree_inputs: activations must be BF16 or F32 alike");
  UGB_REQUIRE(dev, dim % 8 == 0 && vdim % 8 == 0 && dim > 0 && vdim > 0 && dim <= 256 && vdim <= 256 && rot_dims <= dim && rot_dims % 2 == 0 &&
                       heads > 0 && kv_heads > 0 && heads <= 65535 && kv_heads <= 65535, UGB_ERR_SHAPE, "tree_inputs: unsupported shape");
  UGB_REQUIRE(dev, t <= UGB_TREE_MAX, UGB_ERR_UNSUPPORTED, "tree_inputs: %zu nodes, at most %d", t, UGB_TREE_MAX);
  UGB_REQUIRE(dev, b <= (1u << 20) && t_max <= (1u << 30) && t <= t_max, UGB_ERR_SHAPE, "tree_inputs: %zu nodes of %zu sequences, cache depth %zu", t, b, t_max);
  const size_t ld = (heads + kv_heads) * dim + kv_heads * vdim;
  UGB_SLICE(dev, pre, q->dtype, b * t * ld);
  UGB_SLICE(dev, q, q->dtype, b * t * heads * dim);
  UGB_SLICE(dev, kcache, q->dtype, b * kv_heads * t_max * dim);
  UGB_SLICE(dev, vcache, q->dtype, b * kv_heads * t_max * vdim);
  UGB_SLICE(dev, cos_, UGB_F32, t_max * rot_dims / 2);
  UGB_SLICE(dev, sin_, UGB_F32, t_max * rot_dims / 2);
  UGB_SLICE(dev, pos, UGB_I32, b);
  UGB_SLICE(dev, parents, UGB_I32, b * t);
  UGB_REQUIRE(dev, !ugb_overlap({ugb_used(q, b * t * heads * dim), ugb_used(kcache, b * kv_heads * t_max * dim), ugb_used(vcache, b * kv_heads * t_max * vdim)},
                                {ugb_used(pre, b * t * ld), ugb_used(cos_, t_max * rot_dims / 2), ugb_used(sin_, t_max * rot_dims / 2), ugb_used(pos, b),
                                 ugb_used(parents, b * t)}), UGB_ERR_INVALID, "tree_inputs: in place");
  if (b == 0 || t == 0) return UGB_OK;
  UGB_CUDA(dev, cudaSetDevice(dev->ordinal));
  InputParams p;
  p.pre = pre->ptr; p.cos_ = (const float *)cos_->ptr; p.sin_ = (const float *)sin_->ptr; p.pos = (const int *)pos->ptr;
  p.parents = (const int *)parents->ptr; p.q = q->ptr; p.k = kcache->ptr; p.v = vcache->ptr; p.t = (int)t; p.heads = (int)heads;
  p.kv_heads = (int)kv_heads; p.dim = (int)dim; p.vdim = (int)vdim; p.rot = (int)rot_dims; p.interleaved = interleaved != 0;
  p.norm = qk_norm != 0; p.eps = eps; p.t_max = (int)t_max; p.status = dev->status_dev;
  // several nodes share the look at the tree where there are more than fill the GPU, and so many that all CTAs run at once (64 x 64 nodes of 48 heads in
  // 640 CTAs 31.3 us, in the 512 that do 29.7)
  const size_t fill = 4 * (size_t)dev->sm_count;
  size_t per = 1;
  while (per < t && b * ((t + per - 1) / per) > fill) ++per;
  const dim3 grid((unsigned)(b * ((t + per - 1) / per)));
  // rows start at multiples of 8 values: aligned buffers make every piece of 8 aligned (the tables' too, where rot % 16 == 0)
  const bool vec = aligned16(pre->ptr) && aligned16(q->ptr) && aligned16(kcache->ptr) && aligned16(vcache->ptr) && aligned16(cos_->ptr) && aligned16(sin_->ptr);
  const int mode = !vec || (!interleaved && rot_dims % 16) ? SCATTERED : interleaved ? INTERLEAVED : HALVES;
  if (q->dtype == UGB_F32) launch_inputs<float>(mode, grid, dev->stream, p, (int)per);
  else launch_inputs<__nv_bfloat16>(mode, grid, dev->stream, p, (int)per);
  return ugb_after_launch(dev, "tree_inputs_kernel");
}

extern "C" int32_t ugb_cache_keep(ugb_device *dev, ugb_slice *k, ugb_slice *v, const ugb_slice *pos, const ugb_slice *path, const ugb_slice *count,
                                  size_t b, size_t kv_heads, size_t dq, size_t dv, size_t t_max, size_t most) {
  if (!dev) return UGB_ERR_INVALID;
  UGB_REQUIRE(dev, k && v, UGB_ERR_INVALID, "cache_keep: null slice");
  UGB_REQUIRE(dev, k->dtype == v->dtype && (k->dtype == UGB_BF16 || k->dtype == UGB_F32), UGB_ERR_DTYPE, "cache_keep: caches must be BF16 or F32 alike");
  UGB_REQUIRE(dev, dq % 8 == 0 && dv % 8 == 0 && dq > 0 && dv > 0 && dq <= 4096 && dv <= 4096 && kv_heads > 0 && kv_heads <= 65535 && b <= 65535 &&
                       t_max <= (1u << 30), UGB_ERR_SHAPE, "cache_keep: unsupported shape");
  UGB_REQUIRE(dev, most <= UGB_TREE_MAX, UGB_ERR_UNSUPPORTED, "cache_keep: up to %zu nodes, at most %d", most, UGB_TREE_MAX);
  UGB_SLICE(dev, k, k->dtype, b * kv_heads * t_max * dq);
  UGB_SLICE(dev, v, k->dtype, b * kv_heads * t_max * dv);
  UGB_SLICE(dev, pos, UGB_I32, b);
  UGB_SLICE(dev, path, UGB_I32, b * most);
  UGB_SLICE(dev, count, UGB_I32, b);
  UGB_REQUIRE(dev, !ugb_overlap({ugb_used(k, b * kv_heads * t_max * dq), ugb_used(v, b * kv_heads * t_max * dv)},
                                {ugb_used(pos, b), ugb_used(path, b * most), ugb_used(count, b)}), UGB_ERR_INVALID, "cache_keep: the caches overlap, or one and the paths");
  if (b == 0 || most == 0) return UGB_OK;
  UGB_CUDA(dev, cudaSetDevice(dev->ordinal));
  KeepParams p;
  p.k = k->ptr; p.v = v->ptr; p.pos = (const int *)pos->ptr; p.path = (const int *)path->ptr; p.count = (const int *)count->ptr;
  p.kv_heads = (int)kv_heads; p.dq = (int)dq; p.dv = (int)dv; p.t_max = (int)t_max; p.most = (int)most; p.status = dev->status_dev;
  const bool vec = aligned16(k->ptr) && aligned16(v->ptr);
  const size_t size = ugb_dtype_size(k->dtype), pieces = kv_heads * (dq + dv) / (vec ? 16 / size : 1);
  const dim3 grid((unsigned)((pieces + 127) / 128), (unsigned)b);
  if (size == 2) vec ? cache_keep_kernel<uint4, 2><<<grid, 128, 0, dev->stream>>>(p) : cache_keep_kernel<uint16_t, 2><<<grid, 128, 0, dev->stream>>>(p);
  else vec ? cache_keep_kernel<uint4, 4><<<grid, 128, 0, dev->stream>>>(p) : cache_keep_kernel<uint32_t, 4><<<grid, 128, 0, dev->stream>>>(p);
  return ugb_after_launch(dev, "cache_keep_kernel");
}
