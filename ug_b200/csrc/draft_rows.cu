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

template <typename T> __device__ __forceinline__ float to_f32(T x) { return (float)x; }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// 8 consecutive values: one or two 16-byte accesses where VEC says that they are aligned
template <bool VEC> __device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&f)[8]) {
  if constexpr (VEC) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)p[i];
  }
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

// One CTA per node.  Groups of LANES lanes take a head each, 8 dimensions a lane (dim, vdim <= 8 LANES); the partner of a rotated
// dimension is read again, from L1, where it belongs to another lane.
template <typename T, int LANES, bool VEC>
__global__ void __launch_bounds__(256)
tree_inputs_kernel(InputParams p) {
  __shared__ int up[UGB_TREE_MAX];
  const int s = blockIdx.x / p.t, node = blockIdx.x % p.t;
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
  int at = pos;
  for (int j = up[node]; j >= 0; j = up[j]) ++at;
  const int half = p.rot / 2;
  const float *cs = p.cos_ + (size_t)at * half, *sn = p.sin_ + (size_t)at * half;
  const int all = p.heads + 2 * p.kv_heads, turned = p.heads + p.kv_heads;
  const T *pre = (const T *)p.pre + ((size_t)s * p.t + node) * ((size_t)turned * p.dim + (size_t)p.kv_heads * p.vdim);
  const int group = threadIdx.x / LANES, c0 = (threadIdx.x % LANES) * 8;
  for (int h0 = 0; h0 < all; h0 += 256 / LANES) {          // all lanes of a warp stay together for the sums
    const int h = h0 + group;
    const bool rotated = h < turned;
    const int width = rotated ? p.dim : p.vdim;
    const bool on = h < all && c0 < width;
    const T *x = pre + (rotated ? (size_t)h * p.dim : (size_t)turned * p.dim + (size_t)(h - turned) * p.vdim);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 0.f;
    if (on) load8<VEC>(x + c0, f);
    if (on && rotated) {
      if (p.interleaved) {                                 // pairs (2i, 2i + 1): both in this lane
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          if (c0 + e < p.rot) {
            const float c = cs[(c0 + e) / 2], n = sn[(c0 + e) / 2], a = f[e], b = f[e + 1];
            f[e] = a * c - b * n;
            f[e + 1] = b * c + a * n;
          }
      } else if (VEC && half % 8 == 0) {                   // pairs (i, i + half): all 8 partners lie together, on one side
        if (c0 < p.rot) {
          const bool low = c0 < half;
          const int i = low ? c0 : c0 - half;
          float o[8], c[8], n[8];
          load8<VEC>(x + (low ? c0 + half : i), o);
          load8<VEC>(cs + i, c);
          load8<VEC>(sn + i, n);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = low ? f[e] * c[e] - o[e] * n[e] : f[e] * c[e] + o[e] * n[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = c0 + e;
          if (d < p.rot) {
            const bool low = d < half;
            const int i = low ? d : d - half;
            const float o = to_f32(x[low ? d + half : i]);
            f[e] = low ? f[e] * cs[i] - o * sn[i] : f[e] * cs[i] + o * sn[i];
          }
        }
      }
    }
    if (p.norm) {                                          // sum of squares over the lanes of the head, in 32 bits
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (rotated) {
        const float r = 1.0f / sqrtf(ss / (float)p.dim + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= r;
      }
    }
    if (!on) continue;
    const size_t row = pos + node;
    if (h < p.heads) store8<VEC>((T *)p.q + (((size_t)s * p.t + node) * p.heads + h) * p.dim + c0, f);
    else if (rotated) store8<VEC>((T *)p.k + (((size_t)s * p.kv_heads + (h - p.heads)) * p.t_max + row) * p.dim + c0, f);
    else store8<VEC>((T *)p.v + (((size_t)s * p.kv_heads + (h - turned)) * p.t_max + row) * p.vdim + c0, f);
  }
}

template <typename T, bool VEC> void launch_inputs(dim3 grid, cudaStream_t st, const InputParams &p) {
  const int widest = p.dim > p.vdim ? p.dim : p.vdim;
  if (widest <= 64) tree_inputs_kernel<T, 8, VEC><<<grid, 256, 0, st>>>(p);
  else if (widest <= 128) tree_inputs_kernel<T, 16, VEC><<<grid, 256, 0, st>>>(p);
  else tree_inputs_kernel<T, 32, VEC><<<grid, 256, 0, st>>>(p);
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
  UGB_REQUIRE(dev, !ugb_overlap(pre, q) && !ugb_overlap(pre, kcache) && !ugb_overlap(pre, vcache) && !ugb_overlap(q, kcache) && !ugb_overlap(q, vcache) &&
                       !ugb_overlap(kcache, vcache), UGB_ERR_INVALID, "tree_inputs: in place");
  if (b == 0 || t == 0) return UGB_OK;
  UGB_CUDA(dev, cudaSetDevice(dev->ordinal));
  InputParams p;
  p.pre = pre->ptr; p.cos_ = (const float *)cos_->ptr; p.sin_ = (const float *)sin_->ptr; p.pos = (const int *)pos->ptr;
  p.parents = (const int *)parents->ptr; p.q = q->ptr; p.k = kcache->ptr; p.v = vcache->ptr; p.t = (int)t; p.heads = (int)heads;
  p.kv_heads = (int)kv_heads; p.dim = (int)dim; p.vdim = (int)vdim; p.rot = (int)rot_dims; p.interleaved = interleaved != 0;
  p.norm = qk_norm != 0; p.eps = eps; p.t_max = (int)t_max; p.status = dev->status_dev;
  const dim3 grid((unsigned)(b * t));
  // rows start at multiples of 8 values: aligned buffers make every piece of 8 aligned (the tables' too, where half % 8 == 0 asks for it)
  const bool vec = aligned16(pre->ptr) && aligned16(q->ptr) && aligned16(kcache->ptr) && aligned16(vcache->ptr) && aligned16(cos_->ptr) && aligned16(sin_->ptr);
  if (q->dtype == UGB_F32) vec ? launch_inputs<float, true>(grid, dev->stream, p) : launch_inputs<float, false>(grid, dev->stream, p);
  else vec ? launch_inputs<__nv_bfloat16, true>(grid, dev->stream, p) : launch_inputs<__nv_bfloat16, false>(grid, dev->stream, p);
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
  UGB_REQUIRE(dev, !ugb_overlap(k, v), UGB_ERR_INVALID, "cache_keep: the caches overlap");
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
