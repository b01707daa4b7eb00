// Grouped-query attention over a cache whose queries see a part of it: a sliding window beside the first positions, or the committed
// positions and a node's ancestors.
#pragma once
#include "draft_rows.cuh"

struct ugb_masked_attention_args {
  bool f32;                  // T = f32, else bf16
  const void *q;             // T [b][t][heads][dq]
  const void *k, *v;         // T [b][kv_heads][t_max][dq / dv], the new positions' rows included
  void *out;                 // T [b][t][heads][dv] times out_scale
  const int *pos;            // [b] positions ahead of the new ones; -1: no sequence
  const int *parents;        // [b][t]: a tree; null: a window
  int b, t, heads, kv_heads, dq, dv, t_max;
  int sinks, window;
  float scale, out_scale;
};

// What a kernel needs to know of the mask.  Row r of a (sequence, key / value head) is query r / share of the block, head r % share of the
// group, so that a tile of rows reads a tile of keys once for all heads of the group.
struct ugb_mask {
  const int *pos, *parents;
  int t, t_max, sinks, window;
};
constexpr int UGB_MASKED_SPLITS = 256;    // slices of the keys and their parts, at most
struct ugb_masked_params {
  const void *q, *k, *v;
  void *out;
  ugb_mask mask;
  int heads, kv_heads, share, rows, dq, dv, splits;        // rows: t * share, of a sequence and key / value head
  float scale, out_scale;                                  // scale: with log2(e)
  float4 *part_o;                                          // of slices: [splits][b][kv_heads][dv / 4][rows], so that threads of neighbouring rows
                                                           // write and read neighbouring pieces
  float2 *part_ml;                                         // (maximum, sum) [splits][b][kv_heads][rows]
  ugb_status_word *status;
};

#ifdef __CUDACC__
namespace ugb_masked {

__device__ __forceinline__ void raise_invalid(ugb_status_word *status, int detail) {
  if (atomicCAS(&status->code, 0u, (unsigned)UGB_ERR_INVALID) == 0u) status->detail = (unsigned)detail;
}

// The keys that rows of queries i0 .. i1 of a sequence see: positions below `first`, and from `from` to `end` - 1.  All of the rows see those below `high`
// that are not below `low`, or that are first positions of the window's mask.
struct Span { int first, from, end, low, high; };
template <bool TREE> __device__ __forceinline__ Span span_of(const ugb_mask &m, int pos, int i0, int i1) {
  Span s;
  s.end = pos + i1 + 1;
  s.first = 0;
  s.from = 0;
  s.low = 0;
  s.high = pos;
  if constexpr (!TREE) {
    s.low = max(0, pos + i1 - m.window + 1);
    s.high = pos + i0 + 1;
    s.from = max(0, pos + i0 - m.window + 1);
    s.first = min(m.sinks, s.from);
  }
  return s;
}

}  // namespace ugb_masked
#endif

// The tensor-core kernel (masked_attention_tc.cu).  Whether it takes a call; how many items a slice of the keys has, how many run at a time, into
// how many parts each leaves its slice's result and how many query positions it has; its launch.
bool ugb_masked_tc_takes(const ugb_device *dev, const ugb_masked_attention_args &a);
void ugb_masked_tc_shape(const ugb_device *dev, const ugb_masked_attention_args &a, long long *items, long long *slots, int *parts, int *positions);
int32_t ugb_masked_tc_launch(ugb_device *dev, const ugb_masked_attention_args &a, const ugb_masked_params &p);

int32_t ugb_masked_attention(ugb_device *dev, const ugb_masked_attention_args &a);
