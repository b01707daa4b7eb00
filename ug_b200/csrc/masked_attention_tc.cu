// Attention over a window or a tree on the 5th-generation tensor cores (see masked_attention.cuh), bf16 heads of up to 128 values: DQ and DV are 64 or 128,
// what a head lacks of them is filled with zeros by TMA and cut off by it.
//
// One item = up to RT x 128 rows of a (sequence, key / value head) and a slice of the keys they see, in tiles of 128 keys (64 where 64 are enough); a row is
// a query position of one head of the group, so that keys and values are read once for all heads that share them:
//     warp 0        TMA producer: the rows' queries (one box: heads x positions), then key and value tiles into a ring
//     warp 1        MMA issuer:   S = Q K^T of each 128 rows, O += P V, both accumulated in TMEM
//     then 4 warps  softmax of 128 rows each (RT groups): one row per thread, no shuffles; P through shared memory in bf16, the type of V, as the product
//                   takes both in one type (2^-8 of each probability, which the f32 sum does not have: the whole error is 1.4 times that of a result rounded once)
// The scores of the next tile are formed as soon as this tile's are in registers, so that the softmax finds them ready; while one group's softmax runs, the
// other's products do.  O stays in TMEM from the first tile to the last: it is rescaled only where a row's maximum has grown by more than 2^8 since
// it was last (the probabilities are then up to 2^8, which costs bf16 no precision, and the sum is f32), which after the first tiles is hardly ever.
// Up to 32 rows (single positions, small trees) lie four times in the tile, once for each softmax warp, which takes a quarter of every tile's keys: a
// warp's chain per tile is then short enough for HBM.  The quarters are joined as slices of the keys are, by the combine kernel.
// Results leave through shared memory, by TMA.  Rows of V that no row of the item sees are set to zero there: P is zero for them, but 0 x NaN is not.  So is what
// is not finite in rows that only some see; those get it behind the last tile, from memory.  With two groups the warps that are left of the first
// warpgroup do this, while the tile's softmax is on its way (4 x 2048 positions as below 209 us for 204 without looking for what is not finite); a tile
// looked through by the softmax warps of the first group 211 us, and one of single positions, all of them, 68 us for 56.
// Grid: one CTA per item; a CTA that is done takes over the item of one that has not started (cluster launch control), so that its set-up and its
// TMEM are shared by many and long and short items even out.  Every wait on an mbarrier is bounded.
//
// What it is bound by, at two groups of 128-wide heads: a tile of 128 keys takes 4000 cycles, of which its products' reads of shared memory are 3000 and the
// two groups' exponentials 2048; of the rest of a softmax warp's chain, waits, stores and fences are 1400.  4 x 2048 positions over a window of 1024, 32
// heads on 8: 198 to 205 us, 710 to 685 TF/s (beside 198 in one run: 204 without packed arithmetic and three-way maxima, 226 without the registers of the first warpgroup, 260 with the scores
// taken from the tensor memory twice, 219 with a quarter of the exponentials on the FP32 pipe one by one, 202 in pairs).
// Tiles of 128 keys and not 64: the waits, fences and stores of a tile cost a softmax warp 1000 cycles whatever its size, the exponentials of 64 keys
// 950 to 1600; and the products read Q and P from shared memory once per 128 keys.
#include <cuda_bf16.h>

#include <algorithm>

#include "gemm_tcgen05.cuh"
#include "masked_attention.cuh"
#include "tc_ptx.cuh"

namespace {

using namespace ugb_tc;
using namespace ugb_masked;

constexpr int BQ = 128, CB = 64;                           // rows of a group, columns of a block (one 128-byte swizzle row)
constexpr int KEYS = 128;                                  // of a tile
constexpr int BLOCK = 128 * CB * 2;                        // 128 rows of 64 columns: 16 KiB
constexpr int P_BYTES = 2 * BLOCK;                         // 128 rows x 128 keys

// RT 0: up to 32 rows, spread over the four warps of one group.
template <int DQ, int DV, int RT0> struct Shape {
  static constexpr int RT = RT0 ? RT0 : 1;
  // Two groups: the softmax warps are two whole warpgroups, which take registers over from the first one.
  static constexpr int FIRST = RT == 2 ? 4 : 2, THREADS = 32 * FIRST + 128 * RT;    // FIRST: softmax warp
  static constexpr int Q_BYTES = DQ / CB * BLOCK, STAGE = (DQ > DV ? DQ : DV) / CB * BLOCK;     // a stage holds a tile of keys or of values
  static constexpr int O_COL = RT * KEYS;                  // TMEM: S [RT][128], then O [RT][DV]
  static constexpr int TMEM_USED = O_COL + RT * DV, TMEM_COLS = TMEM_USED <= 256 ? 256 : 512;
  static constexpr int FIXED = RT * (Q_BYTES + P_BYTES) + 512 /*barriers*/ + RT * UGB_TREE_MAX * 4;
  static constexpr int CTAS_PER_SM = RT0 <= 1 && DQ + DV == 128 ? 2 : 1;      // more would not fit
  static constexpr int LIMIT = (CTAS_PER_SM == 2 ? 113 : 227) * 1024;
  static constexpr int FIT = (LIMIT - FIXED) / STAGE, STAGES = FIT > 8 ? 8 : FIT;
  static constexpr int TILES = FIXED + STAGES * STAGE;
  // a CTA that takes all of the TMEM is alone on its SM: more than half of the shared memory sees to that
  static constexpr int SMEM_BYTES = CTAS_PER_SM == 1 && TILES < 116 * 1024 ? 116 * 1024 : TILES;
  static_assert(TMEM_USED <= 512 && STAGES >= 3 && SMEM_BYTES <= 227 * 1024, "tile shape");
};

struct Params {
  ugb_masked_params m;
  int pairs, row_tiles, per_group;                         // per_group: rows of a group, share * (128 / share)
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two values at a time, and three: the softmax warps are bound by the instructions they issue.
struct Two { unsigned long long v; };
__device__ __forceinline__ Two two(float x, float y) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void apart(Two a, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Asks for the item of a CTA that has not started; the answer arrives at the barrier (16 bytes).
__device__ __forceinline__ void next_item_request(uint32_t answer, uint32_t bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
// Its block index, or -1.
__device__ __forceinline__ int next_item_answer(uint32_t answer) {
  int x;
  asm volatile(
      "{\n .reg .b128 r;\n .reg .pred p;\n .reg .b32 a, b, c, d;\n"
      " ld.shared.b128 r, [%1];\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n"
      " mov.b32 %0, -1;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {a, b, c, d}, r;\n"
      " @p mov.b32 %0, a;\n}"
      : "=r"(x) : "r"(answer) : "memory");
  return x;
}
// Whether any of the 128 threads of a group says so; a barrier of theirs.
__device__ __forceinline__ bool group_or(int id, bool v) {
  uint32_t r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n barrier.cta.red.or.pred p, %2, 128, q;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(r) : "r"((uint32_t)v), "r"(id) : "memory");
  return r != 0;
}
__device__ __forceinline__ void group_sync(int id) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void tma_store_4d(const CUtensorMap *map, uint32_t src, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void store_read_wait() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// Row `row` of a tile of values, whose key not all rows of the item see: zeros, or zeros for what is not finite.  Whether there was any of that.
template <int DV> __device__ __forceinline__ bool clean_values(uint8_t *stage, int row, bool nobody) {
  uint8_t *const at = stage + row * 128;                   // 16 bytes at a time, others first in every row: no bank conflicts
  if (nobody) {
#pragma unroll
    for (int x = 0; x < DV / 8; ++x) *reinterpret_cast<uint4 *>(at + x / 8 * BLOCK + ((x ^ row) & 7) * 16) = make_uint4(0, 0, 0, 0);
    return false;
  }
  const __nv_bfloat162 zero = __float2bfloat162_rn(0.f);
  __nv_bfloat162 sum = zero;                               // of 0 x value: NaN if any is not finite
#pragma unroll
  for (int x = 0; x < DV / 8; ++x) {
    const uint4 v = *reinterpret_cast<const uint4 *>(at + x / 8 * BLOCK + ((x ^ row) & 7) * 16);
    const __nv_bfloat162 *w = reinterpret_cast<const __nv_bfloat162 *>(&v);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = __hfma2(w[e], zero, sum);
  }
  const uint32_t bits = *reinterpret_cast<const uint32_t *>(&sum);
  if (!(bits & 0x7fff7fffu)) return false;
#pragma unroll 1
  for (int x = 0; x < DV; ++x) {
    uint16_t *v = reinterpret_cast<uint16_t *>(at + x / 64 * BLOCK) + x % 64;
    if ((*v & 0x7f80) == 0x7f80) *v = 0;
  }
  return true;
}
// What is not finite in columns c .. c + 31 of the keys of `seen`, v: the values of its first key.  Hardly ever called.
struct NotFinite { uint32_t plus, minus, nan; };
__device__ __noinline__ NotFinite not_finite(const uint16_t *v, int dv, int c, unsigned long long seen) {
  NotFinite r{0, 0, 0};
  for (; seen; seen &= seen - 1) {
    const uint16_t *x = v + (size_t)(__ffsll((long long)seen) - 1) * dv + c;
    for (int e = 0; e < min(32, dv - c); ++e)
      if ((x[e] & 0x7f80) == 0x7f80) (x[e] & 0x7f ? r.nan : x[e] & 0x8000 ? r.minus : r.plus) |= 1u << e;
  }
  return r;
}
// The lowest n bits, n clamped to 0 .. 64.
__device__ __forceinline__ unsigned long long low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }

// Items in the order of their block index: the last rows of every pair first (they see the most keys), their slices side by side.
struct Item {
  int s, kvh, slice, row0, pos, first, tiles;              // first: of the slice's tiles; tiles: 0 = nothing to compute
  int first_tiles, start;                                  // tiles of the first positions; where the others start
  bool valid;                                              // the sequence exists and its position is inside the cache
  Span span;
  // tile j of the slice: its first key, and whether it has more than 64
  __device__ __forceinline__ int key0(int j) const { return first + j < first_tiles ? (first + j) * KEYS : start + (first + j - first_tiles) * KEYS; }
  __device__ __forceinline__ bool full(int j) const {      // the last of the first tiles may hold the start of the window too
    return (first + j < first_tiles && span.from >= first_tiles * KEYS ? span.first : span.end) - key0(j) > 64;
  }
  // which of the item's stages holds the values of tile j: K(0), then K(j + 1), V(j) for every tile, and V of the last one
  __device__ __forceinline__ int stage_of_values(int j) const { return j + 1 < tiles ? 2 * j + 2 : 2 * j + 1; }
  __device__ __forceinline__ bool nobody_sees(int k) const { return k >= span.first && (k < span.from || k >= span.end); }
  // whether all rows see the keys from k on, n of them
  __device__ __forceinline__ bool all_see(int k, int n, int sinks) const { return k + n <= span.high && (k >= span.low || k + n <= sinks); }
};
template <int RT, bool TREE> __device__ __forceinline__ Item item_of(int idx, const Params &p) {
  Item it;
  it.slice = idx % p.m.splits;
  const int r = idx / p.m.splits, pair = r % p.pairs, tile = p.row_tiles - 1 - r / p.pairs;
  it.s = pair / p.m.kv_heads;
  it.kvh = pair - it.s * p.m.kv_heads;
  it.row0 = tile * RT * p.per_group;
  it.pos = *reinterpret_cast<const volatile int *>(p.m.mask.pos + it.s);
  it.valid = it.pos >= 0 && it.pos <= p.m.mask.t_max - p.m.mask.t;
  it.tiles = it.first = 0;
  if (it.valid) {
    const int last = min(it.row0 + RT * p.per_group, p.m.rows) - 1;
    it.span = span_of<TREE>(p.m.mask, it.pos, it.row0 / p.m.share, last / p.m.share);
    it.first_tiles = (it.span.first + KEYS - 1) / KEYS;
    it.start = max(it.span.from, it.first_tiles * KEYS);
    const int tiles = it.first_tiles + max(0, it.span.end - it.start + KEYS - 1) / KEYS;
    const int per = (tiles + p.m.splits - 1) / p.m.splits;
    it.first = it.slice * per;
    it.tiles = max(0, min(tiles, it.first + per) - it.first);
  }
  return it;
}

template <int DQ, int DV, int RT0, bool TREE>
__global__ void __launch_bounds__((Shape<DQ, DV, RT0>::THREADS), (Shape<DQ, DV, RT0>::CTAS_PER_SM))
masked_attention_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                           const __grid_constant__ CUtensorMap tmO, Params p) {
  using Sh = Shape<DQ, DV, RT0>;
  constexpr int ST = Sh::STAGES, RT = Sh::RT;
  constexpr bool SPREAD = RT0 == 0;
  extern __shared__ __align__(1024) uint8_t smem[];        // all of it: a block of rows starts at a multiple of 1024 bytes
  if (smem_u32(smem) & 1023) {
    if (threadIdx.x == 0 && atomicCAS(&p.m.status->code, 0u, (unsigned)UGB_ERR_UNSUPPORTED) == 0u) p.m.status->detail = 0x5f;
    return;
  }
  uint8_t *q_s = smem, *p_s = q_s + RT * Sh::Q_BYTES, *kv_s = p_s + RT * P_BYTES;
  uint64_t *bars = (uint64_t *)(kv_s + ST * Sh::STAGE);
  uint64_t *q_full = bars, *q_empty = bars + 1, *answer_full = bars + 2, *answer = bars + 4;       // the answer: 16 bytes, aligned
  uint64_t *item_full = bars + 6, *item_empty = bars + 8, *s_full = bars + 10, *s_free = s_full + RT, *p_full = s_free + RT, *o_full = p_full + RT;
  uint64_t *kv_full = o_full + RT, *kv_empty = kv_full + ST, *v_ready = kv_empty + ST, *v_clean = v_ready + 1;
  uint32_t *tmem_slot = (uint32_t *)(v_clean + 1);
  volatile int *abort_flag = (volatile int *)(tmem_slot + 1), *item_slot = (volatile int *)(tmem_slot + 2);      // two entries
  volatile int *not_finite_slot = item_slot + 2;           // of four items in turn: n_it + 1 where values were set to zero
  int(*up)[UGB_TREE_MAX] = (int(*)[UGB_TREE_MAX])((uint8_t *)bars + 512);
  static_assert((12 + 4 * RT + 2 * ST) * 8 + 32 <= 512, "barriers fit");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ugb_status_word *const status = p.m.status;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(q_full), 1);
    mbar_init(smem_u32(q_empty), 1);
    mbar_init(smem_u32(answer_full), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&item_full[i]), 1);
      mbar_init(smem_u32(&item_empty[i]), 1 + 4 * RT + (RT == 2 ? 2 : 0));
    }
    for (int i = 0; i < RT; ++i) {
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&s_free[i]), 4);
      mbar_init(smem_u32(&p_full[i]), 4);
      mbar_init(smem_u32(&o_full[i]), 1);
    }
    for (int i = 0; i < ST; ++i) {
      mbar_init(smem_u32(&kv_full[i]), 1);
      mbar_init(smem_u32(&kv_empty[i]), 1);
    }
    mbar_init(smem_u32(v_ready), 1);
    mbar_init(smem_u32(v_clean), 2);
    *abort_flag = 0;
    for (int i = 0; i < 4; ++i) not_finite_slot[i] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmQ) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmK) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmV) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmO) : "memory");
  }
  if constexpr (SPREAD) {                                  // a row's probabilities outside its warp's quarter of the keys stay zero
    for (int i = threadIdx.x; i < P_BYTES / 16; i += Sh::THREADS) reinterpret_cast<uint4 *>(p_s)[i] = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(Sh::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;

  // The ring's order: K(0), then K(j + 1), V(j) for every tile j, and V of the last one: the order in which the products are issued.
  if (warp < Sh::FIRST) {
  // of 168 registers per thread at the launch: 4 x 96 + 8 x 200 <= 12 x 168
  if constexpr (RT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer --
    if (elect_one()) {
      int g = 0, n_q = 0, idx = blockIdx.x;                // stages filled and items with tiles so far
      for (int n_it = 0;; ++n_it) {
        const int at = n_it & 1;
        if (!mbar_wait(smem_u32(&item_empty[at]), ((uint32_t)(n_it >> 1) & 1u) ^ 1u, abort_flag, status, 0x60)) break;
        item_slot[at] = idx;
        mbar_arrive(smem_u32(&item_full[at]));             // release: the slot is visible to the waiters
        if (idx < 0) break;
        // the next item is asked for now, the answer is looked at behind this one's tiles
        mbar_expect_tx(smem_u32(answer_full), 16);
        next_item_request(smem_u32(answer), smem_u32(answer_full));
        const Item it = item_of<RT, TREE>(idx, p);
        bool alive = true;
        auto load = [&](const CUtensorMap *map, int d, int j) {          // tile j of the keys or values
          const int s = g % ST, n = it.full(j) ? 2 : 1, key0 = it.key0(j);
          if (!mbar_wait(smem_u32(&kv_empty[s]), ((uint32_t)(g / ST) & 1u) ^ 1u, abort_flag, status, 0x61)) { alive = false; return; }
          ++g;
          mbar_expect_tx(smem_u32(&kv_full[s]), (uint32_t)(n * 64 * d * 2));
          for (int c = 0; c < d / CB; ++c)
            for (int h = 0; h < n; ++h)
              tma_load_4d(smem_u32(kv_s + s * Sh::STAGE + c * BLOCK + h * (BLOCK / 2)), map, smem_u32(&kv_full[s]), c * CB, it.kvh, key0 + 64 * h, it.s);
        };
        if (it.tiles > 0) {
          const int i0 = it.row0 / p.m.share, step = p.per_group / p.m.share;
          // the query buffers are free once every S product of the item before has retired
          alive = mbar_wait(smem_u32(q_empty), ((uint32_t)n_q & 1u) ^ 1u, abort_flag, status, 0x62);
          ++n_q;
          if (alive) {
            constexpr int COPIES = SPREAD ? 4 : RT;        // rows 32 apart, or groups
            mbar_expect_tx(smem_u32(q_full), (uint32_t)(COPIES * (DQ / CB) * p.per_group * CB * 2));
            for (int a = 0; a < COPIES; ++a)
              for (int c = 0; c < DQ / CB; ++c)
                tma_load_4d(smem_u32(q_s + a * (SPREAD ? 32 * 128 : Sh::Q_BYTES) + c * BLOCK), &tmQ, smem_u32(q_full), c * CB, it.kvh * p.m.share,
                            SPREAD ? i0 : i0 + a * step, it.s);
            load(&tmK, DQ, 0);
          }
          for (int j = 0; j < it.tiles && alive; ++j) {
            if (j + 1 < it.tiles) load(&tmK, DQ, j + 1);
            if (alive) load(&tmV, DV, j);
          }
        }
        if (!mbar_wait(smem_u32(answer_full), (uint32_t)n_it & 1u, abort_flag, status, 0x64)) break;
        idx = next_item_answer(smem_u32(answer));
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // read before the next answer is written
        if (!alive) break;
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer --
    if (elect_one()) {
      // Q and K both K-major; P K-major, V MN-major ([key][dim] rows, blocks of 64 columns BLOCK apart)
      const uint32_t idesc_s[2] = {make_idesc(BQ, 64, false), make_idesc(BQ, 128, false)}, idesc_o = make_idesc(BQ, DV, true);
      const uint64_t q_desc = make_smem_desc(smem_u32(q_s), 0, 1024), p_desc = make_smem_desc(smem_u32(p_s), 0, 1024);
      const uint64_t k_desc = make_smem_desc(smem_u32(kv_s), 0, 1024), v_desc = make_smem_desc(smem_u32(kv_s), BLOCK, 1024);
      int g = 0, n_q = 0;                                               // stages and items so far
      uint32_t n_s[2] = {0, 0}, n_p[2] = {0, 0};                        // S and P V products of a group so far
      uint32_t n_clean = 0;                                             // tiles of values that were cleaned so far
      for (int n_it = 0;; ++n_it) {
        const int at = n_it & 1;
        if (!mbar_wait(smem_u32(&item_full[at]), (uint32_t)(n_it >> 1) & 1u, abort_flag, status, 0x65)) break;
        const int idx = item_slot[at];
        mbar_arrive(smem_u32(&item_empty[at]));
        if (idx < 0) break;
        const Item it = item_of<RT, TREE>(idx, p);
        if (it.tiles == 0) continue;
        if (!mbar_wait(smem_u32(q_full), (uint32_t)n_q & 1u, abort_flag, status, 0x66)) break;
        ++n_q;
        const bool both = RT == 2 && it.row0 + p.per_group < p.m.rows;
        bool alive = true;
        auto scores = [&](int j) {                                      // S of tile j, of every group
          const int s = g % ST;
          if (!mbar_wait(smem_u32(&kv_full[s]), (uint32_t)(g / ST) & 1u, abort_flag, status, 0x67)) { alive = false; return; }
          ++g;
          const uint64_t kd = k_desc + (uint64_t)(s * (Sh::STAGE >> 4));
          const uint32_t idesc = idesc_s[it.full(j) ? 1 : 0];
#pragma unroll
          for (int a = 0; a < RT; ++a) {
            if (a == 1 && !both) break;
            // the group has taken the scores before out of the tensor memory
            if (!mbar_wait(smem_u32(&s_free[a]), (n_s[a] & 1u) ^ 1u, abort_flag, status, 0x68)) { alive = false; return; }
            ++n_s[a];
            tcgen05_fence_after();
            const uint64_t qd = q_desc + (uint64_t)(a * (Sh::Q_BYTES >> 4));
#pragma unroll
            for (int kk = 0; kk < DQ / UMMA_K; ++kk) {                  // 16 columns are 32 bytes inside the swizzled row
              const uint64_t off = (uint64_t)(((kk / 4) * BLOCK + (kk % 4) * (UMMA_K * 2)) >> 4);
              umma_bf16(tmem + (uint32_t)(a * KEYS), qd + off, kd + off, idesc, kk > 0 ? 1u : 0u);
            }
            umma_commit(smem_u32(&s_full[a]));
          }
          umma_commit(smem_u32(&kv_empty[s]));
          if (j == it.tiles - 1) umma_commit(smem_u32(q_empty));        // no more products read the queries
        };
        scores(0);
        for (int j = 0; j < it.tiles && alive; ++j) {
          if (j + 1 < it.tiles) scores(j + 1);
          if (!alive) break;
          const int s = g % ST;
          if (!mbar_wait(smem_u32(&kv_full[s]), (uint32_t)(g / ST) & 1u, abort_flag, status, 0x69)) { alive = false; break; }
          ++g;
          const uint64_t vd = v_desc + (uint64_t)(s * (Sh::STAGE >> 4));
          const bool full = it.full(j);
          if (RT == 2 && !it.all_see(it.key0(j), full ? KEYS : 64, p.m.mask.sinks)) {
            mbar_arrive(smem_u32(v_ready));
            if (!mbar_wait(smem_u32(v_clean), n_clean & 1u, abort_flag, status, 0x63)) { alive = false; break; }
            ++n_clean;
          }
#pragma unroll
          for (int a = 0; a < RT; ++a) {
            if (a == 1 && !both) break;
            if (!mbar_wait(smem_u32(&p_full[a]), n_p[a] & 1u, abort_flag, status, 0x6a)) { alive = false; break; }
            ++n_p[a];
            tcgen05_fence_after();
            const uint64_t pd = p_desc + (uint64_t)(a * (P_BYTES >> 4));
#pragma unroll
            for (int kk = 0; kk < KEYS / UMMA_K; ++kk) {
              if (kk >= 4 && !full) break;
              // P: 16 keys are 32 bytes inside the swizzled row, 64 keys a block; V: 16 keys are 16 rows
              umma_bf16(tmem + (uint32_t)(Sh::O_COL + a * DV), pd + (uint64_t)(((kk / 4) * BLOCK + (kk % 4) * (UMMA_K * 2)) >> 4),
                        vd + (uint64_t)((kk * (UMMA_K * 128)) >> 4), idesc_o, j > 0 || kk > 0 ? 1u : 0u);
            }
            umma_commit(smem_u32(&o_full[a]));
          }
          if (alive) umma_commit(smem_u32(&kv_empty[s]));
        }
        if (!alive) break;
      }
    }
  } else if (RT == 2) {
    // ------------------------------------------- values of keys that not all rows see --
    // While the softmax of the tile is on its way.  The issuer says when a tile is there: a wait for a stage that it has not got to might take an older phase of its
    // barrier for the one that is meant.
    bool alive = true;
    int g0 = 0;                                            // stages of the CTA so far
    uint32_t n_clean = 0;
    for (int n_it = 0; alive; ++n_it) {
      const int at = n_it & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&item_full[at]), (uint32_t)(n_it >> 1) & 1u, abort_flag, status, 0x6b))) break;
      const int idx = item_slot[at];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&item_empty[at]));
      if (idx < 0) break;
      const Item it = item_of<RT, TREE>(idx, p);
      for (int j = 0; j < it.tiles; ++j) {
        const int key0 = it.key0(j), n_keys = it.full(j) ? KEYS : 64;
        if (it.all_see(key0, n_keys, p.m.mask.sinks)) continue;
        const int g = g0 + it.stage_of_values(j), s = g % ST;
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(v_ready), n_clean & 1u, abort_flag, status, 0x6e) &&
                                         mbar_wait(smem_u32(&kv_full[s]), (uint32_t)(g / ST) & 1u, abort_flag, status, 0x6e))) { alive = false; break; }
        ++n_clean;
        for (int row = threadIdx.x - 64; row < n_keys; row += 64) {
          const bool nobody = it.nobody_sees(key0 + row);
          if ((nobody || !it.all_see(key0 + row, 1, p.m.mask.sinks)) && clean_values<DV>(kv_s + s * Sh::STAGE, row, nobody))
            not_finite_slot[n_it & 3] = n_it + 1;          // the groups are two items behind at most
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(v_clean));
      }
      g0 += 2 * it.tiles;
    }
  }
  } else {
    // -------------------------------------------------------------- softmax warps --
    if constexpr (RT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int a = (warp - Sh::FIRST) / 4, quad = warp & 3, row = quad * 32 + lane;              // TMEM lane = row of the group
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16), s_base = lane_base + (uint32_t)(a * KEYS), o_base = lane_base + (uint32_t)(Sh::O_COL + a * DV);
    uint8_t *const p_group = p_s + a * P_BYTES, *const prow = p_group + row * 128;
    const bool leader = threadIdx.x == 32 * Sh::FIRST + a * 128;     // issues the group's stores
    bool alive = true;
    int g0 = 0;                                            // stages of the CTA so far
    uint32_t n_s = 0, n_o = 0;                             // S and O products of this group so far
    for (int n_it = 0;; ++n_it) {
      const int at = n_it & 1;
      alive = __all_sync(0xffffffffu, mbar_wait(smem_u32(&item_full[at]), (uint32_t)(n_it >> 1) & 1u, abort_flag, status, 0x6b));
      if (!alive) break;
      const int idx = item_slot[at];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&item_empty[at]));
      if (idx < 0) break;
      const Item it = item_of<RT, TREE>(idx, p);
      if (!it.valid) {
        if (it.pos != -1 && leader) raise_invalid(status, it.s);
        const int r = it.row0 + a * p.per_group + (SPREAD ? lane : row);
        if (p.m.part_ml && it.slice == 0 && r < p.m.rows && (!SPREAD || quad == 0) && (SPREAD || row < p.per_group))
          p.m.part_ml[((size_t)it.s * p.m.kv_heads + it.kvh) * p.m.rows + r] = make_float2(NAN, 0.f);       // for the combine kernel: to be left as it is
        continue;
      }
      const int r0 = it.row0 + a * p.per_group, n_rows = min(p.per_group, p.m.rows - r0);      // of this group
      if (n_rows <= 0) { g0 += 2 * it.tiles; continue; }
      const int in_rows = SPREAD ? lane : row;
      const bool mine = in_rows < n_rows;                  // this thread has a row
      const bool busy = SPREAD || quad * 32 < n_rows;      // this warp has rows
      const int i = (r0 + min(in_rows, n_rows - 1)) / p.m.share, n = it.pos + i;
      unsigned long long nodes0 = 0, nodes1 = 0;
      bool bad = false;
      if constexpr (TREE) {
        if (it.tiles > 0) {
          for (int j = row; j < p.m.mask.t; j += 128) {
            const int x = *reinterpret_cast<const volatile int *>(p.m.mask.parents + (size_t)it.s * p.m.mask.t + j);
            up[a][j] = x;
            bad |= x < -1 || x >= j;
          }
          bad = group_or(1 + a, bad);
          if (bad && leader) raise_invalid(status, it.s);
          if (!bad)
            for (int j = i; j >= 0; j = up[a][j]) (j < 64 ? nodes0 : nodes1) |= 1ull << (j & 63);
        }
      }
      // which of the 64 keys from key0 on this row sees
      auto seen_from = [&](int key0) -> unsigned long long {
        if constexpr (TREE) {
          const int rel = key0 - it.pos;                   // node of the first key
          if (rel <= -64) return ~0ull;
          if (rel < 0) return (nodes0 << -rel) | low_bits(-rel);
          if (rel < 64) return (nodes0 >> rel) | (rel ? nodes1 << (64 - rel) : 0ull);
          return rel < 128 ? nodes1 >> (rel - 64) : 0ull;
        } else {
          return low_bits(n - key0 + 1) & (~low_bits(n - p.m.mask.window - key0 + 1) | low_bits(p.m.mask.sinks - key0));
        }
      };
      const float sc = p.m.scale;
      float m_ref = -INFINITY, l = 0.f;
      for (int j = 0; j < it.tiles; ++j) {
        const int key0 = it.key0(j);
        const bool full = it.full(j);
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[a]), n_s & 1u, abort_flag, status, 0x6c))) { alive = false; break; }
        ++n_s;
        if constexpr (SPREAD) {
          const bool some = full || quad < 2;              // a half tile has keys for two warps
          if (some) {
            tcgen05_fence_after();
            uint32_t f[32];
            tmem_ld_32x32b_x32(s_base + 32 * quad, f);
            tmem_ld_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s_free[a]));
            const uint32_t on = (uint32_t)(seen_from(key0 + 64 * (quad / 2)) >> (32 * (quad & 1)));
            if (__any_sync(0xffffffffu, on != ~0u)) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(on >> e & 1u)) f[e] = 0xff800000u;   // -inf
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 32; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(f[e]));
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
            const bool grow = top > m_ref + 8.f;
            float alpha = 1.f;
            if (grow) {
              alpha = ex2(m_ref - top);
              m_ref = top;
              l *= alpha;
            }
            const float neg = m_ref == -INFINITY ? 0.f : -m_ref;
            float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float x = ex2(fmaf(__uint_as_float(f[2 * e]), sc, neg)), y = ex2(fmaf(__uint_as_float(f[2 * e + 1]), sc, neg));
              l4[2 * e & 3] += x;
              l4[(2 * e + 1) & 3] += y;
              const __nv_bfloat162 t = __floats2bfloat162_rn(x, y);
              f[e] = *reinterpret_cast<const uint32_t *>(&t);
            }
            l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
            if (j > 0) {
              if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&o_full[a]), n_o & 1u, abort_flag, status, 0x6d))) { alive = false; break; }
              ++n_o;
              if (__any_sync(0xffffffffu, grow && mine)) {
                tcgen05_fence_after();
#pragma unroll
                for (int c = 0; c < DV; c += 32) {
                  uint32_t o[32];
                  tmem_ld_32x32b_x32(o_base + c, o);
                  tmem_ld_wait();
#pragma unroll
                  for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                  tmem_st_32x32b_x32(o_base + c, o);
                }
                tmem_st_wait();
              }
            }
#pragma unroll
            for (int ch = 0; ch < 4; ++ch)
              *reinterpret_cast<uint4 *>(prow + quad / 2 * BLOCK + (((quad % 2 * 4 + ch) ^ (row & 7)) << 4)) = make_uint4(f[4 * ch], f[4 * ch + 1], f[4 * ch + 2], f[4 * ch + 3]);
          } else {
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s_free[a]));
            if (j > 0) {
              if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&o_full[a]), n_o & 1u, abort_flag, status, 0x6d))) { alive = false; break; }
              ++n_o;
            }
          }
        } else if (busy) {
          tcgen05_fence_after();
          uint32_t f[KEYS];                                // scores, and in their place, two to a register, the probabilities
          {
            uint32_t(*r)[32] = reinterpret_cast<uint32_t(*)[32]>(f);    // what a half tile leaves in the upper columns is replaced below
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_base + 32 * c, r[c]);
          }
          tmem_ld_wait();
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&s_free[a]));             // the next tile's scores may come
          constexpr uint32_t HIDDEN = 0xff800000u;         // -inf
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const unsigned long long seen = h == 1 && !full ? 0ull : seen_from(key0 + 64 * h);
            if (__any_sync(0xffffffffu, seen != ~0ull)) {
              const uint32_t lo = (uint32_t)seen, hi = (uint32_t)(seen >> 32);
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                if (!(lo >> e & 1u)) f[64 * h + e] = HIDDEN;
                if (!(hi >> e & 1u)) f[64 * h + 32 + e] = HIDDEN;
              }
            }
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < KEYS / 2; ++e) mx[e & 3] = max3(mx[e & 3], __uint_as_float(f[2 * e]), __uint_as_float(f[2 * e + 1]));
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;        // sc > 0
          const bool grow = top > m_ref + 8.f;
          float alpha = 1.f;
          if (grow) {
            alpha = ex2(m_ref - top);
            m_ref = top;
            l *= alpha;
          }
          const float neg = m_ref == -INFINITY ? 0.f : -m_ref;          // a row may see nothing of the tiles so far
          const Two sc2 = two(sc, sc), neg2 = two(neg, neg);
          Two sum[2] = {two(0.f, 0.f), two(0.f, 0.f)};
#pragma unroll
          for (int e = 0; e < KEYS / 2; ++e) {
            float x, y;
            apart(fma2(two(__uint_as_float(f[2 * e]), __uint_as_float(f[2 * e + 1])), sc2, neg2), x, y);
            x = ex2(x);
            y = ex2(y);
            sum[e & 1] = add2(sum[e & 1], two(x, y));
            const __nv_bfloat162 t = __floats2bfloat162_rn(x, y);
            f[e] = *reinterpret_cast<const uint32_t *>(&t);
          }
          float x, y;
          apart(add2(sum[0], sum[1]), x, y);
          l += x + y;
          // the product before has retired: its probabilities may be overwritten, and O is at rest
          if (j > 0) {
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&o_full[a]), n_o & 1u, abort_flag, status, 0x6d))) { alive = false; break; }
            ++n_o;
            if (__any_sync(0xffffffffu, grow && mine)) {
              tcgen05_fence_after();
#pragma unroll
              for (int c = 0; c < DV; c += 32) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(o_base + c, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_st_32x32b_x32(o_base + c, o);
              }
              tmem_st_wait();
            }
          } else {
            if (leader) store_read_wait();                 // nor does a store read them, of the item before
            group_sync(1 + a);
          }
#pragma unroll
          for (int ch = 0; ch < KEYS / 8; ++ch) {
            if (ch >= 8 && !full) break;
            *reinterpret_cast<uint4 *>(prow + ch / 8 * BLOCK + ((ch % 8 ^ (row & 7)) << 4)) = make_uint4(f[4 * ch], f[4 * ch + 1], f[4 * ch + 2], f[4 * ch + 3]);
          }
        } else {                                           // no rows: only the barriers' counts
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&s_free[a]));
          if (j > 0) {
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&o_full[a]), n_o & 1u, abort_flag, status, 0x6d))) { alive = false; break; }
            ++n_o;
          } else {
            if (leader) store_read_wait();
            group_sync(1 + a);
          }
        }
        if constexpr (RT == 1) {                           // with two groups, the warps beside the issuer do this
          const int n_keys = full ? KEYS : 64;
          if (!it.all_see(key0, n_keys, p.m.mask.sinks)) {
            const int g = g0 + it.stage_of_values(j), s = g % ST;
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&kv_full[s]), (uint32_t)(g / ST) & 1u, abort_flag, status, 0x6e))) { alive = false; break; }
            const bool nobody = it.nobody_sees(key0 + row);
            if (row < n_keys && (nobody || !it.all_see(key0 + row, 1, p.m.mask.sinks)) && clean_values<DV>(kv_s + s * Sh::STAGE, row, nobody))
              not_finite_slot[n_it & 3] = n_it + 1;
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");    // visible to the tensor core's reads
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_full[a]));
      }
      g0 += 2 * it.tiles;
      if (!alive) break;
      if (it.tiles > 0) {
        alive = __all_sync(0xffffffffu, mbar_wait(smem_u32(&o_full[a]), n_o & 1u, abort_flag, status, 0x6f));
        if (!alive) break;
        ++n_o;
        tcgen05_fence_after();
      }
      const bool zeroed = it.tiles > 0 && not_finite_slot[n_it & 3] == n_it + 1;
      // what was set to zero of values that this row sees, whose weights are above 0.  SPREAD: the other quarters' keys have weights of 0 in this row, too, so that
      // an infinite value that all see is NaN here, and has to be infinite in its quarter and to count nothing in the others.
      auto add_not_finite = [&](uint32_t (&o)[32], int c) {
        bool add = zeroed;
        if constexpr (SPREAD) {
          float any = 0.f;
#pragma unroll
          for (int e = 0; e < 32; ++e) any = fmaf(__uint_as_float(o[e]), 0.f, any);
          add = zeroed || __any_sync(0xffffffffu, any != 0.f && l == l);
        }
        if (!add) return;
        NotFinite all{0, 0, 0};
        const uint16_t *v = (const uint16_t *)p.m.v + ((size_t)it.s * p.m.kv_heads + it.kvh) * p.m.mask.t_max * p.m.dv;
        for (int j = 0; j < it.tiles; ++j) {
          const int key0 = it.key0(j), halves = it.full(j) ? 2 : 1;
          if (!SPREAD && it.all_see(key0, 64 * halves, p.m.mask.sinks)) continue;
          for (int h = 0; h < halves; ++h) {
            unsigned long long seen = seen_from(key0 + 64 * h);
            if (SPREAD) seen &= quad / 2 == h ? 0xffffffffull << (32 * (quad & 1)) : 0ull;
            const NotFinite r = not_finite(v + (size_t)(key0 + 64 * h) * p.m.dv, p.m.dv, c, seen);
            all.plus |= r.plus;
            all.minus |= r.minus;
            all.nan |= r.nan;
          }
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          float x = __uint_as_float(o[e]);
          if (SPREAD && l == l && x != x) x = 0.f;
          if (all.plus >> e & 1u) x += INFINITY;
          if (all.minus >> e & 1u) x -= INFINITY;
          if (all.nan >> e & 1u) x = NAN;
          o[e] = __float_as_uint(x);
        }
      };
      if (!SPREAD && p.m.splits == 1) {
        // every item has tiles then; the probabilities' buffer takes the result, a block of 64 columns after the other
        const float scale = p.m.out_scale / l;             // at least 1: a row sees itself; 0 where all its scores are -inf, which gives NaN
        if (busy) {
#pragma unroll
          for (int c = 0; c < DV; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(o_base + c, o);
            tmem_ld_wait();
            add_not_finite(o, c);
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const __nv_bfloat162 t = __floats2bfloat162_rn(__uint_as_float(o[e + 2 * k]) * scale, __uint_as_float(o[e + 2 * k + 1]) * scale);
                w[k] = *reinterpret_cast<const uint32_t *>(&t);
              }
              *reinterpret_cast<uint4 *>(prow + c / CB * BLOCK + (((c + e) % CB / 8 ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        tcgen05_fence_before();                            // the loads of O are done before this group's next p_full lets it be overwritten
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        group_sync(1 + a);
        if (leader && !bad) {
          for (int c = 0; c < DV / CB; ++c) tma_store_4d(&tmO, smem_u32(p_group + c * BLOCK), c * CB, it.kvh * p.m.share, r0 / p.m.share, it.s);
          store_commit();
        }
      } else if (busy) {
        const size_t pair = (size_t)(SPREAD ? 4 * it.slice + quad : it.slice) * p.pairs + it.s * p.m.kv_heads + it.kvh;
        const int out_row = r0 + in_rows;
        const bool write = mine && !bad;
        if (mine) p.m.part_ml[pair * p.m.rows + out_row] = make_float2(bad ? NAN : m_ref, l);
        if (it.tiles > 0) {
#pragma unroll
          for (int c = 0; c < DV; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(o_base + c, o);
            tmem_ld_wait();
            add_not_finite(o, c);
            if (write) {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                if (c + e < p.m.dv)
                  *reinterpret_cast<uint4 *>(p.m.part_o + (pair * (p.m.dv / 4) + (c + e) / 4) * p.m.rows + out_row) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
        }
        tcgen05_fence_before();
      }
    }
    if (leader) store_wait();                              // before the shared memory goes
    // a wait gave up: the warps that are still at a barrier of the group's leave it, and give up too
    if (!alive) asm volatile("barrier.cta.arrive %0, 128;" ::"r"(1 + a) : "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  ugb_pdl_trigger();                                       // the combine kernel's CTAs may come and wait
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sh::TMEM_COLS) : "memory");
  }
}

template <int DQ, int DV, int RT0, bool TREE>
int32_t launch(ugb_device *dev, const ugb_masked_attention_args &a, const Params &p) {
  using Sh = Shape<DQ, DV, RT0>;
  static bool attr_set[64] = {};
  if (!attr_set[dev->ordinal & 63]) {
    UGB_CUDA(dev, cudaFuncSetAttribute(masked_attention_tc_kernel<DQ, DV, RT0, TREE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM_BYTES));
    attr_set[dev->ordinal & 63] = true;
  }
  CUtensorMap tmQ, tmK, tmV, tmO;
  int32_t rc;
  auto q_map = [&](CUtensorMap *m, const void *base, int d) {      // [b, t, heads, d]: a box is 64 columns of a group's heads for as many positions as 128 rows hold
    const uint64_t dims[4] = {(uint64_t)d, (uint64_t)a.heads, (uint64_t)a.t, (uint64_t)a.b};
    const uint64_t strides[3] = {(uint64_t)d, (uint64_t)a.heads * d, (uint64_t)a.t * a.heads * d};
    const uint32_t box[4] = {(uint32_t)CB, (uint32_t)p.m.share, (uint32_t)(p.per_group / p.m.share), 1};
    return ugb_tc_encode_bf16(dev, m, (const __nv_bfloat16 *)base, 4, dims, strides, box);
  };
  auto kv_map = [&](CUtensorMap *m, const void *base, int d) {     // [b, kv_heads, t_max, d]
    const uint64_t dims[4] = {(uint64_t)d, (uint64_t)a.kv_heads, (uint64_t)a.t_max, (uint64_t)a.b};
    const uint64_t strides[3] = {(uint64_t)a.t_max * d, (uint64_t)d, (uint64_t)a.kv_heads * a.t_max * d};
    const uint32_t box[4] = {(uint32_t)CB, 1, 64, 1};
    return ugb_tc_encode_bf16(dev, m, (const __nv_bfloat16 *)base, 4, dims, strides, box);
  };
  if ((rc = q_map(&tmQ, a.q, a.dq)) || (rc = q_map(&tmO, a.out, a.dv)) || (rc = kv_map(&tmK, a.k, a.dq)) || (rc = kv_map(&tmV, a.v, a.dv))) return rc;
  masked_attention_tc_kernel<DQ, DV, RT0, TREE><<<(unsigned)((long long)p.row_tiles * p.pairs * p.m.splits), Sh::THREADS, Sh::SMEM_BYTES, dev->stream>>>(tmQ, tmK, tmV, tmO, p);
  return ugb_after_launch(dev, "masked_attention_tc_kernel");
}

// Groups of 128 rows in a CTA; 0: up to 32 rows in all, spread, where the sequences alone fill the GPU and the keys may be so many that HBM is the bound: only
// then is it worth joining the quarters (one position each of 64 sequences, 32 heads on 8 of 128: 1000 keys 57.8 us against 56.4 in one group, 4000 keys
// 158 against 182; of one sequence, 32 on 4 of 64, 2000 keys 18.4 against 16.4, 16000 keys 36.9 against 30.2).
int groups_of(const ugb_masked_attention_args &a, int sms) {
  const int share = a.heads / a.kv_heads;
  const long long reach = a.parents ? a.t_max : std::min<long long>(a.t_max, (long long)a.window + a.t + a.sinks);
  return a.t * share <= 32 && reach >= 2048 && (long long)a.b * a.kv_heads >= sms ? 0 : a.t > 128 / share ? 2 : 1;
}
int per_group(const ugb_masked_attention_args &a, int sms) {
  const int share = a.heads / a.kv_heads;
  return groups_of(a, sms) == 0 ? share * a.t : share * (128 / share);
}
int row_tiles(const ugb_masked_attention_args &a, int sms) {
  const int per = per_group(a, sms) * std::max(1, groups_of(a, sms));
  return (a.t * (a.heads / a.kv_heads) + per - 1) / per;
}

template <int DQ, int DV> int32_t launch_any(ugb_device *dev, const ugb_masked_attention_args &a, const Params &p) {
  const int sms = dev->sm_count;
  if (groups_of(a, sms) == 0) return a.parents ? launch<DQ, DV, 0, true>(dev, a, p) : launch<DQ, DV, 0, false>(dev, a, p);
  if (groups_of(a, sms) == 1) return a.parents ? launch<DQ, DV, 1, true>(dev, a, p) : launch<DQ, DV, 1, false>(dev, a, p);
  return a.parents ? launch<DQ, DV, 2, true>(dev, a, p) : launch<DQ, DV, 2, false>(dev, a, p);
}

}  // namespace

bool ugb_masked_tc_takes(const ugb_device *dev, const ugb_masked_attention_args &a) {
  const int sms = dev->sm_count;
  const bool wide = a.dq <= 128 && a.dv <= 128;
  const bool aligned = (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) & 15) == 0;
  return !a.f32 && wide && aligned && a.heads / a.kv_heads <= 128 && a.scale > 0.f &&
         (long long)row_tiles(a, sms) * a.b * a.kv_heads <= 0x7fffffffLL;
}

void ugb_masked_tc_shape(const ugb_device *dev, const ugb_masked_attention_args &a, long long *items, long long *slots, int *parts, int *positions) {
  const int sms = dev->sm_count;
  *items = (long long)row_tiles(a, sms) * a.b * a.kv_heads;
  *parts = groups_of(a, sms) == 0 ? 4 : 1;
  *positions = per_group(a, sms) * std::max(1, groups_of(a, sms)) / (a.heads / a.kv_heads);
  *slots = (long long)(groups_of(a, sms) <= 1 && a.dq <= 64 && a.dv <= 64 ? 2 : 1) * dev->sm_count;
}

int32_t ugb_masked_tc_launch(ugb_device *dev, const ugb_masked_attention_args &a, const ugb_masked_params &m) {
  const int sms = dev->sm_count;
  Params p;
  p.m = m;
  p.pairs = a.b * a.kv_heads; p.row_tiles = row_tiles(a, sms); p.per_group = per_group(a, sms);
  if (a.dq <= 64) return a.dv <= 64 ? launch_any<64, 64>(dev, a, p) : launch_any<64, 128>(dev, a, p);
  return a.dv <= 64 ? launch_any<128, 64>(dev, a, p) : launch_any<128, 128>(dev, a, p);
}
