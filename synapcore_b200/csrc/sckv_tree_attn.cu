// Attention of a tree of drafted tokens over a paged cache, on the
// 5th-generation tensor cores (tcgen05.mma, accumulators in tensor memory).
//
// Node i of sequence b is the query of rows (i, head); its own K/V row sits in
// slot ctx_lens[b] + i. It sees the ctx_lens[b] committed tokens and the nodes
// j whose bit is set in its mask:
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale_log2 q . k_j - m)
//
// with a running reference m (one pass over K and V).
//
// Work. The rows of a kv head are its (node, q head of the group) pairs, in
// groups of up to two query tiles of 128 rows (one for one-byte pools), over
// the sequence's key tiles of 128 keys (8 pages). The key tiles of all
// (sequence, kv head, row group) items form one line that the CTAs share out
// evenly (one persistent CTA per SM), so that few sequences, long ones and
// ragged batches all keep every SM on HBM. An item that a border cuts leaves
// unnormalised partials (at most two per CTA) that a second kernel joins.
//
// With one query tile the two softmax warpgroups take a half of 64 keys of
// every tile each, with their own reference, sum and O accumulator, joined at
// the end of the item; S has two buffers, so the next tile's scores are made
// while this one's are weighed (a whole tile per warpgroup in turn was slower:
// FP8 793 us against 680). With two query tiles each warpgroup owns one and
// both use every K/V tile. An item of at most 64 (32) rows fills the query
// tile with 2 (4) copies of them, and each copy weighs only its 32 (16) keys of
// the half (P is 0 elsewhere): the lanes of tensor memory that would be idle
// share the softmax, whose time per tile falls accordingly, and the copies'
// sums and O are joined like those of the warpgroups. Either way a tile costs 8
// MMAs of 128 x 128 x 16 for S per query tile and 8 for P V (16 with P in two
// parts): narrower S products (64 keys) take the same time each, limited by
// their operands' shared-memory reads (measured 60 - 150 cycles against 64).
//
// 16 warps (a warp runs on SM sub-partition warp % 4):
//   warps 0, 2   producers. 16-bit pools: K, V by TMA; one 4 KiB box per
//                page-head, which a rank-5 view of the pool lays out as 8-row
//                groups [rows 0-7 | 8-15][dims 0-63 | 64-127], so that groups
//                of consecutive pages have one stride. One-byte pools: K and
//                V of a page in one 4 KiB box into a staging ring, half a tile
//                at a time; the scales.
//   warps 3, 13-19  one-byte pools (20 warps): decode a staged page-head each
//                into the f16 rings. int8 codes times their token's fp16 scale
//                (the rounding that the cache's values have); e4m3 codes
//                exactly, their page's scales go to the scores (K) and to P
//                (V). No load from global memory is on its way in these warps:
//                their proxy fence would wait for it (copying and decoding in
//                one warp: FP8 840 us and more).
//   warps 1, 12  issue the MMAs and commits, from one elected lane each: S, and
//                P V (a wait takes ~250 cycles, beside the other's products);
//                with two query tiles warp 1 all of them, each query tile's S
//                behind its P V.
//   warps 4-11   softmax, one thread per query row; they also load Q and
//                write the results.
//
// Measured with several states in turn, so that nothing is left in L2 (floor:
// bytes at a copy's rate): 32 x 4,096 tokens, 16 fp16 heads without groups, 24
// nodes: 184 us (137), 4.9 TB/s: the rings' loads, and ~4,500 cycles per item to
// write it. 64 x 16,384 tokens, 32 / 8 heads, FP8: 714 us (292; 660 in a short run
// at full clocks, 557 of them the copies alone): the staging ring's turns (48 KiB
// on the way), then the chain decoding - S - softmax - P V. 4 x 65,536 tokens, 32 /
// 8 heads, 64 nodes, bf16: 419 us (164, and 246 of tensor time with P in two parts;
// 379 in a short run): the exponentials, 2,048 cycles of a pair of tiles, behind
// the waits for S.
//
// P is held as 2^6 times the weight, so that f16's smallest step is 2^-31 of
// a weight of 1 (m is stale by at most 2^8: P <= 2^14); e4m3 pages multiply it
// by their V scale over a reference that has seen the largest one. P is split
// into hi + lo parts on bf16 pools (rounding 2^-16) and for fp32 outputs (f16:
// 2^-22), which costs a second P V product. For 16-bit outputs the other pools
// have one f16 part, 2^-11 at most: an eighth of a bf16 output's own step.
// Beside an f16 output's it shows (32 x 4,096 tokens against 64 bits: 2.8e-4,
// the output's rounding alone 2.1e-4); two parts cost 203 us instead of 184
// there, 817 instead of 714 (FP8) and 71 instead of 63 (int8). Sums, references
// and O are fp32. int8 codes stand for fp16(code x scale), as the arena's
// dequantisation, gather and the prefill kernel have them (one-token decode
// multiplies in fp32: a difference of 2^-11 of a value at most).
//
// Rows of K/V tiles past the sequence's last node hold anything: their scores
// are masked and their V rows zeroed. A node's V that is not finite must not
// reach rows that do not see it (0 x NaN): such elements are zeroed in the
// tile and added to the rows that see them at the end. Every row sees the
// committed tokens; there a NaN result is looked into (its sum is none).
#include <cuda.h>
#include <math.h>
#include <type_traits>

#include "sckv_geo.cuh"
#include "sckv_mma_common.cuh"
#include "sckv_tcgen05.cuh"

using namespace sckv_geo;
using namespace sckv_mma;
using namespace sckv_tc;

namespace {

constexpr int kHD = 128;
constexpr int kMaskWordsMax = 4;
constexpr int kMaxSeqs = 2048;
constexpr int kRows = 128;                     // rows of a query tile (UMMA M)
constexpr int kHalf = 64;                      // keys of half a K/V tile
constexpr int kKeys = 2 * kHalf;               // keys of a K/V tile
constexpr int kHalfPages = kHalf / SCKV_PAGE_TOKENS;
constexpr int kTilePages = 2 * kHalfPages;
constexpr int kMaxWarps = 20;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 0;                  // S[x] at 128 x
constexpr uint32_t kColO = 256;                // O[w] at 256 + 128 w
constexpr int kWarpProdA = 0, kWarpMma = 1, kWarpProdB = 2, kWarpMma2 = 12;
constexpr int kQHalf = kRows * 128;            // one 64-dim half of a query tile: 16 KiB
constexpr int kQTile = 2 * kQHalf;
constexpr int kPageTile = 4096;                // one page-head in f16 / bf16
constexpr int kHalfSlot = kHalfPages * kPageTile;
constexpr int kSlot = 2 * kHalfSlot;           // a K (or V) tile: 32 KiB
constexpr int kStages = 2;                     // K and V tiles in the MMA's type
constexpr int kScaleSlots = 16;                // one-byte pools: half tiles whose scales are kept

template <int KVDT>
struct TreeCfg {
  static constexpr bool kFP8 = KVDT == SCKV_DTYPE_FP8_E4M3, kINT8 = KVDT == SCKV_DTYPE_INT8;
  static constexpr bool kB8 = kFP8 || kINT8;
  static constexpr bool kBF16 = KVDT == SCKV_DTYPE_BF16;
  static constexpr int kThreads = kB8 ? 640 : 512;
  static constexpr int kSoftRegs = kB8 ? 144 : 176, kGiveRegs = kB8 ? 64 : 80;  // registers after the roles split
  static constexpr int kQTiles = kB8 ? 1 : 2;
  static constexpr int kStaging = kB8 ? 3 : 0;        // staged half tiles of codes (K and V)
  static constexpr int kOffK = kQTiles * kQTile;
  static constexpr int kOffV = kOffK + kStages * kSlot;
  static constexpr int kOffStage = kOffV + kStages * kSlot;
  static constexpr int kOffScale = kOffStage + kStaging * kHalfSlot;
  static constexpr int kOffBar = kOffScale + (kB8 ? kScaleSlots * 256 : 0);
  static constexpr int kNumBars = 4 * kStages + 6 + 6 + 2 * kStaging;
  static constexpr int kOffMl = kOffBar + ((kNumBars * 8 + 15) / 16) * 16;  // float2 [2][128]: m, l of a row
  static constexpr int kOffVref = kOffMl + 2 * kRows * 8;                   // float [2][4]: V scale of a warp's O
  static constexpr int kOffBad = kOffVref + 32;                             // u64 [2][4]: nodes whose V is not finite
  static constexpr int kOffTmem = kOffBad + 64;
  static constexpr int kOffAbort = kOffTmem + 4;
  static constexpr int kOffPartial = kOffTmem + 16;                         // int [warps]
  static constexpr int kOffCum = kOffPartial + kMaxWarps * 4;               // int [n_seqs + 1]
  static constexpr int kFixedSmem = 1024 + kOffCum + 4;                     // + 4 n_seqs
  static_assert(2 * kStages + kStaging < kScaleSlots, "scale slots outlive their half tiles");
};

// What the joining kernel needs of a CTA whose first item began in an earlier one and ends in it.
struct JoinHead {
  int n_parts, c0, slot0, rows, row0, q_base, h, pad;
};

struct TreeParams {
  Geo g;
  int layer;
  const void* q;
  void* out;
  const int32_t* cu_q;
  const int32_t* ctx_lens;
  const int32_t* bt;
  int64_t bt_stride;
  const unsigned long long* mask;
  int mask_words;
  int max_blocks, n_seqs, n_tokens, hq, G;
  uint32_t g_mul;   // 2^32 / G + 1 (0: G is 1)
  int group_shift;  // log2 of a row group's rows: 8, one-byte pools 7
  int q_dtype, out_dtype;
  float scale_log2;
  // workspace: JoinHead [grid], then per CTA two slots of float4 [32][part_rows] (O by 4 dims and row)
  // and float2 [part_rows] (m, l)
  JoinHead* heads;
  float* parts;
  int part_rows;
};

__device__ __forceinline__ int64_t slot_floats(int part_rows) { return (int64_t)part_rows * (kHD + 2); }

// Geometry of one sequence: nodes, committed tokens, key tiles, row groups; false (all zero) if out of range.
__device__ __forceinline__ bool tree_seq(const TreeParams& p, int s, int& n, int& ctx, int& kt, int& groups) {
  const int t0 = __ldg(p.cu_q + s), t1 = __ldg(p.cu_q + s + 1);
  ctx = __ldg(p.ctx_lens + s);
  const int cap = p.max_blocks * SCKV_PAGE_TOKENS;
  n = t1 - t0;
  const bool ok = t0 >= 0 && t1 >= t0 && t1 <= p.n_tokens && n <= 64 * p.mask_words && ctx >= 0 && ctx <= cap - n;
  if (!ok) n = ctx = 0;
  kt = n > 0 ? (ctx + n + kKeys - 1) / kKeys : 0;
  groups = (n * p.G + (1 << p.group_shift) - 1) >> p.group_shift;
  return ok;
}

// Node of row rr of a sequence's group: rr / G. Exact while rr G < 2^32; rr < 256 G.
__device__ __forceinline__ int tree_node(const TreeParams& p, int rr) {
  return p.g_mul ? (int)__umulhi((uint32_t)rr, p.g_mul) : rr;
}
constexpr int kMaxGroup = 4095;

// A CTA's walk over its share of the line of key tiles, one item (or part of one) at a time.
struct TreeWalk {
  int seq, t, t1;
};
struct TreeSeg {
  int seq, h, n, ctx, L;
  int kt, ka, nk;         // the item's key tiles; first one here and how many
  int row0, rows, nq;     // first row of the group, rows of it, query tiles (1 or 2)
  int copies;             // copies of the rows in the query tile (1, 2, 4)
  int q_base, pages;      // first token; pages of the sequence
};

__device__ __forceinline__ bool tree_next(const TreeParams& p, const int* cum, TreeWalk& w, TreeSeg& s) {
  if (w.t >= w.t1) return false;
  while (cum[w.seq + 1] <= w.t) ++w.seq;
  int groups;
  tree_seq(p, w.seq, s.n, s.ctx, s.kt, groups);
  const int rem = w.t - cum[w.seq];
  const int item = rem / s.kt;
  s.seq = w.seq;
  s.ka = rem - item * s.kt;
  s.nk = min(s.kt - s.ka, w.t1 - w.t);
  s.h = item / groups;
  s.row0 = (item - s.h * groups) << p.group_shift;
  s.rows = min(1 << p.group_shift, s.n * p.G - s.row0);
  s.nq = s.rows > kRows ? 2 : 1;
  s.copies = s.rows <= kRows / 4 ? 4 : s.rows <= kRows / 2 ? 2 : 1;
  s.L = s.ctx + s.n;
  s.pages = (s.L + SCKV_PAGE_TOKENS - 1) / SCKV_PAGE_TOKENS;
  s.q_base = __ldg(p.cu_q + s.seq);
  w.t += s.nk;
  return true;
}

// The CTA (of n) whose share of `total` tiles holds tile t; shares begin at total * c / n.
__device__ __forceinline__ int tree_owner(int t, int total, int n) {
  return (int)((((int64_t)t + 1) * n - 1) / total);
}
__device__ __forceinline__ int tree_begin(int c, int total, int n) {
  const int q = total / n, r = total - q * n;  // (32-bit divisions; c, r <= n, the number of SMs)
  return c * q + c * r / n;
}

// 64 bits from bit `off` of a row's view of keys ctx + i: ones for committed tokens (i < 0), the mask for nodes
// i < n, zeros after.
__device__ __forceinline__ unsigned long long tree_window(const unsigned long long* words, int n_words, int n,
                                                          int off) {
  if (off <= -64) return ~0ull;
  auto word = [&](int i) -> unsigned long long {
    if (i >= n_words || 64 * i >= n) return 0ull;
    const unsigned long long live = n - 64 * i >= 64 ? ~0ull : (1ull << (n - 64 * i)) - 1;
    return __ldg(words + i) & live;
  };
  if (off < 0) return ((1ull << -off) - 1) | (word(0) << -off);
  const int i = off >> 6, sh = off & 63;
  return sh ? (word(i) >> sh) | (word(i + 1) << (64 - sh)) : word(i);
}

// Element (node's row, dim) of V as the cache stands for it.
__device__ float tree_v(const Geo& g, int layer, int64_t page, int h, int slot, int d) {
  const int64_t o = row_off(g, layer, page, 1, h, slot) + d;
  if (g.dtype == SCKV_DTYPE_INT8)
    return __half2float(__hmul(__float2half_rn((float)reinterpret_cast<const int8_t*>(g.data)[o]),
                               reinterpret_cast<const __half*>(g.scales)[int8_scale_idx(g, layer, page, 1, h, slot)]));
  if (g.dtype == SCKV_DTYPE_FP8_E4M3)
    return sckv_fp8_to_float(reinterpret_cast<const uint8_t*>(g.data)[o]) *
           reinterpret_cast<const float*>(g.scales)[fp8_scale_idx(g, layer, page, 1, h)];
  return sckv_load_as_float(g.data, o, g.dtype);
}

__device__ __forceinline__ void tree_store4(void* dst, int64_t idx, int dtype, float a, float b, float c, float d) {
  if (dtype == SCKV_DTYPE_F32) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(dst) + idx) = make_float4(a, b, c, d);
  } else {
    const uint2 v = dtype == SCKV_DTYPE_BF16 ? make_uint2(pack2<true>(a, b), pack2<true>(c, d))
                                             : make_uint2(pack2<false>(a, b), pack2<false>(c, d));
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(dst) + idx) = v;
  }
}

// Barriers by their shared-memory address.
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded by SCKV_WAIT_LIMIT_NS; a plain test first (most waits are short), the global timer once per 64 polls.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  if (bar_test(bar, parity)) return true;
  uint64_t t0 = 0;
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (bar_try(bar, parity)) return true;
    const uint64_t t = globaltimer_ns();
    if (t0 == 0) t0 = t;
    else if (t - t0 > SCKV_WAIT_LIMIT_NS) return false;
  }
}
// Every lane of the warp waits; the result is the same on all lanes.
__device__ __forceinline__ bool warp_wait_bar(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, bar_wait(bar, parity));
}
// 5-D tiled TMA load.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x0, int x1, int x2, int x3, int x4,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
      "%6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x0), "r"(x1), "r"(x2), "r"(x3), "r"(x4), "r"(bar)
      : "memory");
}

// 8 / 16 columns of this thread's tensor memory lane.
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ void bar_arrive_n(uint32_t bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(n) : "memory");
}

// 1 on one lane of the (converged) warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(r));
  return r;
}

template <int N>
__device__ __forceinline__ void reg_give() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// kSplit: the weights P in two parts (hi + lo) in tensor memory.
template <int KVDT, bool kSplit>
__global__ void __launch_bounds__(TreeCfg<KVDT>::kThreads, 1)
    tree_attn_kernel(const TreeParams p, const __grid_constant__ CUtensorMap tmap) {
  using C = TreeCfg<KVDT>;
  constexpr bool kBF16 = C::kBF16;
  static_assert(kSplit || !kBF16, "one bf16 part would round a weight by 2^-9");
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // barriers, as shared-memory addresses (8 bytes each)
  const uint32_t bar0 = smem_u32(base + C::kOffBar);
  const uint32_t k_full = bar0;                   // [S] K tile in shared memory
  const uint32_t k_empty = k_full + 8 * kStages;      // [S] the S products that read it finished (commit)
  const uint32_t v_full = k_empty + 8 * kStages;      // [S] V tile in shared memory
  const uint32_t v_empty = v_full + 8 * kStages;      // [S] the PV products that read it finished (commit)
  // set x: one query tile: tile i of the item uses set i & 1; two: query tile w uses set w for every tile
  const uint32_t s_full = v_empty + 8 * kStages;      // [x] S in tensor memory (commit)
  const uint32_t p_full = s_full + 8 * 2;             // [x] P in tensor memory, V tile fixed (8 arrivals)
  const uint32_t pv_done = p_full + 8 * 2;            // [x] PV finished (commit)
  // the item's Q is in shared memory and the O of the item before was read (one arrival per softmax warp), and the PV
  // warp is at the item too
  const uint32_t q_full = pv_done + 8 * 2;
  const uint32_t mma_done = q_full + 8 * 1;           // every issued MMA finished
  // the item's sums are written and its O is complete (one arrival per softmax warp)
  const uint32_t o_full = mma_done + 8 * 1;
  // [w] a piece of O is in the exchange buffer (one arrival per warp of w)
  const uint32_t x_full = o_full + 8 * 1;
  const uint32_t x_done = x_full + 8 * 2;             // the exchange buffer was read (one arrival per softmax warp)
  const uint32_t st_full = x_done + 8 * 1;            // one-byte pools: [SS] staged half tile, scales are there
  const uint32_t st_empty = st_full + 8 * C::kStaging;  // [SS] decoded (one arrival per decoding warp)
  float2* s_ml = reinterpret_cast<float2*>(base + C::kOffMl);
  float* s_vref = reinterpret_cast<float*>(base + C::kOffVref);
  unsigned long long* s_bad = reinterpret_cast<unsigned long long*>(base + C::kOffBad);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base + C::kOffTmem);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(base + C::kOffAbort);
  int* partial = reinterpret_cast<int*>(base + C::kOffPartial);
  int* cum = reinterpret_cast<int*>(base + C::kOffCum);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  pdl_trigger();
  if (warp == kWarpMma) tmem_alloc(tmem_slot, kTmemCols);
  // ---- key tiles per sequence, prefix-summed by the whole CTA
  {
    const int per = (p.n_seqs + C::kThreads - 1) / C::kThreads;
    const int s0 = min(p.n_seqs, (int)threadIdx.x * per), s1 = min(p.n_seqs, s0 + per);
    int local = 0, n, ctx, kt, groups;
    for (int s = s0; s < s1; ++s) {
      if (!tree_seq(p, s, n, ctx, kt, groups) && blockIdx.x == 0)
        sckv_report(p.g.status, SCKV_ERR_BOUNDS, s, KID_TREE_ATTN);
      local += kt * groups * p.g.H;
    }
    // inclusive scan within each warp, then over the warps
    int x = local;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) partial[warp] = x;
    if ((int)threadIdx.x < C::kNumBars) {
      const uint32_t bar = bar0 + 8 * threadIdx.x;
      uint32_t count = 1;
      if (C::kB8 && ((bar >= k_full && bar < k_full + 8 * kStages) || (bar >= v_full && bar < v_full + 8 * kStages))) count = 8;
      if (bar >= p_full && bar < p_full + 16) count = 8;
      if (bar == mma_done) count = 2;
      if (bar == o_full || bar == x_done) count = 8;
      if (bar == q_full) count = 9;
      if (bar == x_full || bar == x_full + 8) count = 4;
      if (C::kB8 && bar >= st_full && bar < st_full + 8 * C::kStaging) count = 2;
      if (C::kB8 && bar >= st_empty && bar < st_empty + 8 * C::kStaging) count = 8;
      bar_init(bar, count);
      fence_mbar_init();
    }
    if (threadIdx.x < 2 * kMaskWordsMax) s_bad[threadIdx.x] = 0;
    if (threadIdx.x == 0) *abort_flag = 0;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < warp; ++i) before += partial[i];
    int run = before + x - local;
    for (int s = s0; s < s1; ++s) {
      cum[s] = run;
      if (s + 1 < s1) {
        tree_seq(p, s, n, ctx, kt, groups);
        run += kt * groups * p.g.H;
      }
    }
    if (threadIdx.x == C::kThreads - 1) cum[p.n_seqs] = before + x;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  }
  const uint32_t tmem = *tmem_slot;
  const int total = cum[p.n_seqs];
  // CTAs that take a share
  const int n_cta = max(1, min((int)gridDim.x, total));
  TreeWalk walk{0, 0, 0};
  if ((int)blockIdx.x < n_cta && total > 0) {
    walk.t = tree_begin(blockIdx.x, total, n_cta);
    walk.t1 = tree_begin(blockIdx.x + 1, total, n_cta);
    int lo = 0, hi = p.n_seqs - 1;
    while (lo < hi) {  // the last sequence that begins at or before t
      const int mid = (lo + hi + 1) >> 1;
      if (cum[mid] <= walk.t) lo = mid; else hi = mid - 1;
    }
    walk.seq = lo;
  }
  const int64_t layer_base = (int64_t)p.layer * p.g.P;
  // Registers: 128 a thread at launch (one-byte pools: 96); the softmax warpgroups take 176 (144) for a row's 64 scores
  // and their P, the others give theirs up: 256 x 80 + 256 x 176 = 512 x 128 (384 x 64 + 256 x 144 = 640 x
  // 96). Each role does it in its own branch, so that the compiler knows the count of every region.
  if (warp == kWarpProdA || warp == kWarpProdB) {
    // ------------------------------------------------------------ producers
    reg_give<C::kGiveRegs>();
    // A lane owns a page of the tile: its id is loaded one tile ahead (and not looked at in the turn that loads it,
    // which would wait for it), and the copies of all pages go out as one instruction (one lane after the other
    // issued them in ~180 cycles each, which paced the kernel).
    const int part = warp == kWarpProdB ? 1 : 0;  // 16-bit: K, V; one-byte: codes, scales
    if (lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap)) : "memory");
    TreeSeg s;
    int g = 0;
    bool aborted = false;
    auto valid_page = [&](int page) -> int {
      if (page >= 0 && page < p.g.P) return page;
      sckv_report(p.g.status, SCKV_ERR_BOUNDS, page, KID_TREE_ATTN);
      return 0;
    };
    if constexpr (!C::kB8) {
      const uint32_t fulls = part ? v_full : k_full, empties = part ? v_empty : k_empty;
      const uint32_t ring = smem_u32(base + (part ? C::kOffV : C::kOffK)) + lane * kPageTile;
      while (!aborted && tree_next(p, cum, walk, s)) {
        const int32_t* bt_row = p.bt + (int64_t)s.seq * p.bt_stride;
        auto there = [&](int j) { return lane < kTilePages && j * kTilePages + lane < s.pages; };
        const int je = s.ka + s.nk;
        int nxt = there(s.ka) ? __ldg(bt_row + s.ka * kTilePages + lane) : 0;
        for (int j = s.ka; j < je; ++j, ++g) {
          const int id = nxt;
          if (j + 1 < je && there(j + 1)) nxt = __ldg(bt_row + (j + 1) * kTilePages + lane);
          const int st = g % kStages;
          if (*abort_flag || (g >= kStages && !warp_wait_bar(empties + 8 * st, ((g / kStages) - 1) & 1))) {
            aborted = true;
            break;
          }
          if (lane == 0) bar_expect(fulls + 8 * st, (uint32_t)min(kTilePages, s.pages - j * kTilePages) * kPageTile);
          __syncwarp();
          if (there(j)) {
            const int slab = (int)(((layer_base + valid_page(id)) * 2 + part) * p.g.H + s.h);
            tma_load(ring + st * kSlot, &tmap, 0, 0, 0, 0, slab, fulls + 8 * st);
          }
          __syncwarp();
        }
      }
      // nothing of ours may still be landing when the CTA retires
      for (int t = g > kStages ? g - kStages : 0; t < g; ++t)
        warp_wait_bar(fulls + 8 * (t % kStages), (t / kStages) & 1);
    } else if (part == 0) {
      const uint32_t ring = smem_u32(base + C::kOffStage) + lane * 4096;
      while (!aborted && tree_next(p, cum, walk, s)) {
        const int32_t* bt_row = p.bt + (int64_t)s.seq * p.bt_stride;
        auto there = [&](int j) { return lane < kHalfPages && j * kHalfPages + lane < s.pages; };
        const int je = 2 * (s.ka + s.nk);
        int nxt = there(2 * s.ka) ? __ldg(bt_row + 2 * s.ka * kHalfPages + lane) : 0;
        for (int j = 2 * s.ka; j < je; ++j, ++g) {
          const int id = nxt;
          if (j + 1 < je && there(j + 1)) nxt = __ldg(bt_row + (j + 1) * kHalfPages + lane);
          const int st = g % C::kStaging;
          if (*abort_flag || (g >= C::kStaging && !warp_wait_bar(st_empty + 8 * st, ((g / C::kStaging) - 1) & 1))) {
            aborted = true;
            break;
          }
          if (lane == 0)
            bar_expect(st_full + 8 * st, (uint32_t)max(0, min(kHalfPages, s.pages - j * kHalfPages)) * 4096u);
          __syncwarp();
          if (there(j))
            tma_load(ring + st * kHalfSlot, &tmap, 0, 0, s.h, 0, (int)(layer_base + valid_page(id)), st_full + 8 * st);
          __syncwarp();
        }
      }
      for (int t = g > C::kStaging ? g - C::kStaging : 0; t < g; ++t)
        warp_wait_bar(st_full + 8 * (t % C::kStaging), (t / C::kStaging) & 1);
    } else {
      // scales of a half tile: int8 four tokens' fp16 per lane (K, V; 4 pages; 4 x 4 tokens); FP8 lanes 0-3 the K,
      // 4-7 the V scales of its pages, a page past the last node scales by 1 (K, masked anyway) and 0 (V). Loaded one
      // half tile ahead, the page ids two.
      const int skv = C::kINT8 ? lane >> 4 : (lane >> 2) & 1, spg = C::kINT8 ? (lane >> 2) & 3 : lane & 3;
      const bool mine = C::kINT8 || lane < 8;
      while (!aborted && tree_next(p, cum, walk, s)) {
        const int32_t* bt_row = p.bt + (int64_t)s.seq * p.bt_stride;
        const int je = 2 * (s.ka + s.nk);
        auto there = [&](int j) { return mine && j < je && j * kHalfPages + spg < s.pages; };
        auto fetch = [&](int j) -> int { return there(j) ? __ldg(bt_row + j * kHalfPages + spg) : 0; };
        auto load_scale = [&](int page, int j) -> uint2 {
          uint2 r = make_uint2(C::kFP8 && skv == 0 ? 0x3f800000u : 0u, 0u);
          if (page < 0 || page >= p.g.P) page = 0;
          const int64_t at = ((layer_base + page) * 2 + skv) * p.g.H + s.h;
          if (there(j)) {
            if (C::kINT8)
              r = __ldg(reinterpret_cast<const uint2*>(p.g.scales) + at * 4 + (lane & 3));
            else
              r.x = __ldg(reinterpret_cast<const uint32_t*>(p.g.scales) + at);
          }
          return r;
        };
        uint2 sc = load_scale(fetch(2 * s.ka), 2 * s.ka);
        int sid = fetch(2 * s.ka + 1);
        for (int j = 2 * s.ka; j < je; ++j, ++g) {
          const int st = g % C::kStaging;
          const uint2 now = sc;
          sc = load_scale(sid, j + 1);
          sid = fetch(j + 2);
          if (*abort_flag || (g >= C::kStaging && !warp_wait_bar(st_empty + 8 * st, ((g / C::kStaging) - 1) & 1))) {
            aborted = true;
            break;
          }
          uint8_t* slot = base + C::kOffScale + (g % kScaleSlots) * 256;
          if (C::kINT8)
            reinterpret_cast<uint2*>(slot)[lane] = now;
          else if (lane < 8)  // (a K scale of 0 would turn masked scores, -inf, into NaN; NaN stays)
            reinterpret_cast<float*>(slot)[lane] =
                skv == 0 && __uint_as_float(now.x) < 1e-30f ? 1e-30f : __uint_as_float(now.x);
          __syncwarp();
          if (lane == 0) bar_arrive(st_full + 8 * st);
        }
      }
    }
    if (aborted && lane == 0) {
      if (!*abort_flag) sckv_report(p.g.status, SCKV_ERR_TIMEOUT, blockIdx.x, KID_TREE_ATTN);
      *abort_flag = 1;
    }
  } else if (C::kB8 && (warp == 3 || warp >= 13)) {
    // ------------------------------------------------------------ decoding of one-byte pages
    // Warp `role` decodes page role & 3 of K (role < 4) or V of each half tile. Lane
    // (quarter, rowbit, c): rows r and r ^ 5 of a quarter's eight lanes keep both the
    // swizzled 16-byte reads and the two 16-byte writes free of bank conflicts.
    reg_give<C::kGiveRegs>();
    if constexpr (C::kB8) {
      const int role = warp == 3 ? 0 : warp - 12;
      const int kv = role >> 2, pg = role & 3;
      const uint32_t fulls = kv ? v_full : k_full;
      const uint32_t empties = kv ? v_empty : k_empty;
      uint8_t* ring = base + (kv ? C::kOffV : C::kOffK);
      const int qt = lane >> 3;
      const int r8 = (lane & 4) ? qt ^ 5 : qt;  // row of the 8-row group
      TreeSeg s;
      int g = 0;  // half tiles
      bool aborted = false;
      while (!aborted && tree_next(p, cum, walk, s)) {
        for (int j = 2 * s.ka; j < 2 * (s.ka + s.nk); ++j, ++g) {
          const int ss = g % C::kStaging, gt = g >> 1, st = gt & 1;
          if (((g & 1) == 0 && gt >= 2 && (*abort_flag || !warp_wait_bar(empties + 8 * st, ((gt >> 1) - 1) & 1))) ||
              !warp_wait_bar(st_full + 8 * ss, (g / C::kStaging) & 1)) {
            aborted = true;
            break;
          }
          if (j * kHalfPages + pg < s.pages) {
            const __half* tok = reinterpret_cast<const __half*>(base + C::kOffScale + (g % kScaleSlots) * 256) +
                                kv * 64 + pg * SCKV_PAGE_TOKENS;
            const uint8_t* src = base + C::kOffStage + ss * kHalfSlot + pg * 4096 + kv * 2048;
            uint8_t* dst = ring + st * kSlot + (g & 1) * kHalfSlot + pg * kPageTile;
            uint4 w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)  // row 8 (e / 2) + r8, codes of dims 64 (e % 2) + 16 (lane % 4) ..
              w[e] = *reinterpret_cast<const uint4*>(src + ((e >> 1) * 8 + r8) * 128 +
                                                     ((((e & 1) * 4 + (lane & 3)) ^ r8) << 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              __half2 s2 = __half2half2(__half(1.f));
              if (C::kINT8) s2 = __half2half2(tok[(e >> 1) * 8 + r8]);
              const uint32_t ws[4] = {w[e].x, w[e].y, w[e].z, w[e].w};
              uint32_t o[8];
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                cvt_b8x4<KVDT>(ws[c], o[2 * c], o[2 * c + 1]);
                if (C::kINT8) {
#pragma unroll
                  for (int k = 0; k < 2; ++k) {
                    const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&o[2 * c + k]), s2);
                    o[2 * c + k] = *reinterpret_cast<const uint32_t*>(&x);
                  }
                }
              }
              uint8_t* d = dst + (e >> 1) * 2048 + (e & 1) * 1024 + r8 * 128;
              const int c = 2 * (lane & 3);
              *reinterpret_cast<uint4*>(d + ((c ^ r8) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<uint4*>(d + (((c + 1) ^ r8) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
            }
            fence_proxy_async_smem();  // read by the tensor cores
          }
          // The staged slot is free too: what was stored needed the loads from it to be complete, and the proxy fence
          // stands between them and the next copy (TMA, the async proxy) into it. A release before the stores has
          // neither.
          __syncwarp();
          if (lane == 0) {
            bar_arrive(fulls + 8 * st);
            bar_arrive(st_empty + 8 * ss);
          }
        }
      }
      if (aborted && lane == 0) {
        if (!*abort_flag) sckv_report(p.g.status, SCKV_ERR_TIMEOUT, blockIdx.x, KID_TREE_ATTN);
        *abort_flag = 1;
      }
    }
  } else if (warp == kWarpMma || warp == kWarpMma2) {
    // ------------------------------------------------------------ MMA issuers
    // A whole warp walks and waits, one elected lane issues (a role on one lane alone measured 1.3 x slower).
    reg_give<C::kGiveRegs>();
    const int mw = warp == kWarpMma2 ? 1 : 0;
    if (mw == 1 && lane == 0) {  // what the joining kernel needs; by a warp that waits long for its first P
      JoinHead hd{};
      TreeWalk w = walk;
      TreeSeg s;
      if (tree_next(p, cum, w, s) && s.ka > 0 && s.ka + s.nk == s.kt) {
        const int first = walk.t - s.ka;  // the item's first tile
        hd.c0 = tree_owner(first, total, n_cta);
        hd.slot0 = tree_begin(hd.c0, total, n_cta) == first ? 0 : 1;
        hd.n_parts = (int)blockIdx.x - hd.c0 + 1;
        hd.rows = s.rows;
        hd.row0 = s.row0;
        hd.q_base = s.q_base;
        hd.h = s.h;
      }
      p.heads[blockIdx.x] = hd;
    }
    __syncwarp();
    const uint32_t el = elect_one();
    constexpr uint32_t kIdescS = instr_desc_f16(kBF16, kKeys, false);
    constexpr uint32_t kIdescPV = instr_desc_f16(kBF16, kHD, true);
    const uint64_t q_desc0 = smem_desc_sw128(smem_u32(base), 16, 1024);
    const uint64_t k_desc0 = smem_desc_sw128(smem_u32(base + C::kOffK), 16, 2048);
    const uint64_t v_desc0 = smem_desc_sw128(smem_u32(base + C::kOffV), 1024, 2048);
    // S[x] = Q tile w . K of slot st
    auto issue_s = [&](int x, int w, int st) {
      const uint64_t qd = desc_advance(q_desc0, (uint32_t)(w * kQTile));
      const uint64_t kd = desc_advance(k_desc0, (uint32_t)(st * kSlot));
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        const int half = ks >> 2, kk = ks & 3;
        umma_ss(tmem + kColS + (uint32_t)(x * kKeys), desc_advance(qd, (uint32_t)(half * kQHalf + kk * 32)),
                desc_advance(kd, (uint32_t)(half * 1024 + kk * 32)), kIdescS, ks > 0);
      }
      bar_commit(s_full + 8 * x);
    };
    // O[w] (+)= P[x], half h . V of slot st, half h
    auto issue_pv = [&](int x, int h, int w, int st, bool first) {
      const uint64_t vd = desc_advance(v_desc0, (uint32_t)(st * kSlot + h * kHalfSlot));
      const uint32_t pa = tmem + kColS + (uint32_t)(x * kKeys + h * kHalf), o = tmem + kColO + (uint32_t)(w * kHD);
#pragma unroll
      for (int pg = 0; pg < kHalfPages; ++pg) {
        // B = V rows of page pg: 128 dims in two 64-dim halves (LBO), 16 keys in two 8-row groups (SBO)
        const uint64_t bdesc = desc_advance(vd, (uint32_t)(pg * kPageTile));
        umma_ts(o, pa + (uint32_t)(pg * 8), bdesc, kIdescPV, (!first || pg > 0) ? 1u : 0u);
        if (kSplit) umma_ts(o, pa + (uint32_t)(pg * 8 + 32), bdesc, kIdescPV, 1u);
      }
    };
    TreeSeg s;
    bool ok = true;
    int gt = 0;              // tiles of earlier items
    int cnt[2] = {0, 0};     // uses of each set in earlier items
    for (int k = 0; ok && tree_next(p, cum, walk, s); ++k) {
      const bool two = C::kQTiles == 2 && s.nq == 2;
      // Both warps begin an item together: the PV warp, which has nothing to do for an item of two query tiles, would
      // otherwise wait for phases of P and V several uses ahead, which their parity cannot tell from earlier ones.
      if (mw == 1 && lane == 0) bar_arrive(q_full);
      if (*abort_flag || !warp_wait_bar(q_full, k & 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (!two && mw == 0) {
        // ---- S of every tile
        for (int i = 0; i < s.nk; ++i) {
          const int g = gt + i, st = g % kStages, x = i & 1, use = cnt[x] + (i >> 1);
          // (S replaces the P that the set's last PV read)
          if (*abort_flag || !warp_wait_bar(k_full + 8 * st, (g / kStages) & 1) ||
              (use > 0 && !warp_wait_bar(pv_done + 8 * x, (use - 1) & 1))) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (el) {
            issue_s(x, 0, st);
            bar_commit(k_empty + 8 * st);
          }
          __syncwarp();
        }
      } else if (!two) {
        // ---- P V of every tile
        for (int i = 0; i < s.nk; ++i) {
          const int g = gt + i, st = g % kStages, x = i & 1, use = cnt[x] + (i >> 1);
          if (*abort_flag || !warp_wait_bar(v_full + 8 * st, (g / kStages) & 1) ||
              !warp_wait_bar(p_full + 8 * x, use & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (el) {
            issue_pv(x, 0, 0, st, i == 0);
            if ((s.ka + i) * kKeys + kHalf < s.L) issue_pv(x, 1, 1, st, i == 0);  // the second half holds keys
            bar_commit(pv_done + 8 * x);
            bar_commit(v_empty + 8 * st);
          }
          __syncwarp();
        }
      } else if (two && mw == 0) {
        // ---- two query tiles: S(i) of each follows its PV(i - 1) into the columns that held its P
        for (int i = 0; ok && i <= s.nk; ++i) {
          const int g = gt + i, st = g % kStages, su = (g + kStages - 1) % kStages;
          if (i < s.nk && (*abort_flag || !warp_wait_bar(k_full + 8 * st, (g / kStages) & 1))) ok = false;
          if (ok && i > 0 && !warp_wait_bar(v_full + 8 * su, ((g - 1) / kStages) & 1)) ok = false;
          for (int w = 0; ok && w < 2; ++w) {
            const int use = cnt[w] + i;
            // (the first S of the item: the set's last PV may be another warp's)
            if (i > 0 ? !warp_wait_bar(p_full + 8 * w, (use - 1) & 1)
                      : use > 0 && !warp_wait_bar(pv_done + 8 * w, (use - 1) & 1)) {
              ok = false;
              break;
            }
            tc_fence_after();
            if (el) {
              if (i > 0) {
                issue_pv(w, 0, w, su, i == 1);
                if ((s.ka + i - 1) * kKeys + kHalf < s.L) issue_pv(w, 1, w, su, false);
                bar_commit(pv_done + 8 * w);
              }
              if (i < s.nk) issue_s(w, w, st);
            }
            __syncwarp();
          }
          if (ok && el) {
            if (i < s.nk) bar_commit(k_empty + 8 * st);
            if (i > 0) bar_commit(v_empty + 8 * su);
          }
          __syncwarp();
        }
      }
      if (!ok) break;
      gt += s.nk;
      cnt[0] += two ? s.nk : (s.nk + 1) >> 1;
      cnt[1] += two ? s.nk : s.nk >> 1;
    }
    if (!ok && lane == 0) {
      if (!*abort_flag) sckv_report(p.g.status, SCKV_ERR_TIMEOUT, blockIdx.x, KID_TREE_ATTN);
      *abort_flag = 1;
    }
    if (el) bar_commit(mma_done);  // every MMA of both warps has finished before the tensor memory is released
    __syncwarp();
    warp_wait_bar(mma_done, 0);
  } else if (warp >= 4 && warp < 12) {
    // ------------------------------------------------------------ softmax, Q, results
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftRegs));
    const int w = (warp - 4) >> 2;     // warpgroup
    const int quad = warp & 3;         // tensor memory lanes 32 quad ..
    const int row = quad * 32 + lane;  // query row of the tile = tensor memory lane
    const int tid = threadIdx.x - 128; // 0 .. 255
    const uint32_t t_row = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t col_o = kColO + (uint32_t)(w * kHD);
    // Q rows of an item into shared memory (128-byte swizzled, K-major): with one
    // query tile all 256 threads load it, with two each warpgroup its own.
    // Rows past the last keep what they have: no other row sees it. (The 16-bit
    // types share one load, which nothing waits for before the last is out.)
    int xchg = 0;  // uses of the exchange buffer
    auto load_q = [&](const TreeSeg& s) -> bool {
      const bool two = C::kQTiles == 2 && s.nq == 2;
      const int n_it = two ? 16 : 8, step = two ? 128 : 256;
      const int t = two ? tid & 127 : tid;
      const int tile_row0 = two ? w * kRows : 0;
      uint8_t* q_tile = base + (two ? w * kQTile : 0);
      const int64_t q0 = ((int64_t)s.q_base * p.hq + (int64_t)s.h * p.G) * kHD + (t & 15) * 8;
      bool ready = true;
#pragma unroll 1
      for (int b8 = 0; b8 < n_it; b8 += 8) {
        uint4 v[8];
        auto at = [&](int i) -> int64_t {  // element of piece i of this thread, -1: past the last row
          const int r = tile_row0 + ((t + (b8 + i) * step) >> 4), rr = s.row0 + r, node = tree_node(p, rr);
          return r < s.rows ? q0 + (int64_t)(node * (p.hq - p.G) + rr) * kHD : -1;
        };
        if (p.q_dtype == SCKV_DTYPE_F32) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int64_t o = at(i);
            if (o >= 0) v[i] = load_q8<kBF16>(p.q, o, SCKV_DTYPE_F32);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int64_t o = at(i);
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (o >= 0) v[i] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + o));
          }
          if (p.q_dtype != (kBF16 ? SCKV_DTYPE_BF16 : SCKV_DTYPE_F16)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = cvt_q8<kBF16>(v[i]);
          }
        }
        // the exchange of the item before lay in the Q tile
        if (b8 == 0 && xchg > 0) ready = warp_wait_bar(x_done, (xchg - 1) & 1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c = t + (b8 + i) * step;
          const int r = c >> 4, half = (c >> 3) & 1, ch = c & 7;
          if (tile_row0 + r < s.rows)
            for (int e = 0; e < kRows; e += kRows / s.copies)
              *reinterpret_cast<uint4*>(q_tile + half * kQHalf + (r + e) * 128 + ((ch ^ (r & 7)) << 4)) = v[i];
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) bar_arrive(q_full);
      return ready;
    };
    bool ok = true;
    int gt = 0;           // tiles of earlier items
    int cnt[2] = {0, 0};  // uses of each set in earlier items
    TreeSeg s;
    bool more = tree_next(p, cum, walk, s);
    if (more) ok = load_q(s);
    // One item (or part of one); false if a wait ran out. kTwo: two query tiles; kCopies: copies of the rows.
    auto run_item = [&](auto two_c, auto copies_c, const int k) -> bool {
      constexpr bool two = decltype(two_c)::value;
      constexpr int R = decltype(copies_c)::value;
      constexpr int kCols = kHalf / R;       // keys of a half that this thread weighs
      constexpr int kPg = kCols / SCKV_PAGE_TOKENS;
      const int copy = row / (kRows / R);
      const int r_in = (two ? w * kRows : 0) + (row & (kRows / R - 1));  // row of the group
      const bool valid = r_in < s.rows;
      const int node = tree_node(p, s.row0 + r_in);
      const int head = s.h * p.G + (s.row0 + r_in) - node * p.G;
      const unsigned long long* mask = p.mask + (int64_t)(s.q_base + (valid ? node : 0)) * p.mask_words;
      const bool live = __any_sync(0xffffffffu, valid);
      unsigned long long* bad = s_bad + (k & 1) * kMaskWordsMax;
      float m = -INFINITY, l = 0.f;
      float vref = 0.f, inv_vref = 0.f;  // FP8: the V scale that this warp's O counts in
      const int32_t* bt_row = p.bt + (int64_t)s.seq * p.bt_stride;
#pragma unroll 1
      for (int i = 0; i < s.nk; ++i) {
        const int x = two ? w : i & 1;
        const int use = cnt[x] + (two ? i : i >> 1);
        const int key0 = (s.ka + i) * kKeys;
        const bool both = key0 + kHalf < s.L;
        // this warpgroup's halves: one query tile: half w; two: both
        const int h0 = two ? 0 : w, nh = two ? (both ? 2 : 1) : (w == 0 || both ? 1 : 0);
        if (*abort_flag || !warp_wait_bar(s_full + 8 * x, use & 1)) return false;
        tc_fence_after();
        float ks[kPg], vs[kPg];
        float alpha = 1.f;
        bool rescale = false;
#pragma unroll
        for (int q = 0; q < kPg; ++q) ks[q] = p.scale_log2;
        if (C::kFP8) {
          // the tile's page scales (written before the codes were decoded, and so before S was made)
          const int slot = (2 * (gt + i) + w) % kScaleSlots;
          const float* sc = reinterpret_cast<const float*>(base + C::kOffScale + slot * 256) + copy * kPg;
          float vm = 0.f;
#pragma unroll
          for (int q = 0; q < kPg; ++q) {
            ks[q] *= sc[q];
            vs[q] = sc[4 + q];
            vm = fmaxf(vm, vs[q]);
          }
          if (vm > vref) {  // (the same for the whole warp) twice the largest: growth below 2 needs no rescale
            if (vref > 0.f) {
              alpha = vref / (2.f * vm);
              rescale = true;
            }
            vref = 2.f * vm;
            inv_vref = __frcp_rn(vref);
          }
        }
        const uint32_t col_s = t_row + kColS + (uint32_t)(x * kKeys);
        if (live && nh > 0) {
          float sv[kCols];
          auto load_half = [&](int h) {
            if constexpr (kCols == 64) {
              uint32_t r0[32], r1[32];
              tmem_ld32(col_s + h * kHalf, r0);
              tmem_ld32(col_s + h * kHalf + 32, r1);
              tc_wait_ld();
#pragma unroll
              for (int c = 0; c < 32; ++c) {
                sv[c] = __uint_as_float(r0[c]);
                sv[32 + c] = __uint_as_float(r1[c]);
              }
            } else if constexpr (kCols == 32) {
              uint32_t r0[32];
              tmem_ld32(col_s + h * kHalf + copy * 32, r0);
              tc_wait_ld();
#pragma unroll
              for (int c = 0; c < 32; ++c) sv[c] = __uint_as_float(r0[c]);
            } else {
              uint32_t r0[16];
              tmem_ld16(col_s + h * kHalf + copy * 16, r0);
              tc_wait_ld();
#pragma unroll
              for (int c = 0; c < 16; ++c) sv[c] = __uint_as_float(r0[c]);
            }
            const int off = key0 + h * kHalf + copy * kCols - s.ctx;
            if (off + kCols > 0) {
              const unsigned long long win = valid ? tree_window(mask, p.mask_words, s.n, off) : 0ull;
              const uint32_t lo = (uint32_t)win, hi = (uint32_t)(win >> 32);
#pragma unroll
              for (int c = 0; c < kCols; ++c) sv[c] = ((c < 32 ? lo : hi) >> (c & 31)) & 1 ? sv[c] : -INFINITY;
            }
          };
          // the row's largest score; the scale is positive
          float pm = -INFINITY;
#pragma unroll 1
          for (int hh = 0; hh < nh; ++hh) {
            load_half(h0 + hh);
            float t = -INFINITY;
#pragma unroll
            for (int q = 0; q < kPg; ++q) {  // (a short chain per page)
              float y = sv[16 * q];
#pragma unroll
              for (int c = 1; c < 15; c += 2) y = fmax3(y, sv[16 * q + c], sv[16 * q + c + 1]);
              y = fmaxf(y, sv[16 * q + 15]);
              t = fmaxf(t, y * ks[q]);
            }
            pm = fmaxf(pm, t);
          }
          // stale reference: it moves when a tile exceeds it by more than 2^8
          if (pm > m + 8.f) {
            if (m != -INFINITY) {
              const float e = ex2_approx(m - pm);
              alpha *= e;
              l *= e;
              rescale = true;
            }
            m = pm;
          }
          if (__any_sync(0xffffffffu, rescale) && i > 0) {
            // O holds PV of this item's earlier tiles: wait for the last, then scale this warp's rows
            const int xp = two ? w : (i - 1) & 1;
            const int usep = cnt[xp] + (two ? i - 1 : (i - 1) >> 1);
            if (!warp_wait_bar(pv_done + 8 * xp, usep & 1)) return false;
            tc_fence_after();
#pragma unroll 1
            for (int cc = 0; cc < 4; ++cc) {
              uint32_t r[32];
              tmem_ld32(t_row + col_o + cc * 32, r);
              tc_wait_ld();
#pragma unroll
              for (int c = 0; c < 32; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) * alpha);
              tmem_st32(t_row + col_o + cc * 32, r);
            }
            tc_wait_st();
            // (the scores' registers were given up for this)
            load_half(h0 + nh - 1);
          }
          // 2^6 times the weight; a row that sees no key yet (m = -inf) has every score -inf: 2^-inf = 0
          const float mm = (m == -INFINITY) ? 0.f : m - 6.f;
          const uint64_t negm2 = f32x2(-mm, -mm), minus1 = f32x2(-1.f, -1.f);
          uint64_t ls2 = f32x2(0.f, 0.f);
#pragma unroll 1
          for (int hh = nh - 1; hh >= 0; --hh) {
            if (two && hh < nh - 1) load_half(h0 + hh);
            const uint32_t pc = col_s + (h0 + hh) * kHalf;
#pragma unroll
            for (int q = 0; q < kPg; ++q) {  // a page (16 keys) at a time
              uint32_t ph[8], plo[8];
              const uint64_t scale2 = f32x2(ks[q], ks[q]);
              uint64_t v2 = 0;
              if (C::kFP8) v2 = f32x2(vs[q] * inv_vref, vs[q] * inv_vref);
#pragma unroll
              for (int d = 0; d < 8; ++d) {
                float x0, x1;
                f32x2_split(fma_f32x2(f32x2(sv[16 * q + 2 * d], sv[16 * q + 2 * d + 1]), scale2, negm2), x0, x1);
                const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
                ls2 = add_f32x2(ls2, f32x2(p0, p1));
                uint64_t w2 = f32x2(p0, p1);
                if (C::kFP8) w2 = mul_f32x2(w2, v2);
                float w0, w1;
                f32x2_split(w2, w0, w1);
                ph[d] = pack2<kBF16>(w0, w1);
                if (kSplit) {
                  // lo = w - hi, exact
                  float h0, h1;
                  if (kBF16) {
                    h0 = __uint_as_float(ph[d] << 16);
                    h1 = __uint_as_float(ph[d] & 0xFFFF0000u);
                  } else {
                    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&ph[d]));
                    h0 = h.x;
                    h1 = h.y;
                  }
                  float l0, l1;
                  f32x2_split(fma_f32x2(f32x2(h0, h1), minus1, w2), l0, l1);
                  plo[d] = pack2<kBF16>(l0, l1);
                }
              }
              tmem_st8(pc + 8 * (copy * kPg + q), ph);
              if (kSplit) tmem_st8(pc + 32 + 8 * (copy * kPg + q), plo);
            }
            if constexpr (R > 1) {  // the keys of the other copies
              const uint32_t z[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
#pragma unroll
              for (int q = 0; q < kHalfPages - kPg; ++q) {
                const int pg = q < copy * kPg ? q : q + kPg;
                tmem_st8(pc + 8 * pg, z);
                if (kSplit) tmem_st8(pc + 32 + 8 * pg, z);
              }
            }
          }
          float ls0, ls1;
          f32x2_split(ls2, ls0, ls1);
          l += ls0 + ls1;
          tc_wait_st();
        }
        if (key0 + kKeys > s.ctx && (!two || w == 0)) {
          // V rows past the last node become 0, and so does what is not finite in a node's row (noted). The V tile of
          // S(i) cannot be replaced before P(i) is written, and the one before it in this slot was complete before S(i)
          // (its PV went out earlier): the wait is for this tile's phase.
          const int st = (gt + i) % kStages;
          if (!warp_wait_bar(v_full + 8 * st, ((gt + i) / kStages) & 1)) return false;
          uint8_t* vt = base + C::kOffV + st * kSlot;
          const int r0 = max(h0 * kHalf, s.ctx - key0), r1 = (h0 + nh) * kHalf;
#pragma unroll 1
          for (int c = row; c < (r1 - r0) * 16; c += 128) {
            const int r = r0 + (c >> 4), ch = c & 15;
            const int key = key0 + r;
            uint4* cell = reinterpret_cast<uint4*>(vt + (r >> 4) * kPageTile + ((r >> 3) & 1) * 2048 + (ch >> 3) * 1024 +
                                                   (r & 7) * 128 + (((ch & 7) ^ (r & 7)) << 4));
            if (key >= s.L) {
              *cell = make_uint4(0u, 0u, 0u, 0u);
            } else {
              constexpr uint32_t kExp = kBF16 ? 0x7F80u : 0x7C00u;
              uint4 xv = *cell;
              uint32_t xs[4] = {xv.x, xv.y, xv.z, xv.w};
              bool hit = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if ((xs[e] & kExp) == kExp) { xs[e] &= 0xFFFF0000u; hit = true; }
                if ((xs[e] & (kExp << 16)) == (kExp << 16)) { xs[e] &= 0x0000FFFFu; hit = true; }
              }
              if (hit) {
                *cell = make_uint4(xs[0], xs[1], xs[2], xs[3]);
                atomicOr(bad + ((key - s.ctx) >> 6), 1ull << ((key - s.ctx) & 63));
              }
            }
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive_n(p_full + 8 * x, two ? 2 : 1);  // 8 arrivals either way
      }
      // ---- the item's result, once its last PV finished
      {
        const int i = s.nk - 1, x = two ? w : i & 1;
        const int use = cnt[x] + (two ? i : i >> 1);
        if (!warp_wait_bar(pv_done + 8 * x, use & 1)) return false;
      }
      s_ml[w * kRows + row] = make_float2(m, l);
      if (lane == 0) s_vref[w * 4 + quad] = C::kFP8 ? vref : 1.f;
      // both warpgroups' O are complete and every S product has finished (a bounded wait, not a named barrier: a
      // warp that gave up must not leave the others waiting)
      tc_fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(o_full);
      if (!warp_wait_bar(o_full, k & 1)) return false;
      tc_fence_after();
      // one query tile: O[0] and O[1] (and the copies) join, warpgroup w writes dims 64 w ..; two: its own rows
      const bool join = !two && s.ka * kKeys + kHalf < s.L;  // a second half held keys
      float f0 = 1.f, f1 = 0.f, M = m, Lsum = l;
      if constexpr (!two) {
        M = -INFINITY;
#pragma unroll
        for (int e = 0; e < R; ++e) {
          const int o = (row & (kRows / R - 1)) + e * (kRows / R);
          M = fmaxf(M, s_ml[o].x);
          if (join) M = fmaxf(M, s_ml[kRows + o].x);
        }
        auto weight = [&](float mx) { return mx == -INFINITY ? 1.f : ex2_approx(mx - M); };
        Lsum = 0.f;
#pragma unroll
        for (int e = 0; e < R; ++e) {
          const int o = (row & (kRows / R - 1)) + e * (kRows / R);
          Lsum = fmaf(s_ml[o].y, weight(s_ml[o].x), Lsum);
          if (join) Lsum = fmaf(s_ml[kRows + o].y, weight(s_ml[kRows + o].x), Lsum);
        }
        f0 = weight(s_ml[row].x);
        if (join) f1 = weight(s_ml[kRows + row].x);
      }
      f0 *= s_vref[two ? w * 4 + quad : quad];
      f1 *= s_vref[4 + quad];
      const bool full = s.nk == s.kt;
      if (full) {
        const float inv = Lsum == 0.f ? 0.f : 1.f / Lsum;  // no key seen: zeros; NaN stays NaN
        f0 *= inv;
        f1 *= inv;
      }
      const int d0 = two ? 0 : 64 * w, nd = two ? kHD : 64;
      const int64_t obase = ((int64_t)(s.q_base + node) * p.hq + head) * kHD;
      float* part = p.parts + (int64_t)(2 * blockIdx.x + (k > 0 ? 1 : 0)) * slot_floats(p.part_rows);
      bool odd = false;  // this thread wrote a NaN, or infinities of both signs
      auto put4 = [&](int d, float a, float b, float c, float e) {
        const float sum = (a + b) + (c + e);
        odd |= sum != sum;
        if (full)
          tree_store4(p.out, obase + d, p.out_dtype, a, b, c, e);
        else
          reinterpret_cast<float4*>(part)[(int64_t)(d >> 2) * p.part_rows + r_in] = make_float4(a, b, c, e);
      };
      // f(word, pos): the nodes that this row sees and whose V is not finite somewhere, by their position
      auto each_bad = [&](auto f) {
#pragma unroll 1
        for (int wd = 0; wd < p.mask_words; ++wd) {
          unsigned long long hit = bad[wd];
          if (hit) hit &= tree_window(mask, p.mask_words, s.n, 64 * wd);
#pragma unroll 1
          for (; hit; hit &= hit - 1) {
            const int pos = s.ctx + 64 * wd + __ffsll((long long)hit) - 1;
            int page = __ldg(bt_row + pos / SCKV_PAGE_TOKENS);
            if (page < 0 || page >= p.g.P) page = 0;
            f(page, pos % SCKV_PAGE_TOKENS);
          }
        }
      };
      // this thread's merged O, 32 dims from d0 + cc
      auto merged = [&](int cc, float (&y)[32]) {
        uint32_t r[32];
        tmem_ld32(t_row + kColO + (two ? w * kHD : 0) + d0 + cc, r);
        tc_wait_ld();
#pragma unroll
        for (int c = 0; c < 32; ++c) y[c] = __uint_as_float(r[c]) * f0;
        if (join) {
          tmem_ld32(t_row + kColO + kHD + d0 + cc, r);
          tc_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; ++c) y[c] = fmaf(__uint_as_float(r[c]), f1, y[c]);
        }
      };
      if constexpr (R == 1) {
        if (live) {
#pragma unroll 1
          for (int cc = 0; cc < nd; cc += 32) {
            float y[32];
            merged(cc, y);
            if (valid) {
#pragma unroll
              for (int c = 0; c < 32; c += 4) put4(d0 + cc + c, y[c], y[c + 1], y[c + 2], y[c + 3]);
            }
            __syncwarp();
          }
          if (valid) {
            each_bad([&](int page, int slot) {
#pragma unroll 1
              for (int d = d0; d < d0 + nd; ++d) {
                const float v = tree_v(p.g, p.layer, page, s.h, slot, d);
                if (isfinite(v)) continue;
                if (full)
                  sckv_store_from_float(p.out, obase + d, p.out_dtype,
                                        sckv_load_as_float(p.out, obase + d, p.out_dtype) + v);
                else
                  part[((int64_t)(d >> 2) * p.part_rows + r_in) * 4 + (d & 3)] += v;
              }
            });
          }
        }
      } else {
        // the copies' rows are added up through the (now idle) Q tiles, 32 dims of each warpgroup at a time and tile:
        // [w][row] of 128 bytes, 16-byte chunks swizzled by the row
        float* xb = reinterpret_cast<float*>(base) + w * kRows * 32;
#pragma unroll 1
        for (int c0 = 0; c0 < nd; c0 += 32 * C::kQTiles) {
          // (a second pass writes what the first has read)
          if (c0 > 0 && !warp_wait_bar(x_done, (xchg - 1) & 1)) return false;
#pragma unroll 1
          for (int b = 0; b < C::kQTiles; ++b) {
            const int cc = c0 + 32 * b;
            float* xt = xb + b * (kQTile / 4);
            float y[32];
            merged(cc, y);
            float4* mine = reinterpret_cast<float4*>(xt + row * 32);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              mine[j ^ (row & 7)] = valid ? make_float4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3])
                                          : make_float4(0.f, 0.f, 0.f, 0.f);
            if (valid && copy == 0) {
              each_bad([&](int page, int slot) {
#pragma unroll 1
                for (int d = 0; d < 32; ++d) {
                  const float v = tree_v(p.g, p.layer, page, s.h, slot, d0 + cc + d);
                  if (!isfinite(v)) xt[row * 32 + (((d >> 2) ^ (row & 7)) << 2) + (d & 3)] += v;
                }
              });
            }
          }
          __syncwarp();
          if (lane == 0) bar_arrive(x_full + 8 * w);
          if (!warp_wait_bar(x_full + 8 * w, xchg & 1)) return false;
          if (valid) {
            const int sub = row & (kRows / R - 1);
#pragma unroll
            for (int b = 0; b < C::kQTiles; ++b) {
#pragma unroll
              for (int jj = 0; jj < 8 / R; ++jj) {
                const int j = copy * (8 / R) + jj;
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int e = 0; e < R; ++e) {
                  const float4 b4 = reinterpret_cast<const float4*>(xb + b * (kQTile / 4) +
                                                                    (sub + e * (kRows / R)) * 32)[j ^ (sub & 7)];
                  a.x += b4.x;
                  a.y += b4.y;
                  a.z += b4.z;
                  a.w += b4.w;
                }
                put4(d0 + c0 + 32 * b + 4 * j, a.x, a.y, a.z, a.w);
              }
            }
          }
          __syncwarp();
          if (lane == 0) bar_arrive(x_done);  // (waited for before the tiles are written again)
          ++xchg;
        }
      }
      // An infinite V of a committed token, which every row sees: 0 x Inf, of a lane that does not weigh its key (a
      // copy's, the lo part of an exact weight, a half whose sum is nothing beside the other's), left NaN where the
      // row's value is that infinity. Each lane looks through 4 dims of this part's committed V.
      if (!C::kFP8 && __any_sync(0xffffffffu, valid && odd && Lsum == Lsum)) {
        auto kind_of = [](float v) -> uint32_t { return v != v ? 4u : v == INFINITY ? 1u : v == -INFINITY ? 2u : 0u; };
        uint32_t kinds = 0;
        const int k1 = min((s.ka + s.nk) * kKeys, s.ctx);
#pragma unroll 4
        for (int key = s.ka * kKeys; key < k1; ++key) {
          int page = __ldg(bt_row + key / SCKV_PAGE_TOKENS);
          if (page < 0 || page >= p.g.P) page = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            kinds |= kind_of(tree_v(p.g, p.layer, page, s.h, key % SCKV_PAGE_TOKENS, 4 * lane + e)) << (4 * e);
        }
#pragma unroll 1
        for (int d = d0; d < d0 + nd; ++d) {
          uint32_t seen = (__shfl_sync(0xffffffffu, kinds, d >> 2) >> (4 * (d & 3))) & 7u;
          if (!valid || seen == 0 || Lsum != Lsum || (R > 1 && ((d & 31) >> 2) / (8 / R) != copy)) continue;
          float* at = part + ((int64_t)(d >> 2) * p.part_rows + r_in) * 4 + (d & 3);
          const float x = full ? sckv_load_as_float(p.out, obase + d, p.out_dtype) : *at;
          if (x == x) continue;
          each_bad([&](int page, int slot) { seen |= kind_of(tree_v(p.g, p.layer, page, s.h, slot, d)); });
          if (seen != 1u && seen != 2u) continue;
          const float v = seen == 1u ? INFINITY : -INFINITY;
          if (full)
            sckv_store_from_float(p.out, obase + d, p.out_dtype, v);
          else
            *at = v;
        }
      }
      if (!full && valid && copy == 0 && (two || w == 0))
        reinterpret_cast<float2*>(part + (int64_t)p.part_rows * kHD)[r_in] = make_float2(M, Lsum);
      // the other flags were last read in the item before and are next set in the one after
      if (tid < kMaskWordsMax) s_bad[((k + 1) & 1) * kMaskWordsMax + tid] = 0;
      tc_fence_before();
      gt += s.nk;
      cnt[0] += two ? s.nk : (s.nk + 1) >> 1;
      cnt[1] += two ? s.nk : s.nk >> 1;
      return true;
    };
    for (int k = 0; ok && more; ++k) {
      constexpr bool kPair = C::kQTiles == 2;
      if (kPair && s.nq == 2)
        ok = run_item(std::integral_constant<bool, kPair>{}, std::integral_constant<int, 1>{}, k);
      else if (s.copies == 1)
        ok = run_item(std::false_type{}, std::integral_constant<int, 1>{}, k);
      else if (s.copies == 2)
        ok = run_item(std::false_type{}, std::integral_constant<int, 2>{}, k);
      else
        ok = run_item(std::false_type{}, std::integral_constant<int, 4>{}, k);
      if (!ok) break;
      more = tree_next(p, cum, walk, s);
      if (more) ok = load_q(s);
    }
    if (!ok) {
      if (lane == 0 && !*abort_flag) sckv_report(p.g.status, SCKV_ERR_TIMEOUT, blockIdx.x, KID_TREE_ATTN);
      if (lane == 0) *abort_flag = 1;
    }
  } else {
    reg_give<C::kGiveRegs>();
  }
  if (warp < 4 || warp >= 12) __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the partials of the items that end in CTA blockIdx.x and began earlier: 16 rows a CTA, 4 dims of a row a
// thread. Eight parts' values are on the way while the parts' references and sums are weighed (one item may have as
// many parts as there are SMs).
constexpr int kJoinRows = 16, kJoinThreads = kJoinRows * kHD / 4, kJoinBatch = 8;

__global__ void __launch_bounds__(kJoinThreads) tree_join_kernel(const TreeParams p) {
  extern __shared__ float2 s_part[];  // [n_parts][kJoinRows]: m, l
  pdl_wait();
  const JoinHead hd = p.heads[blockIdx.x];
  const int rl = threadIdx.x % kJoinRows, dg = threadIdx.x / kJoinRows, r = blockIdx.y * kJoinRows + rl;
  if ((int)blockIdx.y * kJoinRows >= hd.rows || hd.n_parts == 0) return;
  auto slot = [&](int i) { return p.parts + (2 * (hd.c0 + i) + (i == 0 ? hd.slot0 : 0)) * slot_floats(p.part_rows); };
  float4 v[kJoinBatch];
  auto load = [&](int i0) {
#pragma unroll
    for (int e = 0; e < kJoinBatch; ++e)
      if (i0 + e < hd.n_parts && r < hd.rows)
        v[e] = reinterpret_cast<const float4*>(slot(i0 + e))[(int64_t)dg * p.part_rows + r];
  };
  load(0);
  for (int i = dg; i < hd.n_parts; i += kHD / 4)
    s_part[i * kJoinRows + rl] = r < hd.rows ? reinterpret_cast<const float2*>(slot(i) + (int64_t)p.part_rows * kHD)[r]
                                             : make_float2(-INFINITY, 0.f);
  __syncthreads();
  if (r >= hd.rows) return;
  float M = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < hd.n_parts; ++i) M = fmaxf(M, s_part[i * kJoinRows + rl].x);
  float L = 0.f, x0 = 0.f, x1 = 0.f, x2 = 0.f, x3 = 0.f;
  for (int i0 = 0; i0 < hd.n_parts; i0 += kJoinBatch) {
    if (i0 > 0) load(i0);
#pragma unroll
    for (int e = 0; e < kJoinBatch; ++e) {
      if (i0 + e >= hd.n_parts) break;
      const float2 a = s_part[(i0 + e) * kJoinRows + rl];
      // (at least the smallest float: an infinite sum of a part that weighs nothing stays infinite)
      const float f = a.x == -INFINITY ? 1.f : fmaxf(ex2_approx(a.x - M), 1.17549435e-38f);
      L = fmaf(a.y, f, L);
      x0 = fmaf(v[e].x, f, x0);
      x1 = fmaf(v[e].y, f, x1);
      x2 = fmaf(v[e].z, f, x2);
      x3 = fmaf(v[e].w, f, x3);
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;  // no key seen: zeros; NaN stays NaN
  const int rr = hd.row0 + r, node = tree_node(p, rr);
  const int64_t o = ((int64_t)(hd.q_base + node) * p.hq + hd.h * p.G + (rr - node * p.G)) * kHD + 4 * dg;
  tree_store4(p.out, o, p.out_dtype, x0 * inv, x1 * inv, x2 * inv, x3 * inv);
}

// Rank-5 view of a 16-bit pool whose boxes are whole page-heads in 8-row
// groups: dims {64 of the head dim, 8 tokens, 2 halves of the head dim, 2
// groups of tokens, (slab, K|V, head)}, 128-byte swizzle.
int ensure_tree_tmap(sckv_pool* p) {
  if (p->tmap_tree_ready) return SCKV_OK;
  PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
  if (encode == nullptr)
    return sckv_record_error(__FILE__, __LINE__, "cudaGetDriverEntryPoint", "cuTensorMapEncodeTiled not found");
  const cuuint64_t dims[5] = {64, 8, 2, 2, (cuuint64_t)p->num_layers * (cuuint64_t)p->max_pages * 2 * p->num_kv_heads};
  const cuuint64_t strides[4] = {256, 128, 2048, 4096};
  const cuuint32_t box[5] = {64, 8, 2, 2, 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = encode(reinterpret_cast<CUtensorMap*>(p->tmap_tree), CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, p->data, dims,
                            strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    char what[64];
    snprintf(what, sizeof what, "CUresult %d", (int)r);
    return sckv_record_error(__FILE__, __LINE__, "cuTensorMapEncodeTiled", what);
  }
  p->tmap_tree_ready = 1;
  return SCKV_OK;
}

// Rows of a partial slot: a group's rows, at most.
int tree_group_rows(const sckv_pool* p) { return sckv_elem_bytes(p->kv_dtype) == 1 ? kRows : 2 * kRows; }

int tree_part_rows(const sckv_pool* p, int n_tokens, int mask_words, int G) {
  const int64_t rows = (int64_t)(n_tokens < 64 * mask_words ? n_tokens : 64 * mask_words) * G;
  return rows > kRows ? tree_group_rows(p) : kRows;
}

size_t tree_head_bytes(const sckv_pool* p) { return ((size_t)p->num_sms * sizeof(JoinHead) + 255) / 256 * 256; }

template <int KVDT, bool kSplit>
int launch_tree(sckv_pool* p, const TreeParams& t, cudaStream_t stream) {
  using C = TreeCfg<KVDT>;
  const int rc = C::kB8 ? ensure_tmap(p, 1, p->tmap_kv1, &p->tmap1_ready) : ensure_tree_tmap(p);
  if (rc != SCKV_OK) return rc;
  const CUtensorMap* map = reinterpret_cast<const CUtensorMap*>(C::kB8 ? p->tmap_kv1 : p->tmap_tree);
  auto kern = tree_attn_kernel<KVDT, kSplit>;
  const int smem = C::kFixedSmem + 4 * t.n_seqs;
  static_assert(C::kFixedSmem + 4 * kMaxSeqs <= 227 * 1024, "shared memory of the largest batch");
  if (!(p->tree_smem_ready & (1 << kSplit))) {  // the largest batch's, once per pool and kernel
    SCKV_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         C::kFixedSmem + 4 * kMaxSeqs));
    p->tree_smem_ready |= 1 << kSplit;
  }
  kern<<<p->num_sms, C::kThreads, smem, stream>>>(t, *map);
  SCKV_LAUNCH_CHECK();
  SCKV_CUDA_CHECK(sckv_launch_pdl(tree_join_kernel, dim3(p->num_sms, t.part_rows / kJoinRows), dim3(kJoinThreads),
                                  p->num_sms * kJoinRows * sizeof(float2), stream, t));
  SCKV_LAUNCH_CHECK();
  return SCKV_OK;
}

}  // namespace

extern "C" size_t sckv_tree_attn_workspace_bytes(const sckv_pool* p, int n_tokens, int num_q_heads) {
  if (p == nullptr || n_tokens <= 0 || num_q_heads <= 0) return 0;
  const int rows = tree_part_rows(p, n_tokens, kMaskWordsMax, num_q_heads / p->num_kv_heads);
  return tree_head_bytes(p) + (size_t)p->num_sms * 2 * rows * (kHD + 2) * sizeof(float);
}

extern "C" int sckv_tree_attn(sckv_pool* p, int layer, const void* q, int q_dtype, int num_q_heads, int n_seqs,
                              int n_tokens, const int32_t* cu_q, const int32_t* ctx_lens, const int32_t* block_table,
                              int64_t bt_stride, int max_blocks, const uint64_t* tree_mask, int mask_words,
                              float scale, void* out, int out_dtype, void* workspace, size_t workspace_bytes,
                              void* stream) {
  if (p == nullptr || layer < 0 || layer >= p->num_layers || n_seqs < 0 || n_tokens < 0 || num_q_heads <= 0)
    return SCKV_ERR_INVALID_ARG;
  if (num_q_heads % p->num_kv_heads != 0 || mask_words < 1 || mask_words > kMaskWordsMax || !(scale > 0.f))
    return SCKV_ERR_INVALID_ARG;
  if (!is_src_dtype(q_dtype) || !is_src_dtype(out_dtype)) return SCKV_ERR_INVALID_ARG;
  if (p->head_dim != kHD) return SCKV_ERR_UNSUPPORTED;
  if (p->kv_dtype == SCKV_DTYPE_BF16 && q_dtype != SCKV_DTYPE_BF16) return SCKV_ERR_UNSUPPORTED;
  if (n_seqs == 0 || n_tokens == 0) return SCKV_OK;
  if (!q || !out || !cu_q || !ctx_lens || !block_table || !tree_mask || bt_stride < max_blocks || max_blocks <= 0)
    return SCKV_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return SCKV_ERR_ALIGNMENT;
  if (workspace == nullptr || workspace_bytes < sckv_tree_attn_workspace_bytes(p, n_tokens, num_q_heads))
    return SCKV_ERR_INVALID_ARG;
  const int G = num_q_heads / p->num_kv_heads;
  // tile and box numbers are 32-bit
  const int64_t groups = ((int64_t)(n_tokens < 64 * mask_words ? n_tokens : 64 * mask_words) * G + kRows - 1) / kRows;
  if (n_seqs > kMaxSeqs || G > kMaxGroup || max_blocks > INT32_MAX / SCKV_PAGE_TOKENS ||
      (int64_t)n_seqs * (max_blocks / kTilePages + 1) * groups * p->num_kv_heads > INT32_MAX ||
      (int64_t)p->num_layers * p->max_pages * 2 * p->num_kv_heads > INT32_MAX)
    return SCKV_ERR_UNSUPPORTED;
  TreeParams t{};
  t.g = geo_of(p);
  t.layer = layer;
  t.q = q;
  t.out = out;
  t.cu_q = cu_q;
  t.ctx_lens = ctx_lens;
  t.bt = block_table;
  t.bt_stride = bt_stride;
  t.mask = reinterpret_cast<const unsigned long long*>(tree_mask);
  t.mask_words = mask_words;
  t.max_blocks = max_blocks;
  t.n_seqs = n_seqs;
  t.n_tokens = n_tokens;
  t.hq = num_q_heads;
  t.G = G;
  t.g_mul = G == 1 ? 0u : 0xFFFFFFFFu / (uint32_t)G + 1u;
  t.q_dtype = q_dtype;
  t.out_dtype = out_dtype;
  t.scale_log2 = scale * 1.4426950408889634f;
  t.heads = reinterpret_cast<JoinHead*>(workspace);
  t.parts = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(workspace) + tree_head_bytes(p));
  t.group_shift = tree_group_rows(p) == 2 * kRows ? 8 : 7;
  static_assert(kRows == 1 << 7, "rows of a query tile");
  t.part_rows = tree_part_rows(p, n_tokens, mask_words, G);
  SCKV_DEVICE_GUARD(p->device);
  cudaStream_t s = as_stream(stream);
  const bool split = out_dtype == SCKV_DTYPE_F32;  // one f16 part would be all of an fp32 output's error
  switch (p->kv_dtype) {
    case SCKV_DTYPE_F16:
      return split ? launch_tree<SCKV_DTYPE_F16, true>(p, t, s) : launch_tree<SCKV_DTYPE_F16, false>(p, t, s);
    case SCKV_DTYPE_BF16: return launch_tree<SCKV_DTYPE_BF16, true>(p, t, s);
    case SCKV_DTYPE_INT8:
      return split ? launch_tree<SCKV_DTYPE_INT8, true>(p, t, s) : launch_tree<SCKV_DTYPE_INT8, false>(p, t, s);
    case SCKV_DTYPE_FP8_E4M3:
      return split ? launch_tree<SCKV_DTYPE_FP8_E4M3, true>(p, t, s) : launch_tree<SCKV_DTYPE_FP8_E4M3, false>(p, t, s);
    default: return SCKV_ERR_UNSUPPORTED;
  }
}
