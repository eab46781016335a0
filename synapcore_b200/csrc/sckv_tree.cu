// Operators of a speculative decoding step around its attention: q/k norm +
// rotary positions with several axes + K/V append, the move of the accepted
// rows next to the committed ones, and the choice of the accepted path from
// the logits.
#include <math.h>
#include <type_traits>

#include "sckv_geo.cuh"
#include "sckv_tcgen05.cuh"

using namespace sckv_geo;
using sckv_tc::f32x2;
using sckv_tc::f32x2_split;
using sckv_tc::fma_f32x2;
using sckv_tc::mul_f32x2;

namespace {

// ---------------------------------------------------------------------------
// QK-norm + rotary positions with several axes + append, one layer.
//
//   x' = x / sqrt(mean(x^2) + eps) * w                    (q and k, when w is given)
//   a_i = pos[axis[i]][t] / scaling * inv_freq[i],        i < D / 2
//   out = [x1 cos a - x2 sin a, x2 cos a + x1 sin a]      (halves of x')
//
// A token's rotary positions are independent of its page slot: the nodes of a
// drafted tree sit in consecutive slots but rotate by depth, and image tokens
// rotate by (time, height, width).
//
// Bound by HBM: (Hq + 2 Hkv) rows read and written once. A CTA takes `tpb`
// tokens, whose angles are computed once for all heads; eight lanes own a head
// row, each 8 dims of the first half and their 8 partners of the second (two
// 16-byte loads and stores per 16-bit row, rotation without exchange, a norm
// of three shuffles). With q, k and v of one 16-bit type a thread has its next
// row on the way while it works on one, the first before the angles are
// computed and the pages looked up, and what a row needs by address is kept
// per token. The arithmetic runs on packed pairs; the most frequent stall is the
// read of cos, sin and weights from shared memory. 8,192 tokens of 32 + 2 x 8 bf16
// heads: 43.5 us with several states in turn, 4.6 TB/s (71 % of a copy's rate);
// one state over and over 42, two rows on the way and CTAs of 256 threads slower
// (51, 43 us). The angle is formed and reduced to [-pi, pi] in 64 bits (a
// far position times a frequency near 1 has no useful fp32 bits left after the
// reduction); sin and cos then run in fp32.
// ---------------------------------------------------------------------------
constexpr int kRopeThreads = 128;
constexpr int kRopeD = 128;
constexpr int kRopeTokens = 4;   // most tokens of a CTA

struct RopeAxes {
  Geo g;
  int layer;
  const void* q;
  const void* k;
  const void* v;
  int64_t q_stride, k_stride, v_stride;  // elements between tokens
  int q_dtype, src_dtype;
  void* q_out;
  int q_out_dtype;
  float* k_stage;  // FP8 pools: rotated k [n_tokens][H][D], appended (and rounded) by the next launch
  const __half* q_w;
  const __half* k_w;
  float eps;
  const float* inv_freq;
  double inv_scaling;
  const int32_t* positions;
  int64_t pos_stride;
  int n_axes;
  const int32_t* axis_map;
  int hq, n_seqs, n_tokens, tpb;
  const int32_t* cu;
  const int32_t* start_pos;
  const int32_t* bt;
  int64_t bt_stride;
  int max_blocks;
};

// Sum and max over the 8 lanes that own a row (`m`: their lanes).
__device__ __forceinline__ float row_sum(float v, unsigned m) {
  v += __shfl_xor_sync(m, v, 1);
  v += __shfl_xor_sync(m, v, 2);
  return v + __shfl_xor_sync(m, v, 4);
}
__device__ __forceinline__ float row_max(float v, unsigned m) {
  v = fmaxf(v, __shfl_xor_sync(m, v, 1));
  v = fmaxf(v, __shfl_xor_sync(m, v, 2));
  return fmaxf(v, __shfl_xor_sync(m, v, 4));
}

__device__ __forceinline__ void store8(void* dst, int64_t idx, int dtype, const float (&v)[8]) {
  if (dtype == SCKV_DTYPE_F32) {
    float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(dst) + idx);
    o[0] = make_float4(v[0], v[1], v[2], v[3]);
    o[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    store8_16(dst, idx, dtype, v);
  }
}

// One K or V row into its int8 page slot as the arena stores its fp16 pages:
// the fp16 value, quantised per row (s = max(max|x| / 127, 1e-7), fp16 scale).
__device__ __forceinline__ void store_row8_int8(const Geo& g, int layer, int64_t page, int kv, int h, int slot, int l8,
                                                unsigned m, const float (&a)[8], const float (&b)[8]) {
  float x[16], top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = __half2float(__float2half_rn(a[i]));
    x[8 + i] = __half2float(__float2half_rn(b[i]));
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[i]));
  const float s = fmaxf(row_max(top, m) / 127.0f, 1e-7f);
  int8_t* dst = reinterpret_cast<int8_t*>(g.data) + row_off(g, layer, page, kv, h, slot);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    union {
      int8_t c[8];
      uint2 w;
    } u;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      u.c[i] = static_cast<int8_t>(fminf(fmaxf(rintf(x[8 * half + i] / s), -127.0f), 127.0f));
    *reinterpret_cast<uint2*>(dst + half * (kRopeD / 2) + 8 * l8) = u.w;
  }
  if (l8 == 0)
    reinterpret_cast<__half*>(g.scales)[int8_scale_idx(g, layer, page, kv, h, slot)] = __float2half_rn(s);
}

// kDT: the 16-bit type of q, k and v, or -1: any types, not fetched ahead.
template <int kDT>
__global__ void __launch_bounds__(kRopeThreads) rope_axes_kernel(const RopeAxes p) {
  constexpr bool kAhead = kDT >= 0;
  __shared__ __align__(16) float s_cos[kRopeTokens * (kRopeD / 2)], s_sin[kRopeTokens * (kRopeD / 2)];
  __shared__ __align__(16) float s_w[2][kRopeD];
  __shared__ const uint8_t* s_src[kRopeTokens][4];  // head 0 of q, k, v
  __shared__ uint8_t* s_dst[kRopeTokens][4];        // head 0's row of a 16-bit kDT output, or null
  __shared__ int64_t s_page[kRopeTokens];
  __shared__ int s_slot[kRopeTokens];  // -1: not a token of any sequence
  const int t0 = blockIdx.x * p.tpb, nt = min(p.tpb, p.n_tokens - t0);
  const int l8 = threadIdx.x & 7;
  const unsigned m = 0xffu << (threadIdx.x & 24);
  const int H = p.g.H, rows = p.hq + 2 * H;
  constexpr int kStep = kRopeThreads / 8;  // rows of the CTA at once
  auto kind_of = [&](int hr) { return hr < p.hq ? 0 : hr < p.hq + H ? 1 : 2; };  // q, k, v
  auto head_of = [&](int hr, int kind) { return hr - (kind == 0 ? 0 : kind == 1 ? p.hq : p.hq + H); };
  auto src_of = [&](int kind) { return kind == 0 ? p.q : kind == 1 ? p.k : p.v; };
  auto ld_of = [&](int kind) { return kind == 0 ? p.q_stride : kind == 1 ? p.k_stride : p.v_stride; };
  auto wrap = [&](int& tt, int& hr) {
    while (hr >= rows) {
      hr -= rows;
      ++tt;
    }
  };
  int tt = 0, hr = threadIdx.x >> 3;  // the thread's next row: token, row of q | k | v
  wrap(tt, hr);
  uint4 ra = make_uint4(0u, 0u, 0u, 0u), rb = ra;
  if (kAhead && tt < nt) {
    const int kind = kind_of(hr);
    const uint4* x = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(src_of(kind)) +
                                                    (t0 + tt) * ld_of(kind) + head_of(hr, kind) * kRopeD) + l8;
    ra = __ldg(x);
    rb = __ldg(x + kRopeD / 2 / 8);
  }
  for (int i = threadIdx.x; i < nt * (kRopeD / 2); i += kRopeThreads) {
    const int t = t0 + i / (kRopeD / 2), f = i % (kRopeD / 2);
    int axis = __ldg(p.axis_map + f);
    if (axis < 0 || axis >= p.n_axes) {
      if (blockIdx.x == 0) sckv_report(p.g.status, SCKV_ERR_BOUNDS, axis, KID_ROPE_AXES);
      axis = 0;
    }
    const double pos = (double)__ldg(p.positions + axis * p.pos_stride + t) * p.inv_scaling;
    const double a = pos * (double)__ldg(p.inv_freq + f);
    const double r = a - 6.283185307179586 * rint(a * 0.15915494309189535);
    sincosf((float)r, &s_sin[i], &s_cos[i]);
  }
  static_assert(kRopeThreads == kRopeD, "a thread brings its dim's weights");
  if (p.q_w != nullptr) s_w[0][threadIdx.x] = __half2float(p.q_w[threadIdx.x]);
  if (p.k_w != nullptr) s_w[1][threadIdx.x] = __half2float(p.k_w[threadIdx.x]);
  if (kRopeThreads - 1 - (int)threadIdx.x < nt) {
    const int tl = kRopeThreads - 1 - threadIdx.x, t = t0 + tl;
    int slot = -1;
    int64_t page = -1;
    if (t >= __ldg(p.cu) && t < __ldg(p.cu + p.n_seqs)) {
      const int b = sckv_find_seq(p.cu, p.n_seqs, t);
      const int pos = __ldg(p.start_pos + b) + (t - __ldg(p.cu + b));
      page = resolve_page(p.g, p.bt, p.bt_stride, p.max_blocks, b, pos, KID_ROPE_AXES);
      slot = page >= 0 ? pos % SCKV_PAGE_TOKENS : 0;
    }
    s_page[tl] = page;
    s_slot[tl] = slot;
    if (kAhead) {
#pragma unroll
      for (int kind = 0; kind < 3; ++kind) {
        s_src[tl][kind] = reinterpret_cast<const uint8_t*>(src_of(kind)) + t * ld_of(kind) * 2;
        uint8_t* dst = nullptr;
        if (kind == 0 && p.q_out_dtype == kDT)
          dst = reinterpret_cast<uint8_t*>(p.q_out) + (int64_t)t * p.hq * kRopeD * 2;
        if (kind > 0 && p.g.dtype == kDT && page >= 0)
          dst = reinterpret_cast<uint8_t*>(p.g.data) + row_off(p.g, p.layer, page, kind - 1, 0, slot) * 2;
        s_dst[tl][kind] = dst;
      }
    }
  }
  __syncthreads();
  while (tt < nt) {
    const int tl = tt, kind = kind_of(hr), h = head_of(hr, kind), t = t0 + tl;
    const int dt = kAhead ? kDT : kind == 0 ? p.q_dtype : p.src_dtype;
    float a[8], b[8];
    if (kAhead) {
      unpack8(ra, dt, a);
      unpack8(rb, dt, b);
    }
    hr += kStep;
    wrap(tt, hr);
    if (kAhead && tt < nt) {
      const int k2 = kind_of(hr);
      const uint4* x = reinterpret_cast<const uint4*>(s_src[tt][k2] + head_of(hr, k2) * (kRopeD * 2)) + l8;
      ra = __ldg(x);
      rb = __ldg(x + kRopeD / 2 / 8);
    }
    const int64_t page = s_page[tl];
    const int slot = s_slot[tl];
    if (slot < 0 || (kind != 0 && page < 0)) continue;
    if (!kAhead) {
      const int64_t at = t * ld_of(kind) + (int64_t)h * kRopeD + 8 * l8;
      load8(src_of(kind), at, dt, a);
      load8(src_of(kind), at + kRopeD / 2, dt, b);
    }
    if (kind < 2) {
      uint64_t x[4], y[4];  // pairs of the first and the second half
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = f32x2(a[2 * e], a[2 * e + 1]);
        y[e] = f32x2(b[2 * e], b[2 * e + 1]);
      }
      if ((kind == 0 ? p.q_w : p.k_w) != nullptr) {
        uint64_t ss2 = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) ss2 = fma_f32x2(x[e], x[e], fma_f32x2(y[e], y[e], ss2));
        float s0, s1;
        f32x2_split(ss2, s0, s1);
        const float inv = rsqrtf(row_sum(s0 + s1, m) * (1.f / kRopeD) + p.eps);
        const uint64_t inv2 = f32x2(inv, inv);
        const ulonglong2* wa = reinterpret_cast<const ulonglong2*>(&s_w[kind][8 * l8]);
        const ulonglong2* wb = reinterpret_cast<const ulonglong2*>(&s_w[kind][kRopeD / 2 + 8 * l8]);
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const ulonglong2 u = wa[e / 2], v = wb[e / 2];
          x[e] = mul_f32x2(mul_f32x2(x[e], inv2), u.x);
          x[e + 1] = mul_f32x2(mul_f32x2(x[e + 1], inv2), u.y);
          y[e] = mul_f32x2(mul_f32x2(y[e], inv2), v.x);
          y[e + 1] = mul_f32x2(mul_f32x2(y[e + 1], inv2), v.y);
        }
      }
      const ulonglong2* pc = reinterpret_cast<const ulonglong2*>(s_cos + tl * (kRopeD / 2) + 8 * l8);
      const ulonglong2* ps = reinterpret_cast<const ulonglong2*>(s_sin + tl * (kRopeD / 2) + 8 * l8);
      const uint64_t neg = f32x2(-1.f, -1.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t c = e & 1 ? pc[e / 2].y : pc[e / 2].x, sn = e & 1 ? ps[e / 2].y : ps[e / 2].x;
        f32x2_split(fma_f32x2(x[e], c, mul_f32x2(mul_f32x2(y[e], sn), neg)), a[2 * e], a[2 * e + 1]);
        f32x2_split(fma_f32x2(y[e], c, mul_f32x2(x[e], sn)), b[2 * e], b[2 * e + 1]);
      }
    }
    uint8_t* d16 = kAhead ? s_dst[tl][kind] : nullptr;
    if (d16 != nullptr) {
      uint16_t* o = reinterpret_cast<uint16_t*>(d16) + h * (kind == 0 ? kRopeD : SCKV_PAGE_TOKENS * kRopeD) + 8 * l8;
      store8_16(o, 0, dt, a);
      store8_16(o, kRopeD / 2, dt, b);
    } else if (kind == 0) {
      const int64_t o = ((int64_t)t * p.hq + h) * kRopeD + 8 * l8;
      store8(p.q_out, o, p.q_out_dtype, a);
      store8(p.q_out, o + kRopeD / 2, p.q_out_dtype, b);
    } else if (p.g.dtype == SCKV_DTYPE_INT8) {
      store_row8_int8(p.g, p.layer, page, kind - 1, h, slot, l8, m, a, b);
    } else if (p.g.dtype == SCKV_DTYPE_FP8_E4M3) {
      if (kind == 1) {
        const int64_t o = ((int64_t)t * H + h) * kRopeD + 8 * l8;
        store8(p.k_stage, o, SCKV_DTYPE_F32, a);
        store8(p.k_stage, o + kRopeD / 2, SCKV_DTYPE_F32, b);
      }
    } else {
      const int64_t o = row_off(p.g, p.layer, page, kind - 1, h, slot) + 8 * l8;
      store8_16(p.g.data, o, p.g.dtype, a);
      store8_16(p.g.data, o + kRopeD / 2, p.g.dtype, b);
    }
  }
}

// FP8 pools, second launch: one warp per (sequence, K|V, head) folds the new
// rows into its pages (page scales span 16 tokens, so a row cannot be stored
// by itself). K comes from the rotated fp32 rows, V from its source.
__global__ void rope_axes_fp8_kernel(const RopeAxes p) {
  const int units = p.n_seqs * 2 * p.g.H;
  const int u = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (u >= units) return;
  const int h = u % p.g.H, kv = (u / p.g.H) & 1, b = u / (2 * p.g.H);
  const int c0 = __ldg(p.cu), cn = min(__ldg(p.cu + p.n_seqs), p.n_tokens);
  const int t_first = max(__ldg(p.cu + b), max(c0, 0)), t_end = min(__ldg(p.cu + b + 1), cn);
  const int64_t stride = kv ? p.v_stride : (int64_t)p.g.H * kRopeD;
  for (int t = t_first; t < t_end;) {
    const int pos = __ldg(p.start_pos + b) + (t - __ldg(p.cu + b));
    const int slot0 = pos >= 0 ? pos % SCKV_PAGE_TOKENS : 0;
    const int n_new = min(t_end - t, SCKV_PAGE_TOKENS - slot0);
    const int64_t page = resolve_page(p.g, p.bt, p.bt_stride, p.max_blocks, b, pos, KID_ROPE_AXES);
    if (page >= 0)
      fp8_page_head_update(p.g, p.layer, page, kv, h, slot0, n_new, kv ? p.v : (const void*)p.k_stage,
                           (int64_t)t * stride + (int64_t)h * kRopeD, stride, kv ? p.src_dtype : SCKV_DTYPE_F32);
    t += n_new;
  }
}

// ---------------------------------------------------------------------------
// Accepted rows: row ctx + path[j] of a sequence moves to row ctx + j, j <
// n_keep, in every layer, K and V (with the int8 scales). path increases, so
// path[j] >= j: rows only move down, and a row is read before anything lands
// on it when destinations are taken in order.
//
// Bound by HBM (each moved row read and written once, as single rows of 128 or
// 256 bytes). A CTA takes slices (layer, K|V, head) of one sequence: it checks
// the path and looks the moved rows' pages up once, kMoves at a time, and each
// warp moves these rows of its slices: the 16-byte pieces of kMoveBatch loads
// a lane at a time, all loads before the stores. Pieces are taken by slice,
// then by path, so whatever lands on a row was preceded by all of its reads.
// 64 sequences, 3 to 5 moved rows of each (257), 36 layers of 8 bf16 heads, 76
// MB read and written: 21.8 us with several states in turn, 3.5 TB/s (53 % of a
// copy's rate; before the first row come n_keep, the path and the table, one
// after the other). One state over and over, out of L2: 15.9 us with 4 loads a
// lane, 4 warps a CTA and 8 slices a warp; 8 loads or 8 warps 17 us, 4 slices
// 16.9. The rows' offsets are looked up and not computed per piece: index
// arithmetic took 21.6 there.
//
// FP8: a page-head has one scale for its 16 rows. Rows that come from other
// pages are values code * s_src; the destination's scale grows to
// max(s, max|value| / 448) as an append's does, and the rows it already held
// are re-encoded when it grew. A destination page is only a source for rows
// of itself and of earlier pages, so scales are read before they change. One
// warp owns a slice and takes a destination page at a time.
// ---------------------------------------------------------------------------
constexpr int kCompactWarps = 4;
constexpr int kMoves = 256;    // moved rows whose pages are known at a time
constexpr int kMaxSlices = 8;  // slices of a warp
constexpr int kMoveBatch = 4;  // 16-byte pieces that a lane holds

struct Compact {
  Geo g;
  int layer0, n_layers, n_seqs, max_path;
  const int32_t* path;  // [n_seqs][max_path]
  const int32_t* n_keep;
  const int32_t* ctx;
  const int32_t* bt;
  int64_t bt_stride;
  int max_blocks;
  int per_warp;  // slices of a warp (not FP8)
};

// i / d for i < 2^16, 0 < d < 2^16, mul = 2^32 / d + 1
__device__ __forceinline__ uint32_t div_by(uint32_t i, uint32_t mul, uint32_t d) {
  return d == 1 ? i : __umulhi(i, mul);
}

__global__ void __launch_bounds__(kCompactWarps * 32) compact_kernel(const Compact p) {
  const Geo& g = p.g;
  const int n_slices = p.n_layers * 2 * g.H;
  const int groups = (n_slices + kCompactWarps * p.per_warp - 1) / (kCompactWarps * p.per_warp);
  const int b = blockIdx.x / groups, grp = blockIdx.x - b * groups;
  const bool reporter = grp == 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // rows of the pool: of a moved token in slice (layer 0, K, head 0), -1: not moved; and what a slice adds to them
  __shared__ int64_t s_src[kMoves], s_dst[kMoves], s_slice[kCompactWarps][kMaxSlices];
  const int keep = __ldg(p.n_keep + b), ctx = __ldg(p.ctx + b);
  const int32_t* path = p.path + (int64_t)b * p.max_path;
  const int cap = p.max_blocks * SCKV_PAGE_TOKENS;
  if (keep < 0 || keep > p.max_path || ctx < 0 || ctx > cap) {
    if (reporter && threadIdx.x == 0) sckv_report(g.status, SCKV_ERR_BOUNDS, b, KID_COMPACT);
    return;
  }
  // the path increases and stays inside the table; rows 0 .. j0 - 1 do not move
  bool bad = false;
  for (int j = threadIdx.x; j < keep; j += kCompactWarps * 32) {
    const int pj = __ldg(path + j), before = j > 0 ? __ldg(path + j - 1) : -1;
    bad |= pj <= before || pj >= cap - ctx;
  }
  if (__syncthreads_or(bad)) {
    if (reporter && threadIdx.x == 0) sckv_report(g.status, SCKV_ERR_BOUNDS, b, KID_COMPACT);
    return;
  }
  int j0 = 0;  // (an increasing path that left the diagonal stays off it)
  for (int jb = 0; jb < keep; jb += kCompactWarps * 32) {
    const int j = jb + threadIdx.x;
    j0 += __syncthreads_count(j < keep && __ldg(path + j) == j);
  }
  const int32_t* bt = p.bt + (int64_t)b * p.bt_stride;
  const int eb = g.dtype == SCKV_DTYPE_F16 || g.dtype == SCKV_DTYPE_BF16 ? 2 : 1;
  const uint32_t cpr = (uint32_t)(g.D * eb / 16), cpr_mul = (uint32_t)(0x100000000ull / cpr) + 1u;  // pieces of a row
  uint8_t* data = reinterpret_cast<uint8_t*>(g.data);
  __half* hscale = reinterpret_cast<__half*>(g.scales);
  const int sl0 = (grp * kCompactWarps + warp) * p.per_warp, n_mine = max(0, min(p.per_warp, n_slices - sl0));
  if (lane < n_mine) {
    const int sl = sl0 + lane, h = sl % g.H, lk = sl / g.H;
    s_slice[warp][lane] = row_off(g, p.layer0 + (lk >> 1), 0, lk & 1, h, 0) / g.D;
  }
  const int64_t page_rows = (int64_t)2 * g.H * SCKV_PAGE_TOKENS;
  const uint32_t row_bytes = (uint32_t)(g.D * eb);
  for (int jb = j0; jb < keep; jb += kMoves) {
    const int nm = min(kMoves, keep - jb);
    for (int i = threadIdx.x; i < nm; i += kCompactWarps * 32) {
      const int from = ctx + __ldg(path + jb + i), to = ctx + jb + i;
      const int ps = __ldg(bt + from / SCKV_PAGE_TOKENS), pd = __ldg(bt + to / SCKV_PAGE_TOKENS);
      const bool ok = ps >= 0 && ps < g.P && pd >= 0 && pd < g.P;
      if (!ok && reporter) sckv_report(g.status, SCKV_ERR_BOUNDS, pd >= 0 && pd < g.P ? ps : pd, KID_COMPACT);
      s_src[i] = ok ? ps * page_rows + from % SCKV_PAGE_TOKENS : -1;
      s_dst[i] = ok ? pd * page_rows + to % SCKV_PAGE_TOKENS : -1;
    }
    __syncthreads();
    const uint32_t per = (uint32_t)nm * cpr, nm_mul = (uint32_t)(0x100000000ull / nm) + 1u, n = (uint32_t)n_mine * per;
    for (uint32_t i0 = 0; i0 < n; i0 += 32 * kMoveBatch) {
      uint4 r[kMoveBatch];
      __half sc[kMoveBatch];
      int64_t dst[kMoveBatch];
      uint32_t piece[kMoveBatch];
#pragma unroll
      for (int k = 0; k < kMoveBatch; ++k) {
        const uint32_t i = i0 + 32 * k + lane;
        dst[k] = -1;
        if (i >= n) continue;
        const uint32_t row = div_by(i, cpr_mul, cpr);
        const uint32_t sl = div_by(row, nm_mul, nm), j = row - sl * nm;
        const int64_t from = s_src[j], add = s_slice[warp][sl];
        if (from < 0) continue;
        piece[k] = i - row * cpr;
        dst[k] = s_dst[j] + add;
        r[k] = *reinterpret_cast<const uint4*>(data + (from + add) * row_bytes + piece[k] * 16);
        if (g.dtype == SCKV_DTYPE_INT8 && piece[k] == 0) sc[k] = hscale[from + add];  // (one a row)
      }
      __syncwarp();
#pragma unroll
      for (int k = 0; k < kMoveBatch; ++k) {
        if (dst[k] < 0) continue;
        *reinterpret_cast<uint4*>(data + dst[k] * row_bytes + piece[k] * 16) = r[k];
        if (g.dtype == SCKV_DTYPE_INT8 && piece[k] == 0) hscale[dst[k]] = sc[k];
      }
      __syncwarp();
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kCompactWarps * 32) compact_fp8_kernel(const Compact p) {
  const Geo& g = p.g;
  const int lane = threadIdx.x & 31;
  const int64_t units = (int64_t)p.n_seqs * p.n_layers * 2 * g.H;
  int64_t u = (int64_t)blockIdx.x * kCompactWarps + (threadIdx.x >> 5);
  if (u >= units) return;
  const int h = (int)(u % g.H);
  u /= g.H;
  const int kv = (int)(u & 1);
  u >>= 1;
  const int l = (int)(u % p.n_layers), b = (int)(u / p.n_layers);
  const int layer = p.layer0 + l;
  const bool reporter = l == 0 && kv == 0 && h == 0 && lane == 0;
  const int keep = __ldg(p.n_keep + b), ctx = __ldg(p.ctx + b);
  const int32_t* path = p.path + (int64_t)b * p.max_path;
  const int cap = p.max_blocks * SCKV_PAGE_TOKENS;
  if (keep < 0 || keep > p.max_path || ctx < 0 || ctx > cap) {
    if (reporter) sckv_report(g.status, SCKV_ERR_BOUNDS, b, KID_COMPACT);
    return;
  }
  // the path increases and stays inside the table; rows 0 .. j0 - 1 do not move
  bool bad = false;
  int j0 = keep;
  for (int j = lane; j < keep; j += 32) {
    const int pj = __ldg(path + j), before = j > 0 ? __ldg(path + j - 1) : -1;
    bad |= pj <= before || pj >= cap - ctx;
    if (pj != j) j0 = min(j0, j);
  }
  if (__any_sync(0xffffffffu, bad)) {
    if (reporter) sckv_report(g.status, SCKV_ERR_BOUNDS, b, KID_COMPACT);
    return;
  }
  j0 = __reduce_min_sync(0xffffffffu, j0);
  if (j0 >= keep) return;
  const int32_t* bt = p.bt + (int64_t)b * p.bt_stride;
  const int cpr = g.D / 16;  // 16-byte chunks of a row
  uint8_t* data = reinterpret_cast<uint8_t*>(g.data);
  float* fscale = reinterpret_cast<float*>(g.scales);
  for (int blk = (ctx + j0) / SCKV_PAGE_TOKENS; blk <= (ctx + keep - 1) / SCKV_PAGE_TOKENS; ++blk) {
    const int32_t dpage = __ldg(bt + blk);
    if (dpage < 0 || dpage >= g.P) {
      if (reporter) sckv_report(g.status, SCKV_ERR_BOUNDS, dpage, KID_COMPACT);
      continue;
    }
    const int first = blk * SCKV_PAGE_TOKENS - ctx;  // path index of slot 0
    // byte offset of the row that slot `s` takes over, -1 if it keeps its own; its page through *from
    auto source = [&](int s, int32_t* from) -> int64_t {
      const int j = first + s;
      if (j < j0 || j >= keep) return -1;
      const int pos = ctx + __ldg(path + j);
      const int32_t page = __ldg(bt + pos / SCKV_PAGE_TOKENS);
      if (page < 0 || page >= g.P) {
        if (reporter) sckv_report(g.status, SCKV_ERR_BOUNDS, page, KID_COMPACT);
        return -1;
      }
      *from = page;
      return row_off(g, layer, page, kv, h, pos % SCKV_PAGE_TOKENS);
    };
    const int64_t dst0 = row_off(g, layer, dpage, kv, h, 0);
    const float s_dst = fscale[fp8_scale_idx(g, layer, dpage, kv, h)];
    // pass 1: the largest value that comes from another page
    float top = 0.f;
    for (int i = lane; i < SCKV_PAGE_TOKENS * cpr; i += 32) {
      int32_t from = dpage;
      const int64_t off = source(i / cpr, &from);
      if (off < 0 || from == dpage) continue;
      const float sc = fscale[fp8_scale_idx(g, layer, from, kv, h)];
      const uint4 w = *reinterpret_cast<const uint4*>(data + off + (i % cpr) * 16);
      const uint8_t* c = reinterpret_cast<const uint8_t*>(&w);
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(sckv_fp8_to_float(c[e]) * sc));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float s_new = fmaxf(s_dst, top / 448.0f);
    // pass 2: rows in order, 32 / cpr of them at a time (loads before stores)
    for (int i0 = 0; i0 < SCKV_PAGE_TOKENS * cpr; i0 += 32) {
      const int i = i0 + lane;
      int32_t from = dpage;
      int64_t off = i < SCKV_PAGE_TOKENS * cpr ? source(i / cpr, &from) : -1;
      bool store = off >= 0;
      off += (i % cpr) * 16;
      if (!store && i < SCKV_PAGE_TOKENS * cpr && first + i / cpr < j0 && s_new > s_dst) {
        off = dst0 + (int64_t)i * 16;  // a row that stays: re-encoded under the grown scale
        from = dpage;
        store = true;
      }
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if (store) {
        w = *reinterpret_cast<const uint4*>(data + off);
        const float sc = from == dpage ? s_dst : fscale[fp8_scale_idx(g, layer, from, kv, h)];
        if (sc != s_new) {
          uint8_t* c = reinterpret_cast<uint8_t*>(&w);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            c[e] = s_new > 0.f ? sckv_float_to_fp8(sckv_fp8_to_float(c[e]) * sc / s_new) : (uint8_t)0;
        }
      }
      __syncwarp();
      if (store) *reinterpret_cast<uint4*>(data + dst0 + (int64_t)i * 16) = w;
    }
    __syncwarp();
    if (lane == 0 && s_new > s_dst) fscale[fp8_scale_idx(g, layer, dpage, kv, h)] = s_new;
    __syncwarp();
  }
}

// ---------------------------------------------------------------------------
// Greedy check of a drafted tree: t_i = argmax_v logits[i][v] (the lowest
// index of equal values; NaN counts as the largest, as torch.argmax has it),
// then from node 0 on the child whose token is t of its parent, the first of
// equals, until there is none. Bound by HBM (the logits, read once): rows are
// cut into `chunks` of 16-byte pieces (a row's first and last elements that
// fill none go to its first and last chunk) so that few rows still fill the
// GPU. A thread keeps the largest value of its pieces and the first piece that
// holds it, eight 16-bit values by four packed maxima and one comparison, and
// looks its index up at the end. Every CTA leaves its chunk's best as one
// 64-bit word (ordered value, then the complement of the index), and one CTA
// per sequence joins them and walks. 1,152 rows of 151,936 bf16 logits: 66.2
// us with the walk and several states in turn, 5.3 TB/s (81 % of a copy's
// rate). One state over and over, a third of it in L2: 54.9 us; twice the chunks
// 62 us, CTAs of 512 threads 72; single elements instead of pieces 127.
// ---------------------------------------------------------------------------
constexpr int kVerifyThreads = 256;
constexpr int kVerifyMaxNodes = 1024;

// Larger value, then lower index <-> larger word.
__device__ __forceinline__ unsigned long long rank_word(float x, uint32_t idx) {
  x += 0.f;  // -0 counts as 0
  uint32_t b = __float_as_uint(x);
  b = x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)b << 32) | (uint32_t)~idx;
}

template <int DT>
__device__ __forceinline__ float logit_at(const void* base, int64_t i) {
  if (DT == SCKV_DTYPE_F32) return reinterpret_cast<const float*>(base)[i];
  if (DT == SCKV_DTYPE_F16) return __half2float(reinterpret_cast<const __half*>(base)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[i]);
}

__device__ __forceinline__ uint4 ld_once(const uint4* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// Largest value of a piece, NaN if there is one.
template <int DT>
__device__ __forceinline__ float piece_max(const uint4& w) {
  if constexpr (DT == SCKV_DTYPE_F32) {
    float m, a = __uint_as_float(w.x), b = __uint_as_float(w.y), c = __uint_as_float(w.z), d = __uint_as_float(w.w);
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(a), "f"(b));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(c), "f"(d));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(c));
    return m;
  } else if constexpr (DT == SCKV_DTYPE_F16) {
    const __half2* x = reinterpret_cast<const __half2*>(&w);
    const __half2 m = __hmax2_nan(__hmax2_nan(x[0], x[1]), __hmax2_nan(x[2], x[3]));
    return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
  } else {
    const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&w);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(x[0], x[1]), __hmax2_nan(x[2], x[3]));
    return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
  }
}

template <int DT>
__global__ void __launch_bounds__(kVerifyThreads) verify_argmax_kernel(const void* logits, int64_t ld, int vocab,
                                                                       int chunks, unsigned long long* best) {
  const int row = blockIdx.x / chunks, c = blockIdx.x - row * chunks;
  const int64_t base = row * ld;
  constexpr int kEl = DT == SCKV_DTYPE_F32 ? 4 : 2, kPer = 16 / kEl;
  const uint8_t* at = reinterpret_cast<const uint8_t*>(logits) + base * kEl;
  const int head = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(at) & 15)) & 15) / kEl);
  const int pieces = (vocab - head) / kPer, tail0 = head + pieces * kPer;
  const uint4* x = reinterpret_cast<const uint4*>(at + head * kEl);
  const int per = (pieces + chunks - 1) / chunks;
  const int lo = min(pieces, c * per), hi = min(pieces, lo + per);
  unsigned long long w = 0;
  auto single = [&](int i) {
    const unsigned long long y = rank_word(logit_at<DT>(logits, base + i), (uint32_t)i);
    w = y > w ? y : w;
  };
  if (c == 0 && (int)threadIdx.x < head) single(threadIdx.x);
  if (c == chunks - 1 && tail0 + (int)threadIdx.x < vocab) single(tail0 + threadIdx.x);
  int i = lo + threadIdx.x;
  if (i < hi) {
    float top = piece_max<DT>(ld_once(x + i));
    int where = i;
    auto take = [&](float m, int idx) {  // (nothing passes a NaN)
      if (!(m <= top) && top == top) {
        top = m;
        where = idx;
      }
    };
    for (i += kVerifyThreads; i + 3 * kVerifyThreads < hi; i += 4 * kVerifyThreads) {
      uint4 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = ld_once(x + i + e * kVerifyThreads);
#pragma unroll
      for (int e = 0; e < 4; ++e) take(piece_max<DT>(v[e]), i + e * kVerifyThreads);
    }
    for (; i < hi; i += kVerifyThreads) take(piece_max<DT>(ld_once(x + i)), i);
    for (int e = 0; e < kPer; ++e) {
      const int idx = head + where * kPer + e;
      const float y = logit_at<DT>(logits, base + idx);
      if (y == top || (top != top && y != y)) {
        const unsigned long long z = rank_word(y, (uint32_t)idx);
        w = z > w ? z : w;
        break;
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long y = __shfl_xor_sync(0xffffffffu, w, o);
    w = y > w ? y : w;
  }
  __shared__ unsigned long long s[kVerifyThreads / 32];
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = w;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int e = 1; e < kVerifyThreads / 32; ++e) w = s[e] > w ? s[e] : w;
    best[blockIdx.x] = w;
  }
}

struct Verify {
  int chunks, n_tokens, max_path;
  unsigned long long* best;  // [n_tokens][chunks], written by the launch before
  const int32_t* tokens;
  const int32_t* parents;
  const int32_t* cu;
  int32_t* path;
  int32_t* n_keep;
  int32_t* next;
  int32_t* status;
};

// One CTA per sequence joins the chunks' words of its rows, its first warp walks.
__global__ void __launch_bounds__(kVerifyThreads) verify_walk_kernel(const Verify p) {
  __shared__ unsigned long long s_best[kVerifyMaxNodes];
  const int b = blockIdx.x, t0 = __ldg(p.cu + b);
  int n = __ldg(p.cu + b + 1) - t0;
  const bool ok = t0 >= 0 && n >= 0 && n <= kVerifyMaxNodes && t0 + n <= p.n_tokens;
  if (!ok) n = 0;
  for (int i = threadIdx.x; i < n; i += kVerifyThreads) s_best[i] = 0;
  __syncthreads();
  const unsigned long long* words = p.best + (int64_t)t0 * p.chunks;
#pragma unroll 4
  for (int u = threadIdx.x; u < n * p.chunks; u += kVerifyThreads) atomicMax(s_best + u / p.chunks, __ldg(words + u));
  __syncthreads();
  if (threadIdx.x >= 32) return;
  const int lane = threadIdx.x;
  if (!ok && lane == 0) sckv_report(p.status, SCKV_ERR_BOUNDS, b, KID_VERIFY);
  auto best_of = [&](int i) { return (int32_t)~(uint32_t)s_best[i]; };
  int32_t* out = p.path + (int64_t)b * p.max_path;
  int keep = 0, token = -1;
  if (n > 0) {
    int cur = 0;
    if (lane == 0) out[0] = 0;
    keep = 1;
    token = best_of(0);
    while (keep < p.max_path) {
      // the first later node that hangs on `cur` and carries its token
      int child = -1;
      for (int j0 = cur + 1; j0 < n && child < 0; j0 += 32) {
        const int j = j0 + lane;
        const bool hit = j < n && __ldg(p.parents + t0 + j) == cur && __ldg(p.tokens + t0 + j) == token;
        const unsigned m = __ballot_sync(0xffffffffu, hit);
        if (m) child = j0 + __ffs(m) - 1;
      }
      if (child < 0) break;
      if (lane == 0) out[keep] = child;
      ++keep;
      cur = child;
      token = best_of(cur);
    }
  }
  for (int j = keep + lane; j < p.max_path; j += 32) out[j] = -1;
  if (lane == 0) {
    p.n_keep[b] = keep;
    p.next[b] = token;
  }
}

// Cuts per row so that the argmax pass has a few CTAs per SM.
int verify_chunks(int num_sms, int n_tokens, int vocab) {
  const int most = (vocab + 2047) / 2048;  // at least 2048 logits a CTA
  int c = (8 * num_sms + n_tokens - 1) / n_tokens;
  if (c > most) c = most;
  return c < 1 ? 1 : c;
}

// Tokens of a CTA: one until every SM has 16 CTAs (8 are resident), then more,
// whose angles and page lookups are one latency (8,192 tokens of 48 heads, one
// state over and over: 41 us with 3, 44 with 1).
int rope_tokens(int num_sms, int n_tokens) {
  const int n = n_tokens / (16 * num_sms);
  return n < 1 ? 1 : n > kRopeTokens ? kRopeTokens : n;
}

}  // namespace

extern "C" size_t sckv_append_rope_axes_workspace_bytes(const sckv_pool* p, int n_tokens) {
  if (p == nullptr || n_tokens <= 0 || p->kv_dtype != SCKV_DTYPE_FP8_E4M3) return 0;
  return (size_t)n_tokens * p->num_kv_heads * p->head_dim * sizeof(float);
}

extern "C" int sckv_append_rope_axes(sckv_pool* p, int layer, const void* q, int64_t q_stride, void* q_out,
                                     int num_q_heads, int q_dtype, int q_out_dtype, const void* k, int64_t k_stride,
                                     const void* v, int64_t v_stride, int src_dtype, const void* q_norm_w,
                                     const void* k_norm_w, float eps, const float* inv_freq, float rope_scaling,
                                     const int32_t* positions, int64_t pos_stride, int n_axes,
                                     const int32_t* axis_map, int n_seqs, int n_tokens, const int32_t* cu_tokens,
                                     const int32_t* start_pos, const int32_t* block_table, int64_t bt_stride,
                                     int max_blocks, void* workspace, size_t workspace_bytes, void* stream) {
  if (p == nullptr || layer < 0 || layer >= p->num_layers || n_seqs < 0 || n_tokens < 0 || num_q_heads <= 0 ||
      n_axes <= 0)
    return SCKV_ERR_INVALID_ARG;
  if (p->head_dim != kRopeD) return SCKV_ERR_UNSUPPORTED;
  if (!is_src_dtype(src_dtype) || !is_src_dtype(q_dtype) || !is_src_dtype(q_out_dtype)) return SCKV_ERR_INVALID_ARG;
  if (!(rope_scaling > 0.f) || !(eps >= 0.f)) return SCKV_ERR_INVALID_ARG;
  if (n_seqs == 0 || n_tokens == 0) return SCKV_OK;
  if (!q || !q_out || !k || !v || !inv_freq || !positions || !axis_map || !cu_tokens || !start_pos || !block_table ||
      bt_stride < max_blocks || max_blocks <= 0)
    return SCKV_ERR_INVALID_ARG;
  if (q_stride < (int64_t)num_q_heads * kRopeD || k_stride < (int64_t)p->num_kv_heads * kRopeD ||
      v_stride < (int64_t)p->num_kv_heads * kRopeD)
    return SCKV_ERR_INVALID_ARG;
  const int64_t qe = q_dtype == SCKV_DTYPE_F32 ? 4 : 2, se = src_dtype == SCKV_DTYPE_F32 ? 4 : 2;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
        reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(q_norm_w) |
        reinterpret_cast<uintptr_t>(k_norm_w) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      ((q_stride * qe) & 15) || ((k_stride * se) & 15) || ((v_stride * se) & 15))
    return SCKV_ERR_ALIGNMENT;
  const size_t need = sckv_append_rope_axes_workspace_bytes(p, n_tokens);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return SCKV_ERR_INVALID_ARG;
  RopeAxes a{};
  a.g = geo_of(p);
  a.layer = layer;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_dtype = q_dtype;
  a.src_dtype = src_dtype;
  a.q_out = q_out;
  a.q_out_dtype = q_out_dtype;
  a.k_stage = reinterpret_cast<float*>(workspace);
  a.q_w = reinterpret_cast<const __half*>(q_norm_w);
  a.k_w = reinterpret_cast<const __half*>(k_norm_w);
  a.eps = eps;
  a.inv_freq = inv_freq;
  a.inv_scaling = 1.0 / (double)rope_scaling;
  a.positions = positions;
  a.pos_stride = pos_stride;
  a.n_axes = n_axes;
  a.axis_map = axis_map;
  a.hq = num_q_heads;
  a.n_seqs = n_seqs;
  a.n_tokens = n_tokens;
  a.cu = cu_tokens;
  a.start_pos = start_pos;
  a.bt = block_table;
  a.bt_stride = bt_stride;
  a.max_blocks = max_blocks;
  SCKV_DEVICE_GUARD(p->device);
  cudaStream_t s = as_stream(stream);
  a.tpb = rope_tokens(p->num_sms, n_tokens);
  const int blocks = (n_tokens + a.tpb - 1) / a.tpb;
  if (q_dtype != src_dtype || src_dtype == SCKV_DTYPE_F32)
    rope_axes_kernel<-1><<<blocks, kRopeThreads, 0, s>>>(a);
  else if (src_dtype == SCKV_DTYPE_F16)
    rope_axes_kernel<SCKV_DTYPE_F16><<<blocks, kRopeThreads, 0, s>>>(a);
  else
    rope_axes_kernel<SCKV_DTYPE_BF16><<<blocks, kRopeThreads, 0, s>>>(a);
  SCKV_LAUNCH_CHECK();
  if (p->kv_dtype == SCKV_DTYPE_FP8_E4M3) {
    const int64_t units = (int64_t)n_seqs * 2 * p->num_kv_heads;
    rope_axes_fp8_kernel<<<(unsigned)((units + 3) / 4), 128, 0, s>>>(a);
    SCKV_LAUNCH_CHECK();
  }
  return SCKV_OK;
}

extern "C" int sckv_compact_tree(sckv_pool* p, int layer0, int n_layers, int n_seqs, const int32_t* path, int max_path,
                                 const int32_t* n_keep, const int32_t* ctx_lens, const int32_t* block_table,
                                 int64_t bt_stride, int max_blocks, void* stream) {
  if (p == nullptr || layer0 < 0 || n_layers <= 0 || layer0 + n_layers > p->num_layers || n_seqs < 0 || max_path < 0)
    return SCKV_ERR_INVALID_ARG;
  if (n_seqs == 0 || max_path == 0) return SCKV_OK;
  if (!path || !n_keep || !ctx_lens || !block_table || bt_stride < max_blocks || max_blocks <= 0)
    return SCKV_ERR_INVALID_ARG;
  // slices of a warp: as many as leave every SM 32 warps, at most 8 (its pieces are counted in 16 bits)
  const int64_t n_slices = (int64_t)n_layers * 2 * p->num_kv_heads;
  const bool fp8 = p->kv_dtype == SCKV_DTYPE_FP8_E4M3;
  const int64_t share = n_seqs * n_slices / (32 * p->num_sms);
  const int per_warp = fp8 || share < 1 ? 1 : share > kMaxSlices ? kMaxSlices : (int)share;
  Compact c{geo_of(p), layer0, n_layers, n_seqs, max_path, path, n_keep, ctx_lens, block_table, bt_stride, max_blocks,
            per_warp};
  const int64_t blocks = fp8 ? (n_seqs * n_slices + kCompactWarps - 1) / kCompactWarps
                             : n_seqs * ((n_slices + kCompactWarps * per_warp - 1) / (kCompactWarps * per_warp));
  if (blocks > INT32_MAX) return SCKV_ERR_INVALID_ARG;
  SCKV_DEVICE_GUARD(p->device);
  if (fp8)
    compact_fp8_kernel<<<(unsigned)blocks, kCompactWarps * 32, 0, as_stream(stream)>>>(c);
  else
    compact_kernel<<<(unsigned)blocks, kCompactWarps * 32, 0, as_stream(stream)>>>(c);
  SCKV_LAUNCH_CHECK();
  return SCKV_OK;
}

extern "C" size_t sckv_verify_tree_workspace_bytes(const sckv_pool* p, int n_tokens, int vocab) {
  if (p == nullptr || n_tokens <= 0 || vocab <= 0) return 0;
  return (size_t)n_tokens * verify_chunks(p->num_sms, n_tokens, vocab) * sizeof(unsigned long long);
}

extern "C" int sckv_verify_tree(sckv_pool* p, const void* logits, int logits_dtype, int64_t ld, int n_tokens, int vocab,
                                const int32_t* tokens, const int32_t* parents, const int32_t* cu_tokens, int n_seqs,
                                int max_path, int32_t* path, int32_t* n_keep, int32_t* next_token, void* workspace,
                                size_t workspace_bytes, void* stream) {
  if (p == nullptr || !is_src_dtype(logits_dtype) || n_tokens < 0 || vocab <= 0 || ld < vocab || n_seqs < 0 ||
      max_path <= 0)
    return SCKV_ERR_INVALID_ARG;
  if (n_seqs == 0) return SCKV_OK;
  if (!cu_tokens || !path || !n_keep || !next_token) return SCKV_ERR_INVALID_ARG;
  if (n_tokens > 0 && (!logits || !tokens || !parents)) return SCKV_ERR_INVALID_ARG;
  const size_t need = sckv_verify_tree_workspace_bytes(p, n_tokens, vocab);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return SCKV_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(workspace) & 7) return SCKV_ERR_ALIGNMENT;
  const size_t el = logits_dtype == SCKV_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) & (el - 1)) return SCKV_ERR_ALIGNMENT;
  SCKV_DEVICE_GUARD(p->device);
  cudaStream_t s = as_stream(stream);
  Verify a{1, n_tokens, max_path, reinterpret_cast<unsigned long long*>(workspace), tokens, parents,
           cu_tokens, path, n_keep, next_token, p->status};
  if (n_tokens > 0) {
    a.chunks = verify_chunks(p->num_sms, n_tokens, vocab);
    const int64_t blocks = (int64_t)n_tokens * a.chunks;
    if (blocks > INT32_MAX) return SCKV_ERR_INVALID_ARG;
    auto launch = [&](auto dt) {
      verify_argmax_kernel<decltype(dt)::value>
          <<<(unsigned)blocks, kVerifyThreads, 0, s>>>(logits, ld, vocab, a.chunks, a.best);
    };
    if (logits_dtype == SCKV_DTYPE_F32)
      launch(std::integral_constant<int, SCKV_DTYPE_F32>{});
    else if (logits_dtype == SCKV_DTYPE_F16)
      launch(std::integral_constant<int, SCKV_DTYPE_F16>{});
    else
      launch(std::integral_constant<int, SCKV_DTYPE_BF16>{});
    SCKV_LAUNCH_CHECK();
  }
  verify_walk_kernel<<<n_seqs, kVerifyThreads, 0, s>>>(a);
  SCKV_LAUNCH_CHECK();
  return SCKV_OK;
}
