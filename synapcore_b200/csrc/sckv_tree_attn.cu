// Attention of a tree of drafted tokens over a paged cache.
//
// Node i of sequence b is the query of rows (i, head); its own K/V row sits in
// slot ctx_lens[b] + i. It sees the sequence's ctx_lens[b] committed tokens and
// the nodes j whose bit is set in its mask:
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - m)
//
// One CTA per (node, q head); its four warps take every fourth key with an
// online softmax each (4 dims a lane) and merge at the end.
#include <math.h>

#include "sckv_geo.cuh"

using namespace sckv_geo;

namespace {

constexpr int kHD = 128;
constexpr int kWarps = 4;
constexpr int kMaskWordsMax = 4;

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
  int max_blocks, n_seqs, n_tokens, hq;
  int q_dtype, out_dtype;
  float scale_log2;
};

__device__ __forceinline__ void load_row4(const Geo& g, int layer, int64_t page, int kv, int h, int slot, int lane,
                                          float (&x)[4]) {
  const int64_t o = row_off(g, layer, page, kv, h, slot) + 4 * lane;
  if (g.dtype == SCKV_DTYPE_INT8) {
    const float s = __half2float(reinterpret_cast<const __half*>(g.scales)[int8_scale_idx(g, layer, page, kv, h, slot)]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = __half2float(__float2half_rn((float)reinterpret_cast<const int8_t*>(g.data)[o + i] * s));
  } else if (g.dtype == SCKV_DTYPE_FP8_E4M3) {
    const float s = reinterpret_cast<const float*>(g.scales)[fp8_scale_idx(g, layer, page, kv, h)];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = sckv_fp8_to_float(reinterpret_cast<const uint8_t*>(g.data)[o + i]) * s;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = sckv_load_as_float(g.data, o + i, g.dtype);
  }
}

__global__ void __launch_bounds__(kWarps * 32) tree_attn_simple_kernel(const TreeParams p) {
  const int t = blockIdx.x / p.hq, head = blockIdx.x - t * p.hq;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (t < __ldg(p.cu_q) || t >= __ldg(p.cu_q + p.n_seqs)) return;
  const int b = sckv_find_seq(p.cu_q, p.n_seqs, t);
  const int t0 = __ldg(p.cu_q + b), n = __ldg(p.cu_q + b + 1) - t0, ctx = __ldg(p.ctx_lens + b);
  const int cap = p.max_blocks * SCKV_PAGE_TOKENS;
  if (t0 < 0 || ctx < 0 || n < 0 || t0 + n > p.n_tokens || n > 64 * p.mask_words || ctx > cap - n) {
    if (threadIdx.x == 0) sckv_report(p.g.status, SCKV_ERR_BOUNDS, b, KID_TREE_ATTN);
    return;
  }
  const int h = head / (p.hq / p.g.H);
  float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
  const int64_t row = ((int64_t)t * p.hq + head) * kHD;
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = sckv_load_as_float(p.q, row + 4 * lane + i, p.q_dtype) * p.scale_log2;
  float m = -INFINITY, l = 0.f;
  const int32_t* bt = p.bt + (int64_t)b * p.bt_stride;
  for (int k = warp; k < ctx + n; k += kWarps) {
    if (k >= ctx) {
      const int j = k - ctx;
      if (!((p.mask[(int64_t)t * p.mask_words + (j >> 6)] >> (j & 63)) & 1)) continue;
    }
    int32_t page = __ldg(bt + k / SCKV_PAGE_TOKENS);
    if (page < 0 || page >= p.g.P) {
      if (lane == 0) sckv_report(p.g.status, SCKV_ERR_BOUNDS, page, KID_TREE_ATTN);
      page = 0;
    }
    float x[4];
    load_row4(p.g, p.layer, page, 0, h, k % SCKV_PAGE_TOKENS, lane, x);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s = fmaf(q[i], x[i], s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float mn = fmaxf(m, s);
    const float alpha = exp2f(m - mn), w = exp2f(s - mn);
    m = mn;
    l = fmaf(l, alpha, w);
    load_row4(p.g, p.layer, page, 1, h, k % SCKV_PAGE_TOKENS, lane, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(acc[i], alpha, w * x[i]);
  }
  __shared__ float s_acc[kWarps][kHD], s_m[kWarps], s_l[kWarps];
#pragma unroll
  for (int i = 0; i < 4; ++i) s_acc[warp][4 * lane + i] = acc[i];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  const int d = threadIdx.x;
  float M = -INFINITY, L = 0.f, O = 0.f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w]);
  for (int w = 0; w < kWarps; ++w) {
    if (s_m[w] == -INFINITY) continue;
    const float e = exp2f(s_m[w] - M);
    L = fmaf(s_l[w], e, L);
    O = fmaf(s_acc[w][d], e, O);
  }
  sckv_store_from_float(p.out, row + d, p.out_dtype, L == 0.f ? 0.f : O / L)  /* NaN stays NaN */;
}

}  // namespace

extern "C" size_t sckv_tree_attn_workspace_bytes(const sckv_pool* p, int n_tokens, int num_q_heads) {
  (void)p;
  (void)n_tokens;
  (void)num_q_heads;
  return 0;
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
  const size_t need = sckv_tree_attn_workspace_bytes(p, n_tokens, num_q_heads);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return SCKV_ERR_INVALID_ARG;
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
  t.q_dtype = q_dtype;
  t.out_dtype = out_dtype;
  t.scale_log2 = scale * 1.4426950408889634f;
  const int64_t blocks = (int64_t)n_tokens * num_q_heads;
  if (blocks > INT32_MAX) return SCKV_ERR_INVALID_ARG;
  SCKV_DEVICE_GUARD(p->device);
  tree_attn_simple_kernel<<<(unsigned)blocks, kWarps * 32, 0, as_stream(stream)>>>(t);
  SCKV_LAUNCH_CHECK();
  return SCKV_OK;
}
