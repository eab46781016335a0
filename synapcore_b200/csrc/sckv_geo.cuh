// Page geometry and per-row storage shared by the paging and tree kernels:
// offsets of rows and scales, 8-value loads and stores, page lookup, the int8
// row quantiser and the FP8 page-head update.
#pragma once

#include "sckv_internal.cuh"

namespace sckv_geo {

struct Geo {
  int L, H, D;
  int64_t P;
  int dtype;
  void* data;
  void* scales;
  int32_t* status;
};

inline Geo geo_of(const sckv_pool* p) {
  Geo g;
  g.L = p->num_layers;
  g.H = p->num_kv_heads;
  g.D = p->head_dim;
  g.P = p->max_pages;
  g.dtype = p->kv_dtype;
  g.data = p->data;
  g.scales = p->scales;
  g.status = p->status;
  return g;
}

// Element offset of row (layer, page, kv, head, slot) in the pool.
__device__ __forceinline__ int64_t row_off(const Geo& g, int64_t layer, int64_t page, int kv, int h,
                                           int slot) {
  return ((((layer * g.P + page) * 2 + kv) * g.H + h) * SCKV_PAGE_TOKENS + slot) * (int64_t)g.D;
}

// fp8 scale index of (layer, page, kv, head).
__device__ __forceinline__ int64_t fp8_scale_idx(const Geo& g, int64_t layer, int64_t page, int kv,
                                                 int h) {
  return ((layer * g.P + page) * 2 + kv) * g.H + h;
}

// int8 scale index of (layer, page, kv, head, slot).
__device__ __forceinline__ int64_t int8_scale_idx(const Geo& g, int64_t layer, int64_t page, int kv,
                                                  int h, int slot) {
  return (((layer * g.P + page) * 2 + kv) * g.H + h) * SCKV_PAGE_TOKENS + slot;
}

// 8 values of 16 bits as float.
__device__ __forceinline__ void unpack8(const uint4& raw, int dtype, float v[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dtype == SCKV_DTYPE_F16) {
      __half2 h2 = *reinterpret_cast<const __half2*>(&w[i]);
      float2 f = __half22float2(h2);
      v[2 * i] = f.x; v[2 * i + 1] = f.y;
    } else {
      __nv_bfloat162 b2 = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
      float2 f = __bfloat1622float2(b2);
      v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
  }
}

// Load 8 consecutive source values as float.
__device__ __forceinline__ void load8(const void* src, int64_t idx, int dtype, float v[8]) {
  if (dtype == SCKV_DTYPE_F32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(src) + idx);
    float4 a = p[0], b = p[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    unpack8(*reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(src) + idx), dtype, v);
  }
}

// Store 8 floats as 16-bit dtype (16 bytes).
__device__ __forceinline__ void store8_16(void* dst, int64_t idx, int dtype, const float v[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dtype == SCKV_DTYPE_F16) {
      __half2 h2 = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&h2);
    } else {
      __nv_bfloat162 b2 = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&b2);
    }
  }
  *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(dst) + idx) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Resolve the destination page of (seq b, position pos); -1 on error (reported).
__device__ __forceinline__ int64_t resolve_page(const Geo& g, const int32_t* bt, int64_t stride,
                                                int max_blocks, int b, int pos, int kid) {
  if (pos < 0) { sckv_report(g.status, SCKV_ERR_BOUNDS, pos, kid); return -1; }
  int blk = pos / SCKV_PAGE_TOKENS;
  if (blk >= max_blocks) { sckv_report(g.status, SCKV_ERR_BOUNDS, blk, kid); return -1; }
  int32_t page = __ldg(bt + (int64_t)b * stride + blk);
  if (page < 0 || page >= g.P) { sckv_report(g.status, SCKV_ERR_BOUNDS, page, kid); return -1; }
  return page;
}

// ---------------------------------------------------------------------------
// int8 quantisation of one row of D values held by a warp (lane holds D/32).
// quantize_kv_int8_numpy (native/native_engine.py:207-216):
//   s = max(max|x| / 127, 1e-7) in fp32; q = clip(rint(x / s), -127, 127);
//   stored scale = fp16(s).
// ---------------------------------------------------------------------------
template <int VPL>
__device__ __forceinline__ void quant_row_int8(const float x[VPL], int8_t q[VPL], __half* s_out) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) m = fmaxf(m, fabsf(x[i]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float s = fmaxf(m / 127.0f, 1e-7f);
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    float r = rintf(x[i] / s);
    r = fminf(fmaxf(r, -127.0f), 127.0f);
    q[i] = static_cast<int8_t>(r);
  }
  *s_out = __float2half_rn(s);
}

// ---------------------------------------------------------------------------
// fp8 page-head update: one warp owns (layer, page, kv, head) and folds in
// `n_new` new rows starting at slot `slot0` (slots < slot0 hold earlier tokens).
//   s_new = max(s_old, max|x_new| / 448)   (s_old = 0 for a fresh page, slot0 == 0)
//   if s_new > s_old and slot0 > 0: old codes c -> enc(dec(c) * s_old / s_new)
//   new codes = enc(x / s_new); s_new == 0 -> codes 0.
// enc = e4m3 round-to-nearest-even with saturation; dec exact.
// ---------------------------------------------------------------------------
__device__ inline void fp8_page_head_update(const Geo& g, int64_t layer, int64_t page, int kv, int h,
                                     int slot0, int n_new, const void* src, int64_t src_row0,
                                     int64_t src_row_stride, int src_dtype) {
  const int lane = threadIdx.x & 31;
  float* scales = reinterpret_cast<float*>(g.scales);
  const int64_t sidx = fp8_scale_idx(g, layer, page, kv, h);
  const float s_old = (slot0 == 0) ? 0.f : scales[sidx];
  float m = 0.f;
  for (int r = 0; r < n_new; ++r)
    for (int d = lane; d < g.D; d += 32)
      m = fmaxf(m, fabsf(sckv_load_as_float(src, src_row0 + r * src_row_stride + d, src_dtype)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float s_new = fmaxf(s_old, m / 448.0f);
  uint8_t* base = reinterpret_cast<uint8_t*>(g.data) + row_off(g, layer, page, kv, h, 0);
  if (s_new > s_old && slot0 > 0) {
    for (int i = lane; i < slot0 * g.D; i += 32) {
      float x = sckv_fp8_to_float(base[i]) * s_old;
      base[i] = sckv_float_to_fp8(x / s_new);
    }
  }
  for (int r = 0; r < n_new; ++r)
    for (int d = lane; d < g.D; d += 32) {
      float x = sckv_load_as_float(src, src_row0 + r * src_row_stride + d, src_dtype);
      base[(slot0 + r) * g.D + d] = (s_new > 0.f) ? sckv_float_to_fp8(x / s_new) : (uint8_t)0;
    }
  __syncwarp();
  if (lane == 0) scales[sidx] = s_new;
}

inline bool is_src_dtype(int d) { return d == SCKV_DTYPE_F16 || d == SCKV_DTYPE_BF16 || d == SCKV_DTYPE_F32; }

}  // namespace sckv_geo
