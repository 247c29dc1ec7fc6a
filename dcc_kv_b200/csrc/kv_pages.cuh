// Addresses and codes of the paged KV cache (dcc_kv_pages).
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace dcc {

constexpr float kSmallestScale = 1.262177448353619e-29f;  // 2^-96: keeps x / scale and its reciprocal normal

// Row (page, offset) of a position, or -1 where the sequence holds nothing.
struct PageWalk {
  const int32_t* table;  // of one sequence
  int64_t n_pages;
  int32_t page_size, max_pages;
  __device__ __forceinline__ int64_t page_of(int64_t pos, int& off) const {
    if (pos < 0) return -1;
    const int64_t slot = pos < 0x7fffffff ? (int64_t)((uint32_t)pos / (uint32_t)page_size) : pos / page_size;
    if (slot >= max_pages) return -1;
    off = (int)(pos - slot * page_size);
    const int64_t id = table[slot];
    return id >= 0 && id < n_pages ? id : -1;
  }
};

// Index of row `off` of a page for one KV head, in rows.
__device__ __forceinline__ int64_t page_row(const dcc_kv_pages& c, int64_t page, int head, int off) {
  return (page * c.n_kv_heads + head) * c.page_size + off;
}

// Eight codes as values without their scale.
__device__ __forceinline__ void decode_int8x4(uint32_t w, float* out) {
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = (float)(int8_t)(w >> (8 * i));
}
__device__ __forceinline__ void decode_e4m3x4(uint32_t w, float* out) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    out[2 * i] = f.x;
    out[2 * i + 1] = f.y;
  }
}
template <int kFormat>
__device__ __forceinline__ float load_code(const void* base, int64_t i) {
  if constexpr (kFormat == DCC_KV_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
  if constexpr (kFormat == DCC_KV_F32) return static_cast<const float*>(base)[i];
  if constexpr (kFormat == DCC_KV_INT8) return (float)static_cast<const int8_t*>(base)[i];
  if constexpr (kFormat == DCC_KV_E4M3) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<const __nv_fp8_storage_t*>(base)[i], __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half*>(&h));
  }
  return 0.f;
}

inline int check_pages(const dcc_kv_pages* c, const char* what) {
  if (!c) return fail(DCC_ERR_INVALID_ARGUMENT, std::string(what) + ": null cache");
  if (c->format < DCC_KV_BF16 || c->format > DCC_KV_E4M3)
    return fail(DCC_ERR_DTYPE, std::string(what) + ": unknown cache format");
  if (c->n_pages < 0 || c->page_size < 1 || c->n_kv_heads < 1)
    return fail(DCC_ERR_INVALID_ARGUMENT, std::string(what) + ": bad cache sizes");
  if (c->head_dim < 1 || c->head_dim > 128)
    return fail(DCC_ERR_UNSUPPORTED, std::string(what) + ": head_dim must be in [1, 128]");
  if (c->n_kv_heads > 65535) return fail(DCC_ERR_UNSUPPORTED, std::string(what) + ": too many heads");
  const bool scaled = c->format == DCC_KV_INT8 || c->format == DCC_KV_E4M3;
  if (c->n_pages > 0 && (!c->k || !c->v || (scaled && (!c->k_scale || !c->v_scale))))
    return fail(DCC_ERR_INVALID_ARGUMENT, std::string(what) + ": null cache tensor");
  return DCC_OK;
}

}  // namespace dcc
