// What the kernels of the paged key-value cache share (paged_cache.cu, paged_attention.cu, paged_attention_rows.cu).
//
// Elements [pages, G, S, D] of keys and of values, any strides but a dense D; bf16, fp32, or e4m3 with one power of two per token and head, held
// as its biased exponent in a byte [pages, G, S].  table[b][i] is the page of tokens i·S … i·S + S − 1 of sequence b; lengths[b] counts its tokens, the
// new ones included, and of T rows of new tokens the first new_lengths[b] are real: row i sits at position lengths[b] − new_lengths[b] + i.
// Offsets are 64-bit.  Pages outside the cache and positions outside the table are never touched.
#pragma once
#include "sm100.cuh"
#include "api.h"

namespace b200 {

using PagedView = b200_paged_view;

// the power of two of a scale byte
__device__ __forceinline__ float paged_pow2(uint32_t code) {
  return __uint_as_float(code == 255u ? 0x7fffffffu : code == 0u ? 0x00400000u : code << 23);
}
__device__ __forceinline__ int paged_new(const PagedView& c, int b, int T) {
  return c.new_lengths ? max(0, min(c.new_lengths[b], T)) : T;
}
// page of position pos of sequence b, or -1 (and the status word is set) where there is none
__device__ __forceinline__ int paged_page(const PagedView& c, int b, int index) {
  if (index < 0 || index >= c.table_cols) return -1;
  const int page = c.table[b * c.table_row + index];
  if (page < 0 || page >= c.pages) {
    if (c.status) atomicCAS(c.status, 0, STATUS_INDEX_RANGE);
    return -1;
  }
  return page;
}
// value i of a small fp32 (0) or bf16 (1) array
__device__ __forceinline__ float paged_param(const void* p, int type, int i) {
  return type == 0 ? static_cast<const float*>(p)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

}  // namespace b200
