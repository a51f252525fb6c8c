// Device view of a paged KV cache (cq_kv_pages) and its checks, shared by the
// page operators (cq_pages.hip), the row store (cq_paged_kv.hip) and the
// attention over pages (cq_prefix_attention.hip).
#pragma once

#include "cq_device.h"
#include "cq_internal.h"

namespace cq {

constexpr int kMaxSeqs = 1024;          // sequences of a page map, one per thread of the planning block
constexpr int kMaxPages = 1 << 20;
constexpr int kMaxPageTokens = 32768;

// Strides in elements; a page of one head is a layer cache of 1 << shift slots
// (kv_k_offset and its kin with kv_head 0).
struct PageView {
  char* kv[2];            // K, V
  float* scale[2];
  int64_t layer_stride, page_stride, head_stride;
  int n_pages, shift;     // page_tokens = 1 << shift
};

inline PageView page_view(const cq_kv_pages& p) {
  PageView v;
  v.kv[0] = (char*)p.k; v.kv[1] = (char*)p.v;
  v.scale[0] = p.k_scale; v.scale[1] = p.v_scale;
  v.layer_stride = p.layer_stride; v.page_stride = p.page_stride; v.head_stride = p.head_stride;
  v.n_pages = p.n_pages;
  v.shift = __builtin_ctz((unsigned)p.page_tokens);
  return v;
}

inline int pages_geometry_check(int kv_dtype, int64_t n_layers, int64_t n_pages, int64_t page_tokens, int64_t n_kv, int head_dim) {
  if (kv_dtype != CQ_KV_FP16 && kv_dtype != CQ_KV_INT8 && kv_dtype != CQ_KV_FP8) return fail(CQ_EINVAL, "pages: unknown KV cache type");
  if (head_dim != 64 && head_dim != 128) return fail(CQ_EINVAL, "pages: head_dim must be 64 or 128");
  if (n_kv < 1 || n_kv > 64) return fail(CQ_EINVAL, "pages: n_kv_heads outside [1, 64]");
  if (n_layers < 1 || n_layers > 4096) return fail(CQ_EINVAL, "pages: n_layers outside [1, 4096]");
  if (page_tokens < 32 || page_tokens > kMaxPageTokens || (page_tokens & (page_tokens - 1)))
    return fail(CQ_EINVAL, "pages: page_tokens must be a power of two in [32, 32768]");
  if (n_pages < 1 || n_pages > kMaxPages || n_pages * page_tokens >= ((int64_t)1 << 31))
    return fail(CQ_EINVAL, "pages: n_pages outside [1, 2^20], or 2^31 slots or more");
  return CQ_OK;
}

inline bool unaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

inline int pages_check(const cq_kv_pages* p) {
  if (!p) return fail(CQ_EINVAL, "pages: null description");
  CQ_TRY(pages_geometry_check(p->kv_dtype, p->n_layers, p->n_pages, p->page_tokens, p->n_kv_heads, p->head_dim));
  if (!p->k || !p->v || unaligned16(p->k) || unaligned16(p->v)) return fail(CQ_EINVAL, "pages: k and v must be set and aligned to 16 bytes");
  if (p->kv_dtype != CQ_KV_FP16 && (!p->k_scale || !p->v_scale || unaligned16(p->k_scale) || unaligned16(p->v_scale)))
    return fail(CQ_EINVAL, "pages: a one-byte cache needs its scales, aligned to 16 bytes");
  const int64_t unit = 32 * p->head_dim, run = (int64_t)p->page_tokens * p->head_dim;
  const int64_t most = (int64_t)1 << 46;   // keeps the products below 2^63
  const int64_t s[3] = {p->layer_stride, p->page_stride, p->head_stride};
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0 || s[i] > most || s[i] % unit) return fail(CQ_EINVAL, "pages: strides must be multiples of 32 * head_dim");
  if (p->page_stride > most / p->n_pages || p->head_stride > most / 64) return fail(CQ_EINVAL, "pages: strides too large");
  const int64_t heads = (p->n_kv_heads - 1) * p->head_stride + run;    // extent of a page's heads, of a head's pages
  const int64_t pages = (p->n_pages - 1) * p->page_stride + run;
  const bool heads_within = (p->n_kv_heads == 1 || p->head_stride >= run) && (p->n_pages == 1 || p->page_stride >= heads);
  const bool pages_within = (p->n_pages == 1 || p->page_stride >= run) && (p->n_kv_heads == 1 || p->head_stride >= pages);
  if (!heads_within && !pages_within) return fail(CQ_EINVAL, "pages: strides make pages overlap");
  const int64_t extent = (p->n_pages - 1) * p->page_stride + (p->n_kv_heads - 1) * p->head_stride + run;
  if (p->n_layers > 1 && p->layer_stride < extent) return fail(CQ_EINVAL, "pages: strides make layers overlap");
  return CQ_OK;
}

}  // namespace cq
