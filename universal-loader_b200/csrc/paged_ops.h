/*
 * paged_ops.h — what the paged cache operators (rope.cu, tree_attention.cu, pages.cu, logits.cu)
 * share: element types, the checked geometry of a cache, and launch error plumbing.
 */
#pragma once

#include <cuda_bf16.h>

#include <initializer_list>
#include <type_traits>

#include "ulb_internal.h"

namespace ulb {

/* a cache's layout with the default strides filled in (elements) */
struct CacheGeom {
  int n_head_kv, hd, page, page_shift, n_pages, n_seq, max_pages, n_layer;
  long long layer, pstride, head, pos;
};

inline int dtype_bytes(int t) { return t == ULB_TYPE_F32 ? 4 : t == ULB_TYPE_F16 || t == ULB_TYPE_BF16 ? 2 : 0; }

inline int cache_geom(const char* who, const ulb_cache_desc* d, CacheGeom* g) {
  ULB_CHECK(d, ULB_EINVAL, "%s: cache description is NULL", who);
  ULB_CHECK(d->dtype == ULB_TYPE_F16 || d->dtype == ULB_TYPE_BF16, ULB_EUNSUPPORTED,
            "%s: cache type %d (F16 or BF16)", who, d->dtype);
  ULB_CHECK(d->page == 16 || d->page == 32 || d->page == 64 || d->page == 128 || d->page == 256, ULB_EUNSUPPORTED,
            "%s: page of %d positions (16, 32, 64, 128 or 256)", who, d->page);
  ULB_CHECK(d->head_dim > 0 && d->head_dim <= 256 && d->head_dim % 8 == 0, ULB_EUNSUPPORTED,
            "%s: head_dim %d (a multiple of 8 up to 256)", who, d->head_dim);
  ULB_CHECK(d->n_head_kv > 0 && d->n_pages > 0 && d->n_seq > 0 && d->max_pages > 0 && d->n_layer >= 0, ULB_EINVAL,
            "%s: cache of %d layers, %d kv heads, %d pages, table %d x %d", who, d->n_layer, d->n_head_kv, d->n_pages,
            d->n_seq, d->max_pages);
  ULB_CHECK((long long)d->max_pages * d->page <= 0x7fffffffll, ULB_EUNSUPPORTED,
            "%s: %d pages of %d positions pass 2^31 - 1 positions", who, d->max_pages, d->page);
  for (long long st : {(long long)d->layer_stride, (long long)d->page_stride, (long long)d->head_stride,
                       (long long)d->pos_stride})
    ULB_CHECK(st >= 0 && st % 8 == 0, ULB_EINVAL, "%s: cache stride %lld is not a multiple of 8 elements", who, st);
  g->n_head_kv = d->n_head_kv;
  g->hd = d->head_dim;
  g->page = d->page;
  g->page_shift = __builtin_ctz((unsigned)d->page);
  g->n_pages = d->n_pages;
  g->n_seq = d->n_seq;
  g->max_pages = d->max_pages;
  g->n_layer = d->n_layer > 0 ? d->n_layer : 1;
  g->pos = d->pos_stride ? d->pos_stride : d->head_dim;
  g->head = d->head_stride ? d->head_stride : g->pos * d->page;
  g->pstride = d->page_stride ? d->page_stride : g->head * d->n_head_kv;
  g->layer = d->layer_stride ? d->layer_stride : g->pstride * d->n_pages;
  ULB_CHECK(g->pos >= d->head_dim, ULB_EINVAL, "%s: positions %lld elements apart hold %d", who, g->pos, d->head_dim);
  return ULB_OK;
}

/* arrays of 32-bit elements (NULL is aligned): a kernel that reads one at an odd address faults */
inline bool words_aligned(std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    if (reinterpret_cast<uintptr_t>(p) & 3) return false;
  return true;
}
#define ULB_ALIGNED16(p) ((reinterpret_cast<uintptr_t>(p) & 15) == 0)
#define ULB_LAUNCH(what, call)                                                 \
  do {                                                                         \
    const cudaError_t _le = (call);                                            \
    if (_le != cudaSuccess) return ::ulb::cuda_error(_le, what, __FILE__, __LINE__); \
  } while (0)

}  // namespace ulb

#ifdef __CUDACC__
namespace ulb {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

/* two values rounded into one 32-bit word, the first in the low half */
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t u);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}

}  // namespace ulb
#endif
