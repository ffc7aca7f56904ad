/*
 * quant_cache.h — the layout of a cache held in 8 or 4 bits (ulb_quant_desc), checked once, for the
 * kernels that write and read it (head_norm.cu) and attend it (quant_attention.cu).
 */
#pragma once

#include "paged_ops.h"

namespace ulb {

constexpr int kGroup = 32; /* elements that share a scale */

/* bytes of a row: codes and scales, and what a row takes */
constexpr int quant_code_bytes(bool q4, int hd) { return q4 ? hd / 2 : hd; }
constexpr int quant_used_bytes(bool q4, int hd) { return quant_code_bytes(q4, hd) + hd / kGroup * (q4 ? 4 : 2); }
constexpr int quant_row_bytes(bool q4, int hd) { return (quant_used_bytes(q4, hd) + 15) / 16 * 16; }

/* the geometry of a quantised cache as a CacheGeom whose strides count bytes */
inline int quant_geom(const char* who, const ulb_quant_desc* d, CacheGeom* g) {
  ULB_CHECK(d, ULB_EINVAL, "%s: cache description is NULL", who);
  ULB_CHECK(d->format == ULB_TYPE_Q8_0 || d->format == ULB_TYPE_Q4_1, ULB_EUNSUPPORTED, "%s: cache format %d (Q8_0 or Q4_1)", who,
            d->format);
  ULB_CHECK(d->dtype == ULB_TYPE_F16 || d->dtype == ULB_TYPE_BF16, ULB_EUNSUPPORTED, "%s: type %d (F16 or BF16)", who, d->dtype);
  ULB_CHECK(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256, ULB_EUNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", who,
            d->head_dim);
  ULB_CHECK(d->page == 16 || d->page == 32 || d->page == 64 || d->page == 128 || d->page == 256, ULB_EUNSUPPORTED,
            "%s: page of %d positions (16, 32, 64, 128 or 256)", who, d->page);
  ULB_CHECK(d->n_head_kv > 0 && d->n_pages > 0 && d->n_seq > 0 && d->max_pages > 0, ULB_EINVAL,
            "%s: cache of %d kv heads, %d pages, table %d x %d", who, d->n_head_kv, d->n_pages, d->n_seq, d->max_pages);
  ULB_CHECK((long long)d->max_pages * d->page <= 0x7fffffffll, ULB_EUNSUPPORTED, "%s: %d pages of %d positions pass 2^31 - 1 positions",
            who, d->max_pages, d->page);
  g->n_head_kv = d->n_head_kv;
  g->hd = d->head_dim;
  g->page = d->page;
  g->page_shift = __builtin_ctz((unsigned)d->page);
  g->n_pages = d->n_pages;
  g->n_seq = d->n_seq;
  g->max_pages = d->max_pages;
  g->n_layer = 1;
  g->pos = quant_row_bytes(d->format == ULB_TYPE_Q4_1, d->head_dim);
  g->head = g->pos * d->page;
  g->pstride = g->head * d->n_head_kv;
  g->layer = g->pstride * d->n_pages;
  return ULB_OK;
}

}  // namespace ulb
