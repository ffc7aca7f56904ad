/*
 * quant_rows.cu — rows written to a cache held in 8 or 4 bits (ulb_quant_append: norms, rotary positions
 * and GGUF's Q8_0 / Q4_1 blocks in one pass) and read back (ulb_quant_read).  The reference's cache is fp32 on the host
 * (src/inference/model.h:49-77).
 *
 * Work.  Memory bounds both: every element is read once and written once.  The rows are walked as head_norm.cu walks
 * them; a group's range is a maximum (and minimum) over the lanes that hold its 32 elements, by shuffles: four lanes, or
 * eight in the half layout, whose lanes hold runs of two groups (so a handle of that layout has to turn the whole head).
 *
 * Measured: 8190 fp16 rows of 32 and 2 x 8 heads of 128 written in 4 bits and read back 66 us, 3.4 TB/s of what both move
 * (51 % of the copy rate; the write alone 57 to 62 us, in 8 bits 59, the read 12 to 13): the instructions of the rotation, the
 * ranges and the codes beside HBM.  30000 rows in 8 bits: 180 us, read back 38.  64 rows: 15 us, the host's two calls.
 */
#include "head_rows.h"

namespace ulb {
namespace {

/* GGUF's own rounding of a group: fp32 d = max |x| / 127, codes round(x (1 / d)), half away from zero; 4 bits:
   d = (max - min) / 15, codes floor((x - min) (1 / d) + 1/2); d and min are kept in 16 bits */
struct Group {
  float lo, id;
  bool bad; /* a value is not finite: the group reads as NaN */
  __half d, m;
};
template <bool Q4>
__device__ __forceinline__ Group group_of(float hi, float lo) {
  Group g;
  g.bad = hi == INFINITY;
  g.lo = lo;
  const float d = __fdiv_rn(Q4 ? __fsub_rn(hi, lo) : hi, Q4 ? 15.f : 127.f);
  g.id = d == 0.f || g.bad ? 0.f : __fdiv_rn(1.f, d);
  g.d = g.bad ? __ushort_as_half(0x7e00) : __float2half_rn(fminf(d, 65504.f));
  g.m = g.bad ? __ushort_as_half(0x7e00) : __float2half_rn(fmaxf(fminf(lo, 65504.f), -65504.f));
  return g;
}
/* codes of four consecutive elements: a byte each, or as they lie in a word of the group's half of a row */
template <bool Q4>
__device__ __forceinline__ uint32_t codes4(const Group& g, const float* x) {
  uint32_t c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (Q4) {
      c[j] = (uint32_t)max(0, min((int)floorf(__fadd_rn(__fmul_rn(__fsub_rn(x[j], g.lo), g.id), 0.5f)), 15));
    } else {
      const float y = __fmul_rn(x[j], g.id), f = floorf(fabsf(y));
      const int n = min((int)f + (__fsub_rn(fabsf(y), f) >= 0.5f ? 1 : 0), 127);
      c[j] = (uint8_t)(y < 0.f ? -n : n);
    }
    if (g.bad) c[j] = 0;
  }
  return Q4 ? c[0] | c[1] << 16 | c[2] << 4 | c[3] << 20 : c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
}
template <bool Q4>
__device__ __forceinline__ void range4(const float* x, float* hi, float* lo) {
  bool odd = false;
  *hi = Q4 ? x[0] : 0.f;
  *lo = x[0];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    *hi = fmaxf(*hi, Q4 ? x[j] : fabsf(x[j]));
    if (Q4) *lo = fminf(*lo, x[j]);
    odd |= !isfinite(x[j]);
  }
  if (odd) *hi = INFINITY;
}
/*
 * A head's eight elements of each lane into a quantised row (NULL: nowhere).  Either both runs follow one another
 * (four lanes a group) or each lies in a group of its own with the runs of seven other lanes (PAIRS: the half layout
 * where rot / 2 is a multiple of 32 and rot all of the head).
 */
template <bool Q4, bool PAIRS>
__device__ __forceinline__ void quantise8(const float (&x)[8], unsigned char* row, int hd, const Place& at) {
  float hi[2], lo[2];
  range4<Q4>(x, &hi[0], &lo[0]);
  range4<Q4>(x + 4, &hi[1], &lo[1]);
  if (!PAIRS) {
    hi[0] = fmaxf(hi[0], hi[1]);
    lo[0] = fminf(lo[0], lo[1]);
  }
#pragma unroll
  for (int r = 0; r < (PAIRS ? 2 : 1); ++r)
#pragma unroll
    for (int o = 1; o < (PAIRS ? 8 : 4); o <<= 1) {
      hi[r] = fmaxf(hi[r], __shfl_xor_sync(kAll, hi[r], o));
      if (Q4) lo[r] = fminf(lo[r], __shfl_xor_sync(kAll, lo[r], o));
    }
  const Group g0 = group_of<Q4>(hi[0], lo[0]), g1 = PAIRS ? group_of<Q4>(hi[1], lo[1]) : g0;
  const uint32_t w0 = codes4<Q4>(g0, x), w1 = codes4<Q4>(g1, x + 4);
  const int i0 = at.d0 >> 5, i1 = at.d1 >> 5; /* groups */
  const bool first = (at.d0 & 31) == 0;       /* the lane that writes a group's scale */
  if (!Q4) {
    if (!row) return;
    if (PAIRS) {
      *reinterpret_cast<uint32_t*>(row + at.d0) = w0;
      *reinterpret_cast<uint32_t*>(row + at.d1) = w1;
    } else {
      *reinterpret_cast<uint2*>(row + at.d0) = make_uint2(w0, w1);
    }
    if (first) {
      *reinterpret_cast<__half*>(row + hd + 2 * i0) = g0.d;
      if (PAIRS) *reinterpret_cast<__half*>(row + hd + 2 * i1) = g1.d;
    }
  } else {
    /* a word holds four elements of two neighbouring groups: those of the group before or after are 32 on */
    const int to = PAIRS && hd > 64 ? 8 : PAIRS ? 0 : 4; /* lanes to the one that has them (0: this one, its other run) */
    uint32_t y0 = w0 << (8 * (i0 & 1)), y1 = w1 << (8 * (i1 & 1));
    if (to == 0) {
      y0 |= y1;
    } else {
      y0 |= __shfl_xor_sync(kAll, y0, to);
      y1 |= __shfl_xor_sync(kAll, y1, to);
    }
    if (!row) return;
    if (PAIRS) {
      if (!(i0 & 1)) *reinterpret_cast<uint32_t*>(row + (i0 >> 1) * 32 + (at.d0 & 31)) = y0;
      if (to != 0 && !(i1 & 1)) *reinterpret_cast<uint32_t*>(row + (i1 >> 1) * 32 + (at.d1 & 31)) = y1;
    } else if (!(i0 & 1)) {
      *reinterpret_cast<uint2*>(row + (i0 >> 1) * 32 + (at.d0 & 31)) = make_uint2(y0, y1);
    }
    if (first) {
      *reinterpret_cast<__half2*>(row + hd / 2 + 4 * i0) = __halves2half2(g0.d, g0.m);
      if (PAIRS) *reinterpret_cast<__half2*>(row + hd / 2 + 4 * i1) = __halves2half2(g1.d, g1.m);
    }
  }
}

/* where row m's K and V go, in bytes from the pools' begin; -1: nowhere */
__device__ __forceinline__ long long slot_place(const HeadArgs& a, int m) {
  const int s = a.seq[m], at = a.slot[m];
  if (s < 0 || s >= a.g.n_seq || at < 0 || (at >> a.g.page_shift) >= a.g.max_pages) return -1;
  const int page = a.table[(long long)s * a.g.max_pages + (at >> a.g.page_shift)];
  return page < 0 || page >= a.g.n_pages ? -1 : page * a.g.pstride + (at & (a.g.page - 1)) * a.g.pos;
}

template <typename TI, bool Q4, int LPH, bool HALF>
__global__ void __launch_bounds__(kWarps * 32, 2) quant_append_kernel(const __grid_constant__ HeadArgs a, int f16, int wide_in, int wide_out) {
  pdl_wait();
  pdl_trigger();
  __shared__ HeadWeights sw;
  const Place at = place_of<LPH, HALF>(a, threadIdx.x & 31);
  const Pairs pairs = pairs_of<HALF>(a, at);
  const float inv_hd = 1.f / a.hd;
  load_weights(a, &sw);
  const int hs = a.hd * (int)sizeof(TI), run = (at.d1 - at.d0) * (int)sizeof(TI);
  Turn t;
  long long place = -1, o_row = 0;
  walk_rows<Eight<TI>, LPH, sizeof(TI) == 4 ? 2 : 4>(
      a, a.nq + a.nk + a.nv, at.on,
      [&](int m) {
        return HeadBase{(const char*)((const TI*)a.q + m * a.q_row + at.d0), (const char*)((const TI*)a.k + m * a.k_row + at.d0) - (long long)a.nq * hs,
                        (const char*)((const TI*)a.v + m * a.v_row + at.d0) - (long long)(a.nq + a.nk) * hs};
      },
      [&](const HeadBase& from, int h, bool mine) {
        Eight<TI> e = zero8<TI>();
        if (mine) {
          const int kind = kind_of(a, h);
          const char* p = (kind == 0 ? from.q : kind == 1 ? from.k : from.v) + (long long)h * hs;
          load_run((const TI*)p, wide_in, &e.r[0]);
          load_run((const TI*)(p + run), wide_in, &e.r[1]);
        }
        return e;
      },
      [&](int m, int pos) {
        turn_at(pairs, pos, a.mscale, &t);
        place = slot_place(a, m);
        o_row = (long long)m * a.nq;
      },
      [&](int h, bool mine, const Eight<TI>& e) {
        float x[8];
        unpack8(e, x);
        const int kind = kind_of(a, h);
        if (__any_sync(kAll, kind != 2)) { /* some of q or k */
          float y[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = x[j];
          if (a.wq || a.wk) { /* the same for all threads */
            float ss = 0.f, w[8], f = 1.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = __fmaf_rn(x[j], x[j], ss);
            ss = head_sum<LPH>(ss);
            if (kind == 0 ? a.wq != nullptr : a.wk != nullptr) f = rsqrt_near(__fmaf_rn(ss, inv_hd, a.eps));
            lane_weights(sw, kind, at, w); /* ones where there are none */
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] *= f * w[j];
          }
          turn<HALF>(t, 1.f, y);
          if (kind != 2) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = y[j];
          }
        }
        if (__any_sync(kAll, kind != 0)) {
          unsigned char* const r = !mine || kind == 0 || place < 0 ? nullptr
                                   : kind == 1 ? a.kp + place + (long long)(h - a.nq) * a.g.head
                                               : a.vp + place + (long long)(h - a.nq - a.nk) * a.g.head;
          quantise8<Q4, HALF>(x, r, a.hd, at);
        }
        if (!mine || kind != 0) return;
        const long long o = (o_row + h) * a.hd;
        if (f16) {
          store4((__half*)a.oq + o + at.d0, wide_out, x);
          store4((__half*)a.oq + o + at.d1, wide_out, x + 4);
        } else {
          store4((__nv_bfloat16*)a.oq + o + at.d0, wide_out, x);
          store4((__nv_bfloat16*)a.oq + o + at.d1, wide_out, x + 4);
        }
      });
}

/* rows read back: a warp a row (or several), a lane eight elements of a head of K or of V at a time */
template <typename T, bool Q4>
__global__ void __launch_bounds__(kWarps * 32) quant_read_kernel(const __grid_constant__ HeadArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int U = 4;
  const int lane = threadIdx.x & 31, gw = blockIdx.x * kWarps + (threadIdx.x >> 5), part = gw % a.wpr, n_rows = gridDim.x * kWarps / a.wpr;
  const int hd = a.g.hd, per2 = 31 - __clz(hd >> 3), units = a.g.n_head_kv << per2; /* of K, and as many of V; head dims are powers of two */
  for (int m = gw / a.wpr; m < a.M; m += n_rows) {
    const long long place = slot_place(a, m);
    for (int i0 = part * 32 + lane; i0 < 2 * units; i0 += a.wpr * 32 * U) {
      uint2 w[U];
      uint32_t sc[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * a.wpr * 32, v = i >= units, r = i - v * units, h = r >> per2, d0 = (r & ((1 << per2) - 1)) * 8, grp = d0 >> 5;
        w[u] = make_uint2(0, 0);
        sc[u] = 0;
        if (place < 0 || i >= 2 * units) continue;
        const unsigned char* row = (v ? a.vp : a.kp) + place + (long long)h * a.g.head;
        w[u] = *reinterpret_cast<const uint2*>(Q4 ? row + (grp >> 1) * 32 + (d0 & 31) : row + d0);
        if (Q4) sc[u] = *reinterpret_cast<const uint32_t*>(row + hd / 2 + 4 * grp);
        else sc[u] = *reinterpret_cast<const uint16_t*>(row + hd + 2 * grp);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * a.wpr * 32, v = i >= units, r = i - v * units, h = r >> per2, d0 = (r & ((1 << per2) - 1)) * 8, grp = d0 >> 5;
        if (i >= 2 * units) break;
        const float2 dm = unpack2<__half>(sc[u]);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t y = j < 4 ? w[u].x : w[u].y;
          if (!Q4) x[j] = (float)(int8_t)(y >> (8 * (j & 3))) * dm.x;
        }
        if constexpr (Q4) { /* two codes at a time as fp16 integers: 0x6400 | n is 1024 + n, 0x6400 | 16 n is 1024 + 16 n */
#pragma unroll
          for (int j = 0; j < 8; j += 4) {
            const uint32_t y = (j < 4 ? w[u].x : w[u].y) >> (8 * (grp & 1));
            const float2 lo = unpack2<__half>((y & 0x000f000fu) | 0x64006400u), hi = unpack2<__half>((y & 0x00f000f0u) | 0x64006400u);
            x[j] = __fmaf_rn(lo.x - 1024.f, dm.x, dm.y);
            x[j + 1] = __fmaf_rn(lo.y - 1024.f, dm.x, dm.y);
            x[j + 2] = __fmaf_rn(__fmaf_rn(hi.x, 0.0625f, -64.f), dm.x, dm.y);
            x[j + 3] = __fmaf_rn(__fmaf_rn(hi.y, 0.0625f, -64.f), dm.x, dm.y);
          }
        }
        T* o = (T*)(v ? a.ok : a.oq) + ((long long)m * a.g.n_head_kv + h) * hd + d0;
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<uint4*>(o) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
        } else {
          store4(o, true, x);
          store4(o + 4, true, x + 4);
        }
      }
    }
  }
}

template <typename TI, bool Q4, bool HALF>
int launch_append(Ctx* c, HeadArgs& a, int f16, int wide_in, int wide_out) {
  const int lph = lanes_of(a.hd), blocks = plan_rows(c, a, head_steps(a), c->n_sm * 2);
  auto go = [&](auto kern) -> int {
    ULB_LAUNCH("quant append launch", launch_k(c, kern, dim3(blocks), dim3(kWarps * 32), 0, a, f16, wide_in, wide_out));
    return ULB_OK;
  };
  if (lph == 8) return go(quant_append_kernel<TI, Q4, 8, HALF>);
  if (lph == 16) return go(quant_append_kernel<TI, Q4, 16, HALF>);
  return go(quant_append_kernel<TI, Q4, 32, HALF>);
}
template <typename TI>
int pick_append(Ctx* c, HeadArgs& a, bool q4, int f16, int wide_in, int wide_out) {
  if (q4) return a.half ? launch_append<TI, true, true>(c, a, f16, wide_in, wide_out) : launch_append<TI, true, false>(c, a, f16, wide_in, wide_out);
  return a.half ? launch_append<TI, false, true>(c, a, f16, wide_in, wide_out) : launch_append<TI, false, false>(c, a, f16, wide_in, wide_out);
}

}  // namespace
}  // namespace ulb

using namespace ulb;

extern "C" {

int ulb_quant_row_bytes(const ulb_quant_desc* d, int* out) {
  ULB_CHECK(out, ULB_EINVAL, "ulb_quant_row_bytes: NULL argument");
  CacheGeom g;
  ULB_TRY(quant_geom("ulb_quant_row_bytes", d, &g));
  *out = (int)g.pos;
  return ULB_OK;
}

int ulb_quant_pages(const ulb_quant_desc* d, int n_layer, ulb_cache_desc* out) {
  ULB_CHECK(out, ULB_EINVAL, "ulb_quant_pages: NULL argument");
  CacheGeom g;
  ULB_TRY(quant_geom("ulb_quant_pages", d, &g));
  ULB_CHECK(n_layer > 0, ULB_EINVAL, "ulb_quant_pages: %d layers", n_layer);
  *out = ulb_cache_desc{};
  out->dtype = ULB_TYPE_F16;
  out->n_layer = n_layer;
  out->n_head_kv = d->n_head_kv;
  out->head_dim = (int)g.pos / 2; /* rows are multiples of 16 bytes */
  out->page = d->page;
  out->n_pages = d->n_pages;
  out->n_seq = d->n_seq;
  out->max_pages = d->max_pages;
  return ULB_OK;
}

int ulb_quant_append(ulb_ctx* ctx, const ulb_rope* r, const ulb_quant_desc* d, const ulb_quant_append_args* p) {
  ULB_CHECK(ctx && r && p, ULB_EINVAL, "ulb_quant_append: NULL argument");
  HeadArgs a = {};
  ULB_TRY(quant_geom("ulb_quant_append", d, &a.g));
  ULB_TRY(rotary("ulb_quant_append", r, &a));
  ULB_CHECK(!r->half || r->rot == r->hd, ULB_EUNSUPPORTED, "ulb_quant_append: rot_dim %d of head_dim %d in the half layout (all of the head)", r->rot,
            r->hd);
  ULB_CHECK(r->hd == a.g.hd, ULB_EINVAL, "ulb_quant_append: rotary head_dim %d, cache head_dim %d", r->hd, a.g.hd);
  ULB_CHECK(dtype_bytes(p->in_dtype), ULB_EUNSUPPORTED, "ulb_quant_append: type %d (F32, F16 or BF16)", p->in_dtype);
  ULB_CHECK(p->M >= 0 && p->M <= kMaxRows && p->n_head > 0 && p->n_head <= (1 << 20) && a.g.n_head_kv <= (1 << 20), ULB_EINVAL,
            "ulb_quant_append: %d rows of %d and %d heads", p->M, p->n_head, a.g.n_head_kv);
  ULB_CHECK(p->q_row >= 0 && p->k_row >= 0 && p->v_row >= 0, ULB_EINVAL, "ulb_quant_append: negative stride");
  const bool normed = p->q_weight || p->k_weight;
  ULB_CHECK(!normed || (std::isfinite(p->eps) && p->eps >= kMinEps), ULB_EINVAL, "ulb_quant_append: eps %g", (double)p->eps);
  if (p->M == 0) return ULB_OK;
  ULB_CHECK(p->q && p->k && p->v && p->pos && p->row_seq && p->slot && p->block_table && p->q_out && p->k_pool && p->v_pool, ULB_EINVAL,
            "ulb_quant_append: NULL argument");
  const int eb = dtype_bytes(p->in_dtype);
  ULB_CHECK(element_aligned(eb, {p->q, p->k, p->v}) && element_aligned(2, {p->q_out}), ULB_EINVAL, "ulb_quant_append: unaligned pointer");
  ULB_CHECK(words_aligned({p->pos, p->row_seq, p->slot, p->block_table, p->q_weight, p->k_weight}), ULB_EINVAL,
            "ulb_quant_append: unaligned array of 32-bit elements");
  ULB_CHECK(ULB_ALIGNED16(p->k_pool) && ULB_ALIGNED16(p->v_pool), ULB_EINVAL, "ulb_quant_append: the pools must be 16-byte aligned");
  a.eps = normed ? p->eps : 1.f;
  a.M = p->M;
  a.nq = p->n_head;
  a.nk = a.nv = a.g.n_head_kv;
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.q_head = a.k_head = a.v_head = r->hd;
  a.q_row = p->q_row ? p->q_row : (int64_t)a.nq * r->hd;
  a.k_row = p->k_row ? p->k_row : (int64_t)a.nk * r->hd;
  a.v_row = p->v_row ? p->v_row : (int64_t)a.nv * r->hd;
  a.wq = p->q_weight;
  a.wk = p->k_weight;
  a.oq = p->q_out;
  a.pos = p->pos;
  a.seq = p->row_seq;
  a.slot = p->slot;
  a.table = p->block_table;
  a.kp = (unsigned char*)p->k_pool;
  a.vp = (unsigned char*)p->v_pool;
  Ctx* c = &ctx->c;
  ULB_CUDA(cudaSetDevice(c->device));
  const bool q4 = d->format == ULB_TYPE_Q4_1;
  const int f16 = d->dtype == ULB_TYPE_F16, in = wide(eb, {a.q, a.k, a.v}, a.q_row | a.k_row | a.v_row), out = (uintptr_t)a.oq % 8 == 0;
  switch (p->in_dtype) {
    case ULB_TYPE_F32: return pick_append<float>(c, a, q4, f16, in, out);
    case ULB_TYPE_F16: return pick_append<__half>(c, a, q4, f16, in, out);
    default: return pick_append<__nv_bfloat16>(c, a, q4, f16, in, out);
  }
}

int ulb_quant_read(ulb_ctx* ctx, const ulb_quant_desc* d, int dtype, const void* k, const void* v, const int32_t* table,
                   const int32_t* row_seq, const int32_t* slot, int M, void* k_out, void* v_out) {
  ULB_CHECK(ctx, ULB_EINVAL, "ulb_quant_read: NULL context");
  HeadArgs a = {};
  ULB_TRY(quant_geom("ulb_quant_read", d, &a.g));
  ULB_CHECK(dtype_bytes(dtype), ULB_EUNSUPPORTED, "ulb_quant_read: type %d (F32, F16 or BF16)", dtype);
  ULB_CHECK(M >= 0 && M <= kMaxRows, ULB_EINVAL, "ulb_quant_read: %d rows", M);
  if (M == 0) return ULB_OK;
  ULB_CHECK(k && v && table && row_seq && slot && k_out && v_out, ULB_EINVAL, "ulb_quant_read: NULL argument");
  ULB_CHECK(ULB_ALIGNED16(k) && ULB_ALIGNED16(v) && ULB_ALIGNED16(k_out) && ULB_ALIGNED16(v_out), ULB_EINVAL,
            "ulb_quant_read: the pools and outputs must be 16-byte aligned");
  ULB_CHECK(words_aligned({table, row_seq, slot}), ULB_EINVAL, "ulb_quant_read: unaligned array of int32");
  a.M = M;
  a.kp = (unsigned char*)const_cast<void*>(k);
  a.vp = (unsigned char*)const_cast<void*>(v);
  a.table = table;
  a.seq = row_seq;
  a.slot = slot;
  a.oq = k_out;
  a.ok = v_out;
  Ctx* c = &ctx->c;
  ULB_CUDA(cudaSetDevice(c->device));
  ULB_CHECK(a.g.n_head_kv <= (1 << 20), ULB_EUNSUPPORTED, "ulb_quant_read: %d kv heads", a.g.n_head_kv);
  const int blocks = plan_rows(c, a, (2 * a.g.n_head_kv * (a.g.hd >> 3) + 31) / 32, c->n_sm * 16);
  auto go = [&](auto kern) -> int {
    ULB_LAUNCH("quant read launch", launch_k(c, kern, dim3(blocks), dim3(kWarps * 32), 0, a));
    return ULB_OK;
  };
  const bool q4 = d->format == ULB_TYPE_Q4_1;
  switch (dtype) {
    case ULB_TYPE_F32: return q4 ? go(quant_read_kernel<float, true>) : go(quant_read_kernel<float, false>);
    case ULB_TYPE_F16: return q4 ? go(quant_read_kernel<__half, true>) : go(quant_read_kernel<__half, false>);
    default: return q4 ? go(quant_read_kernel<__nv_bfloat16, true>) : go(quant_read_kernel<__nv_bfloat16, false>);
  }
}

}  // extern "C"

ULB_TRACE_UNIT(quant_rows)
