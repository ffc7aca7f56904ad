/*
 * rope.cu — rotary positions as an operator of its own: both pair layouts, part of the head,
 * the usual context scalings, forward and inverse, alone (ulb_rope_apply) or fused with the
 * append of K and V rows to the pages of a cache (ulb_rope_append).  The model forward keeps
 * its own fused form (epilogue.cuh: interleaved, unscaled, from a table of positions);
 * src/shaders/rope.glsl:50-74 of the reference rotates at position 0 only.
 *
 * Angles.  Pair i of a row at position p turns by p f_i.  In fp32 that product is off by
 * p f_i 2^-24 radians (0.008 at p = 131072), so the handle keeps each frequency as the 64-bit
 * fraction F_i = frac(f_i / 2 pi) 2^64 of a turn.  p F_i mod 2^64 is then the angle modulo one
 * turn, exact but for p 2^-65 turns, whatever the sign and size of the int32 position; its top
 * 32 bits, read as a signed number, are the angle in (-pi, pi] for sincospif.  The integer
 * product costs a few instructions, a table of positions would cost 8 bytes a pair and a bound.
 *
 * Work.  One pass: every element is read once and written once, so HBM bounds large calls and
 * launch latency small ones.  A thread owns one unit of a head: E consecutive elements (E / 2
 * interleaved pairs), or the two runs of E elements that form E pairs of the half layout, or E
 * elements past rot_dim that pass through.  It computes the unit's sines once and applies them to
 * HPT heads of the row, all of whose loads are in flight before the first is used.
 * Measured: 16381 fp32 rows of 40 heads of 128 (671 MB) 111 us, 94 % of the copy rate; append of 1024
 * fp32 rows of 80 heads of 128 into bf16 (63 MB) 15.3 us; of 8 rows 3.7 us.
 */
#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

#include "paged_ops.h"

namespace ulb {
namespace {

struct RopeArgs {
  const unsigned long long* turn; /* F_i of the rot / 2 pairs */
  float mscale, sign;
  int half, rot, hd;
  int M, rows_blk;
  int n_units, n_pair_units, n_groups; /* units a head, those of them that rotate, head groups a row */
  int n_head;                          /* heads rotated into `out` (append: q heads) */
  const void *x, *k, *v;
  long long x_row, x_head, k_row, v_row, o_row, o_head;
  void* out;
  const int *pos, *seq, *slot, *table; /* append: seq, slot, table */
  void *kp, *vp;
  CacheGeom g;
};

/* E elements between memory and fp32 registers (E = 8 or 4: whole 8- or 16-byte words) */
template <typename T, int E>
__device__ __forceinline__ void load_e(const T* p, float (&v)[E]) {
  if constexpr (E == 1) {
    v[0] = to_f<T>(*p);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const float4 a = *reinterpret_cast<const float4*>(p + i);
      v[i] = a.x; v[i + 1] = a.y; v[i + 2] = a.z; v[i + 3] = a.w;
    }
  } else {
    uint32_t w[E / 2];
    if constexpr (E == 8) {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    } else {
      const uint2 a = *reinterpret_cast<const uint2*>(p);
      w[0] = a.x; w[1] = a.y;
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 f = unpack2<T>(w[i]);
      v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
  }
}
template <typename T, int E>
__device__ __forceinline__ void store_e(T* p, const float (&v)[E]) {
  if constexpr (E == 1) {
    *p = from_f<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < E; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
    uint32_t w[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    if constexpr (E == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
}

/*
 * A unit is two runs of E elements at offsets d0 and d1 = d0 + rot / 2 (half layout) or one run
 * at d0 (interleaved, pass through); E = 1 takes a single pair of either layout as two runs of
 * one element.
 */
template <typename TI, typename TO, int E, int HPT, bool APPEND>
__global__ void __launch_bounds__(256) rope_kernel(RopeArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int NC = E == 1 ? 1 : E; /* sines a unit needs at most */
  const int per_row = a.n_units * a.n_groups;
  const int row0 = blockIdx.x * a.rows_blk;
  const int n_rows = min(a.rows_blk, a.M - row0);
  for (int t = threadIdx.x; t < n_rows * per_row; t += blockDim.x) {
    const int rr = t / per_row, rest = t - rr * per_row;
    const int grp = rest / a.n_units, u = rest - grp * a.n_units;
    const long long m = row0 + rr;
    const bool turns = u < a.n_pair_units;
    const bool two = turns && (a.half || E == 1);
    int d0, d1 = 0;
    if (!turns) {
      d0 = a.rot + (u - a.n_pair_units) * E;
    } else if (a.half) {
      d0 = u * E;
      d1 = d0 + (a.rot >> 1);
    } else {
      d0 = E == 1 ? 2 * u : u * E;
      d1 = d0 + 1;
    }
    /* every head's loads first */
    float x0[HPT][E], x1[HPT][E];
    const int h0 = grp * HPT;
    const int n_all = APPEND ? a.n_head + 2 * a.g.n_head_kv : a.n_head;
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
      const int h = h0 + i;
      if (h >= n_all) continue;
      const TI* p;
      if (!APPEND || h < a.n_head)
        p = (const TI*)a.x + m * a.x_row + (long long)h * a.x_head;
      else if (h < a.n_head + a.g.n_head_kv)
        p = (const TI*)a.k + m * a.k_row + (long long)(h - a.n_head) * a.hd;
      else
        p = (const TI*)a.v + m * a.v_row + (long long)(h - a.n_head - a.g.n_head_kv) * a.hd;
      load_e<TI, E>(p + d0, x0[i]);
      if (two) load_e<TI, E>(p + d1, x1[i]);
    }
    float co[NC], si[NC];
    if (turns) {
      const long long pos = a.pos[m];
      const int n_pairs = a.half || E == 1 ? E : E / 2, p0 = a.half || E == 1 ? u * E : u * (E / 2);
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        if (j >= n_pairs) break;
        const unsigned long long ph = (unsigned long long)pos * a.turn[p0 + j];
        const float half_turns = (float)(int)(ph >> 32) * 4.656612873077393e-10f; /* 2^-31: the angle / pi */
        sincospif(half_turns, &si[j], &co[j]);
        si[j] *= a.mscale * a.sign;
        co[j] *= a.mscale;
      }
    }
    TO *kd = nullptr, *vd = nullptr;
    if (APPEND && h0 + HPT > a.n_head) {
      const int s = a.seq[m], at = a.slot[m];
      if (s >= 0 && s < a.g.n_seq && at >= 0 && (at >> a.g.page_shift) < a.g.max_pages) {
        const int page = a.table[(long long)s * a.g.max_pages + (at >> a.g.page_shift)];
        if (page >= 0 && page < a.g.n_pages) {
          const long long off = page * a.g.pstride + (at & (a.g.page - 1)) * a.g.pos;
          kd = (TO*)a.kp + off;
          vd = (TO*)a.vp + off;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
      const int h = h0 + i;
      if (h >= n_all) continue;
      TO* p;
      bool rot = turns;
      if (!APPEND || h < a.n_head) {
        p = (TO*)a.out + m * a.o_row + (long long)h * a.o_head;
      } else if (h < a.n_head + a.g.n_head_kv) {
        p = kd ? kd + (h - a.n_head) * a.g.head : nullptr;
      } else {
        p = vd ? vd + (h - a.n_head - a.g.n_head_kv) * a.g.head : nullptr;
        rot = false;
      }
      if (!p) continue;
      if (rot) {
        if (two) {
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const float b = x0[i][j], c = x1[i][j];
            x0[i][j] = b * co[j] - c * si[j];
            x1[i][j] = b * si[j] + c * co[j];
          }
        } else if constexpr (E > 1) {
#pragma unroll
          for (int j = 0; j < E / 2; ++j) {
            const float b = x0[i][2 * j], c = x0[i][2 * j + 1];
            x0[i][2 * j] = b * co[j] - c * si[j];
            x0[i][2 * j + 1] = b * si[j] + c * co[j];
          }
        }
      }
      store_e<TO, E>(p + d0, x0[i]);
      if (two) store_e<TO, E>(p + d1, x1[i]);
    }
  }
}

template <typename TI, typename TO, int E, int HPT, bool APPEND>
int launch_rope(Ctx* c, RopeArgs& a) {
  const int heads = APPEND ? a.n_head + 2 * a.g.n_head_kv : a.n_head;
  const int rest = a.hd - a.rot;
  a.n_pair_units = a.half || E == 1 ? a.rot / 2 / E : a.rot / E;
  a.n_units = a.n_pair_units + rest / E;
  a.n_groups = (heads + HPT - 1) / HPT;
  const long long per_row = (long long)a.n_units * a.n_groups;
  ULB_CHECK(per_row <= (1 << 24), ULB_EUNSUPPORTED, "rope: %d heads of %d elements a row", heads, a.hd);
  a.rows_blk = (int)std::max<long long>(1, 256 / per_row);
  const long long blocks = ((long long)a.M + a.rows_blk - 1) / a.rows_blk;
  const int threads = (int)std::min<long long>(256, (std::min<long long>(a.M, a.rows_blk) * per_row + 31) / 32 * 32);
  ULB_LAUNCH("rope launch", launch_k(c, rope_kernel<TI, TO, E, HPT, APPEND>, dim3((unsigned)blocks), dim3(threads), 0, a));
  return ULB_OK;
}

/* the widest unit that the head split, the strides and the pointers allow */
template <typename TI, typename TO, bool APPEND>
int pick_rope(Ctx* c, RopeArgs& a) {
  long long all = a.x_row | a.x_head | a.o_row | a.o_head | a.hd | (a.half ? a.rot / 2 : a.rot) | (a.hd - a.rot);
  uintptr_t in = (uintptr_t)a.x, out = (uintptr_t)a.out;
  if (APPEND) {
    all |= a.k_row | a.v_row;
    in |= (uintptr_t)a.k | (uintptr_t)a.v;
  }
  const int heads = APPEND ? a.n_head + 2 * a.g.n_head_kv : a.n_head;
  auto fits = [&](int e) {
    return all % e == 0 && in % std::min<size_t>(16, e * sizeof(TI)) == 0 && out % std::min<size_t>(16, e * sizeof(TO)) == 0;
  };
  /* 16 bytes a load (32 a thread, f32 in units of eight, measured 117 us where units of four took 111:
     16381 rows of 40 heads), and several heads a thread once that still fills the device: one pass
     of sines for all of them and as many loads in flight.  1024 rows of 80 heads of 128 (fp32): two heads a
     thread 15.2 us, four 17.8, one 17.6; 16381 rows of 40 take four.  The bounds lie between those sizes and
     are not measured nearer; 16-bit rows follow the same rule. */
  constexpr int W = sizeof(TI) == 4 ? 4 : 8;
  if (fits(W)) {
    const long long full = (long long)c->n_sm * 2048, units = (long long)a.M * heads * (a.hd / W);
    if (units >= 32 * full) return launch_rope<TI, TO, W, 4, APPEND>(c, a);
    if (units >= 4 * full) return launch_rope<TI, TO, W, 2, APPEND>(c, a);
    return launch_rope<TI, TO, W, 1, APPEND>(c, a);
  }
  if (W == 8 && fits(4)) return launch_rope<TI, TO, 4, 2, APPEND>(c, a);
  return launch_rope<TI, TO, 1, 1, APPEND>(c, a);
}

}  // namespace
}  // namespace ulb

using namespace ulb;

static const long double kTwoPi = 6.283185307179586476925286766559005768L;
/* the (fractional) pair that makes t turns over L positions */
static long double pair_with_turns(long double t, long double rot, long double L, long double base) {
  return rot * logl(L / (kTwoPi * t)) / (2.0L * logl(base));
}

extern "C" {

int ulb_rope_create(ulb_ctx* ctx, const ulb_rope_desc* d, const float* ff, ulb_rope** out) {
  ULB_CHECK(ctx && d && out, ULB_EINVAL, "ulb_rope_create: NULL argument");
  *out = nullptr;
  ULB_CHECK(d->head_dim > 0 && d->head_dim <= 1024 && d->rot_dim > 0 && d->rot_dim % 2 == 0 && d->rot_dim <= d->head_dim,
            ULB_EINVAL, "ulb_rope_create: rot_dim %d of head_dim %d (even, at most 1024)", d->rot_dim, d->head_dim);
  ULB_CHECK(d->layout == ULB_ROPE_INTERLEAVED || d->layout == ULB_ROPE_HALF, ULB_EINVAL, "ulb_rope_create: layout %d", d->layout);
  ULB_CHECK(d->scaling >= ULB_ROPE_NONE && d->scaling <= ULB_ROPE_WAVELENGTH, ULB_EINVAL, "ulb_rope_create: scaling %d", d->scaling);
  ULB_CHECK(std::isfinite(d->base) && d->base > 1.0, ULB_EINVAL, "ulb_rope_create: base %g", d->base);
  ULB_CHECK(std::isfinite(d->attn_scale) && d->attn_scale >= 0, ULB_EINVAL, "ulb_rope_create: attn_scale %g", d->attn_scale);
  if (d->scaling != ULB_ROPE_NONE)
    ULB_CHECK(std::isfinite(d->factor) && d->factor > 0, ULB_EINVAL, "ulb_rope_create: factor %g", d->factor);
  if (d->scaling == ULB_ROPE_NTK)
    ULB_CHECK(d->rot_dim > 2, ULB_EINVAL, "ulb_rope_create: NTK scaling of a single pair");
  if (d->scaling == ULB_ROPE_YARN)
    ULB_CHECK(d->orig_len > 0 && d->beta_fast > 0 && d->beta_slow > 0 && std::isfinite(d->orig_len) &&
                  std::isfinite(d->beta_fast) && std::isfinite(d->beta_slow),
              ULB_EINVAL, "ulb_rope_create: YARN with orig_len %g, beta_fast %g, beta_slow %g", d->orig_len, d->beta_fast, d->beta_slow);
  if (d->scaling == ULB_ROPE_WAVELENGTH)
    ULB_CHECK(d->orig_len > 0 && d->low_freq > 0 && d->high_freq > d->low_freq && std::isfinite(d->orig_len) &&
                  std::isfinite(d->high_freq),
              ULB_EINVAL, "ulb_rope_create: WAVELENGTH with orig_len %g, low_freq %g, high_freq %g", d->orig_len, d->low_freq, d->high_freq);
  const int n = d->rot_dim / 2;
  for (int i = 0; ff && i < n; ++i)
    ULB_CHECK(std::isfinite(ff[i]) && ff[i] > 0, ULB_EINVAL, "ulb_rope_create: freq_factors[%d] = %g", i, (double)ff[i]);

  long double base = d->base, m = 1.0L;
  const long double f = d->scaling == ULB_ROPE_NONE ? 1.0L : (long double)d->factor, rot = d->rot_dim, L = d->orig_len;
  if (d->scaling == ULB_ROPE_NTK) base *= powl(f, rot / (rot - 2.0L));
  long double lo = 0, hi = 0;
  if (d->scaling == ULB_ROPE_YARN) {
    lo = floorl(pair_with_turns(d->beta_fast, rot, L, base));
    if (lo < 0) lo = 0;
    hi = ceill(pair_with_turns(d->beta_slow, rot, L, base));
    if (hi > rot - 1) hi = rot - 1;
    m = 0.1L * logl(f) + 1.0L;
  }
  unsigned long long h_turn[512];
  for (int i = 0; i < n; ++i) {
    long double w = powl(base, -2.0L * i / rot);
    if (ff) w /= ff[i];
    if (d->scaling == ULB_ROPE_LINEAR) {
      w /= f;
    } else if (d->scaling == ULB_ROPE_YARN) {
      const long double ramp = (i - lo) / (hi - lo > 0.001L ? hi - lo : 0.001L);
      const long double r = ramp < 0 ? 0.0L : ramp > 1 ? 1.0L : ramp;
      w = w * (1.0L - r) + w / f * r;
    } else if (d->scaling == ULB_ROPE_WAVELENGTH) {
      const long double wave = kTwoPi / w;
      if (wave > L / d->low_freq) {
        w /= f;
      } else if (wave >= L / d->high_freq) {
        const long double x = (L / wave - d->low_freq) / ((long double)d->high_freq - d->low_freq);
        w = (1.0L - x) * w / f + x * w;
      }
    }
    const long double t = w / kTwoPi;
    long double scaled = roundl((t - floorl(t)) * 18446744073709551616.0L);
    h_turn[i] = scaled >= 18446744073709551616.0L ? 0ull : (unsigned long long)scaled;
  }
  Ctx* c = &ctx->c;
  ULB_CUDA(cudaSetDevice(c->device));
  std::unique_ptr<ulb_rope> r(new (std::nothrow) ulb_rope);
  ULB_CHECK(r, ULB_ENOMEM, "ulb_rope_create: host allocation");
  r->owner = ctx;
  r->hd = d->head_dim;
  r->rot = d->rot_dim;
  r->half = d->layout == ULB_ROPE_HALF;
  r->mscale = (float)(d->attn_scale > 0 ? (long double)d->attn_scale : m);
  ULB_TRY(dev_alloc(c, (void**)&r->turn, n * sizeof(unsigned long long)));
  cudaError_t e = cudaMemcpyAsync(r->turn, h_turn, n * sizeof(unsigned long long), cudaMemcpyHostToDevice, c->stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(c->stream); /* h_turn is on this stack */
  if (e != cudaSuccess) {
    dev_free(c, r->turn, n * sizeof(unsigned long long));
    return cuda_error(e, "ulb_rope_create", __FILE__, __LINE__);
  }
  *out = r.release();
  return ULB_OK;
}

int ulb_rope_free(ulb_rope* r) {
  if (!r) return ULB_OK;
  Ctx* c = &r->owner->c;
  cudaSetDevice(c->device);
  dev_free(c, r->turn, r->rot / 2 * sizeof(unsigned long long));
  delete r;
  return ULB_OK;
}

int ulb_rope_apply(ulb_ctx* ctx, const ulb_rope* r, int dtype, const void* x, int64_t x_row, int64_t x_head,
                   const int32_t* pos, int M, int n_head, int inverse, void* out, int64_t out_row, int64_t out_head) {
  ULB_CHECK(ctx && r, ULB_EINVAL, "ulb_rope_apply: NULL argument");
  ULB_CHECK(dtype_bytes(dtype), ULB_EUNSUPPORTED, "ulb_rope_apply: type %d (F32, F16 or BF16)", dtype);
  ULB_CHECK(M >= 0 && n_head > 0, ULB_EINVAL, "ulb_rope_apply: %d rows of %d heads", M, n_head);
  ULB_CHECK(x_row >= 0 && x_head >= 0 && out_row >= 0 && out_head >= 0, ULB_EINVAL, "ulb_rope_apply: negative stride");
  if (M == 0) return ULB_OK;
  ULB_CHECK(x && pos && out, ULB_EINVAL, "ulb_rope_apply: NULL argument");
  const int eb = dtype_bytes(dtype);
  ULB_CHECK((uintptr_t)x % eb == 0 && (uintptr_t)out % eb == 0 && (uintptr_t)pos % 4 == 0, ULB_EINVAL, "ulb_rope_apply: unaligned pointer");
  RopeArgs a = {};
  a.turn = r->turn;
  a.mscale = r->mscale;
  a.sign = inverse ? -1.f : 1.f;
  a.half = r->half;
  a.rot = r->rot;
  a.hd = r->hd;
  a.M = M;
  a.n_head = n_head;
  a.x = x;
  a.out = out;
  a.pos = pos;
  a.x_head = x_head ? x_head : r->hd;
  a.x_row = x_row ? x_row : a.x_head * n_head;
  a.o_head = out_head ? out_head : r->hd;
  a.o_row = out_row ? out_row : a.o_head * n_head;
  ULB_CHECK(x != out || (a.x_head == a.o_head && a.x_row == a.o_row), ULB_EINVAL, "ulb_rope_apply: in place with other strides");
  Ctx* c = &ctx->c;
  ULB_CUDA(cudaSetDevice(c->device));
  switch (dtype) {
    case ULB_TYPE_F32: return pick_rope<float, float, false>(c, a);
    case ULB_TYPE_F16: return pick_rope<__half, __half, false>(c, a);
    default: return pick_rope<__nv_bfloat16, __nv_bfloat16, false>(c, a);
  }
}

int ulb_rope_append(ulb_ctx* ctx, const ulb_rope* r, const ulb_cache_desc* cache, int in_dtype, const void* q,
                    int64_t q_row, const void* k, int64_t k_row, const void* v, int64_t v_row, int n_head,
                    const int32_t* pos, const int32_t* row_seq, const int32_t* slot, const int32_t* table, int M,
                    void* q_out, void* k_pool, void* v_pool) {
  ULB_CHECK(ctx && r, ULB_EINVAL, "ulb_rope_append: NULL argument");
  RopeArgs a = {};
  ULB_TRY(cache_geom("ulb_rope_append", cache, &a.g));
  ULB_CHECK(dtype_bytes(in_dtype), ULB_EUNSUPPORTED, "ulb_rope_append: type %d (F32, F16 or BF16)", in_dtype);
  ULB_CHECK(r->hd == a.g.hd, ULB_EINVAL, "ulb_rope_append: rotary head_dim %d, cache head_dim %d", r->hd, a.g.hd);
  ULB_CHECK(M >= 0 && n_head > 0, ULB_EINVAL, "ulb_rope_append: %d rows of %d heads", M, n_head);
  ULB_CHECK(q_row >= 0 && k_row >= 0 && v_row >= 0, ULB_EINVAL, "ulb_rope_append: negative stride");
  if (M == 0) return ULB_OK;
  ULB_CHECK(q && k && v && pos && row_seq && slot && table && q_out && k_pool && v_pool, ULB_EINVAL, "ulb_rope_append: NULL argument");
  const int eb = dtype_bytes(in_dtype);
  ULB_CHECK((uintptr_t)q % eb == 0 && (uintptr_t)k % eb == 0 && (uintptr_t)v % eb == 0 && (uintptr_t)q_out % 2 == 0, ULB_EINVAL,
            "ulb_rope_append: unaligned pointer");
  ULB_CHECK(words_aligned({pos, row_seq, slot, table}), ULB_EINVAL, "ulb_rope_append: unaligned array of int32");
  ULB_CHECK(ULB_ALIGNED16(k_pool) && ULB_ALIGNED16(v_pool), ULB_EINVAL, "ulb_rope_append: the pools must be 16-byte aligned");
  a.turn = r->turn;
  a.mscale = r->mscale;
  a.sign = 1.f;
  a.half = r->half;
  a.rot = r->rot;
  a.hd = r->hd;
  a.M = M;
  a.n_head = n_head;
  a.x = q;
  a.k = k;
  a.v = v;
  a.x_head = a.o_head = r->hd;
  a.x_row = q_row ? q_row : (int64_t)n_head * r->hd;
  a.k_row = k_row ? k_row : (int64_t)a.g.n_head_kv * r->hd;
  a.v_row = v_row ? v_row : (int64_t)a.g.n_head_kv * r->hd;
  a.o_row = (int64_t)n_head * r->hd;
  a.out = q_out;
  a.pos = pos;
  a.seq = row_seq;
  a.slot = slot;
  a.table = table;
  a.kp = k_pool;
  a.vp = v_pool;
  Ctx* c = &ctx->c;
  ULB_CUDA(cudaSetDevice(c->device));
  if (cache->dtype == ULB_TYPE_F16) switch (in_dtype) {
      case ULB_TYPE_F32: return pick_rope<float, __half, true>(c, a);
      case ULB_TYPE_F16: return pick_rope<__half, __half, true>(c, a);
      default: return pick_rope<__nv_bfloat16, __half, true>(c, a);
    }
  switch (in_dtype) {
    case ULB_TYPE_F32: return pick_rope<float, __nv_bfloat16, true>(c, a);
    case ULB_TYPE_F16: return pick_rope<__half, __nv_bfloat16, true>(c, a);
    default: return pick_rope<__nv_bfloat16, __nv_bfloat16, true>(c, a);
  }
}

}  // extern "C"

ULB_TRACE_UNIT(rope)
