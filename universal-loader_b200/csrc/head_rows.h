/*
 * head_rows.h — rows of heads as head_norm.cu and quant_rows.cu walk them: which elements of a head a lane
 * has, the sums over a head, the rotation of its pairs, and the grid.
 */
#pragma once

#include <algorithm>
#include <cmath>

#include "quant_cache.h"

#ifdef __CUDACC__
namespace ulb {
namespace {

constexpr int kWarps = 8;
constexpr unsigned kAll = 0xffffffffu;

struct HeadArgs {
  const unsigned long long* turn;
  float mscale, eps;
  int half, rot, hd;
  int M, nq, nk, nv; /* heads of a row: q, then k, then v (append) */
  int wpr;           /* warps a row */
  const void *q, *k, *v;
  long long q_row, q_head, k_row, k_head, v_row, v_head;
  const float *wq, *wk; /* NULL (append): not normed */
  void *oq, *ok;
  const int* pos;
  /* gradient */
  const void *gq, *gk;
  float* part; /* [blocks][2][hd] */
  /* quantised cache */
  CacheGeom g;
  const int *seq, *slot, *table;
  unsigned char *kp, *vp;
};

/* four consecutive elements between memory and fp32 registers */
template <typename T, bool VEC>
__device__ __forceinline__ void load4(const T* p, float* v) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_f<T>(p[i]);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    const float2 x = unpack2<T>(a.x), y = unpack2<T>(a.y);
    v[0] = x.x; v[1] = x.y; v[2] = y.x; v[3] = y.y;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store4(T* p, const float* v) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = from_f<T>(v[i]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  }
}
/* sum over the LPH lanes of a head; every lane has it */
template <int LPH>
__device__ __forceinline__ float head_sum(float x) {
#pragma unroll
  for (int o = LPH / 2; o; o >>= 1) x += __shfl_xor_sync(kAll, x, o);
  return x;
}

/*
 * A lane's eight elements of a head are two runs of four at d0 and d1.  Half layout: both sides of four pairs, then eight
 * in a row past rot; interleaved: eight in a row.  So a pair is always in one lane.
 */
struct Place {
  int d0, d1;
  bool on; /* the head has them */
};
template <int LPH, bool HALF>
__device__ __forceinline__ Place place_of(const HeadArgs& a, int lane) {
  const int li = lane % LPH;
  Place p;
  p.d0 = li * 8;
  p.d1 = p.d0 + 4;
  p.on = p.d0 < a.hd;
  if (HALF && p.d0 < a.rot) {
    p.d0 = li * 4;
    p.d1 = p.d0 + (a.rot >> 1);
  }
  return p;
}
/* cosines and sines of the lane's four pairs at a position (1 and 0 past rot), times the factor of what turns */
struct Turn {
  float co[4], si[4];
};
template <bool HALF>
__device__ __forceinline__ void turn_at(const HeadArgs& a, long long pos, const Place& at, Turn* t) {
  const int p0 = HALF ? at.d0 : at.d0 >> 1, n = a.rot >> 1;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    t->co[j] = 1.f;
    t->si[j] = 0.f;
    if (at.on && p0 + j < n) {
      const unsigned long long ph = (unsigned long long)pos * a.turn[p0 + j]; /* rope.cu: modulo one turn */
      float s, c;
      sincospif((float)(int)(ph >> 32) * 4.656612873077393e-10f, &s, &c);
      t->co[j] = c * a.mscale;
      t->si[j] = s * a.mscale;
    }
  }
}
/* sign 1: R y, -1: R^T y */
template <bool HALF>
__device__ __forceinline__ void turn(const Turn& t, float sign, float (&y)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = HALF ? j : 2 * j, k = HALF ? j + 4 : 2 * j + 1;
    const float b = y[i], c = y[k], s = sign * t.si[j];
    y[i] = b * t.co[j] - c * s;
    y[k] = b * s + c * t.co[j];
  }
}

/* the warp's weights of its lanes' elements (NULL: ones) */
__device__ __forceinline__ void lane_weights(const float* w, const Place& at, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = at.on && w ? __ldg(w + (j < 4 ? at.d0 + j : at.d1 + j - 4)) : 1.f;
}

/* the first of a segment's heads that part `part` of a row's warps takes; the segment begins at the row's head `before` */
__device__ __forceinline__ int part_of(int part, int before, int wpr, int hps) {
  const int steps = (before + hps - 1) / hps % wpr;
  return (part >= steps ? part - steps : part - steps + wpr) * hps;
}

/*
 * n heads at x0, `stride` elements apart, of the row that the warp is at: loaded U steps at a time, normed by
 * 1 / sqrt(mean x^2 + eps) and w, turned, and handed to out(head, whether this lane has elements of it, values).
 */
template <typename T, int LPH, bool HALF, int U, typename Load, typename Out>
__device__ __forceinline__ void walk_heads(const HeadArgs& a, const T* x0, long long stride, int n, int first, const Place& at, const Turn& t,
                                           bool normed, const float (&w)[8], bool turns, Load&& load, Out&& out) {
  constexpr int HPS = 32 / LPH;
  const int grp = (threadIdx.x & 31) / LPH;
  const float inv_hd = 1.f / a.hd;
  for (int h0 = first; h0 < n; h0 += a.wpr * HPS * U) {
    float x[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * a.wpr * HPS + grp;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[u][j] = 0.f;
      if (h >= n || !at.on) continue;
      load(x0 + h * stride, x[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h0 + u * a.wpr * HPS >= n) break; /* the whole warp */
      const int h = h0 + u * a.wpr * HPS + grp;
      if (normed) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __fmaf_rn(x[u][j], x[u][j], ss);
        const float f = rsqrtf(__fmaf_rn(head_sum<LPH>(ss), inv_hd, a.eps));
#pragma unroll
        for (int j = 0; j < 8; ++j) x[u][j] *= f * w[j];
      }
      if (turns) turn<HALF>(t, 1.f, x[u]);
      out(h, h < n && at.on, x[u]);
    }
  }
}

/* a grid of whole rows: as many warps a row as it takes to give every SM some, at most one a step of its `steps`; and at
   most `most` blocks, which then walk the rows */
int plan_rows(Ctx* c, HeadArgs& a, int steps, int most) {
  const long long want = (long long)c->n_sm * 32; /* warps */
  int wpr = 1;
  while (wpr < kWarps && wpr < steps && (long long)a.M * wpr < want) wpr *= 2;
  a.wpr = wpr;
  const long long blocks = ((long long)a.M * wpr + kWarps - 1) / kWarps;
  return (int)std::max<long long>(1, std::min<long long>(blocks, most));
}
int lanes_of(int hd) { return hd <= 64 ? 8 : hd <= 128 ? 16 : 32; }
int head_steps(const HeadArgs& a) { return (a.nq + a.nk + a.nv + 32 / lanes_of(a.hd) - 1) / (32 / lanes_of(a.hd)); }

/* what the handle adds, and its limits here */
int rotary(const char* who, const ulb_rope* r, HeadArgs* a) {
  ULB_CHECK(r->hd % 8 == 0 && r->hd <= 256, ULB_EUNSUPPORTED, "%s: head_dim %d (a multiple of 8 up to 256)", who, r->hd);
  ULB_CHECK(!r->half || r->rot % 8 == 0, ULB_EUNSUPPORTED, "%s: rot_dim %d of the half layout (a multiple of 8)", who, r->rot);
  a->turn = r->turn;
  a->mscale = r->mscale;
  a->half = r->half;
  a->rot = r->rot;
  a->hd = r->hd;
  return ULB_OK;
}

/* pointers of elements, weights and positions: aligned to what they hold; wide where all are 16-byte aligned */
bool wide(int eb, std::initializer_list<const void*> rows, long long strides) {
  uintptr_t all = 0;
  for (const void* p : rows) all |= (uintptr_t)p;
  return all % 16 == 0 && strides * eb % 16 == 0;
}
bool element_aligned(int eb, std::initializer_list<const void*> rows) {
  for (const void* p : rows)
    if ((uintptr_t)p % eb) return false;
  return true;
}

}  // namespace
}  // namespace ulb
#endif
