/*
 * head_rows.h — rows of heads as head_norm.cu and quant_rows.cu walk them: which elements of a head a lane
 * has, the sums over a head, the rotation of its pairs, and the grid.
 */
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "quant_cache.h"

#ifdef __CUDACC__
namespace ulb {
namespace {

constexpr int kWarps = 8;
constexpr unsigned kAll = 0xffffffffu;
constexpr int kMaxRows = 1 << 30; /* rows of a call: a row and the grid's step stay in 32 bits */
constexpr float kMinEps = 1.1754943508222875e-38f; /* the smallest normal number: what a norm divides by is one, too */

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

/* a lane's two runs of four elements as they lie in memory */
template <typename T>
struct Eight {
  using Run = std::conditional_t<sizeof(T) == 4, float4, uint2>;
  Run r[2];
};
template <typename T>
__device__ __forceinline__ void load_run(const T* p, bool wide, typename Eight<T>::Run* r) {
  if (wide) {
    *r = *reinterpret_cast<const typename Eight<T>::Run*>(p);
  } else if constexpr (sizeof(T) == 4) {
    *r = make_float4(p[0], p[1], p[2], p[3]);
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    *r = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
  }
}
template <typename T>
__device__ __forceinline__ void unpack8(const Eight<T>& e, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[4 * i] = e.r[i].x; v[4 * i + 1] = e.r[i].y; v[4 * i + 2] = e.r[i].z; v[4 * i + 3] = e.r[i].w;
    } else {
      const float2 x = unpack2<T>(e.r[i].x), y = unpack2<T>(e.r[i].y);
      v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = y.x; v[4 * i + 3] = y.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ Eight<T> zero8() {
  Eight<T> e;
  if constexpr (sizeof(T) == 4) e.r[0] = e.r[1] = make_float4(0.f, 0.f, 0.f, 0.f);
  else e.r[0] = e.r[1] = make_uint2(0, 0);
  return e;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, bool wide, const float* v) {
  if (!wide) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = from_f<T>(v[i]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  }
}
/* 1 / sqrt(x) of a normal positive x, to 2^-22 */
__device__ __forceinline__ float rsqrt_near(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
/* the frequencies of those pairs (zero: does not turn) and which of them do */
struct Pairs {
  unsigned long long f[4];
  bool turns[4];
};
template <bool HALF>
__device__ __forceinline__ Pairs pairs_of(const HeadArgs& a, const Place& at) {
  const int p0 = HALF ? at.d0 : at.d0 >> 1;
  Pairs p;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    p.turns[j] = at.on && p0 + j < (a.rot >> 1);
    p.f[j] = p.turns[j] ? a.turn[p0 + j] : 0;
  }
  return p;
}
__device__ __forceinline__ void turn_at(const Pairs& p, long long pos, float mscale, Turn* t) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned long long ph = (unsigned long long)pos * p.f[j]; /* rope.cu: modulo one turn */
    float s, c;
    sincospif((float)(int)(ph >> 32) * 4.656612873077393e-10f, &s, &c);
    t->co[j] = p.turns[j] ? c * mscale : 1.f;
    t->si[j] = p.turns[j] ? s * mscale : 0.f;
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

/* weights of a block's heads, q's, k's and ones, in shared memory */
struct HeadWeights {
  float w[3][256];
};
__device__ __forceinline__ void load_weights(const HeadArgs& a, HeadWeights* s) {
  for (int i = threadIdx.x; i < 256; i += kWarps * 32) {
    s->w[0][i] = a.wq && i < a.hd ? a.wq[i] : 1.f;
    s->w[1][i] = a.wk && i < a.hd ? a.wk[i] : 1.f;
    s->w[2][i] = 1.f;
  }
  __syncthreads();
}
__device__ __forceinline__ void lane_weights(const HeadWeights& s, int kind, const Place& at, float (&v)[8]) {
  const float4 x = *reinterpret_cast<const float4*>(&s.w[kind][at.d0 & 255]), y = *reinterpret_cast<const float4*>(&s.w[kind][at.d1 & 255]);
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
}

/*
 * The heads of the warp's rows in steps of 32 / LPH heads, U steps (a batch) at a time; while a batch is worked on, the
 * next one's loads are under way, past the end of the row too.  from(m) gives what load(from, h, mine) needs to find head h
 * of row m and return what a lane keeps of it (zeros where it is not `mine`), row(m, position) is called before the row's
 * first batch, work(h, mine, kept) for every step by the whole warp.
 */
template <typename Kept, int LPH, int U, typename From, typename Load, typename Row, typename Work>
__device__ __forceinline__ void walk_rows(const HeadArgs& a, int heads, bool on, From&& from, Load&& load, Row&& row, Work&& work) {
  constexpr int HPS = 32 / LPH;
  const int gw = blockIdx.x * kWarps + (threadIdx.x >> 5), part = gw % a.wpr, lead = part * HPS + (threadIdx.x & 31) / LPH;
  const int n_rows = gridDim.x * kWarps / a.wpr, per = HPS * a.wpr;
  int m = gw / a.wpr, pos = 0, h = lead; /* h: the lane's head in the first step of the batch */
  if (m >= a.M) return;
  Kept now[U], next[U];
  auto src = from(m);
  auto fetch = [&](int h, Kept (&k)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = load(src, h + u * per, on && h + u * per < heads);
  };
  fetch(h, now);
  pos = a.pos[m];
  while (true) {
    if (h == lead) row(m, pos);
    int m2 = m, h2 = h + per * U;
    if (h2 - lead + part * HPS >= heads) { /* the same for the whole warp */
      h2 = lead;
      m2 += n_rows;
      if (m2 < a.M) {
        src = from(m2);
        pos = a.pos[m2];
      }
    }
    if (m2 < a.M) fetch(h2, next);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = h + u * per;
      if (x - lead + part * HPS >= heads) break; /* the whole warp */
      work(x, on && x < heads, now[u]);
    }
    if (m2 >= a.M) return;
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = next[u];
    m = m2;
    h = h2;
  }
}

/* where the q and k (and v) heads of a row are, as addresses of a lane's first run less what comes before the kind's first
   head, so that head h is at base + h stride; strides in bytes */
struct HeadBase {
  const char *q, *k, *v;
};
/* 0: q, 1: k, 2: v */
__device__ __forceinline__ int kind_of(const HeadArgs& a, int h) { return h < a.nq ? 0 : h < a.nq + a.nk ? 1 : 2; }

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
