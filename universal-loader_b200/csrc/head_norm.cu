/*
 * head_norm.cu — RMS norms of the q and k heads with their rotary positions in one pass
 * (ulb_norm_rope_apply), their gradient (ulb_norm_rope_grad), and the same rows written to a cache held
 * in 8 or 4 bits (ulb_quant_append) and read back (ulb_quant_read).  The reference normalises whole rows
 * only (src/shaders/rmsnorm.glsl), and its cache is fp32 on the host (src/inference/model.h:49-77).
 *
 * Mathematics.  With f = 1 / sqrt(mean x^2 + eps), n = x f and g = R^T dy (R^T turns by the negative angle):
 *   y = R (w n),   dx = f (w g - n mean(w g n)),   dw = sum over rows and heads of g n.
 * mean(w g n) = f mean(w g x), so both sums of a head, x^2 and w g x, are taken in one pass.
 *
 * Work.  Memory bounds it: every element is read once and written once (gradient: two reads).  A lane
 * owns eight consecutive elements of a head and 8, 16 or 32 lanes a head, so the sums are shuffles, and the
 * other element of a half-layout pair is the same register of another lane.  A warp keeps to one row, whose
 * sines it computes once for all its heads; the weights stay in registers over the rows.  When there are
 * few rows, several warps share the heads of one.
 */
#include <algorithm>
#include <cmath>

#include "quant_cache.h"

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

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f<T>(p[i]);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_f<T>(v[i]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  }
}
/* sum over the LPH lanes of a head; every lane has it */
template <int LPH>
__device__ __forceinline__ float head_sum(float x) {
#pragma unroll
  for (int o = LPH / 2; o; o >>= 1) x += __shfl_xor_sync(kAll, x, o);
  return x;
}

/* how a lane's eight elements turn at a position: cosines and sines of its pairs (1 and 0 past rot), for the half
   layout the sine's sign on this side of the pair, and the lane that holds the other side */
struct Turn {
  float co[8], si[8];
  int other;
};
template <int LPH>
__device__ __forceinline__ void turn_at(const HeadArgs& a, long long pos, int d0, int lane, Turn* t) {
  const int hr = a.rot >> 1;
  const bool first = d0 < hr, turns = d0 < a.rot;
  const int p0 = a.half ? (first ? d0 : d0 - hr) : d0 >> 1;
  t->other = lane;
  if (a.half && turns) t->other = (lane & ~(LPH - 1)) + ((first ? d0 + hr : d0 - hr) >> 3);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    t->co[j] = 1.f;
    t->si[j] = 0.f;
    if (j >= 4 && !a.half) continue;
    if (turns && p0 + j < hr) {
      const unsigned long long ph = (unsigned long long)pos * a.turn[p0 + j]; /* rope.cu: modulo one turn */
      float s, c;
      sincospif((float)(int)(ph >> 32) * 4.656612873077393e-10f, &s, &c);
      t->co[j] = c * a.mscale;
      t->si[j] = s * a.mscale * (a.half && first ? -1.f : 1.f);
    }
  }
}
/* sign 1: R y, -1: R^T y */
__device__ __forceinline__ void turn(const Turn& t, bool half, float sign, float (&y)[8]) {
  if (half) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float z = __shfl_sync(kAll, y[j], t.other);
      y[j] = y[j] * t.co[j] + z * (sign * t.si[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float b = y[2 * j], c = y[2 * j + 1], s = sign * t.si[j];
      y[2 * j] = b * t.co[j] - c * s;
      y[2 * j + 1] = b * s + c * t.co[j];
    }
  }
}

/*
 * Eight elements of a row into their place of a quantised row (bytes at `row`, NULL: nowhere): four lanes hold a
 * group.  GGUF's own rounding: fp32 d = max |x| / 127, codes round(x (1 / d)), half away from zero, d kept in 16 bits;
 * 4 bits: d = (max - min) / 15, codes floor((x - min) (1 / d) + 1/2).
 */
template <bool Q4>
__device__ __forceinline__ void quantise8(const float (&x)[8], unsigned char* row, int hd, int d0) {
  const int grp = d0 >> 5, u = (d0 >> 3) & 3; /* group, eighth of the group's elements */
  float hi = Q4 ? x[0] : 0.f, lo = x[0];
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    hi = fmaxf(hi, Q4 ? x[j] : fabsf(x[j]));
    if (Q4) lo = fminf(lo, x[j]);
    odd |= !isfinite(x[j]);
  }
  if (odd) hi = INFINITY;
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(kAll, hi, o));
    if (Q4) lo = fminf(lo, __shfl_xor_sync(kAll, lo, o));
  }
  const bool bad = hi == INFINITY; /* a value of the group is not finite: it reads as NaN */
  const float d = __fdiv_rn(Q4 ? __fsub_rn(hi, lo) : hi, Q4 ? 15.f : 127.f);
  const float id = d == 0.f || bad ? 0.f : __fdiv_rn(1.f, d);
  const __half dh = bad ? __ushort_as_half(0x7e00) : __float2half_rn(fminf(d, 65504.f));
  if (!Q4) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = bad ? 0.f : __fmul_rn(x[j], id), f = floorf(fabsf(y));
      const int c = min((int)f + (__fsub_rn(fabsf(y), f) >= 0.5f ? 1 : 0), 127);
      w[j >> 2] |= (uint32_t)(uint8_t)(y < 0.f ? -c : c) << (8 * (j & 3));
    }
    if (!row) return;
    *reinterpret_cast<uint2*>(row + d0) = make_uint2(w[0], w[1]);
    if (u == 0) *reinterpret_cast<__half*>(row + hd + 2 * grp) = dh;
  } else {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        c[j] = bad ? 0u : (uint32_t)max(0, min((int)floorf(__fadd_rn(__fmul_rn(__fsub_rn(x[4 * i + j], lo), id), 0.5f)), 15));
      w[i] = (c[0] | c[1] << 16 | c[2] << 4 | c[3] << 20) << (8 * (grp & 1));
      w[i] |= __shfl_xor_sync(kAll, w[i], 4); /* the other group's half of the word */
    }
    if (!row) return;
    if (!(grp & 1)) *reinterpret_cast<uint2*>(row + (grp >> 1) * 32 + u * 8) = make_uint2(w[0], w[1]);
    if (u == 0)
      *reinterpret_cast<__half2*>(row + hd / 2 + 4 * grp) =
          __halves2half2(dh, bad ? __ushort_as_half(0x7e00) : __float2half_rn(fmaxf(fminf(lo, 65504.f), -65504.f)));
  }
}

enum Dest { TO_ROWS, TO_Q8, TO_Q4 };

/* where row m's K and V go, in bytes from the pools' begin; -1: nowhere */
__device__ __forceinline__ long long slot_place(const HeadArgs& a, int m) {
  const int s = a.seq[m], at = a.slot[m];
  if (s < 0 || s >= a.g.n_seq || at < 0 || (at >> a.g.page_shift) >= a.g.max_pages) return -1;
  const int page = a.table[(long long)s * a.g.max_pages + (at >> a.g.page_shift)];
  return page < 0 || page >= a.g.n_pages ? -1 : page * a.g.pstride + (at & (a.g.page - 1)) * a.g.pos;
}

template <typename TI, typename TO, int LPH, bool VEC, Dest DEST>
__global__ void __launch_bounds__(kWarps * 32) norm_rope_kernel(const __grid_constant__ HeadArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int HPS = 32 / LPH, U = 4; /* heads a warp takes at once, such steps in flight */
  const int lane = threadIdx.x & 31, grp = lane / LPH, d0 = (lane % LPH) * 8;
  const bool on = d0 < a.hd;
  const int gw = blockIdx.x * kWarps + (threadIdx.x >> 5), part = gw % a.wpr, n_rows = gridDim.x * kWarps / a.wpr;
  const int heads = a.nq + a.nk + a.nv;
  float wq[8], wk[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    wq[j] = on && a.wq ? a.wq[d0 + j] : 1.f;
    wk[j] = on && a.wk ? a.wk[d0 + j] : 1.f;
  }
  const float inv_hd = 1.f / a.hd;
  for (int m = gw / a.wpr; m < a.M; m += n_rows) {
    Turn t;
    turn_at<LPH>(a, a.pos[m], d0, lane, &t);
    const long long place = DEST == TO_ROWS ? 0 : slot_place(a, m);
    for (int h0 = part * HPS; h0 < heads; h0 += a.wpr * HPS * U) {
      float x[U][8];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + u * a.wpr * HPS + grp;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[u][j] = 0.f;
        if (h >= heads || !on) continue;
        const TI* p = h < a.nq           ? (const TI*)a.q + m * a.q_row + h * a.q_head
                      : h < a.nq + a.nk ? (const TI*)a.k + m * a.k_row + (h - a.nq) * a.k_head
                                        : (const TI*)a.v + m * a.v_row + (h - a.nq - a.nk) * a.v_head;
        load8<TI, VEC>(p + d0, x[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h0 + u * a.wpr * HPS >= heads) break; /* the whole warp */
        const int h = h0 + u * a.wpr * HPS + grp;
        const bool is_q = h < a.nq, is_v = DEST != TO_ROWS && h >= a.nq + a.nk;
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __fmaf_rn(x[u][j], x[u][j], ss);
        ss = head_sum<LPH>(ss);
        const bool normed = DEST == TO_ROWS || (is_q ? a.wq : a.wk) != nullptr;
        const float f = normed ? __frsqrt_rn(__fmaf_rn(ss, inv_hd, a.eps)) : 1.f;
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = x[u][j] * f * (is_q ? wq[j] : wk[j]);
        turn(t, a.half, 1.f, y);
        if (is_v) {
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = x[u][j];
        }
        if constexpr (DEST != TO_ROWS) {
          const bool kv = h >= a.nq && h < heads;
          if (__any_sync(kAll, kv)) {
            unsigned char* const row = !kv || place < 0 ? nullptr
                                       : (is_v ? a.vp : a.kp) + place + (long long)(h - a.nq - (is_v ? a.nk : 0)) * a.g.head;
            quantise8<DEST == TO_Q4>(y, row, a.hd, d0);
          }
        }
        if (h >= heads || !on) continue;
        if (is_q) store8<TO, VEC>((TO*)a.oq + ((long long)m * a.nq + h) * a.hd + d0, y);
        else if (DEST == TO_ROWS) store8<TO, VEC>((TO*)a.ok + ((long long)m * a.nk + h - a.nq) * a.hd + d0, y);
      }
    }
  }
}

template <typename T, int LPH, bool VEC>
__global__ void __launch_bounds__(kWarps * 32) norm_rope_grad_kernel(const __grid_constant__ HeadArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int HPS = 32 / LPH, U = 2;
  __shared__ float sh[kWarps][2][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = lane / LPH, d0 = (lane % LPH) * 8;
  const bool on = d0 < a.hd;
  const int gw = blockIdx.x * kWarps + warp, part = gw % a.wpr, n_rows = gridDim.x * kWarps / a.wpr;
  const int heads = a.nq + a.nk;
  float wq[8], wk[8], sq[8] = {}, sk[8] = {};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    wq[j] = on && a.M ? a.wq[d0 + j] : 0.f; /* no rows: the weights may be NULL */
    wk[j] = on && a.M && a.nk ? a.wk[d0 + j] : 0.f;
  }
  const float inv_hd = 1.f / a.hd;
  for (int m = gw / a.wpr; m < a.M; m += n_rows) {
    Turn t;
    turn_at<LPH>(a, a.pos[m], d0, lane, &t);
    for (int h0 = part * HPS; h0 < heads; h0 += a.wpr * HPS * U) {
      float x[U][8], y[U][8];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + u * a.wpr * HPS + grp;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[u][j] = y[u][j] = 0.f;
        if (h >= heads || !on) continue;
        if (h < a.nq) {
          load8<T, VEC>((const T*)a.q + m * a.q_row + h * a.q_head + d0, x[u]);
          load8<T, VEC>((const T*)a.gq + ((long long)m * a.nq + h) * a.hd + d0, y[u]);
        } else {
          load8<T, VEC>((const T*)a.k + m * a.k_row + (h - a.nq) * a.k_head + d0, x[u]);
          load8<T, VEC>((const T*)a.gk + ((long long)m * a.nk + h - a.nq) * a.hd + d0, y[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h0 + u * a.wpr * HPS >= heads) break;
        const int h = h0 + u * a.wpr * HPS + grp;
        const bool is_q = h < a.nq;
        turn(t, a.half, -1.f, y[u]); /* g */
        float ss = 0.f, sg = 0.f, gw_[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          gw_[j] = y[u][j] * (is_q ? wq[j] : wk[j]);
          ss = __fmaf_rn(x[u][j], x[u][j], ss);
          sg = __fmaf_rn(gw_[j], x[u][j], sg);
        }
        ss = head_sum<LPH>(ss);
        sg = head_sum<LPH>(sg);
        const float f = __frsqrt_rn(__fmaf_rn(ss, inv_hd, a.eps)), c = f * f * (sg * inv_hd);
        float dx[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          dx[j] = f * (gw_[j] - x[u][j] * c);
          const float dw = y[u][j] * (x[u][j] * f);
          if (is_q) sq[j] += dw; /* zero past the heads */
          else sk[j] += dw;
        }
        if (h >= heads || !on) continue;
        if (is_q) store8<T, VEC>((T*)a.oq + ((long long)m * a.nq + h) * a.hd + d0, dx);
        else store8<T, VEC>((T*)a.ok + ((long long)m * a.nk + h - a.nq) * a.hd + d0, dx);
      }
    }
  }
  /* the block's share of dw: groups of a warp by shuffles, warps in order */
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int o = LPH; o < 32; o <<= 1) {
      sq[j] += __shfl_xor_sync(kAll, sq[j], o);
      sk[j] += __shfl_xor_sync(kAll, sk[j], o);
    }
    if (grp == 0) {
      sh[warp][0][d0 + j] = sq[j];
      sh[warp][1][d0 + j] = sk[j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.hd; i += kWarps * 32) {
    const int w = i / a.hd, d = i - w * a.hd;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kWarps; ++j) s += sh[j][w][d];
    a.part[(long long)blockIdx.x * 2 * a.hd + i] = s;
  }
}

/* dw = the blocks' shares in order: a block takes eight columns, a warp every eighth ... of the shares */
constexpr int kSumCols = 8, kSumWays = 32;
__global__ void __launch_bounds__(kSumCols* kSumWays) norm_rope_sum_kernel(const float* part, int n, int hd, float* dwq, float* dwk) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sh[kSumWays][kSumCols];
  const int c = threadIdx.x % kSumCols, way = threadIdx.x / kSumCols, i = blockIdx.x * kSumCols + c;
  float s = 0.f;
  if (i < 2 * hd)
    for (int b = way; b < n; b += kSumWays) s += __ldcg(part + (long long)b * 2 * hd + i);
  sh[way][c] = s;
  __syncthreads();
  if (way == 0 && i < 2 * hd) {
    s = 0.f;
#pragma unroll
    for (int j = 0; j < kSumWays; ++j) s += sh[j][c];
    if (i < hd) dwq[i] = s;
    else if (dwk) dwk[i - hd] = s;
  }
}

/* rows read back: a thread takes eight elements of a (row, kv head) of K or of V */
template <typename T, bool Q4>
__global__ void __launch_bounds__(256) quant_read_kernel(const __grid_constant__ HeadArgs a) {
  pdl_wait();
  pdl_trigger();
  const int per = a.g.hd >> 3, units = a.g.n_head_kv * per * 2;
  const long long n = (long long)a.M * units;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const int m = (int)(i / units), r = (int)(i - (long long)m * units), pool = r / (units >> 1), hc = r - pool * (units >> 1);
    const int h = hc / per, d0 = (hc - h * per) * 8, grp = d0 >> 5, u = (d0 >> 3) & 3;
    const long long place = slot_place(a, m);
    float x[8] = {};
    if (place >= 0) {
      const unsigned char* row = (pool ? a.vp : a.kp) + place + (long long)h * a.g.head;
      if (!Q4) {
        const uint2 w = *reinterpret_cast<const uint2*>(row + d0);
        const float d = __half2float(*reinterpret_cast<const __half*>(row + a.g.hd + 2 * grp));
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)(int8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3))) * d;
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(row + (grp >> 1) * 32 + u * 8);
        const float2 dm = __half22float2(*reinterpret_cast<const __half2*>(row + a.g.hd / 2 + 4 * grp));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t y = (j < 4 ? w.x : w.y) >> (8 * (grp & 1) + 16 * (j & 1) + 4 * ((j >> 1) & 1));
          x[j] = __fmaf_rn((float)(y & 15u), dm.x, dm.y);
        }
      }
    }
    store8<T, true>((T*)(pool ? a.ok : a.oq) + ((long long)m * a.g.n_head_kv + h) * a.g.hd + d0, x);
  }
}

/* a grid of whole rows: as many warps a row as it takes to give every SM some, at most one a step of heads; and at
   most `most` blocks, which then walk the rows */
int plan_rows(Ctx* c, HeadArgs& a, int lph, int most) {
  const int heads = a.nq + a.nk + a.nv, steps = (heads + 32 / lph - 1) / (32 / lph);
  const long long want = (long long)c->n_sm * 32; /* warps */
  int wpr = 1;
  while (wpr < kWarps && wpr < steps && (long long)a.M * wpr < want) wpr *= 2;
  a.wpr = wpr;
  const long long blocks = ((long long)a.M * wpr + kWarps - 1) / kWarps;
  return (int)std::max<long long>(1, std::min<long long>(blocks, most));
}
int lanes_of(int hd) { return hd <= 64 ? 8 : hd <= 128 ? 16 : 32; }

template <typename TI, typename TO, Dest DEST, bool VEC>
int launch_apply(Ctx* c, HeadArgs& a) {
  const int lph = lanes_of(a.hd), blocks = plan_rows(c, a, lph, c->n_sm * 8);
  auto go = [&](auto kern) -> int {
    ULB_LAUNCH("norm rope launch", launch_k(c, kern, dim3(blocks), dim3(kWarps * 32), 0, a));
    return ULB_OK;
  };
  if (lph == 8) return go(norm_rope_kernel<TI, TO, 8, VEC, DEST>);
  if (lph == 16) return go(norm_rope_kernel<TI, TO, 16, VEC, DEST>);
  return go(norm_rope_kernel<TI, TO, 32, VEC, DEST>);
}
template <typename T, bool VEC>
int launch_grad(Ctx* c, HeadArgs& a, float* dwq, float* dwk) {
  const int lph = lanes_of(a.hd), blocks = plan_rows(c, a, lph, c->n_sm * kNormBlocks);
  auto go = [&](auto kern) -> int {
    ULB_LAUNCH("norm rope gradient launch", launch_k(c, kern, dim3(blocks), dim3(kWarps * 32), 0, a));
    return ULB_OK;
  };
  if (lph == 8) ULB_TRY(go(norm_rope_grad_kernel<T, 8, VEC>));
  else if (lph == 16) ULB_TRY(go(norm_rope_grad_kernel<T, 16, VEC>));
  else ULB_TRY(go(norm_rope_grad_kernel<T, 32, VEC>));
  ULB_LAUNCH("norm rope gradient sum launch", launch_k(c, norm_rope_sum_kernel, dim3((2 * a.hd + kSumCols - 1) / kSumCols),
                                                       dim3(kSumCols * kSumWays), 0, (const float*)a.part, blocks, a.hd, dwq, dwk));
  return ULB_OK;
}

/* what the handle adds, and its limits here */
int rotary(const char* who, const ulb_rope* r, HeadArgs* a) {
  ULB_CHECK(r->hd % 8 == 0 && r->hd <= 256, ULB_EUNSUPPORTED, "%s: head_dim %d (a multiple of 8 up to 256)", who, r->hd);
  ULB_CHECK(!r->half || r->rot % 16 == 0, ULB_EUNSUPPORTED, "%s: rot_dim %d of the half layout (a multiple of 16)", who, r->rot);
  a->turn = r->turn;
  a->mscale = r->mscale;
  a->half = r->half;
  a->rot = r->rot;
  a->hd = r->hd;
  return ULB_OK;
}

int norm_args(const char* who, const ulb_rope* r, const ulb_norm_rope_args* p, HeadArgs* a) {
  ULB_TRY(rotary(who, r, a));
  ULB_CHECK(dtype_bytes(p->dtype), ULB_EUNSUPPORTED, "%s: type %d (F32, F16 or BF16)", who, p->dtype);
  ULB_CHECK(p->M >= 0 && p->n_head > 0 && p->n_head_kv >= 0, ULB_EINVAL, "%s: %d rows of %d and %d heads", who, p->M, p->n_head, p->n_head_kv);
  ULB_CHECK((long long)p->n_head + p->n_head_kv <= (1 << 20), ULB_EUNSUPPORTED, "%s: %d and %d heads", who, p->n_head, p->n_head_kv);
  ULB_CHECK(std::isfinite(p->eps) && p->eps > 0.f, ULB_EINVAL, "%s: eps %g", who, (double)p->eps);
  ULB_CHECK(p->q_row >= 0 && p->q_head >= 0 && p->k_row >= 0 && p->k_head >= 0, ULB_EINVAL, "%s: negative stride", who);
  a->eps = p->eps;
  a->M = p->M;
  a->nq = p->n_head;
  a->nk = p->n_head_kv;
  a->q = p->q;
  a->k = p->k;
  a->q_head = p->q_head ? p->q_head : r->hd;
  a->q_row = p->q_row ? p->q_row : a->q_head * p->n_head;
  a->k_head = p->k_head ? p->k_head : r->hd;
  a->k_row = p->k_row ? p->k_row : a->k_head * p->n_head_kv;
  a->wq = p->q_weight;
  a->wk = p->k_weight;
  a->pos = p->pos;
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

using namespace ulb;

extern "C" {

int ulb_norm_rope_apply(ulb_ctx* ctx, const ulb_rope* r, const ulb_norm_rope_args* p, void* q_out, void* k_out) {
  ULB_CHECK(ctx && r && p, ULB_EINVAL, "ulb_norm_rope_apply: NULL argument");
  HeadArgs a = {};
  ULB_TRY(norm_args("ulb_norm_rope_apply", r, p, &a));
  if (a.M == 0) return ULB_OK;
  ULB_CHECK(p->q && p->q_weight && p->pos && q_out && (a.nk == 0 || (p->k && p->k_weight && k_out)), ULB_EINVAL,
            "ulb_norm_rope_apply: NULL argument");
  const int eb = dtype_bytes(p->dtype);
  if (a.nk == 0) a.k = a.ok = nullptr, a.k_row = a.k_head = 0, a.wk = nullptr, k_out = nullptr;
  ULB_CHECK(element_aligned(eb, {a.q, a.k, q_out, k_out}) && words_aligned({a.wq, a.wk, a.pos}), ULB_EINVAL,
            "ulb_norm_rope_apply: unaligned pointer");
  ULB_CHECK(a.q != q_out || (a.q_head == a.hd && a.q_row == a.q_head * a.nq), ULB_EINVAL, "ulb_norm_rope_apply: q in place of strided rows");
  ULB_CHECK(!a.k || a.k != k_out || (a.k_head == a.hd && a.k_row == a.k_head * a.nk), ULB_EINVAL,
            "ulb_norm_rope_apply: k in place of strided rows");
  a.oq = q_out;
  a.ok = k_out;
  Ctx* c = &ctx->c;
  ULB_CUDA(cudaSetDevice(c->device));
  const bool v = wide(eb, {a.q, a.k, q_out, k_out}, a.q_row | a.q_head | a.k_row | a.k_head);
  switch (p->dtype) {
    case ULB_TYPE_F32: return v ? launch_apply<float, float, TO_ROWS, true>(c, a) : launch_apply<float, float, TO_ROWS, false>(c, a);
    case ULB_TYPE_F16: return v ? launch_apply<__half, __half, TO_ROWS, true>(c, a) : launch_apply<__half, __half, TO_ROWS, false>(c, a);
    default:
      return v ? launch_apply<__nv_bfloat16, __nv_bfloat16, TO_ROWS, true>(c, a) : launch_apply<__nv_bfloat16, __nv_bfloat16, TO_ROWS, false>(c, a);
  }
}

int ulb_norm_rope_grad(ulb_ctx* ctx, const ulb_rope* r, const ulb_norm_rope_args* p, const void* dq_out, const void* dk_out, void* dq,
                       void* dk, float* dwq, float* dwk) {
  ULB_CHECK(ctx && r && p, ULB_EINVAL, "ulb_norm_rope_grad: NULL argument");
  HeadArgs a = {};
  ULB_TRY(norm_args("ulb_norm_rope_grad", r, p, &a));
  ULB_CHECK(dwq && (a.nk == 0 || dwk), ULB_EINVAL, "ulb_norm_rope_grad: NULL argument");
  ULB_CHECK(a.M == 0 || (p->q && p->q_weight && p->pos && dq_out && dq && (a.nk == 0 || (p->k && p->k_weight && dk_out && dk))), ULB_EINVAL,
            "ulb_norm_rope_grad: NULL argument");
  if (a.nk == 0) a.k = nullptr, a.k_row = a.k_head = 0, a.wk = nullptr, dk_out = nullptr, dk = nullptr, dwk = nullptr;
  const int eb = dtype_bytes(p->dtype);
  ULB_CHECK(element_aligned(eb, {a.q, a.k, dq_out, dk_out, dq, dk}) && words_aligned({a.wq, a.wk, a.pos, dwq, dwk}), ULB_EINVAL,
            "ulb_norm_rope_grad: unaligned pointer");
  a.gq = dq_out;
  a.gk = dk_out;
  a.oq = dq;
  a.ok = dk;
  Ctx* c = &ctx->c;
  ULB_CUDA(cudaSetDevice(c->device));
  /* at the first call, whatever its shape, so that any later one can be captured */
  if (!c->norm_ws) ULB_CUDA(cudaMalloc((void**)&c->norm_ws, (size_t)c->n_sm * kNormBlocks * 2 * 256 * sizeof(float)));
  a.part = c->norm_ws;
  const bool v = wide(eb, {a.q, a.k, dq_out, dk_out, dq, dk}, a.q_row | a.q_head | a.k_row | a.k_head);
  switch (p->dtype) {
    case ULB_TYPE_F32: return v ? launch_grad<float, true>(c, a, dwq, dwk) : launch_grad<float, false>(c, a, dwq, dwk);
    case ULB_TYPE_F16: return v ? launch_grad<__half, true>(c, a, dwq, dwk) : launch_grad<__half, false>(c, a, dwq, dwk);
    default: return v ? launch_grad<__nv_bfloat16, true>(c, a, dwq, dwk) : launch_grad<__nv_bfloat16, false>(c, a, dwq, dwk);
  }
}

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
  ULB_CHECK(r->hd == a.g.hd, ULB_EINVAL, "ulb_quant_append: rotary head_dim %d, cache head_dim %d", r->hd, a.g.hd);
  ULB_CHECK(dtype_bytes(p->in_dtype), ULB_EUNSUPPORTED, "ulb_quant_append: type %d (F32, F16 or BF16)", p->in_dtype);
  ULB_CHECK(p->M >= 0 && p->n_head > 0 && p->n_head <= (1 << 20) && a.g.n_head_kv <= (1 << 20), ULB_EINVAL,
            "ulb_quant_append: %d rows of %d and %d heads", p->M, p->n_head, a.g.n_head_kv);
  ULB_CHECK(p->q_row >= 0 && p->k_row >= 0 && p->v_row >= 0, ULB_EINVAL, "ulb_quant_append: negative stride");
  const bool normed = p->q_weight || p->k_weight;
  ULB_CHECK(!normed || (std::isfinite(p->eps) && p->eps > 0.f), ULB_EINVAL, "ulb_quant_append: eps %g", (double)p->eps);
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
  const bool v = wide(eb, {a.q, a.k, a.v}, a.q_row | a.k_row | a.v_row) && ULB_ALIGNED16(a.oq);
  auto to = [&](auto in, auto out, auto dest) -> int {
    using TI = decltype(in);
    using TO = decltype(out);
    constexpr Dest D = decltype(dest)::value;
    return v ? launch_apply<TI, TO, D, true>(c, a) : launch_apply<TI, TO, D, false>(c, a);
  };
  auto in = [&](auto out, auto dest) -> int {
    switch (p->in_dtype) {
      case ULB_TYPE_F32: return to(0.f, out, dest);
      case ULB_TYPE_F16: return to(__half(), out, dest);
      default: return to(__nv_bfloat16(), out, dest);
    }
  };
  const std::integral_constant<Dest, TO_Q8> q8;
  const std::integral_constant<Dest, TO_Q4> q4;
  if (d->dtype == ULB_TYPE_F16) return d->format == ULB_TYPE_Q8_0 ? in(__half(), q8) : in(__half(), q4);
  return d->format == ULB_TYPE_Q8_0 ? in(__nv_bfloat16(), q8) : in(__nv_bfloat16(), q4);
}

int ulb_quant_read(ulb_ctx* ctx, const ulb_quant_desc* d, int dtype, const void* k, const void* v, const int32_t* table,
                   const int32_t* row_seq, const int32_t* slot, int M, void* k_out, void* v_out) {
  ULB_CHECK(ctx, ULB_EINVAL, "ulb_quant_read: NULL context");
  HeadArgs a = {};
  ULB_TRY(quant_geom("ulb_quant_read", d, &a.g));
  ULB_CHECK(dtype_bytes(dtype), ULB_EUNSUPPORTED, "ulb_quant_read: type %d (F32, F16 or BF16)", dtype);
  ULB_CHECK(M >= 0, ULB_EINVAL, "ulb_quant_read: %d rows", M);
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
  const long long n = (long long)M * a.g.n_head_kv * (a.g.hd >> 3) * 2;
  ULB_CHECK((long long)a.g.n_head_kv * (a.g.hd >> 3) * 2 < (1ll << 31), ULB_EUNSUPPORTED, "ulb_quant_read: %d kv heads", a.g.n_head_kv);
  const int blocks = (int)std::min<long long>((n + 255) / 256, (long long)c->n_sm * 64);
  auto go = [&](auto kern) -> int {
    ULB_LAUNCH("quant read launch", launch_k(c, kern, dim3(blocks), dim3(256), 0, a));
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

ULB_TRACE_UNIT(head_norm)
