/*
 * tree_attention.cu — attention of the rows of drafted trees over a paged fp16 / bf16 cache
 * (ulb_tree_attention).  The loop's own attention (attention.cu) knows its own trees of at most
 * 63 nodes, caches of at most 8192 positions in its own layout, and fp16; this operator takes any
 * masks, lengths, page sizes, strides and both 16-bit types.  flash_attention*.glsl of the
 * reference (src/shaders/attention) read a contiguous cache and know no trees.
 *
 * Mathematics.  For row r and head h, s_t = scale q . k_t over the visible keys t,
 * m = max s_t, l = sum exp(s_t - m), o = sum exp(s_t - m) v_t / l.  One pass over the keys: tiles
 * update (m, l, o) with the running maximum, o scaled by exp(m_old - m_new) when it moves.  Two
 * partial results over disjoint keys join the same way, so the keys are split over CTAs and
 * joined by a second small kernel when one CTA a (row tile, kv head) would leave SMs idle.
 *
 * Work of a CTA: RT = 16 WM rows (row = node x head of the GQA group, so a K / V tile is read
 * once for all heads that share it) against the keys of one split, in tiles of 64 keys that
 * stream through a ring of NST shared-memory stages by cp.async.  The 8 (or 4) warps are WM row
 * groups x WK key groups; a key group has its own (m, l, o), joined in shared memory at the end.
 * S = Q K^T and O = P V are mma.sync m16n8k16 with fp32 accumulators; P stays in registers, rounded to
 * fp16 (2^-11 relative a weight, as the output is; see kRaise) or kept as two bf16 parts.
 *
 * Used for head dim 256 and for calls too small for the tcgen05 form (tree_attention_tc.cu, which has
 * the rule).  Measured: 1 row x 500 keys, 32 heads over 4, hd 64: 8.6 us, a launch each for the splits
 * and their join; 64 rows x 300 keys, 32 kv heads of 64: 38 us; 1 row x 30000 keys, 64 heads over 8 of
 * 256 (246 MB): 64 us, 60 % of the copy rate, bound by the two stages that fit at hd 256.
 *
 * Rows of shared memory are hd + 8 elements apart: 16-byte row pitch odd in units of 16 bytes,
 * so the eight rows of an ldmatrix phase fall in eight different bank groups.
 *
 * Tiles past every row's open positions take the masked path: each score's visibility from the
 * row's bits.  A masked key never reaches a result: its score is replaced, its weight is an exact
 * zero, positions past len and unmapped pages are zero-filled, and a V element of such a tile
 * that is not finite is taken out of shared memory and added only to the rows that see it.
 */
#include "tree_attention.h"

#include <cmath>

#include <algorithm>

namespace ulb {
namespace {

constexpr int BK = 64;         /* keys a tile */
constexpr int kTbl = 512;      /* page ids a block holds: a ring, half of it replaced at a time */

__device__ __forceinline__ uint32_t saddr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
/* which of the two elements of a word are infinite or NaN */
template <typename T> __device__ __forceinline__ bool odd_lo(uint32_t w) {
  constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (w & E) == E;
}
template <typename T> __device__ __forceinline__ bool odd_hi(uint32_t w) { return odd_lo<T>(w >> 16); }

/*
 * Weights are exp(s - m + raise): fp16 holds 11 bits of a weight from 2^-14 on, so with the heaviest at
 * 2^14 (65504 is the largest) a weight keeps them down to 2^-28 of it, and what thousands of keys far
 * below one heavy key weigh together is not lost.  The statistics m - raise and l, and so the partials,
 * carry the factor; it drops out of o / l and of m + log l.  Scores in base 2 up to 2^25: past them a
 * maximum rounded to fp32 could leave weights past 65504.
 */
template <typename T> constexpr float kRaise = std::is_same<T, __half>::value ? 14.f : 0.f;

template <int HD, int WM, int WK>
struct Cfg {
  static constexpr int WARPS = WM * WK, NT = WARPS * 32, RT = 16 * WM, KW = BK / WK;
  static constexpr int PITCH = (HD + 8) * 2;                 /* bytes between rows of a tile */
  static constexpr int STAGE = 2 * BK * PITCH;               /* K and V */
  /* stages of the ring: small blocks (one row tile of 16) several to an SM, since a short sequence is
     mostly start and end (64 rows x 300 keys of 32 kv heads: 38 us, 90 with one block an SM) */
  static constexpr int ROOM = WM == 1 ? 50000 : 75000;
  static constexpr int NST = ROOM / STAGE < 2 ? 2 : ROOM / STAGE;
  static constexpr int MIN_BLOCKS = WM > 1 && HD <= 96 ? 2 : 1; /* 64 x 16 rows x 116 keys, hd 64: 22 us, 33 with one */
  static constexpr int OP = HD + 4;                          /* floats between rows of the warps' outputs */
  static constexpr int JOIN = WK * RT * OP * 4;
  static constexpr int SMEM = NST * STAGE > JOIN ? NST * STAGE : JOIN;
  static_assert(NST >= 2 && SMEM <= 200 * 1024, "shared memory");
  static_assert((NST + 1) * BK / 16 + 2 <= kTbl / 2, "the tiles in flight are in the newer half of the page ids");
};

template <typename T, int HD, int WM, int WK>
__global__ void __launch_bounds__(WM* WK * 32, Cfg<HD, WM, WK>::MIN_BLOCKS) tree_attn_kernel(const __grid_constant__ TreeArgs a) {
  using C = Cfg<HD, WM, WK>;
  constexpr int KS = HD / 16, NB = C::KW / 8, DB = HD / 8;
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ int tbl[kTbl];
  __shared__ float sh_m[WK][C::RT], sh_l[WK][C::RT];
  __shared__ int odd_v, n_ids; /* page ids seen so far, of a split of more than kTbl pages */
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int wm = warp / WK, wk = warp % WK;

  int id = blockIdx.x;
  const int rt = id % a.n_tile;
  id /= a.n_tile;
  const int kvh = id % a.g.n_head_kv;
  id /= a.g.n_head_kv;
  const int split = id % a.n_split, s = id / a.n_split;
  const TreeSeq q = tree_seq(a, s);
  const int nq = min(C::RT, q.n * a.G - rt * C::RT); /* queries of this tile: qi = row * G + head of the group */
  if (nq <= 0) return;
  const int k0 = split * a.split_keys;
  if (split > 0 && k0 >= q.len) return;
  const int k1 = q.len - k0 <= a.split_keys ? q.len : k0 + a.split_keys;
  const bool single = q.len <= a.split_keys;
  const int open = tree_open(a, q);

  /* the split's pages */
  const int p0 = k0 >> a.g.page_shift, np = k1 > k0 ? ((k1 - 1) >> a.g.page_shift) - p0 + 1 : 0;
  if (tid == 0) { odd_v = 0; n_ids = kTbl; }
  auto page_ids = [&](int from, int to) { /* is one of them unmapped? */
    int bad = 0;
    for (int i = from + tid; i < to; i += C::NT) {
      const int p = p0 + i < a.g.max_pages ? a.table[(long long)s * a.g.max_pages + p0 + i] : -1;
      const bool ok = p >= 0 && p < a.g.n_pages;
      tbl[i & (kTbl - 1)] = ok ? p : -1;
      bad |= !ok;
    }
    return __syncthreads_or(bad);
  };
  auto page_of = [&](int pos) { return tbl[((pos >> a.g.page_shift) - p0) & (kTbl - 1)]; };
  /* the first tile that the page ids in shared memory do not cover, less the stages ahead */
  auto covered = [&](int have) { return have < np ? (((p0 + have) << a.g.page_shift) - k0) / BK - C::NST : 0x7fffffff; };
  int bad = page_ids(0, min(np, kTbl)), reload = covered(kTbl);

  const T* const kb = (const T*)a.k + kvh * a.g.head;
  const T* const vb = (const T*)a.v + kvh * a.g.head;
  /* one tile into its stage: eight threads a row; rows past k1 or unmapped are zero */
  auto stage = [&](int it) {
    uint8_t* const ks = sm + (it % C::NST) * C::STAGE;
    for (int j = tid >> 3; j < BK; j += C::NT / 8) {
      const int pos = k0 + it * BK + j;
      const int pg = pos < k1 ? page_of(pos) : -1;
      const bool ok = pg >= 0;
      const long long off = ok ? pg * a.g.pstride + (pos & (a.g.page - 1)) * a.g.pos : 0;
      const uint32_t d = saddr(ks + j * C::PITCH);
#pragma unroll
      for (int c = tid & 7; c < HD / 8; c += 8) {
        cp16(d + c * 16, kb + off + c * 8, ok);
        cp16(d + BK * C::PITCH + c * 16, vb + off + c * 8, ok);
      }
    }
  };

  const int n_it = (k1 - k0 + BK - 1) / BK;
#pragma unroll
  for (int i = 0; i < C::NST - 1; ++i) {
    if (i < n_it) stage(i);
    cp_commit();
  }

  /* Q of rows g and g + 8 as A fragments */
  const int qa = rt * C::RT + wm * 16 + g, qb = qa + 8; /* query indexes in the sequence */
  const int lim = rt * C::RT + nq;
  const bool va = qa < lim, vbq = qb < lim;
  const int ia = va ? qa / a.G : 0, ib = vbq ? qb / a.G : 0; /* their rows */
  uint32_t qf[KS][4];
  {
    const T* pa = (const T*)a.q + ((long long)(q.r0 + ia) * a.H + kvh * a.G + (va ? qa % a.G : 0)) * HD;
    const T* pb = (const T*)a.q + ((long long)(q.r0 + ib) * a.H + kvh * a.G + (vbq ? qb % a.G : 0)) * HD;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      qf[i][0] = va ? *reinterpret_cast<const uint32_t*>(pa + i * 16 + 2 * t) : 0u;
      qf[i][1] = vbq ? *reinterpret_cast<const uint32_t*>(pb + i * 16 + 2 * t) : 0u;
      qf[i][2] = va ? *reinterpret_cast<const uint32_t*>(pa + i * 16 + 8 + 2 * t) : 0u;
      qf[i][3] = vbq ? *reinterpret_cast<const uint32_t*>(pb + i * 16 + 8 + 2 * t) : 0u;
    }
  }

  float mA = -INFINITY, mB = -INFINITY, lA = 0.f, lB = 0.f; /* m: the maximum less kRaise */
  float o[DB][4];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;

  for (int it = 0; it < n_it; ++it) {
    cp_wait<C::NST - 2>();
    __syncthreads();
    if (it + C::NST - 1 < n_it) {
      if (it > reload) { /* every 256 pages of a longer split */
        const int have = n_ids;
        bad |= page_ids(have, min(np, have + kTbl / 2));
        reload = covered(have + kTbl / 2);
        if (tid == 0) n_ids = have + kTbl / 2;
      }
      stage(it + C::NST - 1);
    }
    cp_commit();
    uint8_t* const ks = sm + (it % C::NST) * C::STAGE;
    const int tile0 = k0 + it * BK;
    const bool masked = bad || tile0 + BK > open || tile0 + BK > k1;
    bool fix = false;
    if (masked) {
      /* V elements that are not finite leave the tile (see the top) */
      uint8_t* const vs = ks + BK * C::PITCH;
      for (int i = tid; i < BK * (HD / 8); i += C::NT) {
        uint4* const p = reinterpret_cast<uint4*>(vs + (i / (HD / 8)) * C::PITCH + (i % (HD / 8)) * 16);
        uint4 x = *p;
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
        bool any = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (odd_lo<T>(w[e])) { w[e] &= 0xffff0000u; any = true; }
          if (odd_hi<T>(w[e])) { w[e] &= 0x0000ffffu; any = true; }
        }
        if (any) {
          *p = make_uint4(w[0], w[1], w[2], w[3]);
          odd_v = it + 1;
        }
      }
      __syncthreads();
      fix = odd_v == it + 1;
    }

    /* S of this warp's KW keys */
    float sc[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
    const uint32_t kaddr = saddr(ks) + (wk * C::KW + ((lane >> 4) << 3) + (lane & 7)) * C::PITCH + ((lane >> 3) & 1) * 16;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
#pragma unroll
      for (int n = 0; n < NB; n += 2) {
        uint32_t b[4];
        ldsm4(kaddr + n * 8 * C::PITCH + i * 32, b);
        mma<T>(sc[n], qf[i], b[0], b[1]);
        mma<T>(sc[n + 1], qf[i], b[2], b[3]);
      }
    }
    const int key0 = tile0 + wk * C::KW + 2 * t;
    auto sees = [&](int i, int pos) {
      return pos < k1 && page_of(pos) >= 0 && (pos < open || tree_sees(a, q, i, pos));
    };
    if (masked) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int pos = key0 + n * 8 + e;
          if (!sees(ia, pos)) sc[n][e] = -INFINITY;
          if (!sees(ib, pos)) sc[n][2 + e] = -INFINITY;
        }
    }
    /* running maximum, weights */
    float xA = -INFINITY, xB = -INFINITY;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      xA = fmaxf(xA, fmaxf(sc[n][0], sc[n][1]));
      xB = fmaxf(xB, fmaxf(sc[n][2], sc[n][3]));
    }
    xA = fmaxf(xA, __shfl_xor_sync(0xffffffffu, xA, 1));
    xB = fmaxf(xB, __shfl_xor_sync(0xffffffffu, xB, 1));
    xA = fmaxf(xA, __shfl_xor_sync(0xffffffffu, xA, 2));
    xB = fmaxf(xB, __shfl_xor_sync(0xffffffffu, xB, 2));
    const float nA = fmaxf(mA, __fmaf_rn(xA, a.scale2, -kRaise<T>)), nB = fmaxf(mB, __fmaf_rn(xB, a.scale2, -kRaise<T>));
    const float uA = nA == -INFINITY ? 0.f : nA, uB = nB == -INFINITY ? 0.f : nB;
    const float fA = ex2(mA - uA), fB = ex2(mB - uB);
    mA = nA;
    mB = nB;
    lA *= fA;
    lB *= fB;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      sc[n][0] = ex2(__fmaf_rn(sc[n][0], a.scale2, -uA));
      sc[n][1] = ex2(__fmaf_rn(sc[n][1], a.scale2, -uA));
      sc[n][2] = ex2(__fmaf_rn(sc[n][2], a.scale2, -uB));
      sc[n][3] = ex2(__fmaf_rn(sc[n][3], a.scale2, -uB));
      lA += sc[n][0] + sc[n][1];
      lB += sc[n][2] + sc[n][3];
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      o[d][0] *= fA;
      o[d][1] *= fA;
      o[d][2] *= fB;
      o[d][3] *= fB;
    }
    /* O += P V */
    const uint32_t vaddr = saddr(ks) + BK * C::PITCH + (wk * C::KW + ((lane >> 3) & 1) * 8 + (lane & 7)) * C::PITCH + (lane >> 4) * 16;
#pragma unroll
    for (int n = 0; n < NB; n += 2) {
      const uint32_t pf[4] = {pack2<T>(sc[n][0], sc[n][1]), pack2<T>(sc[n][2], sc[n][3]), pack2<T>(sc[n + 1][0], sc[n + 1][1]),
                              pack2<T>(sc[n + 1][2], sc[n + 1][3])};
      /* what bf16 leaves of a weight is a second operand: these calls wait for memory, not for products,
         and the output's own rounding stays the only one */
      constexpr bool REST = std::is_same<T, __nv_bfloat16>::value;
      [[maybe_unused]] uint32_t pr[4] = {};
      if constexpr (REST) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 h = unpack2<T>(pf[e]);
          const float* w = &sc[n + (e >> 1)][2 * (e & 1)];
          pr[e] = pack2<T>(w[0] - h.x, w[1] - h.y);
        }
      }
#pragma unroll
      for (int d = 0; d < DB; d += 2) {
        uint32_t b[4];
        ldsm4t(vaddr + n * 8 * C::PITCH + d * 16, b);
        mma<T>(o[d], pf, b[0], b[1]);
        mma<T>(o[d + 1], pf, b[2], b[3]);
        if constexpr (REST) {
          mma<T>(o[d], pr, b[0], b[1]);
          mma<T>(o[d + 1], pr, b[2], b[3]);
        }
      }
    }
    if (fix) { /* what left the tile, to the rows that see it */
      for (int kk = 0; kk < C::KW; ++kk) {
        const int pos = tile0 + wk * C::KW + kk, from = (lane & ~3) | ((kk & 7) >> 1);
        float pa = 0.f, pb = 0.f;
#pragma unroll
        for (int n = 0; n < NB; ++n)
          if (n == kk >> 3) {
            pa = kk & 1 ? sc[n][1] : sc[n][0];
            pb = kk & 1 ? sc[n][3] : sc[n][2];
          }
        pa = __shfl_sync(0xffffffffu, pa, from);
        pb = __shfl_sync(0xffffffffu, pb, from);
        const int pg = pos < k1 ? page_of(pos) : -1;
        if (pg < 0) continue;
        const T* vr = vb + pg * a.g.pstride + (pos & (a.g.page - 1)) * a.g.pos;
        const bool sa = sees(ia, pos), sb = sees(ib, pos);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = to_f<T>(vr[d * 8 + 2 * t + e]);
            if (isfinite(x)) continue;
            if (sa) o[d][e] += pa * x;
            if (sb) o[d][2 + e] += pb * x;
          }
      }
    }
  }

  /* the WK key groups of a row join in shared memory */
  lA += __shfl_xor_sync(0xffffffffu, lA, 1);
  lB += __shfl_xor_sync(0xffffffffu, lB, 1);
  lA += __shfl_xor_sync(0xffffffffu, lA, 2);
  lB += __shfl_xor_sync(0xffffffffu, lB, 2);
  cp_wait<0>();
  __syncthreads();
  float* const po = reinterpret_cast<float*>(sm);
  const int ra = wm * 16 + g, rb = ra + 8;
  if (t == 0) {
    sh_m[wk][ra] = mA;
    sh_l[wk][ra] = lA;
    sh_m[wk][rb] = mB;
    sh_l[wk][rb] = lB;
  }
#pragma unroll
  for (int d = 0; d < DB; ++d) {
    *reinterpret_cast<float2*>(po + (wk * C::RT + ra) * C::OP + d * 8 + 2 * t) = make_float2(o[d][0], o[d][1]);
    *reinterpret_cast<float2*>(po + (wk * C::RT + rb) * C::OP + d * 8 + 2 * t) = make_float2(o[d][2], o[d][3]);
  }
  __syncthreads();
  for (int i = tid; i < nq * (HD / 4); i += C::NT) {
    const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
    float M = sh_m[0][r];
#pragma unroll
    for (int w = 1; w < WK; ++w) M = fmaxf(M, sh_m[w][r]);
    const float U = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float f = ex2(sh_m[w][r] - U);
      const float4 y = *reinterpret_cast<const float4*>(po + (w * C::RT + r) * C::OP + d);
      L += sh_l[w][r] * f;
      x.x += y.x * f;
      x.y += y.y * f;
      x.z += y.z * f;
      x.w += y.w * f;
    }
    const int qi = rt * C::RT + r;
    const long long at = (long long)(q.r0 + qi / a.G) * a.H + kvh * a.G + qi % a.G;
    if (single) {
      const float inv = L == 0.f ? 0.f : __fdividef(1.f, L); /* 0: the row sees nothing */
      *reinterpret_cast<uint2*>((T*)a.out + at * HD + d) = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
      if (d == 0 && a.lse) a.lse[at] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
    } else {
      const long long ps = at * a.n_split + split;
      __stcg(reinterpret_cast<float4*>(a.po + ps * HD + d), x);
      if (d == 0) __stcg(reinterpret_cast<float2*>(a.pml + ps * 2), make_float2(M, L));
    }
  }
}

constexpr int kJoinThreads = 128;

/*
 * Join the splits of one (row, head): weights of the splits once, then groups of hd / 4 threads
 * add every GR-th split's outputs, and the groups add up in order: the result does not depend on
 * which CTA ran when.  Rows of sequences with one split are complete already.
 */
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) tree_join_kernel(const __grid_constant__ TreeArgs a) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ float sj[]; /* [n_split] weights, then [groups][hd] */
  __shared__ float red[2][kJoinThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hd = a.g.hd;
  const int h = blockIdx.x % a.H, i = blockIdx.x / a.H, s = blockIdx.y;
  const TreeSeq q = tree_seq(a, s);
  if (i >= q.n || q.len <= a.split_keys) return;
  const int ns = (q.len + a.split_keys - 1) / a.split_keys;
  const long long at = (long long)(q.r0 + i) * a.H + h, ps = at * a.n_split;
  float M = -INFINITY;
  for (int u = tid; u < ns; u += kJoinThreads) M = fmaxf(M, __ldcg(a.pml + (ps + u) * 2));
#pragma unroll
  for (int x = 16; x; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
  if (lane == 0) red[0][warp] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float U = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  for (int u = tid; u < ns; u += kJoinThreads) {
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.pml + (ps + u) * 2));
    const float f = ex2(ml.x - U);
    sj[u] = f;
    L += ml.y * f;
  }
#pragma unroll
  for (int x = 16; x; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
  if (lane == 0) red[1][warp] = L;
  __syncthreads();
  L = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  const int w4 = hd / 4, gr = kJoinThreads / w4, grp = tid / w4, d = tid % w4 * 4;
  float* const acc = sj + (a.n_split + 3) / 4 * 4;
  if (grp < gr) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int u = grp; u < ns; u += gr) {
      const float4 y = __ldcg(reinterpret_cast<const float4*>(a.po + (ps + u) * hd + d));
      const float f = sj[u];
      x.x += y.x * f;
      x.y += y.y * f;
      x.z += y.z * f;
      x.w += y.w * f;
    }
    *reinterpret_cast<float4*>(acc + grp * hd + d) = x;
  }
  __syncthreads();
  if (tid < w4) {
    float4 x = *reinterpret_cast<const float4*>(acc + d);
    for (int u = 1; u < gr; ++u) {
      const float4 y = *reinterpret_cast<const float4*>(acc + u * hd + d);
      x.x += y.x;
      x.y += y.y;
      x.z += y.z;
      x.w += y.w;
    }
    const float inv = L == 0.f ? 0.f : __fdividef(1.f, L); /* 0: the row sees nothing */
    *reinterpret_cast<uint2*>((T*)a.out + at * hd + d) = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
    if (tid == 0 && a.lse) a.lse[at] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
  }
}

/*
 * Keys a split.  `units` CTAs (row tiles x kv heads x sequences) walk whole sequences; `slots`
 * run at once.  One sequence: as many splits as fill the slots once.  Several: about four waves,
 * because their lengths differ and short splits let the last wave even out.  Never under 128 keys,
 * never more partials than the workspace holds (one split needs none).
 */
void plan_splits(TreeArgs* a, long long units, int slots) {
  long long want = (a->g.n_seq == 1 ? (long long)slots : 4ll * slots) / std::max(1ll, units);
  want = std::max(1ll, want);
  const long long per = (long long)a->rows * a->H * (a->g.hd + 2);
  want = std::min(want, std::max(1ll, (long long)kTreeWsFloats / std::max(1ll, per) - 1));
  auto round = [](long long x) { return (x + 127) / 128 * 128; };
  const long long keys = std::max(128ll, round((a->max_len + want - 1) / want));
  a->split_keys = (int)keys;
  a->n_split = (int)std::max(1ll, (a->max_len + keys - 1) / keys);
}

template <typename T, int HD, int WM, int WK>
int launch_tree(Ctx* c, TreeArgs& a) {
  using C = Cfg<HD, WM, WK>;
  static uint64_t attr = 0; /* devices it is set on */
  if (!(attr >> (c->device & 63) & 1)) {
    ULB_CUDA(cudaFuncSetAttribute(tree_attn_kernel<T, HD, WM, WK>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    attr |= 1ull << (c->device & 63);
  }
  a.n_tile = (int)(((long long)a.max_rows * a.G + C::RT - 1) / C::RT);
  const long long units = (long long)a.n_tile * a.g.n_head_kv * a.g.n_seq;
  plan_splits(&a, units, c->n_sm);
  if (a.n_split > 1) {
    a.po = c->tree_ws;
    a.pml = c->tree_ws + (long long)a.rows * a.H * a.g.hd * a.n_split;
  }
  const long long blocks = units * a.n_split;
  ULB_CHECK(blocks < (1ll << 31), ULB_EUNSUPPORTED, "ulb_tree_attention: %lld blocks", blocks);
  ULB_LAUNCH("tree attention launch", launch_k(c, tree_attn_kernel<T, HD, WM, WK>, dim3((unsigned)blocks), dim3(C::NT), C::SMEM, a));
  if (a.n_split > 1) {
    const int w4 = HD / 4;
    const size_t smem = ((size_t)(a.n_split + 3) / 4 * 4 + (size_t)(kJoinThreads / w4) * HD) * sizeof(float);
    ULB_LAUNCH("tree join launch", launch_k(c, tree_join_kernel<T>, dim3((unsigned)((long long)a.max_rows * a.H), a.g.n_seq),
                                            dim3(kJoinThreads), smem, a));
  }
  return ULB_OK;
}

template <typename T, int HD>
int pick_tree(Ctx* c, TreeArgs& a) {
  /* the row tile that holds a sequence's queries with the least padding; past 64 the keys are
     read once a tile from L2 */
  const long long nq = (long long)a.max_rows * a.G;
  if (nq <= 16) return launch_tree<T, HD, 1, 4>(c, a);
  if (nq <= 32) return launch_tree<T, HD, 2, 4>(c, a);
  if (nq <= 64 || HD > 128) return launch_tree<T, HD, 4, 2>(c, a);
  if constexpr (HD <= 128) return launch_tree<T, HD, 8, 1>(c, a);
  return ULB_OK;
}

template <typename T>
int pick_dim(Ctx* c, TreeArgs& a) {
  switch (a.g.hd) {
    case 64: return pick_tree<T, 64>(c, a);
    case 80: return pick_tree<T, 80>(c, a);
    case 96: return pick_tree<T, 96>(c, a);
    case 128: return pick_tree<T, 128>(c, a);
    default: return pick_tree<T, 256>(c, a);
  }
}

}  // namespace
}  // namespace ulb

using namespace ulb;

extern "C" int ulb_tree_attention(ulb_ctx* ctx, const ulb_cache_desc* cache, const ulb_tree_desc* d, const void* q, const void* k,
                                  const void* v, const int32_t* table, const int32_t* row_start, const int32_t* prefix,
                                  const int32_t* len, const uint32_t* mask, void* out, float* lse) {
  ULB_CHECK(ctx && d, ULB_EINVAL, "ulb_tree_attention: NULL argument");
  TreeArgs a = {};
  ULB_TRY(cache_geom("ulb_tree_attention", cache, &a.g));
  ULB_CHECK(a.g.hd == 64 || a.g.hd == 80 || a.g.hd == 96 || a.g.hd == 128 || a.g.hd == 256, ULB_EUNSUPPORTED,
            "ulb_tree_attention: head_dim %d (64, 80, 96, 128 or 256)", a.g.hd);
  ULB_CHECK(d->n_head > 0 && d->n_head % a.g.n_head_kv == 0 && d->n_head / a.g.n_head_kv <= 64, ULB_EINVAL,
            "ulb_tree_attention: %d heads over %d kv heads", d->n_head, a.g.n_head_kv);
  ULB_CHECK(d->rows >= 0 && d->max_rows >= 0 && d->max_len >= 0 && d->mask_words >= 0, ULB_EINVAL,
            "ulb_tree_attention: %d rows, at most %d a sequence over %d positions, %d mask words", d->rows, d->max_rows, d->max_len,
            d->mask_words);
  ULB_CHECK(std::isfinite(d->scale) && d->scale > 0.f, ULB_EINVAL, "ulb_tree_attention: scale %g", (double)d->scale);
  ULB_CHECK(a.g.n_seq <= 65535, ULB_EUNSUPPORTED, "ulb_tree_attention: %d sequences (at most 65535)", a.g.n_seq);
  if (d->rows == 0 || d->max_rows == 0) return ULB_OK;
  ULB_CHECK(q && k && v && table && row_start && prefix && len && out, ULB_EINVAL, "ulb_tree_attention: NULL argument");
  ULB_CHECK(!mask == (d->mask_words == 0), ULB_EINVAL, "ulb_tree_attention: mask without mask_words, or the reverse");
  ULB_CHECK(ULB_ALIGNED16(q) && ULB_ALIGNED16(k) && ULB_ALIGNED16(v) && ULB_ALIGNED16(out), ULB_EINVAL,
            "ulb_tree_attention: q, the pools and out must be 16-byte aligned");
  ULB_CHECK(words_aligned({table, row_start, prefix, len, mask, lse}), ULB_EINVAL, "ulb_tree_attention: unaligned array of 32-bit elements");
  a.H = d->n_head;
  a.G = d->n_head / a.g.n_head_kv;
  a.rows = d->rows;
  a.max_rows = std::min(d->max_rows, d->rows);
  a.max_len = std::min(d->max_len, a.g.max_pages * a.g.page);
  ULB_CHECK((long long)a.max_rows * a.G < (1ll << 31) && (long long)d->rows * d->n_head < (1ll << 31), ULB_EUNSUPPORTED,
            "ulb_tree_attention: %d rows of %d heads", d->rows, d->n_head);
  ULB_CHECK(a.max_len <= 0x7fff0000, ULB_EUNSUPPORTED, "ulb_tree_attention: %d positions", a.max_len);
  a.words = d->mask_words;
  a.scale2 = d->scale * kLog2e;
  a.q = q;
  a.k = k;
  a.v = v;
  a.table = table;
  a.row_start = row_start;
  a.prefix = prefix;
  a.len = len;
  a.mask = mask;
  a.out = out;
  a.lse = lse;
  a.err = ctx->c.dev_err;
  Ctx* c = &ctx->c;
  ULB_CUDA(cudaSetDevice(c->device));
  /* at the first call, whatever its shape, so that any later one can be captured */
  if (!c->tree_ws) ULB_CUDA(cudaMalloc((void**)&c->tree_ws, kTreeWsFloats * sizeof(float)));
  if (tree_tc_fits(c, a)) return launch_tree_tc(c, a, cache->dtype == ULB_TYPE_F16);
  return cache->dtype == ULB_TYPE_F16 ? pick_dim<__half>(c, a) : pick_dim<__nv_bfloat16>(c, a);
}

ULB_TRACE_UNIT(tree_attention)
