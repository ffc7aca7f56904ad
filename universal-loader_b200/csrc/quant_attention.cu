/*
 * quant_attention.cu — attention of a step's new rows over a paged cache held in 8 or 4 bits
 * (ulb_quant_attention).  Rows, masks and promises are those of ulb_tree_attention (tree_attention.cu);
 * the reference has no quantised cache (src/inference/model.h:49-77).
 *
 * Mathematics.  A K or V row is d_g c (+ m_g) with integer codes c and a scale (and minimum) a group g of 32
 * elements; 4-bit codes are taken less 8 and m_g as the middle m_g + 8 d_g, so that the weighted codes are no larger than
 * what they add up to (with codes from 0 the rounding of their weights showed 2.4 times the output's own).  Nothing is
 * expanded to 16-bit values:
 *   s_t   = scale sum_g [ d_tg (q_g . c_tg) + m_tg sum(q_g) ]          fp32 sums of exact products
 *   o_gi  = sum_t (p_t d_tg) c_tgi + sum_t p_t m_tg,   p_t = exp(s_t - M)
 * The codes are exact fp16 integers, so the one rounding is that of the weight p_t d_tg to fp16: 2^-11, an eighth of a bf16
 * output's own; fp16 outputs take a second part of each weight, since one part adds as much as the output's rounding (500
 * keys: 3.0e-4 against 64 bits, the rounding alone 2.1e-4).  M is the running
 * maximum of s_t + log d_t (d_t the largest scale of the V row), so weights are at most 2^(RAISE + GROW) whatever the
 * scales are, and fp16 keeps 11 bits of one down to 2^-26 of the heaviest; p_t itself and what it sums to
 * are fp32 (a scale is at least 2^-24, so p_t stays in range).  q is scaled by a power of two a row, which drops out of the
 * scores exactly: the row's largest element comes to [2^15, 2^16), the top of fp16's range, so that the others keep their
 * bits (11 of fp16, 8 of bf16) down to 2^-29 of that power of two and are off by 2^-40 of it below; the elements that
 * 4 bits want as q / 16 (below) down to 2^-25, and 2^-36.  With the largest at 1, as the scores' range alone would have it, an
 * element 2^-17 of it had 7 bits left, or 3.
 *
 * Work.  A K and a V row take 80 (4 bits) or 144 bytes at head_dim 128.  K^T Q and V P are mma.sync m16n8k16 with
 * the codes as the 16-row operand (keys x dims, then dims x keys) and eight queries as columns, so a product wastes
 * nothing on padding at eight queries and a code is unpacked once for all of them.  K's codes are masked out of their word and
 * used as they are: the bits of a small integer n are the fp16 subnormal n 2^-24.  The parts of a score that only the scales
 * give (m_g sum q, or -128 d_g sum q for offset bytes) are one more product, of the scales' own words with those sums in two
 * fp16 parts.  V's codes are centred (one LOP3 or PRMT and one HADD2 or HFMA2 for two), because the sums run over
 * many keys.  The dims a lane takes of a row are four in a row of each 16 for the first product and four of each 32 for the
 * second, so every shared-memory read is a conflict-free 32-bit word of the rows as they lie in HBM (head_dim 256 in 4 bits:
 * two ways).
 *
 * A warp walks 32-key tiles of its own, 16 keys at a time, through its own ring of bulk copies, which one more warp
 * issues for all, a lane a ring.  The tiles of all (sequence, row tile, kv head) units form one line that is cut evenly
 * over the blocks, so lengths may differ as they like; a unit in several blocks leaves a partial in each and the last
 * of them to arrive joins them in order.  While a unit's tiles are worked on, the next unit's rows of q are made.
 *
 * Measured (bf16): 64 sequences of 256 to 8192 keys, 32 heads over 8 of 128, 4 bits: 112 to 118 us, 3.0 to 3.1 TB/s (46 to
 * 47 % of the copy rate); 5 rows over 100001 keys, 64 heads over 8, 8 bits: 137 to 141 us; 1 x 20000 keys 20 (4 bits) and 22
 * us; 64 x 1000 keys in 8 bits 43 us, half of the copy rate; 16 x 4000 keys, 16 heads over 4 of 256, 45 (4 bits) and 41 us; 16
 * rows of a tree over 4000 keys, 8 sequences, 108 and 97 us, as many in a chain 106 and 96.  No pipe is full (54 % of the
 * issue slots): what bounds it is the order of dependent instructions in few warps, about 450 a warp for 16 keys of eight
 * queries in 4 bits, of which unpacking V, the weights of its groups and their transposition are half; with more queries
 * the weights of each 8 more, and past 32 the keys are walked again.  Tried and slower: 16 warps of 128 registers (170 us
 * for the 113 of the time), a warp that feeds itself (135), all 32 keys in one body (the code leaves the instruction
 * cache; 157).
 */
#include "quant_cache.h"
#include "tcgen05.h"
#include "tree_attention.h"

#include <algorithm>
#include <cmath>

namespace ulb {
namespace {

constexpr float kRaise = 12.f, kGrow = 3.9f; /* weights <= 2^15.9 < 65504 */
/* powers of two of a row's largest element and, against elements in [1, 2), of the sums of 32 (<= 64, so < 2^15) as fp16 */
constexpr int kTopQ = 15, kTopSum = 9;
constexpr unsigned kAll = 0xffffffffu;

template <bool Q4, int HD, int NT>
struct QCfg {
  static constexpr int RB = quant_row_bytes(Q4, HD), CB = quant_code_bytes(Q4, HD);
  static constexpr int KT = HD == 256 && !Q4 ? 16 : 32; /* keys a tile */
  static constexpr int STAGE = 2 * KT * RB;
  /*
   * Working warps (one more copies), and blocks on an SM; with the copying warp a block's are a multiple of four wherever the
   * registers do not say otherwise, since they are given out so.  Eight queries: two blocks of 5 hide what a unit costs
   * besides its tiles behind each other's work: 64 sequences of 100 to 1000 keys, 32 kv heads of 64 71 us (one block of 11
   * warps 94, three of 3 64), 64 x 256-8192 keys in 4 bits 113 (105, 121), 64 x 20-100 keys 16 (25, 19).  More queries: the
   * registers of 7 warps.
   */
  static constexpr int W = HD == 256 ? 3 : NT == 1 ? 5 : HD == 64 && NT < 4 ? 11 : 7;
  static constexpr int CTAS = HD == 256 || NT == 1 ? 2 : 1;
  /* what a unit costs besides its tiles, in tiles, and the places of the line a block takes at least: fitted */
  static constexpr int UNIT = NT == 1 && HD < 256 ? 16 : 32, MIN = UNIT / 2;
  static constexpr int RT = 8 * NT; /* queries a CTA */
  static constexpr int NG = HD / kGroup, KS = HD / 16;
  static constexpr int NW = Q4 ? NG : NG / 2, NC = (NW + 3) / 4; /* 32-bit words of a row's scales, products that take them */
  static constexpr int QB = 2 * NT * (KS + NC) * 256; /* bytes of two units' fragments of q */
  static constexpr int QS = QB / 2 / 8;               /* 8-byte words of one unit's */
  static constexpr int ALL = 227 * 1024 / CTAS - 1024 - 2560; /* the SM's, less what a CTA has besides */
  static constexpr int JD0 = HD == 64 || NT > 1 ? 64 : 128; /* dims the warps join at a time, 32 where the ring wants the room */
  static constexpr int JD = (ALL - QB - W * RT * JD0 * 4) / (W * STAGE) >= 2 ? JD0 : 32;
  static constexpr int JB = W * RT * JD * 4;
  static constexpr int ROOM = (ALL - QB - JB) / (W * STAGE);
  static constexpr int NST = ROOM > 6 ? 6 : ROOM;
  static constexpr int SMEM = W * NST * STAGE + QB + JB;
  static_assert(NST >= 2 && W <= 31, "shared memory, a lane a ring");
};

struct QuantPlan {
  int groups, min_tiles;
  int* tail; /* [groups][2]: arrivals at the unit that begins in this CTA and goes on, the slot of its first piece */
};

/* the line of work, in tiles: a unit takes UNIT places before its tiles.  CTA c's stretch. */
struct QLine {
  int total, groups, per, rem;
  __device__ __forceinline__ void cut(int n) {
    groups = n;
    per = total / n;
    rem = total - per * n;
  }
  __device__ __forceinline__ int begin(int c) const { return c * per + min(c, rem); }
  __device__ __forceinline__ int group_of(int place) const {
    const int big = rem * (per + 1);
    return place < big ? place / (per + 1) : rem + (place - big) / per;
  }
};

struct QPiece {
  TreeSeq q;
  int s, kvh, q0, nq;     /* sequence, kv head, first query (row x group + head) of the row tile, queries in it */
  int t0, n, n_tile;      /* tiles [t0, t0 + n) of n_tile */
  int first, last;        /* places of the unit's first and last tiles on the line */
  int nth;                /* pieces of this CTA before it */
};

template <int RT, int KT, int UNIT>
struct QWalk {
  int at, end, base, cnt, s, n_tile, n_pass, nth;
  TreeSeq q;
  __device__ __forceinline__ void load(const TreeArgs& a) {
    q = tree_seq(a, s);
    n_tile = max(1, (q.len + KT - 1) / KT);
    n_pass = (q.n * a.G + RT - 1) / RT;
    cnt = (n_tile + UNIT) * n_pass * a.g.n_head_kv;
  }
  __device__ __forceinline__ bool next(const TreeArgs& a, QPiece* o) {
    while (at < end) {
      while (at >= base + cnt) { /* ends: at < end <= total */
        base += cnt;
        ++s;
        load(a);
      }
      const int len = n_tile + UNIT, u = (at - base) / len, in = at - base - u * len, upto = min(len, in + end - at);
      o->t0 = max(in - UNIT, 0);
      o->n = max(upto - UNIT, 0) - o->t0;
      o->first = base + u * len + UNIT;
      o->last = base + u * len + len - 1;
      at += upto - in;
      if (o->n <= 0) continue; /* none of its tiles yet */
      o->kvh = u / n_pass;
      o->q0 = (u - o->kvh * n_pass) * RT;
      o->nq = min(RT, q.n * a.G - o->q0);
      o->q = q;
      o->s = s;
      o->n_tile = n_tile;
      o->nth = nth++;
      return true;
    }
    return false;
  }
};

__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2(float a, float b) { return pack2<__half>(a, b); }
__device__ __forceinline__ uint32_t lds32(const uint8_t* p) { return *reinterpret_cast<const uint32_t*>(p); }
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t magic) { /* a - magic, fp16 pairs */
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&magic));
  return *reinterpret_cast<const uint32_t*>(&r);
}
/* nibbles at bits 0 and 16 as two fp16 integers n - 8: 0x6400 | n is 1024 + n, 0x6408 is 1032 */
__device__ __forceinline__ uint32_t nib_lo(uint32_t w) { return sub2((w & 0x000f000fu) | 0x64006400u, 0x64086408u); }
/* nibbles at bits 4 and 20: 1024 + 16 n, then x / 16 - 72 */
__device__ __forceinline__ uint32_t nib_hi(uint32_t w) {
  const uint32_t x = (w & 0x00f000f0u) | 0x64006400u, s = 0x2c002c00u, o = 0xd480d480u; /* 1/16, -72 */
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&s), *reinterpret_cast<const __half2*>(&o));
  return *reinterpret_cast<const uint32_t*>(&r);
}
/* bytes lo and lo + 1 of w (offset binary, int8 + 128) as two fp16 integers: 0x64xx is 1024 + xx; 0x6480 is 1152 */
template <int LO> __device__ __forceinline__ uint32_t byte2(uint32_t w) {
  return sub2(__byte_perm(w, 0x64646464u, LO ? 0x4342 : 0x4140), 0x64806480u);
}
/* K's codes need no more than their place: the bits of a small integer n are the subnormal n 2^-24.  (V's sums run over many
   keys, in which an offset that is taken off at the end would cost bits, so its codes are centred.) */
template <int LO> __device__ __forceinline__ uint32_t raw2(uint32_t w) { return __byte_perm(w, 0u, LO ? 0x4342 : 0x4140); }

/* scales of a row (and the middles m + 8 d, which go with codes less 8) */
template <bool Q4, int NG>
__device__ __forceinline__ void row_scales(const uint8_t* p, float (&d)[NG], float (&m)[NG]) {
  if constexpr (Q4) {
#pragma unroll
    for (int i = 0; i < NG; i += 2) {
      const uint2 w = *reinterpret_cast<const uint2*>(p + 4 * i);
      const float2 x = unpack2<__half>(w.x), y = unpack2<__half>(w.y);
      d[i] = x.x;
      m[i] = __fmaf_rn(8.f, x.x, x.y);
      d[i + 1] = y.x;
      m[i + 1] = __fmaf_rn(8.f, y.x, y.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NG; i += 2) {
      const float2 x = unpack2<__half>(lds32(p + 2 * i));
      d[i] = x.x;
      d[i + 1] = x.y;
    }
  }
}

/* the scales alone */
template <bool Q4, int NG>
__device__ __forceinline__ void first_scales(const uint8_t* p, float (&d)[NG]) {
#pragma unroll
  for (int i = 0; i < NG; i += 2) {
    float2 x;
    if constexpr (Q4) {
      const uint2 w = *reinterpret_cast<const uint2*>(p + 4 * i);
      x = make_float2(unpack2<__half>(w.x).x, unpack2<__half>(w.y).x);
    } else {
      x = unpack2<__half>(lds32(p + 2 * i));
    }
    d[i] = x.x;
    d[i + 1] = x.y;
  }
}

template <typename T, bool Q4, int HD, int NT>
__global__ void __launch_bounds__(QCfg<Q4, HD, NT>::W * 32 + 32, QCfg<Q4, HD, NT>::CTAS)
    quant_attn_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ QuantPlan p) {
  using C = QCfg<Q4, HD, NT>;
  constexpr int W = C::W, NG = C::NG, NTH = W * 32 + 32, JD = C::JD, KT = C::KT, US = KT / 16;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ uint64_t full[W][C::NST], empty[W][C::NST];
  __shared__ uint8_t sh_map[W][C::NST]; /* which 16-key halves of a tile are mapped */
  __shared__ float2 sh_ml[2][W][C::RT];
  __shared__ float sh_qs[2][C::RT];
  __shared__ QWalk<C::RT, C::KT, C::UNIT> sh_walk;
  __shared__ QPiece sh_pc[4];
  __shared__ int sh_have[4], sh_s, sh_base, sh_sum[W + 1], sh_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint2* const q_sm = reinterpret_cast<uint2*>(sm + W * C::NST * C::STAGE);
  float* const jb = reinterpret_cast<float*>(sm + W * C::NST * C::STAGE + C::QB);

  if (lane == 0 && warp < W) {
    for (int i = 0; i < C::NST; ++i) {
      mb_init(&full[warp][i], 1);
      mb_init(&empty[warp][i], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 0) { sh_s = 0; sh_base = 0; }
  for (int i = tid; i < 2 * C::QS; i += NTH) q_sm[i] = make_uint2(0, 0); /* scales that a row does not have */
  pdl_wait();
  pdl_trigger();

  /* the line's length, then this CTA's stretch and the sequence that holds its begin */
  QWalk<C::RT, C::KT, C::UNIT> walk;
  auto places_of = [&](int s) {
    if (s >= a.g.n_seq) return 0;
    QWalk<C::RT, C::KT, C::UNIT> w;
    w.s = s;
    w.load(a);
    return w.cnt;
  };
  const int cnt0 = places_of(tid);
  int mine = cnt0;
  for (int s = tid + NTH; s < a.g.n_seq; s += NTH) mine += places_of(s);
  mine = __reduce_add_sync(kAll, mine);
  if (lane == 0) sh_sum[warp] = mine;
  __syncthreads();
  QLine line;
  line.total = 0;
#pragma unroll
  for (int w = 0; w <= W; ++w) line.total += sh_sum[w];
  line.cut(max(1, min(p.groups, (line.total + p.min_tiles - 1) / p.min_tiles)));
  const int grp_id = blockIdx.x;
  walk.at = grp_id < line.groups ? line.begin(grp_id) : line.total;
  walk.end = grp_id < line.groups ? line.begin(grp_id + 1) : line.total;
  {
    int base = 0;
    for (int s0 = 0; s0 < a.g.n_seq && walk.at < walk.end; s0 += NTH) {
      const int c = s0 == 0 ? cnt0 : places_of(s0 + tid);
      int x = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(kAll, x, o);
        if (lane >= o) x += y;
      }
      __syncthreads();
      if (lane == 31) sh_sum[warp] = x;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int w = 0; w <= W; ++w) {
        if (w < warp) x += sh_sum[w];
        all += sh_sum[w];
      }
      const int b = base + x - c;
      if (c > 0 && b <= walk.at && walk.at < b + c) {
        sh_s = s0 + tid;
        sh_base = b;
      }
      base += all;
      if (base > walk.at) break; /* the same for every thread */
    }
    __syncthreads();
  }
  if (walk.at >= walk.end) return; /* the whole CTA */
  walk.s = sh_s;
  walk.base = sh_base;
  walk.nth = 0;
  walk.load(a);

  if (warp == W) {
    /* ------------------------------------------------ the copying warp: a lane feeds a working warp's ring, ahead of its
       use and past the ends of pieces */
    const uint8_t* const kb = (const uint8_t*)a.k;
    const uint8_t* const vb = (const uint8_t*)a.v;
    uint8_t* const ring = sm + min(lane, W - 1) * C::NST * C::STAGE;
    uint64_t *const f_bar = full[min(lane, W - 1)], *const e_bar = empty[min(lane, W - 1)];
    int slot = 0;
    uint32_t phase = 1; /* the first round passes */
    bool ok = true;
    QPiece pc;
    __syncthreads(); /* with the working warps' first */
    while (ok && walk.next(a, &pc)) {
      auto page_at = [&](int pos) {
        const int j = pos >> a.g.page_shift;
        const int x = pos < pc.q.len && j < a.g.max_pages ? a.table[(long long)pc.s * a.g.max_pages + j] : -1;
        return x >= 0 && x < a.g.n_pages ? x : -1;
      };
      const long long h = pc.kvh * a.g.head;
      const int in_page = a.g.page - 1;
      int id0 = -1, id1 = -1;
      auto ids = [&](int i) { /* the pages of tile i, read a round ahead */
        const int pos = (pc.t0 + i) * KT;
        const bool mine = lane < W && i < pc.n;
        id0 = mine ? page_at(pos) : -1;
        id1 = mine && a.g.page == 16 && KT > 16 ? page_at(pos + 16) : id0;
      };
      ids(lane);
      for (int i0 = 0; i0 < pc.n && ok; i0 += W) {
        const int i = i0 + lane, p0 = id0, p1 = id1;
        const bool mine = lane < W && i < pc.n;
        if (i0 + W < pc.n) ids(i + W);
        if (mine) ok = mb_wait(&e_bar[slot], phase);
        ok = __all_sync(kAll, ok);
        if (mine && ok) {
          const int pos = (pc.t0 + i) * KT, rows = min(KT, pc.q.len - pos);
          uint8_t* const d = ring + slot * C::STAGE;
          uint64_t* const bar = &f_bar[slot];
          if (a.g.page == 16) {
            const int r0 = p0 >= 0 ? min(rows, 16) : 0, r1 = KT > 16 && p1 >= 0 ? rows - 16 : 0; /* rows <= 0: none */
            sh_map[lane][slot] = (p0 >= 0 ? 1 : 0) | (p1 >= 0 ? 2 : 0);
            mb_expect(bar, (uint32_t)(2 * (max(r0, 0) + max(r1, 0)) * C::RB));
            if (r0 > 0) {
              bulk_copy(d, kb + p0 * a.g.pstride + h, r0 * C::RB, bar);
              bulk_copy(d + KT * C::RB, vb + p0 * a.g.pstride + h, r0 * C::RB, bar);
            }
            if (r1 > 0) {
              bulk_copy(d + 16 * C::RB, kb + p1 * a.g.pstride + h, r1 * C::RB, bar);
              bulk_copy(d + (KT + 16) * C::RB, vb + p1 * a.g.pstride + h, r1 * C::RB, bar);
            }
          } else {
            const int r = p0 >= 0 ? max(rows, 0) : 0;
            sh_map[lane][slot] = p0 >= 0 ? 3 : 0;
            mb_expect(bar, (uint32_t)(2 * r * C::RB));
            if (r > 0) {
              const long long off = p0 * a.g.pstride + h + (long long)(pos & in_page) * C::RB;
              bulk_copy(d, kb + off, r * C::RB, bar);
              bulk_copy(d + KT * C::RB, vb + off, r * C::RB, bar);
            }
          }
          if (++slot == C::NST) { slot = 0; phase ^= 1; }
        }
      }
    }
    /* no copy is in flight when the CTA ends: the working warps wait for all of them, and this one where they gave up */
    if (!ok) {
      for (int i = 0; i < C::NST; ++i) mb_wait(&f_bar[i], phase ^ (i < slot ? 1u : 0u)); /* this round's, the last one's */
      if (lane == 0) atomicOr(a.err, 8);
    }
    return;
  }
  /* ------------------------------------------------ the working warps */
  uint8_t* const ring = sm + warp * C::NST * C::STAGE;
  bool ok = true;
  /* piece k is in place k % 4; warp 0 looks for piece k + 2 at the end of piece k */
  auto advance = [&](int k) {
    QWalk<C::RT, C::KT, C::UNIT> w = sh_walk;
    QPiece x;
    const bool more = w.next(a, &x);
    __syncwarp();
    if (lane == 0) {
      sh_walk = w;
      sh_pc[k & 3] = x;
      sh_have[k & 3] = more;
    }
    __syncwarp();
  };
  int slot = 0;
  uint32_t phase = 0;
  auto sync_work = [] { asm volatile("bar.sync 1, %0;" ::"n"(W * 32) : "memory"); };
  /* rows of q: scaled by a power of two, as fragments; sums of the groups.  Two buffers: a unit's rows are made while the
     warps before it still work */
  auto load_q = [&](const QPiece& c, int buf) {
    uint2* const qb = q_sm + buf * C::QS;
    uint2* const qc = qb + NT * C::KS * 32; /* second operands of the products with K's scales */
    for (int qi = warp; qi < C::RT; qi += W) {
      constexpr int N4 = HD / 128 > 0 ? HD / 128 : 1; /* runs of four elements a lane */
      float x[N4][4];
      float top = 0.f;
      const int gq = c.q0 + qi;
      const T* src = (const T*)a.q + ((long long)(c.q.r0 + gq / a.G) * a.H + c.kvh * a.G + gq % a.G) * HD;
#pragma unroll
      for (int i = 0; i < N4; ++i) {
        const int d = (i * 32 + lane) * 4;
        uint2 w = make_uint2(0, 0);
        if (qi < c.nq && d < HD) w = *reinterpret_cast<const uint2*>(src + d);
        const float2 u = unpack2<T>(w.x), v = unpack2<T>(w.y);
        x[i][0] = u.x; x[i][1] = u.y; x[i][2] = v.x; x[i][3] = v.y;
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[i][e]));
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
      const int ex = max(-126, min(127, top > 0.f ? ilogbf(top) : 0)), el = kTopQ - ex;
#pragma unroll
      for (int i = 0; i < N4; ++i) {
        const int d = (i * 32 + lane) * 4;
        /* 4 bits: elements 2 and 3 of a word come as 16 n */
        const int eh = Q4 ? el - 4 : el;
        const uint32_t lo = h2(ldexpf(x[i][0], el), ldexpf(x[i][1], el)), hi = h2(ldexpf(x[i][2], eh), ldexpf(x[i][3], eh));
        const float2 u = unpack2<__half>(lo), v = unpack2<__half>(hi);
        float sum = (u.x + u.y) + (Q4 ? 16.f : 1.f) * (v.x + v.y);
#pragma unroll
        for (int o = 4; o; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
        if (d < HD) qb[((qi >> 3) * C::KS + (d >> 4)) * 32 + (qi & 7) * 4 + ((d >> 2) & 3)] = make_uint2(lo, hi);
        /* s has sum(q) m (4 bits), or -128 sum(q) d (codes are offset by 128; the 2^7 comes with the score's factor), of each
           group: the words of a row's scales as operands (d, m) or (d, d of the next), these sums in two parts beside them */
        sum *= (Q4 ? 1.f : -1.f) / (float)(1 << (kTopQ - kTopSum));
        const float next = __shfl_down_sync(kAll, sum, 8), top16 = to_f<__half>(from_f<__half>(sum)), next16 = to_f<__half>(from_f<__half>(next));
        const int word = Q4 ? d >> 5 : d >> 6;
        if (d < HD && d % (Q4 ? 32 : 64) == 0) {
          const int at = ((qi >> 3) * C::NC + (word >> 2)) * 32 + (qi & 7) * 4 + (word & 3);
          qc[at] = Q4 ? make_uint2(h2(0.f, top16), h2(0.f, sum - top16)) : make_uint2(h2(top16, next16), h2(sum - top16, next - next16));
        }
      }
      if (lane == 0) sh_qs[buf][qi] = ldexpf(a.scale2, ex - kTopSum + (Q4 ? 0 : 7));
    }
  };
  if (warp == 0) {
    if (lane == 0) sh_walk = walk;
    __syncwarp();
    advance(0);
  }
  __syncthreads();
  if (sh_have[0]) load_q(sh_pc[0], 0); /* the stretch may hold no tile */
  if (warp == 0) advance(1);
  sync_work();
  for (int k = 0; sh_have[k & 3]; ++k) {
    const int buf = k & 1;
    const QPiece& pc = sh_pc[k & 3];
    const uint2* const qf = q_sm + buf * C::QS;
    const uint2* const qc = qf + NT * C::KS * 32;
    float sc[NT][2], m[NT][2], l[NT][2];
    float om[Q4 ? NG : 1][NT][2];
    float o[HD / 16][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sc[n][e] = sh_qs[buf][n * 8 + 2 * t + e];
        m[n][e] = -INFINITY;
        l[n][e] = 0.f;
        if constexpr (Q4) {
#pragma unroll
          for (int i = 0; i < NG; ++i) om[i][n][e] = 0.f;
        }
      }
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
    const int open = min(tree_open(a, pc.q), pc.q.len);
    constexpr bool QR = NT == 1; /* fragments of q in registers */
    uint2 qr[QR ? C::KS : 1];
    if constexpr (QR) {
#pragma unroll
      for (int i = 0; i < C::KS; ++i) qr[i] = qf[i * 32 + lane];
    }

    const int n_own = (pc.n + W - 1 - warp) / W, first = (pc.t0 + warp) * KT;
    for (int it = 0; it < n_own && ok; ++it) {
      const int pos0 = first + it * W * KT;
      if (!mb_wait_warp(&full[warp][slot], phase)) { ok = false; break; }
      const uint8_t* const kt = ring + slot * C::STAGE;
      const uint8_t* const vt = kt + KT * C::RB;
      const int map = sh_map[warp][slot];
      const bool masked = pos0 + KT > open || map != 3;
#pragma unroll 1
      for (int u = 0; u < US; ++u) { /* 16 keys at a time: half the code, which would not fit the instruction cache */
        const uint8_t *const k0 = kt + (u * 16 + g) * C::RB, *const k1 = k0 + 8 * C::RB, *const vr = vt + (u * 16 + g) * C::RB;
        float s[NT][4];
        /* ---- scores: sums of codes by group, in units of 2^-24 2^kTopQ, and the part that the scales alone give, of 2^kTopSum */
        {
          float d0[NG], d1[NG];
          first_scales<Q4, NG>(k0 + C::CB, d0);
          first_scales<Q4, NG>(k1 + C::CB, d1);
          float c0[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
            c0[n][0] = c0[n][1] = c0[n][2] = c0[n][3] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < C::NC; ++i) {
            uint32_t f[4] = {0, 0, 0, 0};
            if (C::NW % 4 == 0 || i * 4 + t < C::NW) {
              f[0] = f[2] = lds32(k0 + C::CB + i * 16 + 4 * t);
              f[1] = f[3] = lds32(k1 + C::CB + i * 16 + 4 * t);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint2 y = qc[(n * C::NC + i) * 32 + lane];
              mma16(c0[n], f, y.x, y.y);
            }
          }
          auto group = [&](int i, const uint32_t (&a0)[4], const uint32_t (&a1)[4]) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              const uint2 b0 = QR ? qr[(2 * i) % (QR ? C::KS : 1)] : qf[(n * C::KS + 2 * i) * 32 + lane];
              const uint2 b1 = QR ? qr[(2 * i + 1) % (QR ? C::KS : 1)] : qf[(n * C::KS + 2 * i + 1) * 32 + lane];
              mma16(c, a0, b0.x, b0.y);
              mma16(c, a1, b1.x, b1.y);
              s[n][0] = __fmaf_rn(d0[i], c[0], s[n][0]);
              s[n][1] = __fmaf_rn(d0[i], c[1], s[n][1]);
              s[n][2] = __fmaf_rn(d1[i], c[2], s[n][2]);
              s[n][3] = __fmaf_rn(d1[i], c[3], s[n][3]);
            }
          };
          if constexpr (Q4) {
#pragma unroll
            for (int i = 0; i < NG; i += 2) {
              const int at = i * 16 + 4 * t;
              uint32_t x0 = lds32(k0 + at), x1 = lds32(k1 + at), y0 = lds32(k0 + at + 16), y1 = lds32(k1 + at + 16);
              constexpr uint32_t L = 0x000f000fu, H = 0x00f000f0u;
              {
                const uint32_t f0[4] = {x0 & L, x1 & L, x0 & H, x1 & H}, f1[4] = {y0 & L, y1 & L, y0 & H, y1 & H};
                group(i, f0, f1);
              }
              x0 >>= 8; x1 >>= 8; y0 >>= 8; y1 >>= 8;
              {
                const uint32_t f0[4] = {x0 & L, x1 & L, x0 & H, x1 & H}, f1[4] = {y0 & L, y1 & L, y0 & H, y1 & H};
                group(i + 1, f0, f1);
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < NG; ++i) {
              const int at = i * 32 + 4 * t;
              const uint32_t x0 = lds32(k0 + at) ^ 0x80808080u, x1 = lds32(k1 + at) ^ 0x80808080u, y0 = lds32(k0 + at + 16) ^ 0x80808080u,
                             y1 = lds32(k1 + at + 16) ^ 0x80808080u;
              const uint32_t f0[4] = {raw2<0>(x0), raw2<0>(x1), raw2<1>(x0), raw2<1>(x1)}, f1[4] = {raw2<0>(y0), raw2<0>(y1), raw2<1>(y0), raw2<1>(y1)};
              group(i, f0, f1);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = __fmaf_rn(s[n][e], (float)(1 << (24 - kTopQ + kTopSum - (Q4 ? 0 : 7))), c0[n][e]);
        }
        /* ---- V's scales and middles, the logarithm of each row's largest scale */
        float vd[2][NG], vm[2][NG], lg[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          row_scales<Q4, NG>(vr + r * 8 * C::RB + C::CB, vd[r], vm[r]);
          float x = 5.9604645e-8f; /* 2^-24, the smallest scale there is: a row of zeros counts as that */
#pragma unroll
          for (int i = 0; i < NG; i += 2) x = max3(x, vd[r][i], vd[r][i + 1]);
          lg[r] = __log2f(x);
        }
        uint32_t seen[NT][2]; /* of both queries of key g and of key g + 8, as a mask on packed weights */
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          seen[n][0] = seen[n][1] = 0xffffffffu;
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] *= sc[n][e & 1];
        }
        if (masked) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int pos = pos0 + u * 16 + (e >> 1) * 8 + g, qi = pc.q0 + n * 8 + 2 * t + (e & 1);
              const bool see = (map >> u & 1) && pos < pc.q.len && qi < pc.q0 + pc.nq && (pos < open || tree_sees(a, pc.q, qi / a.G, pos));
              if (!see) {
                s[n][e] = -INFINITY;
                seen[n][e >> 1] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
              }
            }
          if constexpr (Q4) { /* a group that is not finite is so in its scale */
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int i = 0; i < NG; ++i)
                if (!isfinite(vm[r][i])) vm[r][i] = 0.f;
          }
        }
        float top[NT][2];
        bool grow = false; /* by the lane's own keys; m is the same in all lanes of a query */
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            top[n][e] = fmaxf(s[n][e] + lg[0], s[n][2 + e] + lg[1]);
            grow |= top[n][e] - kRaise - kGrow > m[n][e];
          }
        if (__any_sync(kAll, grow)) { /* a row's first keys, seldom later */
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) top[n][e] = fmaxf(top[n][e], __shfl_xor_sync(kAll, top[n][e], x));
              const float to = top[n][e] - kRaise;
              if (to - kGrow > m[n][e]) {
                const float f = m[n][e] == -INFINITY ? 0.f : ex2(m[n][e] - to);
                m[n][e] = to;
                l[n][e] *= f;
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) {
                  o[i][n][e] *= f;
                  o[i][n][2 + e] *= f;
                }
                if constexpr (Q4) {
#pragma unroll
                  for (int i = 0; i < NG; ++i) om[i][n][e] *= f;
                }
              }
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mm = m[n][e] == -INFINITY ? 0.f : m[n][e];
            s[n][e] = ex2(s[n][e] - mm);
            s[n][2 + e] = ex2(s[n][2 + e] - mm);
            l[n][e] += s[n][e] + s[n][2 + e];
          }
        /* ---- o += V^T (p d), middles apart */
        const uint8_t* const v0 = vt + (u * 16 + 2 * t) * C::RB;
        auto product = [&](int i, const uint32_t (&f0)[4], const uint32_t (&f1)[4]) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (Q4) {
#pragma unroll
              for (int e = 0; e < 2; ++e) om[i][n][e] = __fmaf_rn(s[n][2 + e], vm[1][i], __fmaf_rn(s[n][e], vm[0][i], om[i][n][e]));
            }
            const float w0 = s[n][0] * vd[0][i], w1 = s[n][1] * vd[0][i], w2 = s[n][2] * vd[1][i], w3 = s[n][3] * vd[1][i];
            const uint32_t y0 = h2(w0, w1) & seen[n][0], y1 = h2(w2, w3) & seen[n][1];
            const uint32_t b0 = transpose8(y0), b1 = transpose8(y1);
            mma16(o[2 * i][n], f0, b0, b1);
            mma16(o[2 * i + 1][n], f1, b0, b1);
            if constexpr (std::is_same<T, __half>::value) { /* what fp16 leaves of a weight is a second operand */
              const float2 z0 = unpack2<__half>(y0), z1 = unpack2<__half>(y1);
              const uint32_t c0 = transpose8(h2(w0 - z0.x, w1 - z0.y) & seen[n][0]), c1 = transpose8(h2(w2 - z1.x, w3 - z1.y) & seen[n][1]);
              mma16(o[2 * i][n], f0, c0, c1);
              mma16(o[2 * i + 1][n], f1, c0, c1);
            }
          }
        };
        if constexpr (Q4) {
#pragma unroll
          for (int i = 0; i < NG; i += 2) {
            const uint8_t* const w = v0 + i * 16 + 4 * g;
            const uint32_t w0 = lds32(w), w1 = lds32(w + C::RB), w2 = lds32(w + 8 * C::RB), w3 = lds32(w + 9 * C::RB);
            uint32_t x0 = __byte_perm(w0, w1, 0x5410), x1 = __byte_perm(w0, w1, 0x7632), y0 = __byte_perm(w2, w3, 0x5410),
                     y1 = __byte_perm(w2, w3, 0x7632); /* elements 0, 2 and 1, 3 of keys 2 t, 2 t + 1 and 2 t + 8, 2 t + 9 */
            {
              const uint32_t f0[4] = {nib_lo(x0), nib_lo(x1), nib_lo(y0), nib_lo(y1)}, f1[4] = {nib_hi(x0), nib_hi(x1), nib_hi(y0), nib_hi(y1)};
              product(i, f0, f1);
            }
            x0 >>= 8; x1 >>= 8; y0 >>= 8; y1 >>= 8;
            {
              const uint32_t f0[4] = {nib_lo(x0), nib_lo(x1), nib_lo(y0), nib_lo(y1)}, f1[4] = {nib_hi(x0), nib_hi(x1), nib_hi(y0), nib_hi(y1)};
              product(i + 1, f0, f1);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            const uint8_t* const w = v0 + i * 32 + 4 * g;
            const uint32_t w0 = lds32(w) ^ 0x80808080u, w1 = lds32(w + C::RB) ^ 0x80808080u, w2 = lds32(w + 8 * C::RB) ^ 0x80808080u,
                           w3 = lds32(w + 9 * C::RB) ^ 0x80808080u;
            const uint32_t x0 = __byte_perm(w0, w1, 0x5140), x1 = __byte_perm(w0, w1, 0x7362), y0 = __byte_perm(w2, w3, 0x5140),
                           y1 = __byte_perm(w2, w3, 0x7362); /* elements 0, 1 and 2, 3, two keys each */
            const uint32_t f0[4] = {byte2<0>(x0), byte2<1>(x0), byte2<0>(y0), byte2<1>(y0)},
                           f1[4] = {byte2<0>(x1), byte2<1>(x1), byte2<0>(y1), byte2<1>(y1)};
            product(i, f0, f1);
          }
        }
      }
      __syncwarp(); /* every lane has read the tile */
      if (lane == 0) mb_arrive(&empty[warp][slot]);
      if (++slot == C::NST) { slot = 0; phase ^= 1; }
    }

    /* ---- the next unit's rows, then the warps join: each scales its sums to the common maximum */
    if (warp == 0) advance(k + 2);
    if (sh_have[(k + 1) & 3]) load_q(sh_pc[(k + 1) & 3], buf ^ 1);
    const QPiece& c = pc;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n][e] += __shfl_xor_sync(kAll, l[n][e], x);
        if (g == 0) sh_ml[buf][warp][n * 8 + 2 * t + e] = make_float2(m[n][e], l[n][e]);
        if constexpr (Q4) {
#pragma unroll
          for (int i = 0; i < NG; ++i) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) om[i][n][e] += __shfl_xor_sync(kAll, om[i][n][e], x);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              o[2 * i + x][n][e] += om[i][n][e];
              o[2 * i + x][n][2 + e] += om[i][n][e];
            }
          }
        }
      }
    sync_work();
    auto joined = [&](int qi, float* M, float* L) { /* of all warps */
      *M = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) *M = fmaxf(*M, sh_ml[buf][w][qi].x);
      const float U = *M == -INFINITY ? 0.f : *M;
      *L = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) *L += sh_ml[buf][w][qi].y * ex2(sh_ml[buf][w][qi].x - U);
    };
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, sh_ml[buf][w][n * 8 + 2 * t + e].x);
        m[n][e] = ex2(m[n][e] - (M == -INFINITY ? 0.f : M)); /* from here on the factor */
      }
    const bool whole = c.n == c.n_tile;
    const int my_slot = c.nth == 0 ? 0 : 1; /* only a CTA's first and last pieces can be parts */
    const long long ps = ((long long)grp_id * 2 + my_slot) * C::RT;
    auto out_row = [&](int qi) { return (long long)(c.q.r0 + (c.q0 + qi) / a.G) * a.H + c.kvh * a.G + (c.q0 + qi) % a.G; };
#pragma unroll
    for (int d0 = 0; d0 < HD; d0 += JD) {
      if (d0) sync_work(); /* the words of the pass before are read */
#pragma unroll
      for (int i = 0; i < JD / 32; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int f = d0 / 16 + 2 * i;
            const float x = m[n][e];
            *reinterpret_cast<float4*>(jb + (warp * C::RT + n * 8 + 2 * t + e) * JD + i * 32 + 4 * g) =
                make_float4(o[f][n][e] * x, o[f][n][2 + e] * x, o[f + 1][n][e] * x, o[f + 1][n][2 + e] * x);
          }
      sync_work();
      for (int i = tid; i < c.nq * (JD / 4); i += W * 32) {
        const int qi = i / (JD / 4), d = (i % (JD / 4)) * 4;
        float4 x = *reinterpret_cast<const float4*>(jb + qi * JD + d);
#pragma unroll
        for (int w = 1; w < W; ++w) {
          const float4 y = *reinterpret_cast<const float4*>(jb + (w * C::RT + qi) * JD + d);
          x.x += y.x;
          x.y += y.y;
          x.z += y.z;
          x.w += y.w;
        }
        float M, L;
        joined(qi, &M, &L);
        if (whole) {
          const float inv = L == 0.f ? 0.f : __fdividef(1.f, L); /* 0: the row sees nothing */
          *reinterpret_cast<uint2*>((T*)a.out + out_row(qi) * HD + d0 + d) = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
          if (d0 + d == 0 && a.lse) a.lse[out_row(qi)] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
        } else {
          __stcg(reinterpret_cast<float4*>(a.po + (ps + qi) * HD + d0 + d), x);
          if (d0 + d == 0) __stcg(reinterpret_cast<float2*>(a.pml + (ps + qi) * 2), make_float2(M, L));
        }
      }
    }
    if (!whole) {
      /* the last of the unit's CTAs to get here joins them, in the order of their keys */
      const int c0 = line.group_of(c.first), pieces = line.group_of(c.last) - c0 + 1;
      if (c.t0 == 0 && tid == 0) p.tail[2 * c0 + 1] = my_slot;
      __threadfence();
      sync_work();
      if (tid == 0) {
        const int n = atomicAdd(&p.tail[2 * c0], 1);
        sh_last = n == pieces - 1;
        if (n == pieces - 1) p.tail[2 * c0] = 0; /* for the next launch */
      }
      sync_work();
      if (sh_last) {
        __threadfence();
        const int slot0 = __ldcg(&p.tail[2 * c0 + 1]);
        auto place = [&](int i, int qi) { return ((long long)(c0 + i) * 2 + (i == 0 ? slot0 : 0)) * C::RT + qi; };
        /* the maximum and the sum of each query first: a warp a query, a lane every 32nd piece */
        for (int qi = warp; qi < c.nq; qi += W) {
          float M = -INFINITY, L = 0.f;
          for (int k = lane; k < pieces; k += 32) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.pml + place(k, qi) * 2));
            const float top = fmaxf(M, ml.x), u = top == -INFINITY ? 0.f : top;
            L = L * ex2(M - u) + ml.y * ex2(ml.x - u);
            M = top;
          }
#pragma unroll
          for (int x = 16; x; x >>= 1) {
            const float m2 = __shfl_xor_sync(kAll, M, x), l2 = __shfl_xor_sync(kAll, L, x), top = fmaxf(M, m2), u = top == -INFINITY ? 0.f : top;
            L = L * ex2(M - u) + l2 * ex2(m2 - u);
            M = top;
          }
          if (lane == 0) sh_ml[buf][0][qi] = make_float2(M, L);
        }
        sync_work();
        for (int i = tid; i < c.nq * (HD / 4); i += W * 32) {
          const int qi = i / (HD / 4), d = (i % (HD / 4)) * 4;
          const float M = sh_ml[buf][0][qi].x, L = sh_ml[buf][0][qi].y, U = M == -INFINITY ? 0.f : M;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
          for (int k = 0; k < pieces; ++k) {
            const float f = ex2(__ldcg(a.pml + place(k, qi) * 2) - U);
            const float4 y = __ldcg(reinterpret_cast<const float4*>(a.po + place(k, qi) * HD + d));
            x.x += y.x * f;
            x.y += y.y * f;
            x.z += y.z * f;
            x.w += y.w * f;
          }
          const float inv = L == 0.f ? 0.f : __fdividef(1.f, L);
          *reinterpret_cast<uint2*>((T*)a.out + out_row(qi) * HD + d) = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
          if (d == 0 && a.lse) a.lse[out_row(qi)] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
        }
      }
    }
    /* what a warp writes next into the other halves of the buffers, others have read before the barriers above */
  }
  if (!ok) { /* no copy is in flight when the CTA ends */
    for (int i = 0; i < C::NST; ++i) mb_wait_warp(&full[warp][slot], phase), slot = slot + 1 == C::NST ? (phase ^= 1, 0) : slot + 1;
    if (lane == 0) atomicOr(a.err, 8);
  }
}

constexpr size_t kQuantWsFloats = (size_t)8 << 20; /* 32 MiB */
constexpr size_t kQuantTail = 4096;                /* of them, ints of arrivals */

template <typename T, bool Q4, int HD, int NT>
int launch_quant(Ctx* c, TreeArgs& a) {
  using C = QCfg<Q4, HD, NT>;
  static uint64_t attr = 0; /* devices it is set on */
  if (!(attr >> (c->device & 63) & 1)) {
    ULB_CUDA(cudaFuncSetAttribute(quant_attn_kernel<T, Q4, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    prefer_max_shared((const void*)quant_attn_kernel<T, Q4, HD, NT>); /* before the launch does it: all of it, for CTAS blocks an SM */
    ULB_CUDA(cudaFuncSetAttribute(quant_attn_kernel<T, Q4, HD, NT>, cudaFuncAttributePreferredSharedMemoryCarveout, 100));
    attr |= 1ull << (c->device & 63);
  }
  const long long units = (long long)a.g.n_seq * a.g.n_head_kv * (((long long)a.max_rows * a.G + C::RT - 1) / C::RT);
  ULB_CHECK(units * (std::max(1, (a.max_len + C::KT - 1) / C::KT) + C::UNIT) < (1ll << 31) - 65536, ULB_EUNSUPPORTED,
            "ulb_quant_attention: %d sequences of %d positions and %d rows", a.g.n_seq, a.max_len, a.max_rows);
  QuantPlan p;
  p.groups = c->n_sm * C::CTAS;
  p.min_tiles = C::MIN;
  const size_t rows = (size_t)p.groups * 2 * C::RT;
  ULB_CHECK(kQuantTail + rows * (HD + 2) <= kQuantWsFloats && 2 * (size_t)p.groups <= kQuantTail, ULB_EUNSUPPORTED,
            "ulb_quant_attention: workspace for %d SMs", c->n_sm);
  p.tail = reinterpret_cast<int*>(c->quant_ws);
  a.po = c->quant_ws + kQuantTail;
  a.pml = a.po + rows * HD;
  ULB_LAUNCH("quant attention launch", launch_k(c, quant_attn_kernel<T, Q4, HD, NT>, dim3(p.groups), dim3(C::W * 32 + 32), C::SMEM, a, p));
  return ULB_OK;
}

template <typename T, bool Q4, int HD>
int pick_rows(Ctx* c, TreeArgs& a) {
  const long long nq = (long long)a.max_rows * a.G;
  if (nq <= 8) return launch_quant<T, Q4, HD, 1>(c, a);
  if (nq <= 16 || HD == 256) return launch_quant<T, Q4, HD, 2>(c, a);
  if constexpr (HD < 256) {
    const long long passes = (nq + 31) / 32;
    if ((nq + passes - 1) / passes <= 24) return launch_quant<T, Q4, HD, 3>(c, a);
    return launch_quant<T, Q4, HD, 4>(c, a);
  }
  return ULB_OK;
}
template <typename T, bool Q4>
int pick_quant(Ctx* c, TreeArgs& a) {
  if (a.g.hd == 64) return pick_rows<T, Q4, 64>(c, a);
  if (a.g.hd == 128) return pick_rows<T, Q4, 128>(c, a);
  return pick_rows<T, Q4, 256>(c, a);
}

}  // namespace
}  // namespace ulb

using namespace ulb;

extern "C" int ulb_quant_attention(ulb_ctx* ctx, const ulb_quant_desc* cache, const ulb_tree_desc* d, const void* q, const void* k,
                                   const void* v, const int32_t* table, const int32_t* row_start, const int32_t* prefix,
                                   const int32_t* len, const uint32_t* mask, void* out, float* lse) {
  ULB_CHECK(ctx && d, ULB_EINVAL, "ulb_quant_attention: NULL argument");
  TreeArgs a = {};
  ULB_TRY(quant_geom("ulb_quant_attention", cache, &a.g));
  ULB_CHECK(d->n_head > 0 && d->n_head % a.g.n_head_kv == 0 && d->n_head / a.g.n_head_kv <= 64, ULB_EINVAL,
            "ulb_quant_attention: %d heads over %d kv heads", d->n_head, a.g.n_head_kv);
  ULB_CHECK(d->rows >= 0 && d->max_rows >= 0 && d->max_len >= 0 && d->mask_words >= 0, ULB_EINVAL,
            "ulb_quant_attention: %d rows, at most %d a sequence over %d positions, %d mask words", d->rows, d->max_rows, d->max_len,
            d->mask_words);
  ULB_CHECK(std::isfinite(d->scale) && d->scale > 0.f, ULB_EINVAL, "ulb_quant_attention: scale %g", (double)d->scale);
  if (d->rows == 0 || d->max_rows == 0) return ULB_OK;
  ULB_CHECK(q && k && v && table && row_start && prefix && len && out, ULB_EINVAL, "ulb_quant_attention: NULL argument");
  ULB_CHECK(!mask == (d->mask_words == 0), ULB_EINVAL, "ulb_quant_attention: mask without mask_words, or the reverse");
  ULB_CHECK(ULB_ALIGNED16(q) && ULB_ALIGNED16(k) && ULB_ALIGNED16(v) && ULB_ALIGNED16(out), ULB_EINVAL,
            "ulb_quant_attention: q, the pools and out must be 16-byte aligned");
  ULB_CHECK(words_aligned({table, row_start, prefix, len, mask, lse}), ULB_EINVAL, "ulb_quant_attention: unaligned array of 32-bit elements");
  a.H = d->n_head;
  a.G = d->n_head / a.g.n_head_kv;
  a.rows = d->rows;
  a.max_rows = std::min(d->max_rows, d->rows);
  a.max_len = std::min(d->max_len, a.g.max_pages * a.g.page);
  ULB_CHECK((long long)a.max_rows * a.G < (1ll << 31) && (long long)d->rows * d->n_head < (1ll << 31), ULB_EUNSUPPORTED,
            "ulb_quant_attention: %d rows of %d heads", d->rows, d->n_head);
  ULB_CHECK(a.max_len <= 0x7fff0000, ULB_EUNSUPPORTED, "ulb_quant_attention: %d positions", a.max_len);
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
  if (!c->quant_ws) { /* at the first call, whatever its shape, so that any later one can be captured */
    float* ws = nullptr;
    ULB_CUDA(cudaMalloc((void**)&ws, kQuantWsFloats * sizeof(float)));
    const cudaError_t e = cudaMemsetAsync(ws, 0, kQuantTail * sizeof(int), c->stream);
    if (e != cudaSuccess) {
      cudaFree(ws);
      return cuda_error(e, "ulb_quant_attention", __FILE__, __LINE__);
    }
    c->quant_ws = ws;
  }
  if (cache->dtype == ULB_TYPE_F16) return cache->format == ULB_TYPE_Q4_1 ? pick_quant<__half, true>(c, a) : pick_quant<__half, false>(c, a);
  return cache->format == ULB_TYPE_Q4_1 ? pick_quant<__nv_bfloat16, true>(c, a) : pick_quant<__nv_bfloat16, false>(c, a);
}

ULB_TRACE_UNIT(quant_attention)
