/*
 * tree_attention_tc.cu — ulb_tree_attention on the 5th-generation tensor cores, for head
 * dims up to 128 (80 and 96 run in tiles of 128 whose other columns the copies fill with zeros:
 * nothing is read for them).  Same mathematics and masking as tree_attention.cu.
 *
 * A CTA works on 64-key tiles with M = 128 query rows a stream, two streams at a time, each
 * with its own running (m, l, o) and its own softmax warpgroup (one thread a row):
 *   PAIR = false  (at most 128 queries a kv head): both streams hold the same rows and take the
 *                 even and the odd tiles; they join in shared memory at the end
 *   PAIR = true   (more): the streams hold neighbouring tiles of 128 rows and share every K / V
 *                 tile, which halves what shared memory and L2 have to deliver
 * so that one stream's products run while the other stream's weights are computed.  Per tile:
 * S = Q K^T (tcgen05.mma, both operands in shared memory, fp32 in TMEM); the row's thread reads
 * S, updates m and l, writes P (rounded to the cache's type) over S in TMEM; O += P V with P read
 * from TMEM and V as the tile TMA wrote it (keys x hd, the MN-major operand).  O stays in TMEM; it
 * is rescaled only when a row's maximum has grown by more than 2^GROW since the last time (weights
 * stay below 2^(RAISE + GROW), sums are fp32, so the result is the same ratio).
 *
 * Warps: 0 and 3 copy K and V tiles by TMA (pages -> 128-byte-swizzled tiles, one box a page, pages
 * that are unmapped or past the end read as zero through an out-of-range coordinate), 1 and 2 issue
 * the MMAs of a stream each and the commits that free tiles, 4 - 7 and 8 - 11 softmax; they also take V
 * elements that are not finite out of masked tiles.  Barriers carry it: K / V tiles full and free, S full,
 * P full, O += P V done (looked at only to rescale O); the order in which the warps pass the rings is
 * tree_plan.h's.  A stream has two score buffers; one thread issues its MMAs and they complete in order,
 * so a buffer is free for the tile after the next once the product that reads its weights has been
 * issued, and the scores of the next tile are there while weights are computed (128-key tiles with one
 * buffer, weights handed over in halves, took 339 us where this took 300).
 *
 * Weights are rounded to 16 bits once: two parts, as the mma.sync form keeps of bf16, would double the
 * second product, which here is half of the tensor cores' work.  Against 64 bits the outputs are off by
 * 2.3e-3 relative in bf16 and 2.8e-4 in fp16, of which 1.7e-3 and 2.1e-4 are the output's own rounding.
 *
 * Work is cut evenly over the lengths: the tiles of all (sequence, kv head) pairs form one line, every CTA
 * (group of CTAs, when more than 256 rows need several row tiles: its members walk the same keys side by
 * side, so K / V come from HBM once) takes an equal stretch of it and walks whole sequences and pieces
 * of two.  A pair that falls into several stretches leaves one partial a stretch, joined by a small
 * kernel.  It is not cut over rows: a group has as many members as the longest of the sequences has row
 * tiles, members without rows of a sequence pass it by, and causal rows walk the keys after their last.
 *
 * Measured: 64 rows x 64 heads (8 kv heads of 128) x 131072 keys 286 us, 961 TFLOP/s (58 % of the measured
 * burst): the round trip between products and softmax, with two streams of two score buffers, which is
 * what TMEM holds, bounds it (tensor pipe 55 %, exponentials 45 %).  64 sequences of 256 to 4096 keys with
 * 8 to 16 rows, 32 heads over 8: 128 us, 4.6 TB/s of K and V: HBM and some 6 us a (sequence, kv head).
 * 63 rows x 8191 keys, 32 kv heads: 40 us, of which 12 are a CTA's start and end and 5 the join.
 * 160 to 190 bytes a thread are spilled at the 168 registers of the launch, which are what the compiler
 * allots to every role, whatever the split at run time gives.
 *
 * Every mbarrier wait has a limit: past it a role raises bit 3 of the device error word,
 * arrives nowhere and issues nothing any more, so that the others run into theirs; the CTA still
 * waits (bounded) for its MMAs before it frees TMEM.
 */
#include "tree_attention.h"

#include <cuda.h>

#include <algorithm>
#include <mutex>

namespace ulb {
namespace {

constexpr int TK = 64;         /* keys a tile */
constexpr int TQ = 128;        /* query rows a stream: M */
constexpr int kThreads = 384;  /* 4 role warps, 2 x 4 softmax warps */
constexpr int kPairCost = 16;   /* what a pair costs besides its tiles, in tiles */
constexpr int kMinTiles = 12;  /* places of the line a group takes at least */
constexpr int kJoinRows = 8;   /* rows a block of the join kernel: a warp each */
constexpr int kOddWords = 32;  /* bits for 1024 positions */

__device__ __forceinline__ uint32_t sa(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mb_init(uint64_t* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(sa(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void mb_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(sa(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mb_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(sa(b)) : "memory");
}
__device__ __forceinline__ bool mb_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(sa(b)), "r"(parity) : "memory");
  return ok != 0;
}
/* wait for the phase with this parity; false after kTries looks, each of which the hardware may stretch
   (seconds in all; reading a clock between looks costs more than the looks) */
constexpr int kTries = 1 << 21;
__device__ __forceinline__ bool mb_wait(uint64_t* b, uint32_t parity) {
  for (int i = 0; i < kTries; ++i)
    if (mb_try(b, parity)) return true;
  return false;
}
/* the same for a converged warp, one answer for all lanes (a vote: a shuffle would queue behind the
   softmax warps' exponentials, as every shared-memory operation does, for some 300 cycles) */
__device__ __forceinline__ bool mb_wait_warp(uint64_t* b, uint32_t parity) { return __all_sync(0xffffffffu, mb_wait(b, parity)); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(sa(b)) : "memory");
}
__device__ __forceinline__ void tma4(void* dst, const CUtensorMap* m, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               ::"r"(sa(dst)), "l"(m), "r"(x), "r"(y), "r"(z), "r"(w), "r"(sa(bar)) : "memory");
}
/* one lane of a converged warp: the compiler knows that what the branch holds runs once, and keeps
   the operands of tcgen05 instructions in uniform registers (under `lane == 0` each MMA took about
   70 cycles to issue) */
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
/* D (TMEM) (+)= A (shared) B (shared) and D (+)= A (TMEM) B (shared), K = 16 */
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n}\n"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}\n"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u) : "memory");
}
/* 32 consecutive columns of the thread's TMEM lane */
__device__ __forceinline__ void tm_ld(uint32_t t, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
               "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                 "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
                 "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
                 "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(t));
}
__device__ __forceinline__ void tm_st(uint32_t t, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
               "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
               ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
               "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
               "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
               "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(t) : "memory");
}
__device__ __forceinline__ void tm_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
/* two fp32 operations in one instruction */
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
/* the 256 softmax threads */
__device__ __forceinline__ void sync_softmax() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

/* shared-memory descriptors of 128-byte-swizzled tiles (rows of 64 elements, 8-row groups 1024 bytes
   apart): K-major (Q, K: a row is an index of M or N, its 64 elements 64 of hd), and MN-major
   (V: a row is a key = K index, its 64 elements 64 of N; the next 64 of N one half tile on) */
__device__ __forceinline__ uint64_t desc_k(uint32_t s) {
  return (uint64_t)((s >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t s) {
  return (uint64_t)((s >> 4) & 0x3FFFu) | ((uint64_t)((TK * 128) >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
/* byte of 16-byte chunk c (of 8) of row r in a half tile */
__device__ __forceinline__ uint32_t sw128(int r, int c) { return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4)); }

template <int HD, bool PAIR>
struct TcCfg {
  static constexpr int TILE = TK * HD * 2;            /* bytes of a K or V tile */
  static constexpr int QTILE = TQ * HD * 2;
  static constexpr int NQ = PAIR ? 2 : 1;
  static constexpr int NK = HD == 64 ? 8 : PAIR ? 5 : 6; /* K tiles in the ring */
  static constexpr int NV = HD == 64 ? 8 : PAIR ? 5 : 6;
  static constexpr int STAGE = NQ * QTILE >= 32768 ? 0 : 32768; /* outputs pass through Q's place, or their own */
  static constexpr int SMEM = NQ * QTILE + (NK + NV) * TILE + STAGE + 1024; /* + alignment slack */
  static constexpr int RT = PAIR ? 256 : 128;         /* queries a CTA */
  static_assert(SMEM <= 226 * 1024, "shared memory");
};

/* what the launch adds to TreeArgs */
struct TcPlan {
  int members, groups_max; /* CTAs that walk the same keys side by side, such groups in the grid */
  int min_tiles;           /* tiles of the line a group takes at least */
  struct TcTail* tail;     /* [groups][members] */
};
/* the head of a pair that goes on in the next groups: what the join kernel needs */
struct TcTail {
  int pieces, slot, r0, nq, q0, kvh, pad0, pad1; /* pieces 0: none */
};

/* The line of work, in tiles.  A (sequence, kv head, pass) takes kPairCost places before its tiles, for what
   it costs besides them: its rows are loaded, its outputs joined and written.  Group c's stretch. */
struct Line {
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
/* places of one sequence, its tiles a pair and passes over its rows */
__device__ __forceinline__ int seq_places(const TreeArgs& a, const TcPlan& p, const TreeSeq& q, int RT, int* n_tile, int* n_pass) {
  *n_tile = max(1, (q.len + TK - 1) / TK);
  const int rows = RT * p.members;
  *n_pass = q.n * a.G <= rows ? (q.n > 0 ? 1 : 0) : (q.n * a.G + rows - 1) / rows;
  return (*n_tile + kPairCost) * *n_pass * a.g.n_head_kv;
}

struct Piece {
  TreeSeq q;
  int s, kvh, q0, nq; /* sequence, kv head, first query (row x group + head) of the tile, queries in it */
  int t0, n, n_tile;  /* tiles [t0, t0 + n) of n_tile */
  int last;           /* place of the pair's last tile on the line */
  int nth;            /* pieces of this CTA before it */
};

/* walks the pieces of one CTA; every role runs the same walk */
template <int RT>
struct Walk {
  int at, end, base, cnt, s, n_tile, n_pass, member, nth;
  TreeSeq q;
  __device__ __forceinline__ void load(const TreeArgs& a, const TcPlan& p) {
    q = tree_seq(a, s);
    cnt = seq_places(a, p, q, RT, &n_tile, &n_pass);
  }
  __device__ __forceinline__ bool next(const TreeArgs& a, const TcPlan& p, Piece* o) {
    while (at < end) {
      while (at >= base + cnt) { /* ends: at < end <= total */
        base += cnt;
        ++s;
        load(a, p);
      }
      const int len = n_tile + kPairCost, u = (at - base) / len, in = at - base - u * len;
      const int upto = min(len, in + end - at);
      o->t0 = max(in - kPairCost, 0);
      o->n = max(upto - kPairCost, 0) - o->t0;
      o->last = base + u * len + len - 1;
      at += upto - in;
      o->kvh = n_pass == 1 ? u : u / n_pass;
      o->q0 = ((n_pass == 1 ? 0 : u % n_pass) * p.members + member) * RT;
      o->nq = min(RT, q.n * a.G - o->q0);
      if (o->nq <= 0 || o->n <= 0) continue; /* this member has no rows of the sequence, or no tile yet */
      o->q = q;
      o->s = s;
      o->n_tile = n_tile;
      o->nth = nth++;
      return true;
    }
    return false;
  }
};

/* which of positions [pos, pos + 32) row i sees; pages says which 16-position blocks of the tile are
   mapped, rel = pos within the tile */
__device__ __forceinline__ uint32_t sees32(const TreeArgs& a, const TreeSeq& q, int i, int pos, uint32_t blocks, int rel) {
  uint32_t v = 0xffffffffu;
  if (a.words == 0) {
    const int n = q.len - q.n + i - pos + 1;
    v = n <= 0 ? 0u : n >= 32 ? v : (1u << n) - 1u;
  } else {
    const int j = pos - q.prefix;
    if (j > -32) {
      const uint32_t* m = a.mask + (long long)(q.r0 + i) * a.words;
      const int w = j >> 5;
      auto word = [&](int k) { return k < 0 ? 0xffffffffu : k >= a.words ? 0u : m[k]; };
      const uint32_t lo = word(w), hi = word(w + 1);
      v = __funnelshift_r(lo, hi, j & 31);
    }
  }
  const int left = q.len - pos;
  if (left < 32) v &= left <= 0 ? 0u : (1u << left) - 1u;
  const uint32_t b = blocks >> (rel >> 4);
  if (!(b & 1u)) v &= 0xffff0000u;
  if (!(b & 2u)) v &= 0x0000ffffu;
  return v;
}

/*
 * What infinities and NaN of V at the marked positions of [from, upto) add to columns [d0, d0 + 32) of row
 * i's sum, if the row sees them.  Not inlined: with it in the kernel, 64 rows x 131072 keys took 342 us for 330.
 */
template <typename T>
__device__ __noinline__ void add_odd(const TreeArgs& a, TreeSeq q, const uint32_t* marks, int s, int kvh, int i, const T* qr, int from,
                                     int upto, int d0, float m, float* o) {
  const int hd = a.g.hd;
  for (int w = 0; w < kOddWords; ++w)
    for (uint32_t bits = marks[w]; bits; bits &= bits - 1)
      for (int pos = from + ((w * 32 + __ffs(bits) - 1 - from) & (32 * kOddWords - 1)); pos < upto; pos += 32 * kOddWords) {
        const int j = pos >> a.g.page_shift;
        const int pg = j < a.g.max_pages ? a.table[(long long)s * a.g.max_pages + j] : -1;
        if (pg < 0 || pg >= a.g.n_pages || !tree_sees(a, q, i, pos)) continue;
        const long long off = pg * a.g.pstride + (pos & (a.g.page - 1)) * a.g.pos + kvh * a.g.head;
        const T *kr = (const T*)a.k + off, *vr = (const T*)a.v + off + d0;
        bool hit = false;
        for (int e = 0; e < min(32, hd - d0); ++e) hit |= !isfinite(to_f<T>(vr[e]));
        if (!hit) continue;
        float sc = 0.f;
        for (int e = 0; e < hd; ++e) sc = __fmaf_rn(to_f<T>(qr[e]), to_f<T>(kr[e]), sc);
        const float wt = ex2(__fmaf_rn(sc, a.scale2, -(m == -INFINITY ? 0.f : m)));
        for (int e = 0; e < min(32, hd - d0); ++e) {
          const float x = to_f<T>(vr[e]);
          if (!isfinite(x)) o[e] += wt * x;
        }
      }
}

template <typename T, int HD, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const __grid_constant__ TreeArgs a,
                   const __grid_constant__ TcPlan p) {
  using C = TcCfg<HD, PAIR>;
  constexpr bool F16 = std::is_same<T, __half>::value;
  /* Weights are at most 2^(RAISE + GROW): fp16, whose largest number is just under 2^16, holds 11 bits of one
     down to 2^-26 of the maximum (tree_attention.cu, kRaise); bf16 has the range without.  fp16, 64 rows x 64
     heads x 131072 keys: 290 us (331 with scores four times as wide), with GROW 3 300 (346), with 2 320 (356). */
  constexpr float RAISE = F16 ? 12.f : 0.f, GROW = F16 ? 3.9f : 8.f;
  constexpr uint32_t FMT = F16 ? 0u : (1u << 7) | (1u << 10);
  constexpr uint32_t ID_S = (1u << 4) | FMT | ((TK >> 3) << 17) | ((128 >> 4) << 24);
  constexpr uint32_t ID_O = (1u << 4) | FMT | (1u << 16) | ((HD >> 3) << 17) | ((128 >> 4) << 24);
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t k_full[C::NK], k_free[C::NK], v_full[C::NV], v_free[C::NV], s_full[2][2], p_full[2][2], o_done[2][2], v_seen[2],
      piece[2], q_full, mma_done;
  __shared__ uint32_t tmem_sh;
  __shared__ int sh_s, sh_base, sh_sum[kThreads / 32];
  __shared__ uint32_t odd[2][kOddWords + 1]; /* of a piece (its number modulo 2): which positions modulo 1024, before len, lost a V element; any */
  uint8_t* const sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* const q_sm = sm;
  uint8_t* const k_sm = sm + C::NQ * C::QTILE;
  uint8_t* const v_sm = k_sm + C::NK * C::TILE;
  uint8_t* const stage_sm = C::STAGE ? v_sm + C::NV * C::TILE : q_sm;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hd = HD == 64 ? 64 : a.g.hd; /* HD = 128: 80, 96 or 128, the tiles' columns past it are zeros */

  /* nothing here depends on earlier kernels */
  if (tid == 0) {
    for (int i = 0; i < C::NK; ++i) { mb_init(&k_full[i], 1); mb_init(&k_free[i], 2); }
    for (int i = 0; i < C::NV; ++i) { mb_init(&v_full[i], 1); mb_init(&v_free[i], 2); }
    for (int i = 0; i < 2; ++i) {
      mb_init(&v_seen[i], 1);
      mb_init(&piece[i], 1);
      for (int b = 0; b < 2; ++b) { mb_init(&s_full[i][b], 1); mb_init(&p_full[i][b], 4); mb_init(&o_done[i][b], 1); }
    }
    mb_init(&q_full, 8);
    mb_init(&mma_done, 2);
    sh_s = 0;
    sh_base = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < 2 * (kOddWords + 1)) odd[tid / (kOddWords + 1)][tid % (kOddWords + 1)] = 0;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sa(&tmem_sh)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();
  if (tid == 0) p.tail[blockIdx.x].pieces = 0;
  /* the line's length, then this group's place on it */
  auto places_of = [&](int s) {
    int nt, np;
    return s < a.g.n_seq ? seq_places(a, p, tree_seq(a, s), C::RT, &nt, &np) : 0;
  };
  const int cnt0 = places_of(tid);
  int mine = cnt0;
  for (int s = tid + kThreads; s < a.g.n_seq; s += kThreads) mine += places_of(s);
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) sh_sum[warp] = mine;
  tc_before();
  __syncthreads();
  tc_after();
  Line line;
  line.total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) line.total += sh_sum[w];
  line.cut(max(1, min(p.groups_max, (line.total + p.min_tiles - 1) / p.min_tiles)));
  const int grp = blockIdx.x / p.members, member = blockIdx.x % p.members;
  Walk<C::RT> walk;
  walk.at = grp < line.groups ? line.begin(grp) : line.total;
  walk.end = grp < line.groups ? line.begin(grp + 1) : line.total;
  {
    int base = 0;
    for (int s0 = 0; s0 < a.g.n_seq && walk.at < walk.end; s0 += kThreads) { /* the sequence that holds the stretch's begin */
      const int c = s0 == 0 ? cnt0 : places_of(s0 + tid);
      int x = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      __syncthreads();
      if (lane == 31) sh_sum[warp] = x;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
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
  const uint32_t tmem = tmem_sh;
  walk.s = sh_s;
  walk.base = sh_base;
  walk.member = member;
  walk.nth = 0;
  walk.load(a, p);
  Piece pc = {};
  bool ok = true;
  /* stream X's tiles of a piece of n: PAIR all of them (none without rows), else every second */
  auto n_of = [&](int X) { return PAIR ? (X == 0 || pc.nq > 128 ? pc.n : 0) : (pc.n + 1 - X) >> 1; };

  /* registers: 128 x 104 + 256 x 200 = 384 x 168, what the block was launched with */
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 0 || warp == 3) {
      /* ------------------------------------------------ TMA: warp 0 the K tiles, warp 3 the V tiles, in order.
         Asking for a free slot, issuing and looking up pages take some 750 cycles a tile, so each
         has a warp and the page ids are read a tile ahead. */
      const CUtensorMap* const map = warp == 0 ? &mk : &mv;
      uint8_t* const ring = warp == 0 ? k_sm : v_sm;
      uint64_t* const full = warp == 0 ? k_full : v_full;
      uint64_t* const free = warp == 0 ? k_free : v_free;
      const int nring = warp == 0 ? C::NK : C::NV;
      int slot = 0, issued = 0;
      uint32_t phase = 1; /* of the free barrier: the first round passes */
      const int rows = min(a.g.page, TK), boxes = TK / rows;
      constexpr int MB = TK / 16;
      while (ok && walk.next(a, p, &pc)) {
        const int* const tb = a.table + (long long)pc.s * a.g.max_pages;
        int pg[MB]; /* pages of the next tile; n_pages, out of range, reads zeros */
        auto ids = [&](int t) {
          const int pos = (pc.t0 + t) * TK; /* at most len + 63 */
#pragma unroll
          for (int i = 0; i < MB; ++i) {
            const int at = pos + i * rows, j = at >> a.g.page_shift;
            pg[i] = i < boxes && t < pc.n && at < pc.q.len && j < a.g.max_pages ? tb[j] : -1;
          }
        };
        ok = ring_copy(pc.n, ids, [&]() { return mb_wait_warp(&free[slot], phase); }, [&](int t) {
          if (elect()) {
            const int pos = ((pc.t0 + t) * TK) & (a.g.page - 1);
            uint8_t* const d = ring + slot * C::TILE;
            mb_expect(&full[slot], (uint32_t)C::TILE);
#pragma unroll
            for (int i = 0; i < MB; ++i) {
              if (i >= boxes) break;
              const int page = pg[i] >= 0 && pg[i] < a.g.n_pages ? pg[i] : a.g.n_pages;
#pragma unroll
              for (int h = 0; h < HD / 64; ++h) tma4(d + i * rows * 128 + h * TK * 128, map, h * 64, pos, pc.kvh, page, &full[slot]);
            }
          }
          __syncwarp();
          ++issued;
          if (++slot == nring) { slot = 0; phase ^= 1; }
        });
      }
      /* no copy is in flight when the CTA ends, whatever happened: the last round's tiles, in turn */
      for (int c = max(0, issued - nring); c < issued; ++c) ok &= mb_wait_warp(&full[c % nring], (c / nring) & 1);
    } else {
      /* ------------------------------------------------ MMA issue: a warp a stream walks, one elected lane
         issues, in the order of ring_issue.  What one thread does for a tile (waits, MMAs, commits) takes
         about as long as its arithmetic, so descriptors are a base plus a constant and ring places are
         counted.  A parity wait can tell a phase from the one before and after only, so nobody may skip
         one: both warps look at every K and V tile, and a tile is free when both have (the stream that
         does not use it at once).  On a wait that fails the warp stops; nothing is issued after that. */
      const int X = warp - 1;
      uint32_t qp = 0, pp = 0; /* phases of q_full, and of p_full[X][b] in bit b */
      int ks = 0, vs = 0;      /* next tile of the rings, and its phase */
      uint32_t kp = 0, vp = 0;
      const uint64_t dq = desc_k(sa(q_sm)) + (PAIR ? X * (C::QTILE >> 4) : 0), dk = desc_k(sa(k_sm)), dv = desc_mn(sa(v_sm));
      const uint32_t ds = tmem + X * 128, dov = tmem + 256 + X * HD;
      while (ok && walk.next(a, p, &pc)) {
        ok = mb_wait_warp(&q_full, qp);
        qp ^= 1;
        const int n = n_of(X), clear = min(tree_open(a, pc.q), pc.q.len);
        auto step_k = [&]() { if (++ks == C::NK) { ks = 0; kp ^= 1; } };
        auto step_v = [&]() { if (++vs == C::NV) { vs = 0; vp ^= 1; } };
        auto wait_k = [&]() { return mb_wait_warp(&k_full[ks], kp); };
        auto wait_v = [&]() { return mb_wait_warp(&v_full[vs], vp); };
        auto pass_k = [&]() {
          if (!wait_k()) return false;
          if (lane == 0) mb_arrive(&k_free[ks]);
          step_k();
          return true;
        };
        auto pass_v = [&]() {
          if (!wait_v()) return false;
          if (lane == 0) mb_arrive(&v_free[vs]);
          step_v();
          return true;
        };
        auto qk = [&](int b) { /* scores of the next K tile into buffer b (one lane) */
          const uint64_t k0 = dk + ks * (C::TILE >> 4);
#pragma unroll
          for (int j = 0; j < HD / 16; ++j)
            mma_ss(ds + b * TK, dq + (((j >> 2) * (TQ * 128) + (j & 3) * 32) >> 4), k0 + (((j >> 2) * (TK * 128) + (j & 3) * 32) >> 4), ID_S,
                   j > 0);
          commit(&s_full[X][b]);
          commit(&k_free[ks]);
        };
        ok = ok && ring_issue<PAIR>(
            X, n, pc.n, pass_k, pass_v, wait_k, wait_v,
            [&](int b) {
              tc_after();
              if (elect()) qk(b);
              __syncwarp();
              step_k();
            },
            [&](int vt) { /* masked: the softmax warps look it over */
              if ((pc.t0 + vt + 1) * TK > clear && lane == 0) mb_arrive(&v_seen[X]);
            },
            [&](int b) {
              if (!mb_wait_warp(&p_full[X][b], (pp >> b) & 1)) return false;
              pp ^= 1u << b;
              return true;
            },
            [&](int b, int i, bool more) {
              tc_after();
              if (elect()) {
                const uint64_t v0 = dv + vs * (C::TILE >> 4);
                const uint32_t pa = ds + b * TK;
                mma_ts(dov, pa, v0, ID_O, i > 0);
#pragma unroll
                for (int j = 1; j < TK / 16; ++j) mma_ts(dov, pa + j * 8, v0 + ((j * 2048) >> 4), ID_O, 1);
                commit(&o_done[X][b]);
                commit(&v_free[vs]);
                if (more) qk(b);
              }
              __syncwarp();
              step_v();
              if (more) step_k();
            });
        /* the piece is through, without tiles too: the softmax warps wait for it, so they cannot start two
           pieces while this warp has not seen one */
        if (ok && elect()) commit(&piece[X]);
        __syncwarp();
      }
      /* everything issued completes before TMEM is freed */
      if (elect()) commit(&mma_done);
      __syncwarp();
      ok = mb_wait_warp(&mma_done, 0) && ok;
    }
  } else {
    /* ------------------------------------------------ softmax: one thread a row */
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int X = (warp - 4) >> 2, row = tid - 128 - X * 128; /* stream, row of its tile = TMEM lane */
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t to = tmem + lanes + 256 + X * HD;
    constexpr int n_blk = TK / 16; /* 16-position blocks of a tile */
    uint32_t used = 0;       /* V tiles of earlier pieces */
    uint32_t sp = 0, op = 0, vsp = 0; /* phases of s_full[X][b] and o_done[X][b] in bit b, of piece and v_seen */
    constexpr int QW = C::NQ * TQ * (HD / 8) / 256; /* 16-byte words of Q a thread */
    auto q_at = [&](const Piece& c, int j, int* r, int* ch) { /* word j of this thread; null past the tile's queries and past hd */
      const int i = tid - 128 + j * 256;
      *r = i / (HD / 8);
      *ch = i % (HD / 8);
      const int qi = c.q0 + *r;
      return *r < c.nq && *ch * 8 < hd ? (const T*)a.q + ((long long)(c.q.r0 + qi / a.G) * a.H + c.kvh * a.G + qi % a.G) * hd + *ch * 8
                                       : nullptr;
    };
    bool have = walk.next(a, p, &pc);
    while (have) {
      auto mapped = [&](long long pos) { /* or past the end */
        if (pos >= pc.q.len) return true;
        const int j = (int)(pos >> a.g.page_shift);
        const int x = j < a.g.max_pages ? a.table[(long long)pc.s * a.g.max_pages + j] : -1;
        return x >= 0 && x < a.g.n_pages;
      };
      /* is some page of the piece unmapped?  A page a lane, its load under way beside those of Q */
      const int j0 = ((pc.t0 * TK) >> a.g.page_shift) + lane, j1 = (min((pc.t0 + pc.n) * TK, pc.q.len) - 1) >> a.g.page_shift;
      const int page0 = j0 <= j1 && j0 < a.g.max_pages ? a.table[(long long)pc.s * a.g.max_pages + j0] : j0 <= j1 ? -1 : 0;
      {
        uint4 qx[QW];
        int r, ch;
#pragma unroll
        for (int j = 0; j < QW; ++j) {
          const T* src = q_at(pc, j, &r, &ch);
          qx[j] = src ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < QW; ++j) {
          q_at(pc, j, &r, &ch);
          *reinterpret_cast<uint4*>(q_sm + (r >> 7) * C::QTILE + (ch >> 3) * (TQ * 128) + sw128(r & 127, ch & 7)) = qx[j];
        }
      }
      bool holes = page0 < 0 || page0 >= a.g.n_pages;
      for (int j = j0 + 32; j <= j1; j += 32) holes |= !mapped((long long)j << a.g.page_shift);
      holes = __any_sync(0xffffffffu, holes);
      fence_async();
      __syncwarp();
      if (lane == 0 && ok) mb_arrive(&q_full);

      const int r = (PAIR ? X * 128 : 0) + row, qi = pc.q0 + r;
      const bool live = r < pc.nq, warp_live = r - lane < pc.nq;
      const int ri = live ? qi / a.G : 0;
      const int n = n_of(X), open = tree_open(a, pc.q);
      if (live && a.words > 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.mask + (long long)(pc.q.r0 + ri) * a.words));
      float m = -INFINITY, l = 0.f; /* m: the maximum that weights are taken against, less RAISE */
      for (int i = 0; i < n && ok; ++i) {
        const int t = pc.t0 + (PAIR ? i : 2 * i + X), pos = t * TK;
        const int b = i & 1;
        const uint32_t ts = tmem + lanes + X * 128 + b * TK;
        const bool masked = (t + 1) * TK > open || pos + TK > pc.q.len;
        uint32_t blocks = 0xffffffffu; /* which 16-position blocks of the tile are mapped */
        if (holes) blocks = __ballot_sync(0xffffffffu, lane >= n_blk || mapped(pos + lane * 16));
        const bool cut = masked || blocks != 0xffffffffu;
        uint32_t see[TK / 32];
        if (cut) { /* looked up while the scores are computed */
#pragma unroll
          for (int c = 0; c < TK; c += 32) see[c / 32] = sees32(a, pc.q, ri, pos + c, blocks, c);
        }
        if (!mb_wait_warp(&s_full[X][b], (sp >> b) & 1)) { ok = false; break; }
        tc_after();
        if (warp_live) {
          uint32_t sr[TK];
#pragma unroll
          for (int c = 0; c < TK; c += 32) tm_ld(ts + c, sr + c);
          tm_ld_wait();
          if (cut) {
#pragma unroll
            for (int c = 0; c < TK; ++c)
              if (!((see[c / 32] >> (c & 31)) & 1u)) sr[c] = 0xff800000u; /* -inf */
          }
          /* weights against the maximum so far, the tile's own maximum beside them: only when a row's
             has grown by more than 2^GROW (its first tile, seldom later) are they taken again */
          uint32_t pk[TK / 2];
          float sum = 0.f, top = 0.f;
          auto weights = [&](float u) {
            const uint64_t sc2 = two(a.scale2, a.scale2), mu = two(-u, -u);
            uint64_t l0 = two(0.f, 0.f), l1 = l0;
            float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
            for (int c = 0; c < TK; c += 4) {
              const float2 e0 = both(fma2(two(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), sc2, mu));
              const float2 e1 = both(fma2(two(__uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3])), sc2, mu));
              const float p0 = ex2(e0.x), p1 = ex2(e0.y), p2 = ex2(e1.x), p3 = ex2(e1.y);
              x0 = max3(x0, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
              x1 = max3(x1, __uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3]));
              l0 = add2(l0, two(p0, p1));
              l1 = add2(l1, two(p2, p3));
              pk[c / 2] = pack2<T>(p0, p1);
              pk[c / 2 + 1] = pack2<T>(p2, p3);
            }
            const float2 y = both(add2(l0, l1));
            sum = y.x + y.y;
            top = fmaxf(x0, x1);
          };
          weights(m == -INFINITY ? 0.f : m);
          const bool grow = __fmaf_rn(top, a.scale2, -m) > RAISE + GROW; /* m -inf: a first key */
          if (__any_sync(0xffffffffu, grow)) {
            const float to_m = __fmaf_rn(top, a.scale2, -RAISE), f = grow ? (m == -INFINITY ? 0.f : ex2(m - to_m)) : 1.f;
            if (grow) m = to_m;
            l *= f;
            if (i > 0) { /* the first product overwrites O; products before the last are complete */
              if (!mb_wait_warp(&o_done[X][b ^ 1], ((sp >> (b ^ 1)) & 1) ^ 1)) ok = false;
              tc_after();
              uint32_t or_[32];
#pragma unroll
              for (int c = 0; c < HD; c += 32) {
                tm_ld(to + c, or_);
                tm_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) or_[e] = __float_as_uint(__uint_as_float(or_[e]) * f);
                tm_st(to + c, or_);
              }
            }
            weights(m == -INFINITY ? 0.f : m);
          }
          l += sum;
          tm_st(ts, pk); /* over the scores */
        }
        if (masked) {
          /* V elements of a masked tile that are not finite leave it before the product reads it.  With
             PAIR both streams look; what one has cleared the other finds clear, and no product of a
             stream starts before that stream has looked at the whole tile. */
          const uint32_t cvt = used + (uint32_t)(t - pc.t0);
          ok = mb_wait_warp(&v_seen[X], vsp) && ok;
          vsp ^= 1;
          uint4* const v = reinterpret_cast<uint4*>(v_sm + cvt % C::NV * C::TILE);
          constexpr uint32_t E = F16 ? 0x7c00u : 0x7f80u;
          const int lo = max(0, min(open, pc.q.len) - pos); /* first key of the tile that some row does not see */
          auto clear = [&](int j) {
            const uint4 x = v[j];
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
            bool hit = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if ((w[e] & E) == E) { w[e] &= 0xffff0000u; hit = true; }
              if (((w[e] >> 16) & E) == E) { w[e] &= 0x0000ffffu; hit = true; }
            }
            if (hit) {
              const int at = pos + (j >> 3) % TK; /* a key has 8 words in each half */
              if (at < pc.q.len) {
                atomicOr(&odd[pc.nth & 1][(at >> 5) % kOddWords], 1u << (at & 31));
                odd[pc.nth & 1][kOddWords] = 1;
              }
              v[j] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          };
          for (int j = lo * 8 + row; j < TK * 8 && ok; j += 128) {
            clear(j);
            if (HD == 128) clear(TK * 8 + j);
          }
          fence_async();
        }
        if (warp_live) tm_st_wait();
        tc_before();
        __syncwarp();
        if (lane == 0 && ok) mb_arrive(&p_full[X][b]);
        sp ^= 1u << b;
      }
      /* ---- the piece's end; the next one's rows are brought into L2 meanwhile */
      const Piece c = pc;
      have = walk.next(a, p, &pc);
      if (have) {
#pragma unroll 1
        for (int j = 0; j < QW; ++j) {
          int r1, ch1;
          const T* src = q_at(pc, j, &r1, &ch1);
          if (src && (ch1 & 7) == 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(src));
        }
      }
      if (ok) ok = mb_wait_warp(&piece[X], op);
      op ^= 1;
      used += c.n;
      tc_before();
      sync_softmax(); /* both streams are through: Q may be replaced, O of either is whole */
      tc_after();
      if (tid - 128 <= kOddWords) odd[(c.nth & 1) ^ 1][tid - 128] = 0; /* for the next piece */
      const bool whole = c.n == c.n_tile;
      const int slot = c.nth == 0 ? 0 : 1; /* only a CTA's first and last pieces can be parts */
      if (!whole && c.t0 == 0 && tid == 128) { /* the head of a pair that goes on in the next groups */
        TcTail& tl = p.tail[blockIdx.x];
        tl.slot = slot;
        tl.r0 = c.q.r0;
        tl.nq = c.nq;
        tl.q0 = c.q0;
        tl.kvh = c.kvh;
        tl.pieces = line.group_of(c.last) - grp + 1;
      }
      /* PAIR false: the streams' rows are the same and their lanes of TMEM too, so each warpgroup joins
         and writes half of hd */
      float f = 1.f, g = 0.f;
      if (!PAIR) {
        float2* const ml = reinterpret_cast<float2*>(q_sm);
        ml[X * TQ + row] = make_float2(m, l);
        sync_softmax();
        const float2 o1 = ml[(X ^ 1) * TQ + row];
        if (HD == 128) sync_softmax(); /* read, before the outputs pass through the same place */
        const float top = fmaxf(m, o1.x), u = top == -INFINITY ? 0.f : top;
        f = ex2(m - u);
        g = ex2(o1.x - u);
        l = l * f + o1.y * g;
        m = top;
      }
      const bool own = n > 0, other = !PAIR && (X == 0 ? c.n > 1 : true);
      const long long at = live ? (long long)(c.q.r0 + ri) * a.H + c.kvh * a.G + qi % a.G : 0;
      const long long ps = ((long long)blockIdx.x * 2 + slot) * C::RT + r;
      const float inv = l == 0.f ? 0.f : __fdividef(1.f, l); /* 0: the row sees nothing */
      if (warp_live && ok) {
        constexpr int COLS = PAIR ? HD : HD / 2;
        uint4* const stage = reinterpret_cast<uint4*>(stage_sm) + (warp - 4) * 256;
#pragma unroll 1
        for (int d0 = PAIR ? 0 : X * COLS; d0 < (PAIR ? HD : (X + 1) * COLS); d0 += 32) {
          if (d0 >= hd) break;
          uint32_t u[32];
          float o[32];
          tm_ld(tmem + lanes + 256 + X * HD + d0, u); /* whatever was there, where the stream had no tile */
          tm_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = own ? __uint_as_float(u[e]) * f : 0.f;
          if (!PAIR) {
            tm_ld(tmem + lanes + 256 + (X ^ 1) * HD + d0, u);
            tm_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] += other ? __uint_as_float(u[e]) * g : 0.f;
          }
          if (odd[c.nth & 1][kOddWords] && live) { /* values taken out of masked tiles go to the rows that see them */
            float more[32] = {};
            const int from = max(c.t0 * TK, min(open, c.q.len) / TK * TK), upto = min(c.q.len, (c.t0 + c.n) * TK);
            add_odd<T>(a, c.q, odd[c.nth & 1], c.s, c.kvh, ri, (const T*)a.q + at * hd, from, upto, d0, m, more);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] += more[e];
          }
          /* 32 rows x 32 columns change sides in shared memory, so that a row leaves in one piece (a lane
             writing its own row takes a transaction every 16 bytes): 16-byte word w of row y at w ^ y */
          if (whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              stage[lane * 4 + (e ^ ((lane >> 1) & 3))] =
                  make_uint4(pack2<T>(o[8 * e] * inv, o[8 * e + 1] * inv), pack2<T>(o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                             pack2<T>(o[8 * e + 4] * inv, o[8 * e + 5] * inv), pack2<T>(o[8 * e + 6] * inv, o[8 * e + 7] * inv));
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int y = k * 8 + (lane >> 2), w = lane & 3;
              const long long row_at = __shfl_sync(0xffffffffu, at, y);
              const uint4 x = stage[y * 4 + (w ^ ((y >> 1) & 3))];
              if (r - lane + y < c.nq && d0 + w * 8 < hd) *reinterpret_cast<uint4*>((T*)a.out + row_at * hd + d0 + w * 8) = x;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              stage[lane * 8 + (e ^ (lane & 7))] = make_uint4(__float_as_uint(o[4 * e]), __float_as_uint(o[4 * e + 1]),
                                                              __float_as_uint(o[4 * e + 2]), __float_as_uint(o[4 * e + 3]));
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int y = k * 4 + (lane >> 3), w = lane & 7;
              const uint4 x = stage[y * 8 + (w ^ (y & 7))];
              if (r - lane + y < c.nq) __stcg(reinterpret_cast<uint4*>(a.po + (ps - lane + y) * HD + d0 + w * 4), x);
            }
          }
          __syncwarp(); /* the words may be replaced, the next TMEM load is the whole warp's */
        }
        if (live && (PAIR || X == 0)) {
          if (!whole) __stcg(reinterpret_cast<float2*>(a.pml + ps * 2), make_float2(m, l));
          else if (a.lse) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        }
      }
      tc_before();
      sync_softmax(); /* each has read the other's O, and Q's place is free again */
    }
  }
  tc_before();
  __syncthreads();
  if (!ok && lane == 0) atomicOr(a.err, 8);
  if (warp == 1) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

/* join the pieces of a pair that several groups worked on: a warp a row, pieces in order */
template <typename T, int HD>
__global__ void __launch_bounds__(kJoinRows * 32) tree_tc_join_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ TcPlan p, int RT) {
  pdl_wait();
  pdl_trigger();
  const TcTail t = p.tail[blockIdx.x];
  const int r = blockIdx.y * kJoinRows + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t.pieces == 0 || r >= t.nq) return;
  auto place = [&](int i) { return ((long long)(blockIdx.x + i * p.members) * 2 + (i == 0 ? t.slot : 0)) * RT + r; };
  float M = -INFINITY;
  for (int i = lane; i < t.pieces; i += 32) M = fmaxf(M, __ldcg(a.pml + place(i) * 2));
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float U = M == -INFINITY ? 0.f : M;
  constexpr int E = HD / 32;
  float x[E] = {}, L = 0.f;
#pragma unroll 4
  for (int i = 0; i < t.pieces; ++i) {
    const long long at = place(i);
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.pml + at * 2));
    float y[E];
    if constexpr (E == 4) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(a.po + at * HD + lane * 4));
      y[0] = v.x; y[1] = v.y; y[2] = v.z; y[3] = v.w;
    } else {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(a.po + at * HD + lane * 2));
      y[0] = v.x; y[1] = v.y;
    }
    const float f = ex2(ml.x - U);
    L += ml.y * f;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] += y[e] * f;
  }
  const float inv = L == 0.f ? 0.f : __fdividef(1.f, L);
  const int qi = t.q0 + r;
  const long long at = (long long)(t.r0 + qi / a.G) * a.H + t.kvh * a.G + qi % a.G;
  const int hd = a.g.hd;
  if (lane == 0 && a.lse) a.lse[at] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
  if (lane * E >= hd) return;
  T* out = (T*)a.out + at * hd + lane * E;
  if constexpr (E == 4) *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(x[0] * inv, x[1] * inv), pack2<T>(x[2] * inv, x[3] * inv));
  else *reinterpret_cast<uint32_t*>(out) = pack2<T>(x[0] * inv, x[1] * inv);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
  static std::once_flag once;
  static EncodeTiledFn fn = nullptr;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)f;
  });
  return fn;
}

/* K or V pool as [page][head][position][hd], a box = 64 of hd x the positions of a page in a tile */
int pool_map(const TreeArgs& a, bool f16, const void* pool, CUtensorMap* m) {
  EncodeTiledFn enc = encode_tiled();
  ULB_CHECK(enc, ULB_ECUDA, "ulb_tree_attention: no cuTensorMapEncodeTiled entry point");
  const CacheGeom& g = a.g;
  const cuuint64_t dim[4] = {(cuuint64_t)g.hd, (cuuint64_t)g.page, (cuuint64_t)g.n_head_kv, (cuuint64_t)g.n_pages};
  const cuuint64_t str[3] = {(cuuint64_t)g.pos * 2, (cuuint64_t)g.head * 2, (cuuint64_t)g.pstride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)std::min(g.page, TK), 1, 1}, es[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(pool), dim, str,
                         box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  ULB_CHECK(r == CUDA_SUCCESS, ULB_EINVAL, "ulb_tree_attention: the cache's layout has no tensor map (CUresult %d)", (int)r);
  return ULB_OK;
}

/* the longest line a call can have */
long long line_most(const TreeArgs& a, int RT, int n_sm) {
  const long long tiles = ((long long)a.max_rows * a.G + RT - 1) / RT, members = std::min<long long>(tiles, n_sm);
  return (long long)a.g.n_seq * a.g.n_head_kv * (std::max(1, (a.max_len + TK - 1) / TK) + kPairCost) * ((tiles + members - 1) / members);
}

template <typename T, int HD, bool PAIR>
int launch_tc(Ctx* c, TreeArgs& a) {
  using C = TcCfg<HD, PAIR>;
  static uint64_t attr = 0; /* devices it is set on */
  if (!(attr >> (c->device & 63) & 1)) {
    ULB_CUDA(cudaFuncSetAttribute(tree_tc_kernel<T, HD, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    attr |= 1ull << (c->device & 63);
  }
  CUtensorMap mk, mv;
  constexpr bool f16 = std::is_same<T, __half>::value;
  ULB_TRY(pool_map(a, f16, a.k, &mk));
  ULB_TRY(pool_map(a, f16, a.v, &mv));
  TcPlan p;
  const long long tiles = ((long long)a.max_rows * a.G + C::RT - 1) / C::RT;
  p.members = (int)std::min<long long>(tiles, c->n_sm);
  p.groups_max = c->n_sm / p.members;
  p.min_tiles = kMinTiles;
  const int grid = p.groups_max * p.members;
  const size_t rows = (size_t)grid * 2 * C::RT;
  ULB_CHECK(rows * (HD + 2) + (size_t)grid * 8 <= kTreeWsFloats, ULB_EUNSUPPORTED, "ulb_tree_attention: workspace for %d SMs", c->n_sm);
  a.po = c->tree_ws;
  a.pml = a.po + rows * HD;
  p.tail = reinterpret_cast<TcTail*>(a.pml + rows * 2);
  ULB_LAUNCH("tree attention launch", launch_k(c, tree_tc_kernel<T, HD, PAIR>, dim3(grid), dim3(kThreads), C::SMEM, mk, mv, a, p));
  /* a launch that one group covers leaves nothing to join */
  const long long most = line_most(a, C::RT, c->n_sm);
  if (most > p.min_tiles && p.groups_max > 1)
    ULB_LAUNCH("tree join launch", launch_k(c, tree_tc_join_kernel<T, HD>, dim3(grid, C::RT / kJoinRows), dim3(kJoinRows * 32), 0, a, p, C::RT));
  return ULB_OK;
}

template <typename T>
int pick_tc(Ctx* c, TreeArgs& a) {
  const bool pair = (long long)a.max_rows * a.G > 128;
  if (a.g.hd == 64) return pair ? launch_tc<T, 64, true>(c, a) : launch_tc<T, 64, false>(c, a);
  return pair ? launch_tc<T, 128, true>(c, a) : launch_tc<T, 128, false>(c, a);
}

}  // namespace

/*
 * When this form runs, by queries a kv head and bytes of K and V (every sequence as long as the longest):
 * from 65 queries on; from 17 with 16 MB or more; below with 64 MB or more in sequences of 2048
 * positions or more.  Otherwise starting up (barriers, TMEM, tensor maps, two pipelines to fill) and
 * what a (sequence, kv head) costs besides its tiles outweigh the tensor cores.  Measured here / mma.sync
 * form, us (rows x keys): 1 x 500, 8 queries 14.3 / 8.6; 1 x 4000, 8 queries 17.3 / 8.4; 64 x 1 x 1000 mha
 * 167 / 80; 16 x 1 x 2000, 4 queries 32.6 / 34.4; 64 x 1 x 4000, 4 queries 114 / 149; 1 x 8000 mha 34 / 47;
 * 8 x 16 x 1000, 64 queries 21.7 / 33.6; 1 x 63 x 2000 mha 22.6 / 27.7.  From 65 queries on, with the join
 * (sequences x rows x keys): 64 x 70 x 170, 32 kv heads of 128 154 / 290, of 64 115 / 162; 64 x 20 x 170, 80 queries
 * 52 / 87; 16 x 20 x 500 30 / 72; 1 x 70 x 1000 mha 26 / 32; 4 x 33 x 300, 132 queries 30 / 36; 1 x 9 x 200, 72 queries
 * 20 / 23; but 1 x 16 x 2000, 128 queries 27 / 26, 1 x 64 x 1000, 512 queries 40 / 36 and 1 x 128 x 600, 512
 * queries 37 / 30: one sequence of few keys leaves most SMs without a stretch.
 * The line is counted in 32 bits.
 */
bool tree_tc_fits(const Ctx* c, const TreeArgs& a) {
  const long long nq = (long long)a.max_rows * a.G, bytes = 4ll * a.g.n_seq * a.max_len * a.g.n_head_kv * a.g.hd;
  if (a.g.hd > 128) return false;
  if (nq <= 16 && (bytes < (64ll << 20) || a.max_len < 2048)) return false;
  if (nq <= 64 && bytes < (16ll << 20)) return false;
  return line_most(a, nq > 128 ? 256 : 128, c->n_sm) < (1ll << 31) - 65536;
}

int launch_tree_tc(Ctx* c, TreeArgs& a, bool f16) { return f16 ? pick_tc<__half>(c, a) : pick_tc<__nv_bfloat16>(c, a); }

}  // namespace ulb

ULB_TRACE_UNIT(tree_attention_tc)
