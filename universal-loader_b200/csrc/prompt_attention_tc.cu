/*
 * prompt_attention_tc.cu — ulb_prompt_attention on the 5th-generation tensor cores, for head dims up to
 * 128 (80 and 96 run in tiles of 128 whose other columns the copies fill with zeros).  Same mathematics and masking as
 * prompt_attention.cu; the roles, rings and barriers are those of tree_attention_tc.cu, over rows of packed sequences in place
 * of pages.
 *
 * A CTA works on 64-key tiles with M = 128 queries (row x head of the group) a stream, two streams, each with its running
 * (m, l, o), its softmax warpgroup (one thread a query) and a warp that issues its MMAs:
 *   PAIR = true   256 queries: the streams hold neighbouring tiles of 128 and share every K / V tile
 *   PAIR = false  128 queries: both hold the same and take the even and the odd tiles; they join in shared memory
 * S = Q K^T (both operands in shared memory, fp32 in TMEM); the query's thread reads S, updates m and l, writes P in the rows' type
 * over S; O += P V with P from TMEM and V as the tile TMA wrote it.  O is rescaled only when a maximum has grown by more than
 * 2^GROW.  Weights are rounded to 16 bits once, since both operands of the product are of the rows' type and a second part
 * would double it: bf16 outputs are off by 2.1e-3 to 2.3e-3 relative against 64 bits, fp16 ones by 2.4e-4 to 2.7e-4, of which
 * 1.65e-3 and 2.0e-4 are the output's own rounding.  K and V rows come by TMA from wherever a sequence begins; what a
 * tile holds of the next sequence is masked, its infinities and NaN taken out of V with those past the diagonal.
 *
 * Work.  A unit is a (sequence, row tile, share of its keys, kv head) and walks the keys up to its last row's only.  The row
 * tiles of all sequences are sorted by their keys in a small kernel, and a CTA takes every G-th of that list in
 * turns that run back and forth, so all end together whatever the lengths; what fits the SMs once needs no list.  Few units
 * with many keys are cut into shares, joined by a third kernel.
 *
 * Measured: four prompts of 2157 to 6001 rows, 32 heads over 8 of 128 (618 GFLOP): 647 to 732 us, 0.84 to 0.96 PFLOP/s (52 to
 * 58 % of the burst rate, 61 to 69 % of the sustained one: the clock falls to 1.4 GHz under the power cap, by how much differs
 * between runs and GPUs); 513 rows after 30000 keys 276 to 309 us; 4096 rows 150 us at head dim 128 (0.92 PFLOP/s), 148
 * at 96 and at 80, whose tiles hold as many columns, 135 at 64; 2000 rows 48 us; 500 rows of 32 heads over 4 of 64 11 us; 16
 * prompts of 200 to 400 rows 60 to 63 us.  A pair of 64-key tiles takes 1700 to 1980 cycles: 1240 of them on the tensor pipe
 * (products with 64 columns read Q from shared memory every time), 1024 of exponentials, which overlap in part.  What a unit
 * costs besides is not overlapped with the next one: its rows in (4000 to 6000 cycles) and its outputs out (5000), most of a short prompt's time.  Tried and slower:
 * scores and weights in separate columns, so that the next tile's scores start as soon as these are read (827 us for 770 at
 * the time); the next unit's rows held in registers while the outputs leave (spills; 16 short prompts 88 us for 70).
 *
 * Every mbarrier wait has a limit: past it a role raises bit 3 of the device error word, arrives nowhere and issues nothing any
 * more, so that the others run into theirs; the CTA still waits (bounded) for its MMAs before it frees TMEM.
 */
#include "tcgen05.h"
#include "prompt_attention.h"

#include <algorithm>

namespace ulb {
namespace {

constexpr int TK = 64;         /* keys a tile */
constexpr int TQ = 128;        /* query rows a stream: M */
constexpr int kThreads = 384;  /* 4 role warps, 2 x 4 softmax warps */
constexpr int kJoinRows = 8;   /* rows a block of the join kernel: a warp each */
constexpr int kOddWords = 32;  /* bits for 1024 positions */

/* the 256 softmax threads */
__device__ __forceinline__ void sync_softmax() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

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

/* what the launch adds to PromptArgs.  A unit is a (sequence, row tile, share of its keys, kv head). */
struct PromptPlan {
  int shares;          /* the keys of a row tile are cut into so many */
  int row_tiles;       /* of the longest sequence */
  int direct;          /* every CTA takes the unit of its index, without a list */
  const int2* list;    /* (sequence, row tile), the most keys first; a unit for each share and kv head.  Null: one sequence, from
                          its last row tile on */
  const int* n_list;   /* entries there */
  float *po, *pml;     /* partials of (sequence, row tile, kv head, share): outputs, (max, sum) */
};

struct Piece {
  PromptSeq q;
  int s, kvh, q0, nq; /* sequence, kv head, first query (row x group + head) of the tile, queries in it */
  int rt, share;
  int t0, n, n_tile;  /* tiles [t0, t0 + n) of n_tile */
  int open;           /* keys that all its rows see */
  int nth;            /* pieces of this CTA before it */
};

/* a row tile's queries and its keys: all its rows see the first `open`, none sees more than n_tile tiles hold */
__device__ __forceinline__ bool row_tile(const PromptArgs& a, int s, int rt, int RT, Piece* o) {
  o->q = prompt_seq(a, s);
  o->s = s;
  o->rt = rt;
  o->q0 = rt * RT;
  o->nq = min(RT, o->q.n * a.G - o->q0);
  if (o->nq <= 0) return false;
  o->open = prompt_seen(o->q, div_group(a, o->q0));
  o->n_tile = max(1, (prompt_seen(o->q, div_group(a, o->q0 + o->nq - 1)) + TK - 1) / TK);
  return true;
}
__device__ __forceinline__ void share_of(int n_tile, int share, int shares, int* t0, int* n) {
  *t0 = (int)((long long)n_tile * share / shares);
  *n = (int)((long long)n_tile * (share + 1) / shares) - *t0;
}

/* walks the pieces of one CTA; every role runs the same walk.  Of a list that is sorted by length a CTA takes places
   c, 2 G - 1 - c, 2 G + c, 4 G - 1 - c ...: its share of every length */
template <int RT>
struct Walk {
  int turn, nth;
  __device__ __forceinline__ bool next(const PromptArgs& a, const PromptPlan& p, Piece* o) {
    const int G = gridDim.x, c = blockIdx.x;
    const int per = a.KV * p.shares;
    int n_entry = 0;
    if (!p.direct) n_entry = p.list ? *p.n_list : (prompt_seq(a, 0).n * a.G + RT - 1) / RT;
    const int total = (int)min((long long)n_entry * per, 0x7ffe0000ll);
    for (;; ) {
      const int at = turn * G + (turn & 1 ? G - 1 - c : c);
      int s, rt, u;
      if (p.direct) {
        if (turn++ > 0) return false;
        const int e = at / per;
        u = at - e * per;
        s = e % a.n_seq;
        rt = e / a.n_seq;
      } else {
        if (turn * G >= total) return false;
        ++turn;
        if (at >= total) continue;
        const int e = at / per;
        u = at - e * per;
        const int2 x = p.list ? p.list[e] : make_int2(0, n_entry - 1 - e);
        s = x.x;
        rt = x.y;
      }
      if (!row_tile(a, s, rt, RT, o)) continue;
      o->share = u / a.KV;
      o->kvh = u - o->share * a.KV;
      share_of(o->n_tile, o->share, p.shares, &o->t0, &o->n);
      if (o->n <= 0) continue;
      o->nth = nth++;
      return true;
    }
  }
};

/* which of positions [pos, pos + 32) a row that sees `seen` keys sees */
__device__ __forceinline__ uint32_t sees32(int seen, int pos) {
  const int n = seen - pos;
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

/*
 * What infinities and NaN of V at the marked positions of [from, upto) add to columns [d0, d0 + 32) of the sum
 * of a row that sees the keys below upto.  Not inlined, for the registers of the kernel's own loops.
 */
template <typename T>
__device__ __noinline__ void add_odd(const PromptArgs& a, PromptSeq q, const uint32_t* marks, int kvh, const T* qr, int from, int upto, int d0,
                                     float m, float* o) {
  const int hd = a.hd;
  for (int w = 0; w < kOddWords; ++w)
    for (uint32_t bits = marks[w]; bits; bits &= bits - 1)
      for (int pos = from + ((w * 32 + __ffs(bits) - 1 - from) & (32 * kOddWords - 1)); pos < upto; pos += 32 * kOddWords) {
        const T *kr = (const T*)a.k + (q.k0 + pos) * a.k_row + kvh * hd, *vr = (const T*)a.v + (q.k0 + pos) * a.v_row + kvh * hd + d0;
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
    prompt_tc_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const __grid_constant__ PromptArgs a,
                   const __grid_constant__ PromptPlan p) {
  using C = TcCfg<HD, PAIR>;
  constexpr bool F16 = std::is_same<T, __half>::value;
  /* weights are at most 2^(RAISE + GROW): fp16, whose largest number is just under 2^16, holds 11 bits of one down to 2^-26 of
     the maximum (tree_attention.cu, kRaise); bf16 has the range without */
  constexpr float RAISE = F16 ? 12.f : 0.f, GROW = F16 ? 3.9f : 8.f;
  constexpr uint32_t FMT = F16 ? 0u : (1u << 7) | (1u << 10);
  constexpr uint32_t ID_S = (1u << 4) | FMT | ((TK >> 3) << 17) | ((128 >> 4) << 24);
  constexpr uint32_t ID_O = (1u << 4) | FMT | (1u << 16) | ((HD >> 3) << 17) | ((128 >> 4) << 24);
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t k_full[C::NK], k_free[C::NK], v_full[C::NV], v_free[C::NV], s_full[2][2], p_full[2][2], o_done[2][2], v_seen[2],
      piece[2], q_full, mma_done;
  __shared__ uint32_t tmem_sh;
  __shared__ uint32_t odd[2][kOddWords + 1]; /* of a piece (its number modulo 2): which positions modulo 1024, before len, lost a V element; any */
  uint8_t* const sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* const q_sm = sm;
  uint8_t* const k_sm = sm + C::NQ * C::QTILE;
  uint8_t* const v_sm = k_sm + C::NK * C::TILE;
  uint8_t* const stage_sm = C::STAGE ? v_sm + C::NV * C::TILE : q_sm;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hd = HD == 64 ? 64 : a.hd; /* HD = 128: 80, 96 or 128, the tiles' columns past it are zeros */

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
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < 2 * (kOddWords + 1)) odd[tid / (kOddWords + 1)][tid % (kOddWords + 1)] = 0;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sa(&tmem_sh)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();
  tc_before();
  __syncthreads();
  tc_after();
  Walk<C::RT> walk;
  walk.turn = 0;
  walk.nth = 0;
  const uint32_t tmem = tmem_sh;
  Piece pc = {};
  bool ok = true;
  /* stream X's tiles of a piece of n: PAIR all of them (none without rows), else every second */
  auto n_of = [&](int X) { return PAIR ? (X == 0 || pc.nq > 128 ? pc.n : 0) : (pc.n + 1 - X) >> 1; };

  /* registers: 128 x 104 + 256 x 200 = 384 x 168, what the block was launched with */
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 0 || warp == 3) {
      /* ------------------------------------------------ TMA: warp 0 the K tiles, warp 3 the V tiles, in order.
         A warp each: asking for a free slot and issuing take some hundreds of cycles a tile. */
      const CUtensorMap* const map = warp == 0 ? &mk : &mv;
      uint8_t* const ring = warp == 0 ? k_sm : v_sm;
      uint64_t* const full = warp == 0 ? k_full : v_full;
      uint64_t* const free = warp == 0 ? k_free : v_free;
      const int nring = warp == 0 ? C::NK : C::NV;
      int slot = 0, issued = 0;
      uint32_t phase = 1; /* of the free barrier: the first round passes */
      while (ok && walk.next(a, p, &pc)) {
        if (warp == 3) /* its rows of q are wanted soon: a line a lane */
          for (int i = lane; i * 64 < pc.nq * hd; i += 32) {
            const int qi = pc.q0 + i * 64 / hd, row = div_group(a, qi);
            asm volatile("prefetch.global.L2 [%0];" ::"l"((const T*)a.q + (pc.q.r0 + row) * a.q_row + (pc.kvh * a.G + qi - row * a.G) * hd + i * 64 % hd));
          }
        ok = ring_copy(pc.n, [](int) {}, [&]() { return mb_wait_warp(&free[slot], phase); }, [&](int t) {
          if (elect()) {
            const int at = pc.q.k0 + (pc.t0 + t) * TK; /* rows past the sequence's, too: masked; past the array: zeros */
            uint8_t* const d = ring + slot * C::TILE;
            mb_expect(&full[slot], (uint32_t)C::TILE);
#pragma unroll
            for (int h = 0; h < HD / 64; ++h) tma3(d + h * TK * 128, map, h * 64, pc.kvh, at, &full[slot]);
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
      const uint64_t dq = desc_k(sa(q_sm)) + (PAIR ? X * (C::QTILE >> 4) : 0), dk = desc_k(sa(k_sm)), dv = desc_mn<TK>(sa(v_sm));
      const uint32_t ds = tmem + X * 128, dov = tmem + 256 + X * HD;
      while (ok && walk.next(a, p, &pc)) {
        ok = mb_wait_warp(&q_full, qp);
        qp ^= 1;
        const int n = n_of(X), clear = pc.open;
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
    uint32_t used = 0;       /* V tiles of earlier pieces */
    uint32_t sp = 0, op = 0, vsp = 0; /* phases of s_full[X][b] and o_done[X][b] in bit b, of piece and v_seen */
    constexpr int QW = C::NQ * TQ * (HD / 8) / 256; /* 16-byte words of Q a thread */
    bool have = walk.next(a, p, &pc);
    while (have) {
      { /* the rows of Q: word j of this thread; zeros past the tile's queries and past hd */
        uint4 qx[QW];
#pragma unroll
        for (int j = 0; j < QW; ++j) {
          const int i = tid - 128 + j * 256, r = i / (HD / 8), ch = i % (HD / 8), qi = pc.q0 + r, row = div_group(a, qi);
          const T* src = (const T*)a.q + (pc.q.r0 + row) * a.q_row + (pc.kvh * a.G + qi - row * a.G) * hd + ch * 8;
          qx[j] = r < pc.nq && ch * 8 < hd ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < QW; ++j) {
          const int i = tid - 128 + j * 256, r = i / (HD / 8), ch = i % (HD / 8);
          *reinterpret_cast<uint4*>(q_sm + (r >> 7) * C::QTILE + (ch >> 3) * (TQ * 128) + sw128(r & 127, ch & 7)) = qx[j];
        }
      }
      fence_async();
      __syncwarp();
      if (lane == 0 && ok) mb_arrive(&q_full);

      const int r = (PAIR ? X * 128 : 0) + row, qi = pc.q0 + r;
      const bool live = r < pc.nq, warp_live = r - lane < pc.nq;
      const int ri = live ? div_group(a, qi) : 0, head = qi - ri * a.G;
      const int n = n_of(X), open = pc.open, seen = prompt_seen(pc.q, ri);
      float m = -INFINITY, l = 0.f; /* m: the maximum that weights are taken against, less RAISE */
      for (int i = 0; i < n && ok; ++i) {
        const int t = pc.t0 + (PAIR ? i : 2 * i + X), pos = t * TK;
        const int b = i & 1;
        const uint32_t ts = tmem + lanes + X * 128 + b * TK;
        const bool masked = (t + 1) * TK > open;
        if (!mb_wait_warp(&s_full[X][b], (sp >> b) & 1)) { ok = false; break; }
        tc_after();
        if (warp_live) {
          uint32_t sr[TK];
#pragma unroll
          for (int c = 0; c < TK; c += 32) tm_ld(ts + c, sr + c);
          tm_ld_wait();
          if (masked) {
#pragma unroll
            for (int c0 = 0; c0 < TK; c0 += 32) {
              const uint32_t see = sees32(seen, pos + c0);
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (!((see >> c) & 1u)) sr[c0 + c] = 0xff800000u; /* -inf */
            }
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
          if (i == 0) { /* nothing to go by: the maximum first */
            float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
            for (int c = 0; c < TK; c += 4) {
              x0 = max3(x0, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
              x1 = max3(x1, __uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3]));
            }
            m = __fmaf_rn(fmaxf(x0, x1), a.scale2, -RAISE);
          }
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
          const int lo = max(0, open - pos); /* first key of the tile that some row does not see */
          auto clear = [&](int j) {
            const uint4 x = v[j];
            /* an exponent of all ones carries into the sign's place */
            constexpr uint32_t N = 0x7fff7fffu, C1 = F16 ? 0x04000400u : 0x00800080u;
            if (!((((x.x & N) + C1) | ((x.y & N) + C1) | ((x.z & N) + C1) | ((x.w & N) + C1)) & 0x80008000u)) return;
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
      /* ---- the piece's end */
      const Piece c = pc;
      have = walk.next(a, p, &pc);
      if (ok) ok = mb_wait_warp(&piece[X], op);
      op ^= 1;
      used += c.n;
      tc_before();
      sync_softmax(); /* both streams are through: Q may be replaced, O of either is whole */
      tc_after();
      if (tid - 128 <= kOddWords) odd[(c.nth & 1) ^ 1][tid - 128] = 0; /* for the next piece */
      const bool whole = p.shares == 1;
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
      const long long at = live ? (long long)(c.q.r0 + ri) * a.H + c.kvh * a.G + head : 0;
      const long long ps = ((((long long)c.s * p.row_tiles + c.rt) * a.KV + c.kvh) * p.shares + c.share) * C::RT + r;
      const float inv = l == 0.f ? 0.f : __fdividef(1.f, l); /* 0: the row sees nothing */
      if (warp_live && ok) {
        constexpr int COLS = PAIR ? HD : HD / 2;
        uint4* const stage = reinterpret_cast<uint4*>(stage_sm) + (warp - 4) * 256;
        long long row_at[4]; /* of the rows whose words this lane writes */
#pragma unroll
        for (int k = 0; k < 4; ++k) row_at[k] = __shfl_sync(0xffffffffu, at, k * 8 + (lane >> 2));
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
            const int from = max(c.t0 * TK, open / TK * TK), upto = min(seen, (c.t0 + c.n) * TK);
            add_odd<T>(a, c.q, odd[c.nth & 1], c.kvh, (const T*)a.q + (c.q.r0 + ri) * a.q_row + (c.kvh * a.G + head) * hd, from, upto, d0, m, more);
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
              const uint4 x = stage[y * 4 + (w ^ ((y >> 1) & 3))];
              if (r - lane + y < c.nq && d0 + w * 8 < hd) *reinterpret_cast<uint4*>((T*)a.out + row_at[k] * hd + d0 + w * 8) = x;
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
              if (r - lane + y < c.nq) __stcg(reinterpret_cast<uint4*>(p.po + (ps - lane + y) * HD + d0 + w * 4), x);
            }
          }
          __syncwarp(); /* the words may be replaced, the next TMEM load is the whole warp's */
        }
        if (live && (PAIR || X == 0)) {
          if (!whole) __stcg(reinterpret_cast<float2*>(p.pml + ps * 2), make_float2(m, l));
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

/* join the shares of a (sequence, row tile, kv head): a warp a row, shares in order */
template <typename T, int HD, int RT>
__global__ void __launch_bounds__(kJoinRows * 32) prompt_join_kernel(const __grid_constant__ PromptArgs a, const __grid_constant__ PromptPlan p) {
  pdl_wait();
  pdl_trigger();
  const int unit = blockIdx.x, kvh = unit % a.KV, rt = unit / a.KV % p.row_tiles, s = unit / a.KV / p.row_tiles;
  const int r = blockIdx.y * kJoinRows + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  Piece c;
  if (!row_tile(a, s, rt, RT, &c) || r >= c.nq) return;
  auto place = [&](int i) { return ((long long)unit * p.shares + i) * RT + r; };
  auto some = [&](int i) {
    int t0, n;
    share_of(c.n_tile, i, p.shares, &t0, &n);
    return n > 0;
  };
  float M = -INFINITY;
  for (int i = lane; i < p.shares; i += 32)
    if (some(i)) M = fmaxf(M, __ldcg(p.pml + place(i) * 2));
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float U = M == -INFINITY ? 0.f : M;
  constexpr int E = HD / 32;
  float x[E] = {}, L = 0.f;
  for (int i = 0; i < p.shares; ++i) {
    if (!some(i)) continue;
    const long long at = place(i);
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.pml + at * 2));
    float y[E];
    if constexpr (E == 4) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p.po + at * HD + lane * 4));
      y[0] = v.x; y[1] = v.y; y[2] = v.z; y[3] = v.w;
    } else {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(p.po + at * HD + lane * 2));
      y[0] = v.x; y[1] = v.y;
    }
    const float f = ex2(ml.x - U);
    L += ml.y * f;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] += y[e] * f;
  }
  const float inv = L == 0.f ? 0.f : __fdividef(1.f, L);
  const int qi = c.q0 + r;
  const long long at = (long long)(c.q.r0 + qi / a.G) * a.H + kvh * a.G + qi % a.G;
  const int hd = a.hd;
  if (lane == 0 && a.lse) a.lse[at] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
  if (lane * E >= hd) return;
  T* out = (T*)a.out + at * hd + lane * E;
  if constexpr (E == 4) *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(x[0] * inv, x[1] * inv), pack2<T>(x[2] * inv, x[3] * inv));
  else *reinterpret_cast<uint32_t*>(out) = pack2<T>(x[0] * inv, x[1] * inv);
}

/*
 * The row tiles of all sequences, the most keys first (to 1 / 1024 of the most there are): a counting sort by one block,
 * a warp a sequence.  The order inside a step of it is that of the atomics; it decides which CTA takes a unit and no result.
 */
constexpr int kSteps = 1024;
template <int RT>
__global__ void __launch_bounds__(1024) prompt_order_kernel(const __grid_constant__ PromptArgs a, int2* list, int* n_list, int cap) {
  pdl_wait();
  pdl_trigger();
  __shared__ int at[kSteps], sums[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int most = max(1, (a.max_k + TK - 1) / TK);
  at[tid] = 0;
  __syncthreads();
  auto each = [&](auto&& f) {
    for (int s = warp; s < a.n_seq; s += 32) {
      const PromptSeq q = prompt_seq(a, s);
      const int n = (q.n * a.G + RT - 1) / RT;
      for (int rt = lane; rt < n; rt += 32) {
        Piece c;
        row_tile(a, s, rt, RT, &c);
        f(s, rt, kSteps - 1 - (int)((long long)(min(c.n_tile, most) - 1) * kSteps / most));
      }
    }
  };
  each([&](int, int, int step) { atomicAdd(&at[step], 1); });
  __syncthreads();
  const int c = at[tid];
  int x = c;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  for (int w = 0; w < warp; ++w) x += sums[w];
  at[tid] = x - c;
  if (tid == kSteps - 1) *n_list = min(x, cap);
  __syncthreads();
  each([&](int s, int rt, int step) {
    const int i = atomicAdd(&at[step], 1);
    if (i < cap) list[i] = make_int2(s, rt);
  });
}

/* K or V as [row][head][hd], a box = 64 of hd x the rows of a tile */
int rows_map(const PromptArgs& a, bool f16, const void* rows, long long stride, CUtensorMap* m) {
  EncodeTiledFn enc = encode_tiled();
  ULB_CHECK(enc, ULB_ECUDA, "ulb_prompt_attention: no cuTensorMapEncodeTiled entry point");
  const cuuint64_t dim[3] = {(cuuint64_t)a.hd, (cuuint64_t)a.KV, (cuuint64_t)a.k_rows};
  const cuuint64_t str[2] = {(cuuint64_t)a.hd * 2, (cuuint64_t)stride * 2};
  const cuuint32_t box[3] = {64, 1, TK}, es[3] = {1, 1, 1};
  const CUresult r = enc(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(rows), dim, str, box,
                         es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  ULB_CHECK(r == CUDA_SUCCESS, ULB_EINVAL, "ulb_prompt_attention: the rows' layout has no tensor map (CUresult %d)", (int)r);
  return ULB_OK;
}

constexpr int kShareTiles = 16; /* tiles a share has at least */
/*
 * Into how many shares the keys of a row tile are cut: as many as fill the SMs best.  Units that are as many as the SMs
 * four times over stay whole (sorted by length they even out); a share costs a twentieth more for what it leaves to join.
 * The lengths are on the device, so every sequence counts as the longest, which is wrong for a long chunk with short
 * sequences beside it: 513 rows after 30000 keys take 276 us alone and 512 with one sequence of 10 rows beside them, 1 row
 * after 20000 keys 27 alone and 184 with 15 (such a chunk is quicker in a call of its own; the header says so).  Counts that
 * the host could make instead were no better: row tiles that q_rows can hold gave 297 to 520 us for these by chance of the
 * waves, and 195 for 151 on three chunks of 300 rows after 8000 keys with five of 40 rows; k_rows / max_k sequences cut far too
 * finely where max_k is a loose bound.
 */
int pick_shares(long long units, int tiles, int n_sm, long long most) {
  if (units >= 4ll * n_sm) return 1;
  int best = 1;
  double time = 1e30;
  for (int s = 1; s <= 64 && (s == 1 || (tiles / s >= kShareTiles && units * s <= most)); ++s) {
    const double waves = (double)((units * s + n_sm - 1) / n_sm), t = waves / s * (s > 1 ? 1.05 : 1.0);
    if (t < time - 1e-9) {
      time = t;
      best = s;
    }
  }
  return best;
}

template <typename T, int HD, bool PAIR>
int launch_tc(Ctx* c, const PromptArgs& a) {
  using C = TcCfg<HD, PAIR>;
  static uint64_t attr = 0; /* devices it is set on */
  if (!(attr >> (c->device & 63) & 1)) {
    ULB_CUDA(cudaFuncSetAttribute(prompt_tc_kernel<T, HD, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    attr |= 1ull << (c->device & 63);
  }
  CUtensorMap mk, mv;
  constexpr bool f16 = std::is_same<T, __half>::value;
  ULB_TRY(rows_map(a, f16, a.k, a.k_row, &mk));
  ULB_TRY(rows_map(a, f16, a.v, a.v_row, &mv));
  PromptPlan p = {};
  p.row_tiles = (int)(((long long)a.max_q * a.G + C::RT - 1) / C::RT);
  const long long units = (long long)a.n_seq * p.row_tiles * a.KV;
  p.shares = pick_shares(units, (a.max_k + TK - 1) / TK, c->n_sm, (long long)kTreeWsFloats / 2 / (C::RT * (HD + 2)));
  p.direct = units * p.shares <= c->n_sm;
  float* ws = a.ws;
  if (p.shares > 1) { /* at most half of the workspace */
    p.po = ws;
    p.pml = p.po + units * p.shares * C::RT * HD;
    ws = p.pml + units * p.shares * C::RT * 2;
  }
  if (!p.direct) {
    /* whatever q_start holds: room for every row tile of every sequence, or for what q_rows can hold (ranges that overlap lose
       rows then) */
    const long long room = ((long long)kTreeWsFloats - (ws - a.ws) - 4) / 2, all = (long long)a.n_seq * p.row_tiles;
    const long long entries = std::min<long long>(all, (long long)a.q_rows * a.G / C::RT + a.n_seq);
    ULB_CHECK(entries <= room && entries * a.KV * p.shares < 0x7ffe0000ll, ULB_EUNSUPPORTED, "ulb_prompt_attention: %d sequences of %d rows",
              a.n_seq, a.max_q);
    const int cap = (int)std::min<long long>(std::min(all, room), 0x7ffe0000ll);
    if (a.n_seq > 1) {
      int* const n_list = reinterpret_cast<int*>(ws);
      int2* const list = reinterpret_cast<int2*>(ws + 4);
      p.n_list = n_list;
      p.list = list;
      ULB_LAUNCH("prompt order launch", launch_k(c, prompt_order_kernel<C::RT>, dim3(1), dim3(1024), 0, a, list, n_list, cap));
    }
  }
  const int grid = p.direct ? (int)(units * p.shares) : c->n_sm;
  ULB_LAUNCH("prompt attention launch", launch_k(c, prompt_tc_kernel<T, HD, PAIR>, dim3(grid), dim3(kThreads), C::SMEM, mk, mv, a, p));
  if (p.shares > 1)
    ULB_LAUNCH("prompt join launch", launch_k(c, prompt_join_kernel<T, HD, C::RT>, dim3((unsigned)units, C::RT / kJoinRows), dim3(kJoinRows * 32), 0, a, p));
  return ULB_OK;
}

template <typename T>
int pick_tc(Ctx* c, const PromptArgs& a) {
  /* 256 queries a CTA share each K / V tile; where that leaves half of the SMs without a unit, and the keys are too few to be
     cut into shares, 128 a CTA: 500 rows of 32 heads over 4 12.2 us against 17.0, but 513 rows after 30000 keys (shares) 303
     against 278 */
  const long long units = (long long)a.n_seq * (((long long)a.max_q * a.G + 255) / 256) * a.KV;
  const bool pair = (long long)a.max_q * a.G > 128 && (units * 2 > c->n_sm || a.max_k >= 2 * kShareTiles * TK);
  if (a.hd == 64) return pair ? launch_tc<T, 64, true>(c, a) : launch_tc<T, 64, false>(c, a);
  return pair ? launch_tc<T, 128, true>(c, a) : launch_tc<T, 128, false>(c, a);
}

}  // namespace

/*
 * When this form runs: head dims up to 128 and more than 128 keys.  Below, encoding the tensor maps on the host and starting up
 * cost more than the tensor cores give: 1 to 128 rows of as many keys 9.4 us here, 8.8 as mma.sync; 8 x 50-100 rows 12.9 /
 * 13.5; 1 x 16 rows x 1016 keys, 32 kv heads 16.8 / 32; 1 row x 5001 keys 23 / 140.
 */
bool prompt_tc_fits(const PromptArgs& a) { return a.hd <= 128 && a.max_k > 128; }

int launch_prompt_tc(Ctx* c, const PromptArgs& a, bool f16) { return f16 ? pick_tc<__half>(c, a) : pick_tc<__nv_bfloat16>(c, a); }

}  // namespace ulb

ULB_TRACE_UNIT(prompt_attention_tc)
