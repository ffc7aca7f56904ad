/*
 * prompt_attention.cu — causal attention of packed prompts (ulb_prompt_attention): the entry point, and
 * the mma.sync form of the kernel.  The reference's flash_attention*.glsl (src/shaders/attention) know
 * one sequence of a fixed cache.
 *
 * Mathematics.  For row i of a sequence's n and head h, over the keys t <= len - n + i: s_t = scale q . k_t,
 * m = max s_t, l = sum exp(s_t - m), o = sum exp(s_t - m) v_t / l, in one pass with the running maximum.
 *
 * Work of a CTA: RT = 16 WM queries (row x head of the group, so a K / V tile serves all heads that share it) against
 * the keys up to the last row's, in tiles of 64 keys through a ring of cp.async stages.  The warps are WM row
 * groups x WK key groups; a key group has its own (m, l, o), joined in shared memory.  Weights stay in
 * registers, rounded to the rows' type once: V has that type, and a second part of each weight would be half as many products
 * again.  Outputs are off by 1.9e-3 (bf16) and 2.4e-4 (fp16) against 64 bits, of which 1.6e-3 and 2.0e-4 are their own rounding.
 *
 * Used for head_dim 256 and for calls of at most 128 keys (prompt_attention_tc.cu, which has the rule): 64 rows of 32 heads over
 * 8 of 64 9 us, the host's call; as the only form four prompts of 2 to 6 thousand rows of head_dim 128 took 2960 us.  At
 * head_dim 256, 4096 rows of 32 heads over 8 take 1155 us (0.24 PFLOP/s), 500 rows 35 us: one CTA of 8 warps an SM (registers and
 * shared memory), whose products, loads and softmax wait for each other (26 % of the issue slots, mma.sync's pipe 40 % of the time).
 *
 * What a row does not see never reaches its result: scores past its last key are replaced, keys past the tile's last
 * are zero-filled (the rows there belong to the next sequence), and an element of V in a tile on the diagonal that is
 * not finite is taken out and added to the rows that see it.
 */
#include "prompt_attention.h"

#include <algorithm>
#include <cmath>

namespace ulb {
namespace {

constexpr int BK = 64; /* keys a tile */

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
/* weights are exp(s - m + raise): fp16 keeps 11 bits of one down to 2^-28 of the heaviest (tree_attention.cu) */
template <typename T> constexpr float kRaise = std::is_same<T, __half>::value ? 14.f : 0.f;

template <int HD, int WM, int WK>
struct Cfg {
  static constexpr int NT = WM * WK * 32, RT = 16 * WM, KW = BK / WK;
  static constexpr int PITCH = (HD + 8) * 2; /* bytes between rows of a tile: odd in units of 16 */
  static constexpr int STAGE = 2 * BK * PITCH;
  static constexpr int NST = 2;
  static constexpr int OP = HD + 4;
  static constexpr int JOIN = WK > 1 ? WK * RT * OP * 4 : 0;
  static constexpr int SMEM = NST * STAGE > JOIN ? NST * STAGE : JOIN;
  static_assert(SMEM <= 200 * 1024, "shared memory");
};

template <typename T, int HD, int WM, int WK>
__global__ void __launch_bounds__(WM* WK * 32) prompt_kernel(const __grid_constant__ PromptArgs a, int n_tile) {
  using C = Cfg<HD, WM, WK>;
  constexpr int KS = HD / 16, NB = C::KW / 8, DB = HD / 8;
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ float sh_m[WK][C::RT], sh_l[WK][C::RT];
  __shared__ int odd_v;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int wm = warp / WK, wk = warp % WK;
  int id = blockIdx.x;
  const int kvh = id % a.KV;
  id /= a.KV;
  const int s = id % a.n_seq, rt = n_tile - 1 - id / a.n_seq; /* the longest row tiles first */
  const PromptSeq q = prompt_seq(a, s);
  const int q0 = rt * C::RT, nq = min(C::RT, q.n * a.G - q0); /* queries of this tile: qi = row * G + head of the group */
  if (nq <= 0) return;
  const int k1 = prompt_seen(q, (q0 + nq - 1) / a.G), open = prompt_seen(q, q0 / a.G);
  if (tid == 0) odd_v = 0;

  const T* const kb = (const T*)a.k + q.k0 * a.k_row + kvh * HD;
  const T* const vb = (const T*)a.v + q.k0 * a.v_row + kvh * HD;
  auto stage = [&](int it) { /* one tile into its stage: eight threads a row; rows past k1 are zero */
    uint8_t* const ks = sm + (it % C::NST) * C::STAGE;
    for (int j = tid >> 3; j < BK; j += C::NT / 8) {
      const int pos = it * BK + j;
      const bool ok = pos < k1;
      const long long row = ok ? pos : 0;
      const uint32_t d = saddr(ks + j * C::PITCH);
#pragma unroll
      for (int c = tid & 7; c < HD / 8; c += 8) {
        cp16(d + c * 16, kb + row * a.k_row + c * 8, ok);
        cp16(d + BK * C::PITCH + c * 16, vb + row * a.v_row + c * 8, ok);
      }
    }
  };
  const int n_it = (k1 + BK - 1) / BK;
#pragma unroll
  for (int i = 0; i < C::NST - 1; ++i) {
    if (i < n_it) stage(i);
    cp_commit();
  }

  /* Q of rows g and g + 8 as A fragments */
  const int qa = q0 + wm * 16 + g, qb = qa + 8, lim = q0 + nq;
  const bool va = qa < lim, vbq = qb < lim;
  const int ia = va ? qa / a.G : 0, ib = vbq ? qb / a.G : 0;
  const int na = prompt_seen(q, ia), nb = prompt_seen(q, ib);
  uint32_t qf[KS][4];
  {
    const T* pa = (const T*)a.q + (q.r0 + ia) * a.q_row + (kvh * a.G + (va ? qa % a.G : 0)) * HD;
    const T* pb = (const T*)a.q + (q.r0 + ib) * a.q_row + (kvh * a.G + (vbq ? qb % a.G : 0)) * HD;
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
    if (it + C::NST - 1 < n_it) stage(it + C::NST - 1);
    cp_commit();
    uint8_t* const ks = sm + (it % C::NST) * C::STAGE;
    const int tile0 = it * BK;
    const bool masked = tile0 + BK > open;
    bool fix = false;
    if (masked) { /* V elements that are not finite leave the tile (see the top) */
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

    float sc[NB][4]; /* S of this warp's KW keys */
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
    if (masked) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int pos = key0 + n * 8 + e;
          if (pos >= na) sc[n][e] = -INFINITY;
          if (pos >= nb) sc[n][2 + e] = -INFINITY;
        }
    }
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
    const uint32_t vaddr = saddr(ks) + BK * C::PITCH + (wk * C::KW + ((lane >> 3) & 1) * 8 + (lane & 7)) * C::PITCH + (lane >> 4) * 16;
#pragma unroll
    for (int n = 0; n < NB; n += 2) {
      const uint32_t pf[4] = {pack2<T>(sc[n][0], sc[n][1]), pack2<T>(sc[n][2], sc[n][3]), pack2<T>(sc[n + 1][0], sc[n + 1][1]),
                              pack2<T>(sc[n + 1][2], sc[n + 1][3])};
#pragma unroll
      for (int d = 0; d < DB; d += 2) {
        uint32_t b[4];
        ldsm4t(vaddr + n * 8 * C::PITCH + d * 16, b);
        mma<T>(o[d], pf, b[0], b[1]);
        mma<T>(o[d + 1], pf, b[2], b[3]);
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
        if (pos >= k1) continue; /* the same for all lanes */
        const T* vr = vb + pos * a.v_row;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = to_f<T>(vr[d * 8 + 2 * t + e]);
            if (isfinite(x)) continue;
            if (pos < na) o[d][e] += pa * x;
            if (pos < nb) o[d][2 + e] += pb * x;
          }
      }
    }
  }

  lA += __shfl_xor_sync(0xffffffffu, lA, 1);
  lB += __shfl_xor_sync(0xffffffffu, lB, 1);
  lA += __shfl_xor_sync(0xffffffffu, lA, 2);
  lB += __shfl_xor_sync(0xffffffffu, lB, 2);
  auto place = [&](int qi) { return (long long)(q.r0 + qi / a.G) * a.H + kvh * a.G + qi % a.G; };
  if constexpr (WK == 1) {
    const float iA = lA == 0.f ? 0.f : __fdividef(1.f, lA), iB = lB == 0.f ? 0.f : __fdividef(1.f, lB); /* 0: sees nothing */
    const long long pa = place(qa), pb = place(qb);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      if (va) *reinterpret_cast<uint32_t*>((T*)a.out + pa * HD + d * 8 + 2 * t) = pack2<T>(o[d][0] * iA, o[d][1] * iA);
      if (vbq) *reinterpret_cast<uint32_t*>((T*)a.out + pb * HD + d * 8 + 2 * t) = pack2<T>(o[d][2] * iB, o[d][3] * iB);
    }
    if (a.lse && t == 0) {
      if (va) a.lse[pa] = lA == 0.f ? -INFINITY : (mA + log2f(lA)) * kLn2;
      if (vbq) a.lse[pb] = lB == 0.f ? -INFINITY : (mB + log2f(lB)) * kLn2;
    }
  } else {
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
      const long long at = place(q0 + r);
      const float inv = L == 0.f ? 0.f : __fdividef(1.f, L);
      *reinterpret_cast<uint2*>((T*)a.out + at * HD + d) = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
      if (d == 0 && a.lse) a.lse[at] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
    }
  }
}

template <typename T, int HD, int WM, int WK>
int launch_prompt(Ctx* c, const PromptArgs& a) {
  using C = Cfg<HD, WM, WK>;
  static uint64_t attr = 0; /* devices it is set on */
  if (!(attr >> (c->device & 63) & 1)) {
    ULB_CUDA(cudaFuncSetAttribute(prompt_kernel<T, HD, WM, WK>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    attr |= 1ull << (c->device & 63);
  }
  const long long n_tile = ((long long)a.max_q * a.G + C::RT - 1) / C::RT, blocks = n_tile * a.KV * a.n_seq;
  ULB_CHECK(blocks < (1ll << 31), ULB_EUNSUPPORTED, "ulb_prompt_attention: %d sequences of %d rows", a.n_seq, a.max_q);
  ULB_LAUNCH("prompt attention launch", launch_k(c, prompt_kernel<T, HD, WM, WK>, dim3((unsigned)blocks), dim3(C::NT), C::SMEM, a, (int)n_tile));
  return ULB_OK;
}

template <typename T>
int pick_dim(Ctx* c, const PromptArgs& a) {
  switch (a.hd) {
    case 64: return launch_prompt<T, 64, 4, 1>(c, a);
    case 80: return launch_prompt<T, 80, 4, 1>(c, a);
    case 96: return launch_prompt<T, 96, 4, 1>(c, a);
    case 128: return launch_prompt<T, 128, 4, 1>(c, a);
    default: return launch_prompt<T, 256, 4, 2>(c, a);
  }
}

}  // namespace
}  // namespace ulb

using namespace ulb;

extern "C" int ulb_prompt_attention(ulb_ctx* ctx, const ulb_prompt_desc* d, const void* q, const void* k, const void* v,
                                    const int32_t* q_start, const int32_t* k_start, void* out, float* lse) {
  ULB_CHECK(ctx && d, ULB_EINVAL, "ulb_prompt_attention: NULL argument");
  ULB_CHECK(d->dtype == ULB_TYPE_F16 || d->dtype == ULB_TYPE_BF16, ULB_EUNSUPPORTED, "ulb_prompt_attention: type %d (F16 or BF16)", d->dtype);
  ULB_CHECK(d->head_dim == 64 || d->head_dim == 80 || d->head_dim == 96 || d->head_dim == 128 || d->head_dim == 256, ULB_EUNSUPPORTED,
            "ulb_prompt_attention: head_dim %d (64, 80, 96, 128 or 256)", d->head_dim);
  ULB_CHECK(d->n_head > 0 && d->n_head_kv > 0 && d->n_head % d->n_head_kv == 0 && d->n_head / d->n_head_kv <= 64, ULB_EINVAL,
            "ulb_prompt_attention: %d heads over %d kv heads", d->n_head, d->n_head_kv);
  ULB_CHECK(d->n_seq >= 0 && d->q_rows >= 0 && d->k_rows >= 0 && d->max_q >= 0 && d->max_k >= 0, ULB_EINVAL,
            "ulb_prompt_attention: %d sequences of at most %d rows and %d keys in %d and %d", d->n_seq, d->max_q, d->max_k, d->q_rows, d->k_rows);
  ULB_CHECK(std::isfinite(d->scale) && d->scale > 0.f, ULB_EINVAL, "ulb_prompt_attention: scale %g", (double)d->scale);
  PromptArgs a = {};
  a.H = d->n_head;
  a.KV = d->n_head_kv;
  a.G = a.H / a.KV;
  a.hd = d->head_dim;
  unsigned log = 0;
  while ((1 << log) < a.G) ++log;
  a.g_mul = log ? (unsigned)(((1ull << (31 + log)) + a.G - 1) / a.G) : 0;
  a.g_shift = log ? log - 1 : 0;
  a.q_row = d->q_row ? d->q_row : (long long)a.H * a.hd;
  a.k_row = d->k_row ? d->k_row : (long long)a.KV * a.hd;
  a.v_row = d->v_row ? d->v_row : (long long)a.KV * a.hd;
  ULB_CHECK(a.q_row >= (long long)a.H * a.hd && a.k_row >= (long long)a.KV * a.hd && a.v_row >= (long long)a.KV * a.hd && a.q_row % 8 == 0 &&
                a.k_row % 8 == 0 && a.v_row % 8 == 0,
            ULB_EINVAL, "ulb_prompt_attention: rows %lld, %lld and %lld elements apart (multiples of 8 that hold the heads)", a.q_row,
            a.k_row, a.v_row);
  if (d->n_seq == 0 || d->q_rows == 0 || d->max_q == 0) return ULB_OK;
  ULB_CHECK(q && q_start && k_start && out && (d->k_rows == 0 || (k && v)), ULB_EINVAL, "ulb_prompt_attention: NULL argument");
  ULB_CHECK(ULB_ALIGNED16(q) && ULB_ALIGNED16(k) && ULB_ALIGNED16(v) && ULB_ALIGNED16(out), ULB_EINVAL,
            "ulb_prompt_attention: q, k, v and out must be 16-byte aligned");
  ULB_CHECK(words_aligned({q_start, k_start, lse}), ULB_EINVAL, "ulb_prompt_attention: unaligned array of 32-bit elements");
  ULB_CHECK((long long)d->q_rows * a.H < (1ll << 31) && d->k_rows <= 0x7fff0000, ULB_EUNSUPPORTED, "ulb_prompt_attention: %d rows of %d heads, %d keys",
            d->q_rows, a.H, d->k_rows);
  a.n_seq = d->n_seq;
  a.q_rows = d->q_rows;
  a.k_rows = d->k_rows;
  a.max_q = std::min(d->max_q, d->q_rows);
  a.max_k = std::min(d->max_k, d->k_rows);
  a.scale2 = d->scale * kLog2e;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_start = q_start;
  a.k_start = k_start;
  a.out = out;
  a.lse = lse;
  Ctx* c = &ctx->c;
  a.err = c->dev_err;
  ULB_CUDA(cudaSetDevice(c->device));
  /* at the first call, whatever its shape, so that any later one can be captured */
  if (!c->tree_ws) ULB_CUDA(cudaMalloc((void**)&c->tree_ws, kTreeWsFloats * sizeof(float)));
  a.ws = c->tree_ws;
  if (prompt_tc_fits(a)) return launch_prompt_tc(c, a, d->dtype == ULB_TYPE_F16);
  return d->dtype == ULB_TYPE_F16 ? pick_dim<__half>(c, a) : pick_dim<__nv_bfloat16>(c, a);
}

ULB_TRACE_UNIT(prompt_attention)
