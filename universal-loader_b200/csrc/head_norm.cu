/*
 * head_norm.cu — RMS norms of the q and k heads with their rotary positions in one pass
 * (ulb_norm_rope_apply) and their gradient (ulb_norm_rope_grad).  The reference normalises whole rows only
 * (src/shaders/rmsnorm.glsl).
 *
 * Mathematics.  With f = 1 / sqrt(mean x^2 + eps), n = x f and g = R^T dy (R^T turns by the negative angle):
 *   y = R (w n),   dx = f (w g - n mean(w g n)),   dw = sum over rows and heads of g n.
 * mean(w g n) = f mean(w g x), so both sums of a head, x^2 and w g x, are taken in one pass.  f comes from the hardware's
 * reciprocal square root (2^-22) and every sum is fp32: fp32 gradients are off by 1.6e-7 against 64 bits, where sums in 64
 * bits would leave 7e-8; 16-bit rows by their own rounding.
 *
 * Work.  Memory bounds it: every element is read once and written once (gradient: two reads).  A lane owns eight
 * elements of a head, both sides of four pairs, and 8, 16 or 32 lanes a head, so the sums are shuffles and pairs turn in
 * registers.  A warp keeps to one row, whose sines it computes once for all its heads, and has the next batch of heads
 * under way while it works on one; the weights are in shared memory.  When there are few rows, several warps share the heads
 * of one.  The sums of dw stay in registers over all rows of a warp, and a second small kernel adds the blocks in order.
 *
 * Measured: 16381 bf16 rows of 32 and 8 heads of 128 68 to 70 us, 4.8 TB/s (73 to 75 % of the copy rate); their gradient 102
 * to 108 us (71 to 75 %); in fp32 117 and 170 us (87 and 90 %); 1000 fp32 rows' gradient 19 us, of which the second kernel is 4;
 * 8 rows 5 us, a launch.  About 160 instructions a warp for two heads of 128 bound the forward pass beside HBM.  Two blocks
 * an SM with four steps of heads in flight; three blocks 76 us, three with two steps 69, four 88 to 93.
 */
#include "head_rows.h"

namespace ulb {
namespace {

template <typename T, int LPH, bool HALF>
__global__ void __launch_bounds__(kWarps * 32, 2) norm_rope_kernel(const __grid_constant__ HeadArgs a, int wide) {
  pdl_wait();
  pdl_trigger();
  __shared__ HeadWeights sw;
  const Place at = place_of<LPH, HALF>(a, threadIdx.x & 31);
  const Pairs pairs = pairs_of<HALF>(a, at);
  const float inv_hd = 1.f / a.hd;
  load_weights(a, &sw);
  const int qs = (int)a.q_head * (int)sizeof(T), ks = (int)a.k_head * (int)sizeof(T), os = a.hd * (int)sizeof(T);
  const int run = (at.d1 - at.d0) * (int)sizeof(T); /* bytes between a lane's runs */
  Turn t;
  char *oq = nullptr, *ok = nullptr;
  walk_rows<Eight<T>, LPH, sizeof(T) == 4 ? 2 : 4>(
      a, a.nq + a.nk, at.on,
      [&](int m) {
        return HeadBase{(const char*)((const T*)a.q + m * a.q_row + at.d0), (const char*)((const T*)a.k + m * a.k_row + at.d0) - (long long)a.nq * ks,
                        nullptr};
      },
      [&](const HeadBase& from, int h, bool mine) {
        Eight<T> e = zero8<T>();
        if (mine) {
          const bool is_q = h < a.nq;
          const char* p = (is_q ? from.q : from.k) + (long long)h * (is_q ? qs : ks);
          load_run((const T*)p, wide, &e.r[0]);
          load_run((const T*)(p + run), wide, &e.r[1]);
        }
        return e;
      },
      [&](int m, int pos) {
        turn_at(pairs, pos, a.mscale, &t);
        oq = (char*)((T*)a.oq + (long long)m * a.nq * a.hd + at.d0);
        ok = (char*)((T*)a.ok + ((long long)m * a.nk - a.nq) * a.hd + at.d0);
      },
      [&](int h, bool mine, const Eight<T>& e) {
        float x[8], w[8];
        unpack8(e, x);
        const bool is_q = h < a.nq;
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __fmaf_rn(x[j], x[j], ss);
        const float f = rsqrt_near(__fmaf_rn(head_sum<LPH>(ss), inv_hd, a.eps));
        lane_weights(sw, is_q ? 0 : 1, at, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= f * w[j];
        turn<HALF>(t, 1.f, x);
        if (!mine) return;
        char* o = (is_q ? oq : ok) + (long long)h * os;
        store4((T*)o, wide, x);
        store4((T*)(o + run), wide, x + 4);
      });
}

/* x and the gradient of the output */
template <typename T>
struct Both {
  Eight<T> x, y;
};
template <typename T, int LPH, bool HALF>
__global__ void __launch_bounds__(kWarps * 32, 2) norm_rope_grad_kernel(const __grid_constant__ HeadArgs a, int wide) {
  pdl_wait();
  pdl_trigger();
  __shared__ HeadWeights sw;
  __shared__ float sh[kWarps][2][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = lane / LPH;
  const Place at = place_of<LPH, HALF>(a, lane);
  const Pairs pairs = pairs_of<HALF>(a, at);
  const float inv_hd = 1.f / a.hd;
  load_weights(a, &sw);
  const int qs = (int)a.q_head * (int)sizeof(T), ks = (int)a.k_head * (int)sizeof(T), os = a.hd * (int)sizeof(T);
  const int run = (at.d1 - at.d0) * (int)sizeof(T);
  float sq[8] = {}, sk[8] = {};
  Turn t;
  char *oq = nullptr, *ok = nullptr;
  struct Source {
    const char *q, *k, *gq, *gk;
  };
  walk_rows<Both<T>, LPH, sizeof(T) == 4 ? 1 : 2>(
      a, a.nq + a.nk, at.on,
      [&](int m) {
        const long long oq = (long long)m * a.nq * a.hd + at.d0, ok = ((long long)m * a.nk - a.nq) * a.hd + at.d0;
        return Source{(const char*)((const T*)a.q + m * a.q_row + at.d0), (const char*)((const T*)a.k + m * a.k_row + at.d0) - (long long)a.nq * ks,
                      (const char*)((const T*)a.gq + oq), (const char*)((const T*)a.gk + ok)};
      },
      [&](const Source& from, int h, bool mine) {
        Both<T> e = {zero8<T>(), zero8<T>()};
        if (mine) {
          const bool is_q = h < a.nq;
          const char* p = (is_q ? from.q : from.k) + (long long)h * (is_q ? qs : ks);
          const char* g = (is_q ? from.gq : from.gk) + (long long)h * os;
          load_run((const T*)p, wide, &e.x.r[0]);
          load_run((const T*)(p + run), wide, &e.x.r[1]);
          load_run((const T*)g, wide, &e.y.r[0]);
          load_run((const T*)(g + run), wide, &e.y.r[1]);
        }
        return e;
      },
      [&](int m, int pos) {
        turn_at(pairs, pos, a.mscale, &t);
        oq = (char*)((T*)a.oq + (long long)m * a.nq * a.hd + at.d0);
        ok = (char*)((T*)a.ok + ((long long)m * a.nk - a.nq) * a.hd + at.d0);
      },
      [&](int h, bool mine, const Both<T>& e) {
        float x[8], y[8], w[8];
        unpack8(e.x, x);
        unpack8(e.y, y);
        const bool is_q = h < a.nq;
        turn<HALF>(t, -1.f, y); /* g */
        lane_weights(sw, is_q ? 0 : 1, at, w);
        float ss = 0.f, sg = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          w[j] *= y[j];
          ss = __fmaf_rn(x[j], x[j], ss);
          sg = __fmaf_rn(w[j], x[j], sg);
        }
        ss = head_sum<LPH>(ss);
        sg = head_sum<LPH>(sg);
        /* dx as f (w g - n mean(w g n)) with n = x f: f alone may be 2^63 or 2^-63, f^3 is no fp32 number then */
        const float f = rsqrt_near(__fmaf_rn(ss, inv_hd, a.eps)), c = f * (sg * inv_hd);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= f;
        /* y n, of the kind whose sum it belongs to (zero past the heads); both in one warp where heads are not whole steps: the
           other kind's sum keeps its value, whatever y n is */
        if (__all_sync(kAll, is_q)) {
#pragma unroll
          for (int j = 0; j < 8; ++j) sq[j] = __fmaf_rn(y[j], x[j], sq[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float to = __fmaf_rn(y[j], x[j], is_q ? sq[j] : sk[j]);
            sq[j] = is_q ? to : sq[j];
            sk[j] = is_q ? sk[j] : to;
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = f * __fmaf_rn(-x[j], c, w[j]);
        if (!mine) return;
        char* o = (is_q ? oq : ok) + (long long)h * os;
        store4((T*)o, wide, x);
        store4((T*)(o + run), wide, x + 4);
      });
  /* the block's share of dw: groups of a warp by shuffles, warps in order */
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int o = LPH; o < 32; o <<= 1) {
      sq[j] += __shfl_xor_sync(kAll, sq[j], o);
      sk[j] += __shfl_xor_sync(kAll, sk[j], o);
    }
    if (grp == 0 && at.on) {
      sh[warp][0][j < 4 ? at.d0 + j : at.d1 + j - 4] = sq[j];
      sh[warp][1][j < 4 ? at.d0 + j : at.d1 + j - 4] = sk[j];
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

template <typename T, bool HALF>
int launch_apply(Ctx* c, HeadArgs& a, int wide) {
  const int lph = lanes_of(a.hd), blocks = plan_rows(c, a, head_steps(a), c->n_sm * 2);
  auto go = [&](auto kern) -> int {
    ULB_LAUNCH("norm rope launch", launch_k(c, kern, dim3(blocks), dim3(kWarps * 32), 0, a, wide));
    return ULB_OK;
  };
  if (lph == 8) return go(norm_rope_kernel<T, 8, HALF>);
  if (lph == 16) return go(norm_rope_kernel<T, 16, HALF>);
  return go(norm_rope_kernel<T, 32, HALF>);
}
template <typename T>
int pick_apply(Ctx* c, HeadArgs& a, int wide) { return a.half ? launch_apply<T, true>(c, a, wide) : launch_apply<T, false>(c, a, wide); }
template <typename T, bool HALF>
int launch_grad(Ctx* c, HeadArgs& a, int wide, float* dwq, float* dwk) {
  const int lph = lanes_of(a.hd), blocks = plan_rows(c, a, head_steps(a), c->n_sm * kNormBlocks);
  auto go = [&](auto kern) -> int {
    ULB_LAUNCH("norm rope gradient launch", launch_k(c, kern, dim3(blocks), dim3(kWarps * 32), 0, a, wide));
    return ULB_OK;
  };
  if (lph == 8) ULB_TRY(go(norm_rope_grad_kernel<T, 8, HALF>));
  else if (lph == 16) ULB_TRY(go(norm_rope_grad_kernel<T, 16, HALF>));
  else ULB_TRY(go(norm_rope_grad_kernel<T, 32, HALF>));
  ULB_LAUNCH("norm rope gradient sum launch", launch_k(c, norm_rope_sum_kernel, dim3((2 * a.hd + kSumCols - 1) / kSumCols),
                                                       dim3(kSumCols * kSumWays), 0, (const float*)a.part, blocks, a.hd, dwq, dwk));
  return ULB_OK;
}
template <typename T>
int pick_grad(Ctx* c, HeadArgs& a, int wide, float* dwq, float* dwk) {
  return a.half ? launch_grad<T, true>(c, a, wide, dwq, dwk) : launch_grad<T, false>(c, a, wide, dwq, dwk);
}

int norm_args(const char* who, const ulb_rope* r, const ulb_norm_rope_args* p, HeadArgs* a) {
  ULB_TRY(rotary(who, r, a));
  ULB_CHECK(dtype_bytes(p->dtype), ULB_EUNSUPPORTED, "%s: type %d (F32, F16 or BF16)", who, p->dtype);
  ULB_CHECK(p->M >= 0 && p->n_head > 0 && p->n_head_kv >= 0, ULB_EINVAL, "%s: %d rows of %d and %d heads", who, p->M, p->n_head, p->n_head_kv);
  ULB_CHECK((long long)p->n_head + p->n_head_kv <= (1 << 20) && p->M <= kMaxRows, ULB_EUNSUPPORTED, "%s: %d rows of %d and %d heads", who, p->M,
            p->n_head, p->n_head_kv);
  ULB_CHECK(std::isfinite(p->eps) && p->eps >= kMinEps, ULB_EINVAL, "%s: eps %g", who, (double)p->eps);
  ULB_CHECK(p->q_row >= 0 && p->q_head >= 0 && p->k_row >= 0 && p->k_head >= 0, ULB_EINVAL, "%s: negative stride", who);
  ULB_CHECK(p->q_head < (1 << 28) && p->k_head < (1 << 28), ULB_EUNSUPPORTED, "%s: heads %lld and %lld elements apart (under 2^28)", who,
            (long long)p->q_head, (long long)p->k_head);
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
  const int v = wide(eb, {a.q, a.k, q_out, k_out}, a.q_row | a.q_head | a.k_row | a.k_head);
  switch (p->dtype) {
    case ULB_TYPE_F32: return pick_apply<float>(c, a, v);
    case ULB_TYPE_F16: return pick_apply<__half>(c, a, v);
    default: return pick_apply<__nv_bfloat16>(c, a, v);
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
  if (a.M == 0) a.wq = a.wk = nullptr; /* nothing is read */
  a.gq = dq_out;
  a.gk = dk_out;
  a.oq = dq;
  a.ok = dk;
  Ctx* c = &ctx->c;
  ULB_CUDA(cudaSetDevice(c->device));
  /* at the first call, whatever its shape, so that any later one can be captured */
  if (!c->norm_ws) ULB_CUDA(cudaMalloc((void**)&c->norm_ws, (size_t)c->n_sm * kNormBlocks * 2 * 256 * sizeof(float)));
  a.part = c->norm_ws;
  const int v = wide(eb, {a.q, a.k, dq_out, dk_out, dq, dk}, a.q_row | a.q_head | a.k_row | a.k_head);
  switch (p->dtype) {
    case ULB_TYPE_F32: return pick_grad<float>(c, a, v, dwq, dwk);
    case ULB_TYPE_F16: return pick_grad<__half>(c, a, v, dwq, dwk);
    default: return pick_grad<__nv_bfloat16>(c, a, v, dwq, dwk);
  }
}

}  // extern "C"

ULB_TRACE_UNIT(head_norm)
