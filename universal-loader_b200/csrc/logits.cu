/*
 * logits.cu — logits between the LM head and the sampler: penalties for repeated tokens,
 * presence and frequency, biases, and packed grammar masks, for plain rows and for the nodes of
 * drafted trees, whose contexts differ by their path only.  GenerationConfig carries
 * presence / frequency penalties in the reference (src/api/inference_api.h:14-22) that nothing
 * reads.
 *
 * One pass over the logits: each is read once and written once as fp32, HBM bounds large
 * calls.  A block owns a slice of the vocabulary of one sequence.  It first counts the sequence's
 * history over that slice in shared memory (integer atomics: any order gives the same counts;
 * bit 0 seen, bits 1-31 times generated), then turns each count into what steps 1 and 2 need,
 * the amount to subtract (frequency n + presence), -0 for a token that was only seen and +0 for
 * one that was not.  So the counts never travel through global memory, the rows of a tree, which
 * share them, count once, and a logit costs one compare, one select and one FMA.  Biases get a
 * second slice of shared memory, summed in list order, in the blocks that have any.
 *
 * Then each warp takes (row, chunk of the slice) units, all of a chunk's loads in flight at once,
 * the first unit's issued before the counting.  What a node's path adds is settled apart, so that
 * the loop over the logits stays short: the nodes whose token lies in the slice (few) are listed
 * once a block; a unit asks its row's ancestor bits for those, computes their logits from the
 * input, and stores them over the others' after its loop.
 *
 * Measured: 504 tree rows x 128256 (fp16 in, 308 MB) 78 us, 64 rows x 128256 (fp32) 24.5 us, one row x
 * 32000 5 us: 62 %, 42 % and a launch.  Instructions bound the first (some 70 for four tokens a lane),
 * with occupancy: five blocks an SM (48 registers, 36 bytes of them spilled) and one unit in flight a warp,
 * 96 us with two in flight and three blocks; the second is mostly the counting's latency in each of its blocks.
 */
#include <algorithm>

#include "paged_ops.h"

namespace ulb {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxNodes = 1024; /* 32 mask words */
constexpr int kMaxSlice = 4096; /* 32 KB of counts and biases: several blocks an SM */

struct LogitsGeom {
  int slice, chunk, n_slice; /* tokens a block, tokens a warp unit */
  int nodes;                 /* 32 * mask_words: nodes a row's bits can name */
};
/* loads of a unit in flight a lane, each of V tokens */
constexpr int unit_loads(int V) { return V == 4 ? 4 : 8; }

template <typename T, int V>
__device__ __forceinline__ void load_logits(const T* p, float (&x)[V]) {
  if constexpr (V == 1) {
    x[0] = to_f<T>(*p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  } else {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    const float2 f = unpack2<T>(a.x), g = unpack2<T>(a.y);
    x[0] = f.x; x[1] = f.y; x[2] = g.x; x[3] = g.y;
  }
}

/* steps 1 and 2 given what to subtract (`less`, +0: token not seen); x * (1 / rep) is within 1.5
   ulp of x / rep, and the FMA rounds product and difference once */
__device__ __forceinline__ float penal(float x, uint32_t less, float rep, float inv_rep) {
  const float y = __fmaf_rn(x, x > 0.f ? inv_rep : rep, -__uint_as_float(less));
  return less ? y : x;
}
/* what to subtract from a token seen before and generated `made` times */
__device__ __forceinline__ uint32_t less_of(int made, float pres, float freq) {
  const float f = made > 0 ? __fmaf_rn(freq, (float)made, pres) : 0.f;
  return f == 0.f ? 0x80000000u : __float_as_uint(f);
}

template <typename T, int V>
__global__ void __launch_bounds__(kWarps * 32, 5) logits_kernel(const __grid_constant__ ulb_logits_args a, LogitsGeom g) {
  pdl_wait();
  pdl_trigger();
  constexpr int U = unit_loads(V);
  extern __shared__ __align__(16) uint32_t sm[];
  uint32_t* const less = sm;                                       /* [slice] counts, then what to subtract */
  float* const bias = reinterpret_cast<float*>(sm + g.slice);      /* [slice], where the sequence has biases */
  int* const node_at = reinterpret_cast<int*>(sm + 2 * g.slice);   /* [nodes] places of the nodes of this slice */
  int* const node_id = node_at + g.nodes;                          /* [nodes] which nodes */
  uint32_t* const node_cnt = reinterpret_cast<uint32_t*>(node_id + g.nodes); /* [nodes] their tokens' counts */
  __shared__ int n_here;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  /* this warp's path tokens in its chunk: which listed node, its new logit */
  int* const list = node_id + (2 + 2 * warp) * g.nodes;
  float* const list_x = reinterpret_cast<float*>(list + g.nodes);
  const int s = blockIdx.x / g.n_slice, t0 = (blockIdx.x % g.n_slice) * g.slice;
  const int n_tok = min(g.slice, a.V - t0);
  const int r0 = max(0, a.row_start[s]), r1 = min(a.rows, a.row_start[s + 1]);
  if (r0 >= r1) return;
  const int n_chunk = (n_tok + g.chunk - 1) / g.chunk, n_unit = n_chunk * (r1 - r0);
  const int words = (a.V + 31) >> 5;

  auto allow_of = [&](int r) -> const uint32_t* {
    if (!a.allow) return nullptr;
    const int ai = a.row_allow ? a.row_allow[r] : r;
    return ai >= 0 && ai < a.n_allow ? a.allow + (long long)ai * words : nullptr;
  };
  struct Unit {
    int r, c0, c1; /* row, tokens [c0, c1) of the slice */
    float x[U][V];
    uint32_t ok[U];
  };
  auto load_unit = [&](int unit, Unit& n) {
    n.r = r0 + unit / n_chunk;
    n.c0 = (unit % n_chunk) * g.chunk;
    n.c1 = min(n.c0 + g.chunk, n_tok);
    const int i0 = n.c0 + lane * V;
    const T* in = reinterpret_cast<const T*>(a.in) + (long long)n.r * a.ld_in + t0 + i0;
    if (n.c1 - n.c0 == 32 * V * U) { /* a whole unit: no bounds */
#pragma unroll
      for (int u = 0; u < U; ++u) load_logits<T, V>(in + u * 32 * V, n.x[u]);
      const uint32_t* allow = allow_of(n.r);
      if (allow) {
        allow += (t0 + i0) >> 5;
#pragma unroll
        for (int u = 0; u < U; ++u) n.ok[u] = allow[u * V] >> ((t0 + i0) & 31);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) n.ok[u] = 0xffffffffu;
      }
      return;
    }
    const uint32_t* allow = allow_of(n.r);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * 32 * V;
      if (V == 1 || i + V <= n.c1) {
        if (i < n.c1) load_logits<T, V>(in + u * 32 * V, n.x[u]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) n.x[u][e] = i + e < n.c1 ? to_f<T>(in[u * 32 * V + e]) : 0.f;
      }
      n.ok[u] = allow && i < n.c1 ? allow[(t0 + i) >> 5] >> ((t0 + i) & 31) : 0xffffffffu;
    }
  };
  Unit cur;
  int unit = warp;
  if (unit < n_unit) load_unit(unit, cur);

  /* the first tokens of the history and biases travel with them */
  const int b0 = a.bias_start ? a.bias_start[s] : 0, b1 = a.bias_start ? a.bias_start[s + 1] : 0;
  const int h0 = a.history ? a.history_start[s] : 0, nh = a.history ? a.history_start[s + 1] - h0 : 0;
  const int np = a.history && a.prompt ? a.prompt[s] : 0;
  constexpr int HB = 8, HS = kWarps * 32;
  int t[HB];
  auto load_history = [&](int i0) {
#pragma unroll
    for (int u = 0; u < HB; ++u) t[u] = i0 + u * HS < nh ? a.history[(long long)h0 + i0 + u * HS] : -1;
  };
  load_history(tid);
  int bt = -1, bp = -1;
  float bv = 0.f;
  auto load_bias = [&](int i) {
    bt = a.bias_tokens[i];
    bp = i > b0 ? a.bias_tokens[i - 1] : -1;
    bv = a.bias_values[i];
  };
  if (b0 + tid < b1) load_bias(b0 + tid);
  for (int i = tid * 4; i < g.slice; i += kWarps * 32 * 4) {
    *reinterpret_cast<uint4*>(less + i) = make_uint4(0, 0, 0, 0);
    if (b1 > b0) *reinterpret_cast<uint4*>(bias + i) = make_uint4(0, 0, 0, 0);
  }
  if (tid == 0) n_here = 0;
  float rep = 1.f, pres = 0.f, freq = 0.f;
  if (a.params) {
    rep = a.params[3 * s];
    pres = a.params[3 * s + 1];
    freq = a.params[3 * s + 2];
  }
  const float inv_rep = __fdiv_rn(1.f, rep);
  __syncthreads();
  const int n_node = min(g.nodes, r1 - r0);
  for (int i = tid; i < n_node; i += HS) {
    const unsigned at = (unsigned)a.node_tokens[r0 + i] - (unsigned)t0;
    if (at < (unsigned)n_tok) {
      const int l = atomicAdd(&n_here, 1);
      node_at[l] = (int)at;
      node_id[l] = i;
    }
  }
  for (int i0 = tid; i0 < nh; i0 += HS * HB) {
    if (i0 != tid) load_history(i0);
#pragma unroll
    for (int u = 0; u < HB; ++u) {
      const unsigned at = (unsigned)t[u] - (unsigned)t0;
      if (at >= (unsigned)n_tok) continue; /* -1 too: t0 and n_tok are small */
      if (i0 + u * HS < np) atomicOr(&less[at], 1u);
      else atomicAdd(&less[at], 2u);
    }
  }
  bool biased = false;
  for (int i = b0 + tid; i < b1; i += HS) {
    if (i != b0 + tid) load_bias(i);
    const unsigned at = (unsigned)bt - (unsigned)t0;
    if (at >= (unsigned)n_tok || bp == bt) continue; /* the first of equal ids adds them */
    for (int j = i + 1; j < b1 && a.bias_tokens[j] == bt; ++j) bv += a.bias_values[j];
    bias[at] = bv;
    biased = true;
  }
  biased = __syncthreads_or(biased);
  const int n_at = n_here;
  for (int l = tid; l < n_at; l += kWarps * 32) node_cnt[l] = less[node_at[l]];
  if (n_at) __syncthreads();
  for (int i = tid * 4; i < n_tok; i += HS * 4) {
    uint4 w = *reinterpret_cast<const uint4*>(less + i);
    if (!(w.x | w.y | w.z | w.w)) continue;
    if (w.x) w.x = less_of((int)(w.x >> 1), pres, freq);
    if (w.y) w.y = less_of((int)(w.y >> 1), pres, freq);
    if (w.z) w.z = less_of((int)(w.z >> 1), pres, freq);
    if (w.w) w.w = less_of((int)(w.w >> 1), pres, freq);
    *reinterpret_cast<uint4*>(less + i) = w;
  }
  __syncthreads();

  while (unit < n_unit) {
    const int r = cur.r, c0 = cur.c0, c1 = cur.c1;
    int n_list = 0;
    if (n_at) {
      for (int l0 = 0; l0 < n_at; l0 += 32) {
        const int l = l0 + lane;
        bool hit = false;
        if (l < n_at) {
          const int at = node_at[l], j = node_id[l];
          hit = at >= c0 && at < c1 && ((a.mask[(long long)r * a.mask_words + (j >> 5)] >> (j & 31)) & 1u);
        }
        const uint32_t hits = __ballot_sync(0xffffffffu, hit);
        if (hit) list[n_list + __popc(hits & ((1u << lane) - 1u))] = l;
        n_list += __popc(hits);
      }
      __syncwarp();
      const uint32_t* const allow = n_list ? allow_of(r) : nullptr;
      for (int l = lane; l < n_list; l += 32) {
        const int at = node_at[list[l]], tok = t0 + at;
        const uint32_t w = node_cnt[list[l]];
        int made = (int)(w >> 1);
        for (int m = 0; m < n_list; ++m) made += node_at[list[m]] == at;
        float y = penal(to_f<T>(reinterpret_cast<const T*>(a.in)[(long long)r * a.ld_in + tok]), less_of(made, pres, freq), rep, inv_rep);
        if (biased) y += bias[at];
        if (allow && !((allow[tok >> 5] >> (tok & 31)) & 1u)) y = -INFINITY;
        list_x[l] = y;
      }
      __syncwarp();
    }
    float* const out = a.out + (long long)r * a.ld_out + t0;
    const bool whole = c1 - c0 == 32 * V * U;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = c0 + (u * 32 + lane) * V;
      if (!whole && i >= c1) continue;
      float(&x)[V] = cur.x[u];
      uint32_t w[V];
      if constexpr (V == 4) {
        const uint4 q = *reinterpret_cast<const uint4*>(less + i); /* past n_tok: zero */
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
      } else {
        w[0] = less[i];
      }
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) any |= w[e];
      if (any) {
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = penal(x[e], w[e], rep, inv_rep);
      }
      if (biased) {
        if constexpr (V == 4) {
          const float4 f = *reinterpret_cast<const float4*>(bias + i);
          x[0] += f.x; x[1] += f.y; x[2] += f.z; x[3] += f.w;
        } else {
          x[0] += bias[i];
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (!((cur.ok[u] >> e) & 1u)) x[e] = -INFINITY;
      if (V == 1) {
        out[i] = x[0];
      } else if (whole || i + V <= c1) {
        *reinterpret_cast<float4*>(out + i) = make_float4(x[0], x[1 % V], x[2 % V], x[3 % V]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (i + e < c1) out[i + e] = x[e];
      }
    }
    if (n_list) {
      __syncwarp();
      for (int l = lane; l < n_list; l += 32) out[node_at[list[l]]] = list_x[l];
      __syncwarp();
    }
    unit += kWarps;
    if (unit < n_unit) load_unit(unit, cur);
  }
}

template <typename T, int V>
int launch_logits(Ctx* c, const ulb_logits_args& a) {
  /* slices: trees (eight rows or more) about 18 blocks an SM, at most five of them at once, so that the last
     wave wastes little; fewer rows, which do not pay for many countings, larger ones: a unit a warp */
  const long long want = (long long)c->n_sm * 18;
  long long slice = ((long long)a.V * a.n_seq + want - 1) / want;
  if (a.max_rows >= kWarps) slice = (slice + 511) / 512 * 512;
  else slice = slice <= 1024 ? 1024 : kMaxSlice;
  slice = std::min<long long>(slice, kMaxSlice);
  LogitsGeom g;
  g.slice = (int)std::min<long long>(slice, (a.V + 127) / 128 * 128);
  g.n_slice = (a.V + g.slice - 1) / g.slice;
  /* a unit: what a lane's loads cover, less when a sequence has too few rows for every warp */
  const int full = 32 * V * unit_loads(V);
  g.chunk = a.max_rows >= kWarps ? full : std::min(full, std::max(128, (g.slice * a.max_rows / kWarps + 127) / 128 * 128));
  g.nodes = a.node_tokens ? 32 * a.mask_words : 0;
  const size_t smem = (size_t)(2 * g.slice + g.nodes * (3 + 2 * kWarps)) * 4;
  const long long blocks = (long long)g.n_slice * a.n_seq;
  ULB_CHECK(blocks < (1ll << 31), ULB_EUNSUPPORTED, "ulb_logits_process: %d sequences of %d tokens", a.n_seq, a.V);
  static uint64_t attr = 0; /* devices it is set on */
  if (!(attr >> (c->device & 63) & 1)) {
    ULB_CUDA(cudaFuncSetAttribute(logits_kernel<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  (2 * kMaxSlice + kMaxNodes * (3 + 2 * kWarps)) * 4));
    attr |= 1ull << (c->device & 63);
  }
  ULB_LAUNCH("logits launch", launch_k(c, logits_kernel<T, V>, dim3((unsigned)blocks), dim3(kWarps * 32), smem, a, g));
  return ULB_OK;
}

template <typename T>
int pick_logits(Ctx* c, const ulb_logits_args& a) {
  /* four tokens a load when every row starts on a whole word of four */
  if (a.ld_in % 4 == 0 && a.ld_out % 4 == 0 && (uintptr_t)a.in % (4 * sizeof(T)) == 0 && (uintptr_t)a.out % 16 == 0)
    return launch_logits<T, 4>(c, a);
  return launch_logits<T, 1>(c, a);
}

}  // namespace
}  // namespace ulb

using namespace ulb;

extern "C" int ulb_logits_process(ulb_ctx* ctx, const ulb_logits_args* a) {
  ULB_CHECK(ctx && a, ULB_EINVAL, "ulb_logits_process: NULL argument");
  ULB_CHECK(dtype_bytes(a->dtype), ULB_EUNSUPPORTED, "ulb_logits_process: type %d (F32, F16 or BF16)", a->dtype);
  ULB_CHECK(a->V > 0 && a->n_seq >= 0 && a->rows >= 0 && a->max_rows >= 0 && a->mask_words >= 0 && a->n_allow >= 0, ULB_EINVAL,
            "ulb_logits_process: V %d, %d sequences, %d rows (at most %d each), %d mask words, %d grammars", a->V, a->n_seq,
            a->rows, a->max_rows, a->mask_words, a->n_allow);
  ULB_CHECK(a->ld_in >= a->V && a->ld_out >= a->V, ULB_EINVAL, "ulb_logits_process: rows %d and %d apart hold %d logits",
            a->ld_in, a->ld_out, a->V);
  if (a->rows == 0 || a->n_seq == 0) return ULB_OK;
  ULB_CHECK(a->in && a->out && a->row_start, ULB_EINVAL, "ulb_logits_process: NULL logits or row_start");
  ULB_CHECK(!a->history == !a->history_start, ULB_EINVAL, "ulb_logits_process: history without history_start, or the reverse");
  ULB_CHECK(!a->node_tokens || (a->mask && a->mask_words > 0), ULB_EINVAL, "ulb_logits_process: node_tokens without masks");
  ULB_CHECK(!a->node_tokens || a->mask_words <= kMaxNodes / 32, ULB_EUNSUPPORTED, "ulb_logits_process: %d mask words (at most %d)",
            a->mask_words, kMaxNodes / 32);
  ULB_CHECK(!a->bias_start || (a->bias_tokens && a->bias_values), ULB_EINVAL, "ulb_logits_process: bias_start without biases");
  const int eb = dtype_bytes(a->dtype);
  ULB_CHECK((uintptr_t)a->in % eb == 0 && (uintptr_t)a->out % 4 == 0, ULB_EINVAL, "ulb_logits_process: unaligned pointer");
  ULB_CHECK(words_aligned({a->row_start, a->params, a->history, a->history_start, a->prompt, a->node_tokens, a->mask, a->bias_start,
                           a->bias_tokens, a->bias_values, a->allow, a->row_allow}),
            ULB_EINVAL, "ulb_logits_process: unaligned array of 32-bit elements");
  ULB_CHECK((const void*)a->in != (const void*)a->out || (a->dtype == ULB_TYPE_F32 && a->ld_in == a->ld_out), ULB_EINVAL,
            "ulb_logits_process: in place needs F32 logits and equal leading dimensions");
  Ctx* c = &ctx->c;
  ULB_CUDA(cudaSetDevice(c->device));
  switch (a->dtype) {
    case ULB_TYPE_F32: return pick_logits<float>(c, *a);
    case ULB_TYPE_F16: return pick_logits<__half>(c, *a);
    default: return pick_logits<__nv_bfloat16>(c, *a);
  }
}

ULB_TRACE_UNIT(logits)
