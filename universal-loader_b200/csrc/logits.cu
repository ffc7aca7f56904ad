/*
 * logits.cu — logits between the LM head and the sampler: penalties for repeated tokens,
 * presence and frequency, biases, and packed grammar masks, for plain rows and for the nodes of
 * drafted trees, whose contexts differ by their path only.  GenerationConfig carries
 * presence / frequency penalties in the reference (src/api/inference_api.h:14-22) that nothing
 * reads.
 *
 * One pass over the logits: each is read once and written once as fp32, HBM bounds large
 * calls.  A block owns a slice of the vocabulary of one sequence and first counts the
 * sequence's history over that slice in shared memory (integer atomics: any order gives the
 * same counts), one word a token:
 *   bit 0 seen (prompt or generated), bits 1-30 times generated, bit 31 has a bias
 * so the counts never travel through global memory and the rows of a tree, which share them,
 * count once.  Then each warp takes (row, chunk of the slice) units.  Four tokens whose words are
 * all zero and whose grammar bits are set are copied; only the others take the arithmetic.  The
 * tokens of a node's path come from the row's ancestor bits: a warp collects those that fall in
 * its chunk (mostly none) in a list of its own and adds them to the counts as it goes.
 */
#include <algorithm>

#include "paged_ops.h"

namespace ulb {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxNodes = 1024; /* 32 mask words */

struct LogitsGeom {
  int slice, chunk, n_slice; /* tokens a block, tokens a warp unit */
  int nodes;                 /* 32 * mask_words: nodes a row's bits can name */
};

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

/* one token's logit: word = its count word, more = its count on the row's path */
__device__ __forceinline__ float change(float x, uint32_t word, int more, float rep, float pres, float freq,
                                        const ulb_logits_args& a, int b0, int b1, int tok) {
  const int made = (int)((word & 0x7fffffffu) >> 1) + more;
  if ((word & 1u) || made > 0) x = x > 0.f ? __fdiv_rn(x, rep) : x * rep;
  if (made > 0) x = x - freq * (float)made - pres;
  if (word >> 31) {
    int lo = b0, hi = b1;
    while (lo < hi) {
      const int mid = lo + ((hi - lo) >> 1);
      if (a.bias_tokens[mid] < tok) lo = mid + 1;
      else hi = mid;
    }
    float b = 0.f;
    for (; lo < b1 && a.bias_tokens[lo] == tok; ++lo) b += a.bias_values[lo];
    x += b;
  }
  return x;
}

template <typename T, int V>
__global__ void __launch_bounds__(kWarps * 32) logits_kernel(const __grid_constant__ ulb_logits_args a, LogitsGeom g) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ uint32_t sm[];
  uint32_t* const cnt = sm;                                  /* [slice] */
  int* const node_tok = reinterpret_cast<int*>(sm + g.slice); /* [nodes] */
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* const list = node_tok + g.nodes + warp * g.nodes; /* this warp's path tokens in its chunk */
  const int s = blockIdx.x / g.n_slice, t0 = (blockIdx.x % g.n_slice) * g.slice;
  const int n_tok = min(g.slice, a.V - t0);
  const int r0 = max(0, a.row_start[s]), r1 = min(a.rows, a.row_start[s + 1]);
  if (r0 >= r1) return;

  for (int i = tid; i < g.slice; i += kWarps * 32) cnt[i] = 0;
  const int n_node = min(g.nodes, r1 - r0);
  for (int i = tid; i < n_node; i += kWarps * 32) node_tok[i] = a.node_tokens[r0 + i];
  const int b0 = a.bias_start ? a.bias_start[s] : 0, b1 = a.bias_start ? a.bias_start[s + 1] : 0;
  float rep = 1.f, pres = 0.f, freq = 0.f;
  if (a.params) {
    rep = a.params[3 * s];
    pres = a.params[3 * s + 1];
    freq = a.params[3 * s + 2];
  }
  __syncthreads();
  if (a.history) {
    const int h0 = a.history_start[s], n = a.history_start[s + 1] - h0, np = a.prompt ? a.prompt[s] : 0;
    for (int i0 = tid; i0 < n; i0 += kWarps * 32 * 8) {
      int t[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * kWarps * 32;
        t[u] = i < n ? a.history[(long long)h0 + i] : -1;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const unsigned at = (unsigned)t[u] - (unsigned)t0;
        if (t[u] < 0 || at >= (unsigned)n_tok) continue;
        if (i0 + u * kWarps * 32 < np) atomicOr(&cnt[at], 1u);
        else atomicAdd(&cnt[at], 2u);
      }
    }
  }
  for (int i = b0 + tid; i < b1; i += kWarps * 32) {
    const unsigned at = (unsigned)a.bias_tokens[i] - (unsigned)t0;
    if (at < (unsigned)n_tok) atomicOr(&cnt[at], 0x80000000u);
  }
  __syncthreads();

  const int n_chunk = (n_tok + g.chunk - 1) / g.chunk;
  const int words = (a.V + 31) >> 5;
  for (int unit = warp; unit < n_chunk * (r1 - r0); unit += kWarps) {
    const int r = r0 + unit / n_chunk, c0 = (unit % n_chunk) * g.chunk, c1 = min(c0 + g.chunk, n_tok);
    int n_list = 0;
    for (int w = 0; w * 32 < n_node; ++w) {
      const uint32_t bits = a.mask[(long long)r * a.mask_words + w];
      const int j = w * 32 + lane;
      const int at = j < n_node ? node_tok[j] - t0 : -1;
      const bool hit = ((bits >> lane) & 1u) && at >= c0 && at < c1;
      const uint32_t hits = __ballot_sync(0xffffffffu, hit);
      if (hit) list[n_list + __popc(hits & ((1u << lane) - 1u))] = at;
      n_list += __popc(hits);
    }
    __syncwarp();
    const uint32_t* allow = nullptr;
    if (a.allow) {
      const int ai = a.row_allow ? a.row_allow[r] : r;
      if (ai >= 0 && ai < a.n_allow) allow = a.allow + (long long)ai * words;
    }
    const T* in = reinterpret_cast<const T*>(a.in) + (long long)r * a.ld_in + t0;
    float* out = a.out + (long long)r * a.ld_out + t0;
    constexpr int U = V == 1 ? 8 : 4; /* loads in flight */
    for (int i0 = c0 + lane * V; i0 < c1; i0 += 32 * V * U) {
      float x[U][V];
      uint32_t ok[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * 32 * V;
        if (i < c1) {
          if (V == 1 || i + V <= c1) {
            load_logits<T, V>(in + i, x[u]);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) x[u][e] = i + e < c1 ? to_f<T>(in[i + e]) : 0.f;
          }
          ok[u] = allow ? allow[(t0 + i) >> 5] >> ((t0 + i) & 31) : 0xffffffffu;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * 32 * V;
        if (i >= c1) continue;
        uint32_t any = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) any |= i + e < c1 ? cnt[i + e] : 0u;
        if (any || n_list) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (i + e >= c1) continue;
            int more = 0;
            for (int l = 0; l < n_list; ++l) more += list[l] == i + e;
            x[u][e] = change(x[u][e], cnt[i + e], more, rep, pres, freq, a, b0, b1, t0 + i + e);
          }
        }
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (!((ok[u] >> e) & 1u)) x[u][e] = -INFINITY;
        if (V == 1) {
          out[i] = x[u][0];
        } else if (i + V <= c1) {
          *reinterpret_cast<float4*>(out + i) = make_float4(x[u][0], x[u][1 % V], x[u][2 % V], x[u][3 % V]);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (i + e < c1) out[i + e] = x[u][e];
        }
      }
    }
    __syncwarp(); /* the list is this unit's */
  }
}

template <typename T, int V>
int launch_logits(Ctx* c, const ulb_logits_args& a) {
  /* slices: about four blocks an SM over the whole call, at least 128 tokens a warp, at most 64 KB of counts */
  const long long want = (long long)c->n_sm * 4;
  long long slice = ((long long)a.V * a.n_seq + want - 1) / want;
  slice = std::min<long long>(std::max<long long>((slice + 1023) / 1024 * 1024, 1024), 16384);
  LogitsGeom g;
  g.slice = (int)std::min<long long>(slice, (a.V + 127) / 128 * 128);
  g.n_slice = (a.V + g.slice - 1) / g.slice;
  g.chunk = a.max_rows >= kWarps ? 1024 : std::min(1024, std::max(128, (g.slice * a.max_rows / kWarps + 127) / 128 * 128));
  g.nodes = a.node_tokens ? 32 * a.mask_words : 0;
  const size_t smem = (size_t)(g.slice + g.nodes * (1 + kWarps)) * 4;
  const long long blocks = (long long)g.n_slice * a.n_seq;
  ULB_CHECK(blocks < (1ll << 31), ULB_EUNSUPPORTED, "ulb_logits_process: %d sequences of %d tokens", a.n_seq, a.V);
  static bool attr = false;
  if (!attr) {
    ULB_CUDA(cudaFuncSetAttribute(logits_kernel<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  (16384 + kMaxNodes * (1 + kWarps)) * 4));
    attr = true;
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
