/*
 * prompt_attention.h — what the two kernels of ulb_prompt_attention share: arguments, and the rows and
 * keys of a sequence.
 */
#pragma once

#include "paged_ops.h"
#include "tree_attention.h"

namespace ulb {

struct PromptArgs {
  int H, KV, G, hd;            /* query heads, kv heads, query heads a kv head */
  unsigned g_mul, g_shift;     /* n / G = mulhi(n, g_mul) >> g_shift for 0 <= n < 2^31, G > 1 */
  int n_seq, q_rows, k_rows, max_q, max_k;
  long long q_row, k_row, v_row; /* elements between rows */
  float scale2;                /* scale log2(e): scores live in the base-2 domain */
  const void *q, *k, *v;
  const int *q_start, *k_start;
  void* out;
  float* lse;
  int* err;
  float* ws;                   /* the context's partials (kTreeWsFloats) */
};

#ifdef __CUDACC__
/* one sequence of a call: rows r0 .. r0 + n of q, keys k0 .. k0 + len of k and v; row i sees keys <= len - n + i */
struct PromptSeq {
  int r0, n, k0, len;
};
__device__ __forceinline__ PromptSeq prompt_seq(const PromptArgs& a, int s) {
  PromptSeq q;
  q.n = rows_of(a.q_start[s], a.q_start[s + 1], a.q_rows, a.max_q, &q.r0);
  q.len = rows_of(a.k_start[s], a.k_start[s + 1], a.k_rows, a.max_k, &q.k0);
  return q;
}
/*
 * n / G.  With 2^L >= G > 2^(L - 1) and m = ceil(2^(31 + L) / G), n m / 2^(31 + L) is n / G and less than
 * n 2^L / (G 2^(31 + L)) < 1 / G more, so its whole part is that of n / G.
 */
__device__ __forceinline__ int div_group(const PromptArgs& a, int n) {
  return a.G == 1 ? n : (int)(__umulhi((unsigned)n, a.g_mul) >> a.g_shift);
}
/* keys that row i sees: [0, prompt_seen) */
__device__ __forceinline__ int prompt_seen(const PromptSeq& q, int i) { return min(max(q.len - q.n + i + 1, 0), q.len); }
#endif

/* the tcgen05 form (prompt_attention_tc.cu) */
bool prompt_tc_fits(const PromptArgs& a);
int launch_prompt_tc(Ctx* c, const PromptArgs& a, bool f16);

}  // namespace ulb
