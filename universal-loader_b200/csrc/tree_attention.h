/*
 * tree_attention.h — what the two kernels of ulb_tree_attention share: arguments, visibility of
 * a key to a row, and the layout of split partials.
 */
#pragma once

#include "paged_ops.h"
#include "tree_plan.h"

namespace ulb {

struct TreeArgs {
  CacheGeom g;
  int H, G;                  /* query heads, query heads a kv head */
  int rows, max_rows, max_len, words;
  float scale2;              /* scale log2(e): scores live in the base-2 domain */
  int split_keys, n_split;   /* keys a split (a multiple of 128), splits of the longest sequence */
  int n_tile;                /* row tiles of the longest sequence */
  const void *q, *k, *v;
  const int *table, *row_start, *prefix, *len;
  const uint32_t* mask;
  void* out;
  float* lse;
  float *po, *pml;           /* partials of (row, head, split): [hd] outputs, (max, sum) */
  int* err;
};

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

#ifdef __CUDACC__
/* one sequence of a call, every field checked against the call's sizes */
struct TreeSeq {
  int r0, n, len, prefix; /* first row, rows, cached positions, positions before the tree */
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int s) {
  TreeSeq q;
  q.n = rows_of(a.row_start[s], a.row_start[s + 1], a.rows, a.max_rows, &q.r0);
  q.len = min(max(a.len[s], 0), a.max_len);
  q.prefix = min(max(a.prefix[s], 0), q.len);
  return q;
}
/* does row i of the sequence see position pos < len?  (prefix positions: yes) */
__device__ __forceinline__ bool tree_sees(const TreeArgs& a, const TreeSeq& q, int i, int pos) {
  if (a.words == 0) return pos <= q.len - q.n + i;
  const int j = pos - q.prefix;
  if (j < 0) return true;
  if (j >= 32 * a.words) return false;
  return (a.mask[(long long)(q.r0 + i) * a.words + (j >> 5)] >> (j & 31)) & 1u;
}
/* positions that every row of the sequence sees: [0, tree_open) */
__device__ __forceinline__ int tree_open(const TreeArgs& a, const TreeSeq& q) {
  return a.words == 0 ? max(q.len - q.n + 1, 0) : q.prefix;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
#endif

/* the tcgen05 form (tree_attention_tc.cu): head dims up to 128 */
bool tree_tc_fits(const Ctx* c, const TreeArgs& a);
int launch_tree_tc(Ctx* c, TreeArgs& a, bool f16);

/* floats of split partials a context holds for this operator (128 MiB) */
constexpr size_t kTreeWsFloats = (size_t)32 << 20;

}  // namespace ulb
