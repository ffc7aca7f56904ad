/*
 * tree_plan.h — the parts of the tree attention that hold no CUDA types, as functions the kernels
 * call with their own waits, copies and products and the CPU tests with a model of the barriers.
 */
#pragma once

#ifdef __CUDACC__
#define ULB_ROLE __device__ __forceinline__
#else
#define ULB_ROLE inline
#endif

namespace ulb {

/* rows of a sequence from its places in row_start, whatever those hold: *r0 and the answer name rows
   of [0, rows), at most max_rows */
ULB_ROLE int rows_of(int begin, int end, int rows, int max_rows, int* r0) {
  const int b = begin < 0 ? 0 : begin > rows ? rows : begin, e = end < b ? b : end > rows ? rows : end;
  *r0 = b;
  return e - b < max_rows ? e - b : max_rows;
}

/*
 * The order in which the issuing warp of stream X passes the K and V rings in a piece of `tiles`
 * tiles, n of them its own: all (PAIR) or every second (t % 2 == X).  A ring's place is free when
 * both streams have passed it, so a stream may not run ahead in one ring while the other stream waits
 * for it in the other ring: a tile that is not its own is passed next to one of its own in the
 * same ring, and a stream that has no tile at all passes K and V in turn.
 *
 *   pass_k(), pass_v()  wait for the next tile of a ring and free it unused
 *   wait_k(), wait_v()  wait for the next tile of a ring, which is the stream's own
 *   scores(b)           scores of that K tile into buffer b; frees the tile
 *   look(t)             V tile t of the piece is there (the softmax warps look a masked one over)
 *   wait_p(b)           weights of buffer b
 *   product(b, i, more) product i with them; frees the V tile; then, where `more`, scores(b)
 *
 * All but look, scores and product say whether the wait ended; after one that did not, nothing is
 * called any more and the answer is false.
 */
template <bool PAIR, typename PassK, typename PassV, typename WaitK, typename WaitV, typename Scores, typename Look, typename WaitP,
          typename Product>
ULB_ROLE bool ring_issue(int X, int n, int tiles, PassK&& pass_k, PassV&& pass_v, WaitK&& wait_k, WaitV&& wait_v, Scores&& scores,
                         Look&& look, WaitP&& wait_p, Product&& product) {
  if (n == 0) {
    for (int t = 0; t < tiles; ++t)
      if (!pass_k() || !pass_v()) return false;
    return true;
  }
  int kt = 0, vt = 0; /* tiles of the piece passed so far */
  auto others = [&](int t) { return !PAIR && t < tiles && (t & 1) != X; };
  auto next_k = [&]() { /* to this stream's next K tile, or the end */
    for (; others(kt); ++kt)
      if (!pass_k()) return false;
    return true;
  };
  auto next_v = [&]() {
    for (; others(vt); ++vt)
      if (!pass_v()) return false;
    return true;
  };
  for (int i = 0; i < n && i < 2; ++i) {
    if (!next_k() || !wait_k()) return false;
    scores(i);
    ++kt;
  }
  for (int i = 0; i < n; ++i) {
    const int b = i & 1;
    const bool more = i + 2 < n;
    /* the rings first, they are mostly ready; then the weights */
    if (!next_v() || !wait_v()) return false;
    look(vt);
    if (more && (!next_k() || !wait_k())) return false;
    if (!wait_p(b)) return false;
    product(b, i, more);
    ++vt;
    if (more) ++kt;
  }
  return next_k() && next_v();
}

/*
 * What a copying warp does with the n tiles of a piece: a place is waited for, then filled; look(t)
 * reads ahead what the copy of tile t needs.  After a wait that did not end, nothing is copied any more
 * (the place may still be read) and the answer is false.
 */
template <typename Look, typename WaitFree, typename Copy>
ULB_ROLE bool ring_copy(int n, Look&& look, WaitFree&& wait_free, Copy&& copy) {
  look(0);
  for (int t = 0; t < n; ++t) {
    if (!wait_free()) return false;
    copy(t);
    look(t + 1);
  }
  return true;
}

}  // namespace ulb
