/*
 * pages.cu — moving K / V between the pages of a cache, in every layer at once: whole or partly
 * filled pages (copy on write of forked sequences, defragmentation) and single positions (the
 * accepted path of a drafted tree brought to its sequence positions), and the device side of the
 * page book (page_book.h).  The loop's own tree compaction (model.cu) knows full trees and its
 * own layout only; the reference has no pages (src/inference/model.h:49-77).
 *
 * Both kernels are copies: every byte is read once and written once, HBM bounds them, and there
 * is nothing to compute.  All loads of a thread are issued before its first store.  Measured: 16 pages of
 * 256 positions in 32 layers of 8 heads of 128 (572 MB moved) 93 us, 96 % of the copy rate (with streaming
 * hints on loads and stores 96 us); 64 paths in 16 layers 4.5 us, a launch.
 */
#include <algorithm>
#include <memory>
#include <new>

#include "page_book.h"
#include "paged_ops.h"

namespace ulb {
namespace {

constexpr int kInlineMoves = 64;
struct MoveList { PageMove m[kInlineMoves]; };
constexpr int kInlineEntries = 128;
struct EntryList { int at[kInlineEntries], page[kInlineEntries]; };

constexpr int kCopyThreads = 256, kCopyUnroll = 8; /* 16-byte words a thread has in flight */

/*
 * One block = one move's words [y * 2048, + 2048) of one (layer, pool, head): positions x hd
 * elements, contiguous when positions follow one another (FLAT) or hd / 8 words a position.
 */
template <bool FLAT>
__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(CacheGeom g, uint4* k, uint4* v, const int* moves,
                                                                  const __grid_constant__ MoveList inl, int n_chunk) {
  pdl_wait();
  pdl_trigger();
  const int chunk = blockIdx.x % n_chunk;
  int id = blockIdx.x / n_chunk;
  const int h = id % g.n_head_kv;
  id /= g.n_head_kv;
  const int pool = id & 1, l = id >> 1, i = blockIdx.y;
  PageMove mv;
  if (moves) {
    mv.src = moves[3 * i];
    mv.dst = moves[3 * i + 1];
    mv.positions = moves[3 * i + 2];
  } else {
    mv = inl.m[i];
  }
  if (mv.src < 0 || mv.src >= g.n_pages || mv.dst < 0 || mv.dst >= g.n_pages) return;
  const int wpp = g.hd >> 3; /* words a position */
  const int n = min(max(mv.positions, 0), g.page) * wpp;
  uint4* base = pool ? v : k;
  const long long lh = (l * g.layer + h * g.head) >> 3;
  const uint4* src = base + lh + ((mv.src * g.pstride) >> 3);
  uint4* dst = base + lh + ((mv.dst * g.pstride) >> 3);
  const int w0 = chunk * (kCopyThreads * kCopyUnroll) + threadIdx.x;
  uint4 x[kCopyUnroll];
  long long off[kCopyUnroll];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u) {
    const int w = w0 + u * kCopyThreads;
    off[u] = FLAT ? (long long)w : (long long)(w / wpp) * (g.pos >> 3) + w % wpp;
    if (w < n) x[u] = src[off[u]];
  }
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (w0 + u * kCopyThreads < n) dst[off[u]] = x[u];
}

constexpr int kPathTile = 64; /* path positions whose places a block holds at a time */

/*
 * One block = one (sequence, layer, pool): the places of the path's positions once, in shared
 * memory, then each thread walks the path for its 16-byte words of the heads.  A word's sources
 * ascend and none is below its destination, so a thread that reads four positions before it
 * writes four never reads a place already written; no thread touches another's words.
 */
__global__ void __launch_bounds__(256) pages_compact_kernel(CacheGeom g, uint4* k, uint4* v, const int* table,
                                                            const int* base, const int* count, const int* src, int max_src) {
  pdl_wait();
  pdl_trigger();
  __shared__ long long from[kPathTile], to[kPathTile];
  const int s = blockIdx.y, pool = blockIdx.x & 1, l = blockIdx.x >> 1;
  const int n = min(count[s], max_src);
  const long long b0 = base[s];
  uint4* const p = (pool ? v : k) + ((l * g.layer) >> 3);
  const int wpp = g.hd >> 3, words = g.n_head_kv * wpp;
  auto place = [&](long long pos) -> long long { /* in words; -1: unmapped */
    if (pos < 0 || (pos >> g.page_shift) >= g.max_pages) return -1;
    const int pg = table[(long long)s * g.max_pages + (pos >> g.page_shift)];
    return pg < 0 || pg >= g.n_pages ? -1 : (pg * g.pstride + (pos & (g.page - 1)) * g.pos) >> 3;
  };
  for (int i0 = 0; i0 < n; i0 += kPathTile) {
    const int m = min(kPathTile, n - i0);
    __syncthreads();
    for (int i = threadIdx.x; i < m; i += blockDim.x) {
      const int sl = src[(long long)s * max_src + i0 + i];
      long long a = sl < 0 ? -1 : place(b0 + sl);
      const long long d = place(b0 + i0 + i);
      if (a == d || d < 0) a = -1;
      from[i] = a;
      to[i] = d;
    }
    __syncthreads();
    for (int w = threadIdx.x; w < words; w += blockDim.x) {
      const long long ho = (long long)(w / wpp) * (g.head >> 3) + w % wpp;
      for (int i = 0; i < m; i += 4) {
        uint4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + u < m && from[i + u] >= 0) x[u] = p[from[i + u] + ho];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + u < m && from[i + u] >= 0) p[to[i + u] + ho] = x[u];
      }
    }
  }
}

__global__ void pages_table_kernel(int* table, const __grid_constant__ EntryList e, int n) {
  pdl_wait();
  pdl_trigger();
  if ((int)threadIdx.x < n) table[e.at[threadIdx.x]] = e.page[threadIdx.x];
}

int launch_copy(Ctx* c, const CacheGeom& g, void* k, void* v, const int* moves, const MoveList& inl, int n) {
  const int wpp = g.hd / 8, n_chunk = (g.page * wpp + kCopyThreads * kCopyUnroll - 1) / (kCopyThreads * kCopyUnroll);
  const long long gx = (long long)n_chunk * g.n_head_kv * 2 * g.n_layer;
  ULB_CHECK(gx < (1ll << 31), ULB_EUNSUPPORTED, "ulb_pages_copy: %d layers of %d heads", g.n_layer, g.n_head_kv);
  for (int i0 = 0; i0 < n; i0 += 65535) {
    const int m = std::min(65535, n - i0);
    const int* at = moves ? moves + (size_t)3 * i0 : nullptr;
    if (g.pos == g.hd)
      ULB_LAUNCH("pages_copy launch", launch_k(c, pages_copy_kernel<true>, dim3((unsigned)gx, m), dim3(kCopyThreads), 0, g,
                                               (uint4*)k, (uint4*)v, at, inl, n_chunk));
    else
      ULB_LAUNCH("pages_copy launch", launch_k(c, pages_copy_kernel<false>, dim3((unsigned)gx, m), dim3(kCopyThreads), 0, g,
                                               (uint4*)k, (uint4*)v, at, inl, n_chunk));
  }
  return ULB_OK;
}

}  // namespace
}  // namespace ulb

using namespace ulb;

struct ulb_pages {
  ulb_ctx* owner = nullptr;
  CacheGeom g;
  void *k = nullptr, *v = nullptr;
  int* table = nullptr;
  PageBook book;
  ulb_pages(int n_pages, int n_seq, int max_pages, int page) : book(n_pages, n_seq, max_pages, page) {}
};

/* enqueue what a change of the book asks of the device: copies first, then the table */
static int pages_enqueue(ulb_pages* p, const PageWork& w) {
  Ctx* c = &p->owner->c;
  ULB_CUDA(cudaSetDevice(c->device));
  for (size_t i = 0; i < w.moves.size(); i += kInlineMoves) {
    MoveList l = {};
    const int n = (int)std::min<size_t>(kInlineMoves, w.moves.size() - i);
    std::copy(w.moves.begin() + i, w.moves.begin() + i + n, l.m);
    ULB_TRY(launch_copy(c, p->g, p->k, p->v, nullptr, l, n));
  }
  for (size_t i = 0; i < w.entries.size(); i += kInlineEntries) {
    EntryList l = {};
    const int n = (int)std::min<size_t>(kInlineEntries, w.entries.size() - i);
    for (int j = 0; j < n; ++j) {
      l.at[j] = w.entries[i + j].seq * p->g.max_pages + w.entries[i + j].index;
      l.page[j] = w.entries[i + j].page;
    }
    ULB_LAUNCH("pages table launch", launch_k(c, pages_table_kernel, dim3(1), dim3(kInlineEntries), 0, p->table, l, n));
  }
  return ULB_OK;
}

/* run a change of the book; a failed host allocation comes back as a status */
template <typename F>
static int pages_change(const char* who, ulb_pages* p, F&& change) {
  try {
    PageWork w;
    const PageRc rc = change(&w);
    ULB_CHECK(rc != PageRc::kBadArg, ULB_EINVAL, "%s: sequence or position out of range, or the state does not allow it", who);
    ULB_CHECK(rc != PageRc::kNoPages, ULB_ENOMEM, "%s: %d free pages are too few", who, p->book.free_pages());
    return pages_enqueue(p, w);
  } catch (const std::bad_alloc&) {
    return set_error(ULB_ENOMEM, "%s: host allocation", who);
  }
}

extern "C" {

int ulb_pages_copy(ulb_ctx* ctx, const ulb_cache_desc* cache, void* k, void* v, const int32_t* moves, int n) {
  ULB_CHECK(ctx, ULB_EINVAL, "ulb_pages_copy: NULL context");
  CacheGeom g;
  ULB_TRY(cache_geom("ulb_pages_copy", cache, &g));
  ULB_CHECK(n >= 0, ULB_EINVAL, "ulb_pages_copy: %d moves", n);
  if (n == 0) return ULB_OK;
  ULB_CHECK(k && v && moves, ULB_EINVAL, "ulb_pages_copy: NULL argument");
  ULB_CHECK(ULB_ALIGNED16(k) && ULB_ALIGNED16(v), ULB_EINVAL, "ulb_pages_copy: the pools must be 16-byte aligned");
  ULB_CHECK(words_aligned({moves}), ULB_EINVAL, "ulb_pages_copy: unaligned array of int32");
  ULB_CUDA(cudaSetDevice(ctx->c.device));
  return launch_copy(&ctx->c, g, k, v, moves, MoveList{}, n);
}

int ulb_pages_compact(ulb_ctx* ctx, const ulb_cache_desc* cache, void* k, void* v, const int32_t* table,
                      const int32_t* base, const int32_t* count, const int32_t* src, int max_src) {
  ULB_CHECK(ctx, ULB_EINVAL, "ulb_pages_compact: NULL context");
  CacheGeom g;
  ULB_TRY(cache_geom("ulb_pages_compact", cache, &g));
  ULB_CHECK(max_src >= 0, ULB_EINVAL, "ulb_pages_compact: max_src %d", max_src);
  if (max_src == 0) return ULB_OK;
  ULB_CHECK(k && v && table && base && count && src, ULB_EINVAL, "ulb_pages_compact: NULL argument");
  ULB_CHECK(ULB_ALIGNED16(k) && ULB_ALIGNED16(v), ULB_EINVAL, "ulb_pages_compact: the pools must be 16-byte aligned");
  ULB_CHECK(words_aligned({table, base, count, src}), ULB_EINVAL, "ulb_pages_compact: unaligned array of int32");
  ULB_CHECK(g.n_seq <= 65535, ULB_EUNSUPPORTED, "ulb_pages_compact: %d sequences (at most 65535)", g.n_seq);
  Ctx* c = &ctx->c;
  ULB_CUDA(cudaSetDevice(c->device));
  const int words = g.n_head_kv * g.hd / 8, threads = std::min(256, (words + 31) / 32 * 32);
  ULB_LAUNCH("pages_compact launch", launch_k(c, pages_compact_kernel, dim3(2u * g.n_layer, g.n_seq), dim3(threads), 0, g,
                                              (uint4*)k, (uint4*)v, (const int*)table, (const int*)base, (const int*)count,
                                              (const int*)src, max_src));
  return ULB_OK;
}

int ulb_pages_create(ulb_ctx* ctx, const ulb_cache_desc* cache, void* k, void* v, ulb_pages** out) {
  ULB_CHECK(ctx && out, ULB_EINVAL, "ulb_pages_create: NULL argument");
  *out = nullptr;
  CacheGeom g;
  ULB_TRY(cache_geom("ulb_pages_create", cache, &g));
  ULB_CHECK(k && v && ULB_ALIGNED16(k) && ULB_ALIGNED16(v), ULB_EINVAL, "ulb_pages_create: the pools must be 16-byte aligned");
  ULB_CHECK((long long)g.n_seq * g.max_pages < (1ll << 31), ULB_EUNSUPPORTED, "ulb_pages_create: table %d x %d", g.n_seq, g.max_pages);
  Ctx* c = &ctx->c;
  ULB_CUDA(cudaSetDevice(c->device));
  try {
    std::unique_ptr<ulb_pages> p(new ulb_pages(g.n_pages, g.n_seq, g.max_pages, g.page));
    p->owner = ctx;
    p->g = g;
    p->k = k;
    p->v = v;
    const size_t bytes = (size_t)g.n_seq * g.max_pages * sizeof(int);
    ULB_TRY(dev_alloc(c, (void**)&p->table, bytes));
    const cudaError_t e = cudaMemsetAsync(p->table, 0xff, bytes, c->stream);
    if (e != cudaSuccess) {
      dev_free(c, p->table, bytes);
      return cuda_error(e, "ulb_pages_create", __FILE__, __LINE__);
    }
    *out = p.release();
    return ULB_OK;
  } catch (const std::bad_alloc&) {
    return set_error(ULB_ENOMEM, "ulb_pages_create: host allocation");
  }
}

int ulb_pages_free(ulb_pages* p) {
  if (!p) return ULB_OK;
  Ctx* c = &p->owner->c;
  cudaSetDevice(c->device);
  dev_free(c, p->table, (size_t)p->g.n_seq * p->g.max_pages * sizeof(int));
  delete p;
  return ULB_OK;
}

int ulb_pages_reserve(ulb_pages* p, int seq, int from, int to) {
  ULB_CHECK(p, ULB_EINVAL, "ulb_pages_reserve: NULL argument");
  return pages_change("ulb_pages_reserve", p, [&](PageWork* w) { return p->book.reserve(seq, from, to, w); });
}

int ulb_pages_fork(ulb_pages* p, int src, int dst, int n) {
  ULB_CHECK(p, ULB_EINVAL, "ulb_pages_fork: NULL argument");
  return pages_change("ulb_pages_fork", p, [&](PageWork* w) { return p->book.fork(src, dst, n, w); });
}

int ulb_pages_truncate(ulb_pages* p, int seq, int n) {
  ULB_CHECK(p, ULB_EINVAL, "ulb_pages_truncate: NULL argument");
  return pages_change("ulb_pages_truncate", p, [&](PageWork* w) { return p->book.truncate(seq, n, w); });
}

int ulb_pages_defrag(ulb_pages* p, int* used) {
  ULB_CHECK(p, ULB_EINVAL, "ulb_pages_defrag: NULL argument");
  int n = 0;
  const int rc = pages_change("ulb_pages_defrag", p, [&](PageWork* w) {
    p->book.defrag(w, &n);
    return PageRc::kOk;
  });
  if (rc == ULB_OK && used) *used = n;
  return rc;
}

int ulb_pages_info(const ulb_pages* p, const int32_t** table, int* n_free, int seq, int* mapped) {
  ULB_CHECK(p, ULB_EINVAL, "ulb_pages_info: NULL argument");
  ULB_CHECK(seq < 0 || p->book.seq_ok(seq), ULB_EINVAL, "ulb_pages_info: sequence %d", seq);
  if (table) *table = p->table;
  if (n_free) *n_free = p->book.free_pages();
  if (mapped && seq >= 0) *mapped = (int)p->book.pages(seq).size();
  return ULB_OK;
}

}  // extern "C"

ULB_TRACE_UNIT(pages)
