/*
 * page_book.h — which page holds which positions of which sequence, with pages shared between
 * forked sequences (reference counts).  The device side (block table, page copies) is pages.cu;
 * the speculative loop's slots use the simpler PagePool of paging.h, which never shares.
 *
 * Every call either succeeds or changes nothing.  What the device has to do comes back as a
 * list of table entries to set and a list of page copies; copies name destinations that were
 * free, so within one call no page is both read and written.
 *
 * Host-only (no CUDA types): unit tested on the CPU.
 */
#pragma once

#include <vector>

namespace ulb {

struct PageEntry { int seq, index, page; };        /* table[seq][index] = page (-1: unmapped) */
struct PageMove { int src, dst, positions; };
struct PageWork {
  std::vector<PageEntry> entries;
  std::vector<PageMove> moves;
};
enum class PageRc { kOk, kBadArg, kNoPages };

class PageBook {
 public:
  PageBook(int n_pages, int n_seq, int max_pages, int page)
      : max_pages_(max_pages), page_(page), n_free_(n_pages), low_(0), ref_(n_pages, 0), seqs_(n_seq) {}

  /* positions [0, to) mapped, the pages of [from, to) held by this sequence alone */
  PageRc reserve(int s, int from, int to, PageWork* w) {
    if (!seq_ok(s) || from < 0 || to < from || pages_of(to) > max_pages_) return PageRc::kBadArg;
    std::vector<int>& have = seqs_[s];
    const int n = (int)have.size(), want = pages_of(to), first = from / page_;
    std::vector<int> shared;
    for (int j = first; to > from && j < want && j < n; ++j)
      if (ref_[have[j]] > 1) shared.push_back(j);
    const int need = (int)shared.size() + (want > n ? want - n : 0);
    if (n_free_ < need) return PageRc::kNoPages;
    w->entries.reserve(w->entries.size() + need);
    w->moves.reserve(w->moves.size() + shared.size());
    if (want > n) have.reserve(want);
    for (int j : shared) {
      const int p = take(), keep = from - j * page_;
      if (keep > 0) w->moves.push_back({have[j], p, keep});
      --ref_[have[j]];
      have[j] = p;
      w->entries.push_back({s, j, p});
    }
    for (int j = n; j < want; ++j) {
      const int p = take();
      have.push_back(p);
      w->entries.push_back({s, j, p});
    }
    return PageRc::kOk;
  }

  /* dst, which holds nothing, shares src's pages of positions [0, n) */
  PageRc fork(int src, int dst, int n, PageWork* w) {
    if (!seq_ok(src) || !seq_ok(dst) || src == dst || n < 0 || !seqs_[dst].empty()) return PageRc::kBadArg;
    const long long k = ((long long)n + page_ - 1) / page_;
    if (k > (long long)seqs_[src].size()) return PageRc::kBadArg;
    w->entries.reserve(w->entries.size() + (size_t)k);
    seqs_[dst].assign(seqs_[src].begin(), seqs_[src].begin() + k);
    for (int j = 0; j < (int)k; ++j) {
      ++ref_[seqs_[dst][j]];
      w->entries.push_back({dst, j, seqs_[dst][j]});
    }
    return PageRc::kOk;
  }

  /* the pages past position n go back */
  PageRc truncate(int s, int n, PageWork* w) {
    if (!seq_ok(s) || n < 0) return PageRc::kBadArg;
    std::vector<int>& have = seqs_[s];
    const long long keep = ((long long)n + page_ - 1) / page_;
    if (keep >= (long long)have.size()) return PageRc::kOk;
    w->entries.reserve(w->entries.size() + have.size() - (size_t)keep);
    for (int j = (int)keep; j < (int)have.size(); ++j) {
      w->entries.push_back({s, j, -1});
      if (--ref_[have[j]] == 0) {
        ++n_free_;
        if (have[j] < low_) low_ = have[j];
      }
    }
    have.resize((size_t)keep);
    return PageRc::kOk;
  }

  /* every page in use below *used */
  void defrag(PageWork* w, int* used) {
    const int n = (int)ref_.size() - n_free_;
    std::vector<int> to(ref_.size(), -1);
    int hole = 0;
    for (int p = n; p < (int)ref_.size(); ++p)
      if (ref_[p] > 0) {
        while (ref_[hole] > 0) ++hole;
        to[p] = hole++;
        w->moves.push_back({p, to[p], page_});
      }
    for (int s = 0; s < (int)seqs_.size(); ++s)
      for (int j = 0; j < (int)seqs_[s].size(); ++j)
        if (to[seqs_[s][j]] >= 0) w->entries.push_back({s, j, to[seqs_[s][j]]});
    /* nothing below allocates */
    for (const PageEntry& e : w->entries) seqs_[e.seq][e.index] = e.page;
    for (const PageMove& m : w->moves) {
      ref_[m.dst] = ref_[m.src];
      ref_[m.src] = 0;
    }
    low_ = n;
    *used = n;
  }

  int free_pages() const { return n_free_; }
  bool seq_ok(int s) const { return s >= 0 && s < (int)seqs_.size(); }
  const std::vector<int>& pages(int s) const { return seqs_[s]; }
  int refs(int p) const { return ref_[p]; }

 private:
  int pages_of(int n) const { return (int)(((long long)n + page_ - 1) / page_); }
  int take() {
    while (ref_[low_] > 0) ++low_;
    --n_free_;
    ref_[low_] = 1;
    return low_;
  }

  int max_pages_, page_;
  int n_free_, low_;        /* free pages; no page below low_ is free */
  std::vector<int> ref_;    /* sequences holding each page, 0: free */
  std::vector<std::vector<int>> seqs_;
};

}  // namespace ulb
