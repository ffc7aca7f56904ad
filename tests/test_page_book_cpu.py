"""The page book (page_book.h) on the CPU: sharing, copy on write, roll-back, refusals that change
nothing, lowest page first, and defragmentation, against a model that keeps whole sequences."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DRIVER = r'''
#include <cassert>
#include <cstdio>
#include <map>
#include <random>
#include "page_book.h"
using namespace ulb;
#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main() {
  {
    PageBook b(6, 3, 4, 16);
    PageWork w;
    CHECK(b.reserve(0, 0, 40, &w) == PageRc::kOk && w.entries.size() == 3 && w.moves.empty());
    CHECK(b.pages(0) == (std::vector<int>{0, 1, 2}) && b.free_pages() == 3);
    w = {};
    CHECK(b.fork(0, 1, 35, &w) == PageRc::kOk && b.pages(1) == b.pages(0) && b.refs(2) == 2 && b.free_pages() == 3);
    w = {};
    /* the tail page is shared: 3 of its positions move to a page of the sequence's own */
    CHECK(b.reserve(1, 35, 36, &w) == PageRc::kOk && w.moves.size() == 1);
    CHECK(w.moves[0].src == 2 && w.moves[0].dst == 3 && w.moves[0].positions == 3 && b.refs(2) == 1);
    w = {};
    CHECK(b.reserve(1, 36, 37, &w) == PageRc::kOk && w.moves.empty() && w.entries.empty());
    /* a write that starts on a page edge copies nothing of that page */
    CHECK(b.reserve(1, 16, 17, &w) == PageRc::kOk && w.moves.empty() && w.entries.size() == 1 && b.pages(1)[1] == 4);
    w = {};
    CHECK(b.reserve(2, 0, 33, &w) == PageRc::kNoPages && b.free_pages() == 1 && b.pages(2).empty() && w.entries.empty());
    CHECK(b.reserve(0, 0, 65, &w) == PageRc::kBadArg && b.reserve(3, 0, 1, &w) == PageRc::kBadArg);
    CHECK(b.reserve(0, 2, 1, &w) == PageRc::kBadArg && b.reserve(-1, 0, 0, &w) == PageRc::kBadArg);
    CHECK(b.fork(0, 1, 1, &w) == PageRc::kBadArg && b.fork(0, 2, 49, &w) == PageRc::kBadArg && b.fork(0, 0, 1, &w) == PageRc::kBadArg);
    CHECK(b.truncate(0, 17, &w) == PageRc::kOk && b.pages(0).size() == 2 && b.refs(2) == 0 && b.free_pages() == 2);
    CHECK(b.truncate(0, 17, &w) == PageRc::kOk && b.truncate(0, -1, &w) == PageRc::kBadArg);
    w = {};
    CHECK(b.truncate(0, 0, &w) == PageRc::kOk && b.refs(0) == 1 && b.free_pages() == 3); /* page 0 is sequence 1's */
    w = {};
    int used = -1;
    b.defrag(&w, &used);
    CHECK(used == 3 && b.free_pages() == 3);
    for (int p : b.pages(1)) CHECK(p < 3);
    for (const PageMove& m : w.moves) CHECK(m.src >= 3 && m.dst < 3 && m.positions == 16);
    w = {};
    CHECK(b.reserve(0, 0, 16, &w) == PageRc::kOk && b.pages(0)[0] == 3); /* lowest free page */
  }
  /* random changes: page contents follow the work lists, sequences keep their words */
  std::mt19937 r(7);
  const int P = 30, S = 5, M = 9, Z = 16;
  PageBook b(P, S, M, Z);
  std::vector<std::vector<int>> page(P, std::vector<int>(Z, 0)), word(S), table(S, std::vector<int>(M, -1));
  int next = 1;
  for (int step = 0; step < 20000; ++step) {
    PageWork w;
    const int s = r() % S, what = r() % 8;
    int from = 0, to = 0;
    bool wrote = false;
    if (what < 4) {
      from = what < 2 ? (int)word[s].size() : (int)(r() % (word[s].size() + 1));
      to = std::min(from + (int)(r() % 40), M * Z);
      const int before = b.free_pages();
      const PageRc rc = b.reserve(s, from, to, &w);
      CHECK(rc != PageRc::kBadArg);
      if (rc == PageRc::kNoPages) { CHECK(before == b.free_pages() && w.entries.empty() && w.moves.empty()); continue; }
      wrote = true;
    } else if (what == 4) {
      const int d = r() % S;
      if (d == s || !b.pages(d).empty()) continue;
      const int n = r() % (word[s].size() + 1);
      CHECK(b.fork(s, d, n, &w) == PageRc::kOk);
      word[d].assign(word[s].begin(), word[s].begin() + n);
    } else if (what < 7) {
      const int n = r() % 2 ? r() % (word[s].size() + 1) : 0;
      CHECK(b.truncate(s, n, &w) == PageRc::kOk);
      word[s].resize(n);
    } else {
      int used;
      b.defrag(&w, &used);
      CHECK(used + b.free_pages() == P);
    }
    std::vector<int> src(P, 0);
    for (const PageMove& m : w.moves) src[m.src] = 1;
    for (const PageMove& m : w.moves) { CHECK(!src[m.dst]); src[m.dst] |= 2; }
    for (const PageMove& m : w.moves) for (int i = 0; i < m.positions; ++i) page[m.dst][i] = page[m.src][i];
    for (const PageEntry& e : w.entries) table[e.seq][e.index] = e.page;
    if (wrote && to > from) {
      word[s].resize(from);
      for (int t = from; t < to; ++t) {
        CHECK(b.refs(table[s][t / Z]) == 1);
        page[table[s][t / Z]][t % Z] = next;
        word[s].push_back(next++);
      }
    }
    std::map<int, int> held;
    for (int q = 0; q < S; ++q) {
      for (int j = 0; j < M; ++j) CHECK(table[q][j] == (j < (int)b.pages(q).size() ? b.pages(q)[j] : -1));
      for (int p : b.pages(q)) ++held[p];
      for (int t = 0; t < (int)word[q].size(); ++t) CHECK(page[table[q][t / Z]][t % Z] == word[q][t]);
    }
    int n = 0;
    for (int p = 0; p < P; ++p) { CHECK(b.refs(p) == (held.count(p) ? held[p] : 0)); n += b.refs(p) == 0; }
    CHECK(n == b.free_pages());
  }
  std::printf("ok\n");
  return 0;
}
'''


def test_page_book(tmp_path):
    src = tmp_path / "pb.cpp"
    src.write_text(DRIVER)
    exe = tmp_path / "pb"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I" + os.path.join(ROOT, "universal-loader_b200", "csrc"),
                    "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
