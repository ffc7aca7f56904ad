"""The host-side parts of the tree attention (tree_plan.h) on the CPU: the very functions that the
kernels call, driven by a model of their barriers."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(tmp_path, source):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(source)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "universal-loader_b200", "csrc"),
                    "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


# Each role's waits and signals in its own order; a role runs until its next wait is not met.  The copies
# of K and of V, the issuing warps and the softmax warps of two streams walk several pieces.
ISSUE = r'''
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>
#include "tree_plan.h"

enum Op { kWaitK, kWaitV, kFreeK, kFreeV, kScores, kLook, kWaitP, kProduct };
struct Ev { Op op; int arg; };

template <bool PAIR>
std::vector<Ev> script(int X, int n, int tiles, bool* whole) {
  std::vector<Ev> e;
  auto on = [&](Op op, int arg) { e.push_back({op, arg}); return true; };
  *whole = ulb::ring_issue<PAIR>(
      X, n, tiles, [&] { return on(kWaitK, 0) && on(kFreeK, 0); }, [&] { return on(kWaitV, 0) && on(kFreeV, 0); },
      [&] { return on(kWaitK, 0); }, [&] { return on(kWaitV, 0); }, [&](int b) { on(kScores, b), on(kFreeK, 0); },
      [&](int t) { on(kLook, t); }, [&](int b) { return on(kWaitP, b); },
      [&](int b, int i, bool more) {
        on(kProduct, i), on(kFreeV, 0);
        if (more) on(kScores, b), on(kFreeK, 0);
      });
  return e;
}

#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s (PAIR %d NK %d NV %d, %d pieces, first %d tiles, n1 %d)\n", __LINE__, #c, \
  (int)PAIR, NK, NV, (int)tiles.size(), tiles[0], (int)n1[0]); return false; } } while (0)

/* pieces of tiles[p]; n1[p]: stream 1 has rows (PAIR); masked[p]: V tiles of the piece from there are looked over */
template <bool PAIR>
bool walk(int NK, int NV, const std::vector<int>& tiles, const std::vector<char>& n1, const std::vector<int>& masked) {
  const int P = (int)tiles.size();
  int total = 0;
  for (int t : tiles) total += t;
  int loaded_k = 0, loaded_v = 0;
  struct Stream {
    int piece = 0, at = 0, seen_k = 0, seen_v = 0, free_k = 0, free_v = 0;  /* issuing warp; tiles waited for and freed */
    int scores = 0, looked = 0, products = 0, weights = 0, s_piece = 0;    /* of the piece; s_piece: the softmax warps' piece */
    std::vector<std::vector<Ev>> ev;
    std::vector<int> n;
  } st[2];
  for (int X = 0; X < 2; ++X)
    for (int p = 0; p < P; ++p) {
      st[X].n.push_back(PAIR ? (X == 0 || n1[p] ? tiles[p] : 0) : (tiles[p] + 1 - X) / 2);
      bool whole = false;
      st[X].ev.push_back(script<PAIR>(X, st[X].n[p], tiles[p], &whole));
      CHECK(whole);
    }
  for (bool moved = true; moved;) {
    moved = false;
    while (loaded_k < total && loaded_k - std::min(st[0].free_k, st[1].free_k) < NK) ++loaded_k, moved = true;
    while (loaded_v < total && loaded_v - std::min(st[0].free_v, st[1].free_v) < NV) ++loaded_v, moved = true;
    for (Stream& s : st) {
      while (s.piece < P && s.piece <= std::min(st[0].s_piece, st[1].s_piece)) { /* its queries are there */
        const std::vector<Ev>& e = s.ev[s.piece];
        if (s.at == (int)e.size()) {
          ++s.piece, s.at = 0, moved = true;
          break; /* the counts below are the piece's until the softmax warps are through */
        }
        const Ev v = e[s.at];
        if (v.op == kWaitK && s.seen_k == loaded_k) break;
        if (v.op == kWaitV && s.seen_v == loaded_v) break;
        if (v.op == kWaitP && s.weights <= s.products) break;
        if (v.op == kWaitK) ++s.seen_k;
        if (v.op == kWaitV) ++s.seen_v;
        if (v.op == kFreeK) ++s.free_k;
        if (v.op == kFreeV) ++s.free_v;
        if (v.op == kScores) {
          CHECK(s.scores - s.products <= 2 && v.arg == (s.scores & 1)); /* the buffer's earlier product has been issued */
          ++s.scores;
        }
        if (v.op == kLook) {
          CHECK(v.arg == (PAIR ? s.looked : 2 * s.looked + (int)(&s - st)));
          ++s.looked;
        }
        if (v.op == kWaitP) CHECK(v.arg == (s.products & 1));
        if (v.op == kProduct) CHECK(v.arg == s.products++ && s.seen_v > 0);
        CHECK(s.free_k <= s.seen_k && s.free_v <= s.seen_v);
        ++s.at;
        moved = true;
      }
      /* weights of tile i: its scores, and a masked V tile */
      if (s.s_piece < P && s.piece >= s.s_piece) {
        while (s.weights < s.n[s.s_piece] && s.scores > s.weights &&
               ((PAIR ? s.weights : 2 * s.weights + (int)(&s - st)) < masked[s.s_piece] || s.looked > s.weights))
          ++s.weights, moved = true;
      }
    }
    /* the piece's end: both issuing warps and both softmax warpgroups are through */
    const int p = st[0].s_piece;
    if (p < P && st[0].piece == p + 1 && st[1].piece == p + 1) {
      for (Stream& s : st) {
        CHECK(s.scores == s.n[p] && s.products == s.n[p] && s.weights == s.n[p] && s.looked == s.n[p]);
        s.scores = s.products = s.weights = s.looked = 0;
        ++s.s_piece;
      }
      moved = true;
    }
  }
  CHECK(st[0].s_piece == P && st[1].s_piece == P); /* else every role waits for another */
  CHECK(loaded_k == total && st[0].free_k == total && st[1].free_k == total && st[0].free_v == total && st[1].free_v == total);
  return true;
}

template <bool PAIR>
bool all(int NK, int NV) {
  for (int n = 1; n <= 70; ++n)
    for (int one = 0; one < 2; ++one)
      for (int m : {0, n / 2, n - 1, n})
        if (!walk<PAIR>(NK, NV, {n}, {(char)one}, {m})) return false;
  std::mt19937 r(NK * 10 + PAIR);
  for (int c = 0; c < 400; ++c) {
    std::vector<int> tiles, masked;
    std::vector<char> n1;
    for (int p = 1 + r() % 6; p > 0; --p) {
      tiles.push_back(1 + r() % (r() % 2 ? 4 : 60));
      n1.push_back(r() % 2);
      masked.push_back(r() % (tiles.back() + 1));
    }
    if (!walk<PAIR>(NK, NV, tiles, n1, masked)) return false;
  }
  return true;
}

int main() {
  for (int nk = 3; nk <= 8; ++nk)
    for (int nv = 2; nv <= 8; ++nv)
      if (!all<false>(nk, nv) || !all<true>(nk, nv)) return 1;
  std::printf("ok\n");
}
'''


def test_no_role_waits_for_itself(tmp_path):
    """Pieces of any length, both streams with rows or one without: every K and V tile is copied, used and
    freed in rings of any depth that the kernels have, with masked tiles and without."""
    run(tmp_path, ISSUE)


# A wait that is not met ends the issuing role: nothing is issued or freed after it.
STOP = r'''
#include <cstdio>
#include "tree_plan.h"
template <bool PAIR> int stop(int X, int n, int tiles, int fail) {
  int waits = 0, after = 0;
  bool failed = false;
  auto wait = [&] { after += failed; failed = failed || waits++ == fail; return !failed; };
  auto act = [&] { after += failed; };
  const bool whole = ulb::ring_issue<PAIR>(X, n, tiles, wait, wait, wait, wait, [&](int) { act(); }, [&](int) { act(); },
                                           [&](int) { return wait(); }, [&](int, int, bool) { act(); });
  return after || whole == failed;
}
int main() {
  for (int tiles = 1; tiles < 20; ++tiles)
    for (int fail = 0; fail < 70; ++fail)
      for (int X = 0; X < 2; ++X) {
        if (stop<false>(X, (tiles + 1 - X) / 2, tiles, fail) || stop<true>(X, tiles, tiles, fail) || stop<true>(X, 0, tiles, fail)) {
          std::printf("%d tiles, wait %d\n", tiles, fail);
          return 1;
        }
      }
  std::printf("ok\n");
}
'''


def test_a_failed_wait_ends_the_issuing_role(tmp_path):
    run(tmp_path, STOP)


COPY = r'''
#include <cstdio>
#include "tree_plan.h"
int main() {
  for (int n = 0; n < 20; ++n)
    for (int fail = 0; fail <= n; ++fail) {
      int waits = 0, copies = 0, looks = 0, bad = 0;
      const bool whole = ulb::ring_copy(
          n, [&](int t) { bad += t != looks++; }, [&] { return waits++ != fail; },
          [&](int t) { bad += t != copies++ || copies > fail || looks != t + 1; });
      if (bad || copies != (fail < n ? fail : n) || whole != (fail >= n)) {
        std::printf("%d tiles, wait %d: %d copies\n", n, fail, copies);
        return 1;
      }
    }
  std::printf("ok\n");
}
'''


def test_a_failed_wait_ends_the_copies(tmp_path):
    """A place that was not seen free is not copied into, nor any after it."""
    run(tmp_path, COPY)


ROWS = r'''
#include <climits>
#include <cstdio>
#include "tree_plan.h"
int main() {
  const int at[] = {INT_MIN, INT_MIN + 1, -1000, -1, 0, 1, 5, 99, 100, 101, 4000, INT_MAX - 1, INT_MAX};
  const int sizes[] = {0, 1, 7, 100, INT_MAX};
  for (int rows : sizes)
    for (int most : sizes)
      for (int b : at)
        for (int e : at) {
          int r0 = -7;
          const int n = ulb::rows_of(b, e, rows, most, &r0);
          const long long lo = b < 0 ? 0 : b, hi = e < rows ? e : rows;  /* the rows that [b, e) and [0, rows) share */
          const long long want = hi > lo ? (hi - lo < most ? hi - lo : most) : 0;
          if (n != want || r0 < 0 || r0 > rows || (n > 0 && r0 != lo) || (long long)r0 + n > rows) {
            std::printf("[%d, %d) of %d, at most %d: %d rows from %d\n", b, e, rows, most, n, r0);
            return 1;
          }
        }
  std::printf("ok\n");
}
'''


def test_rows_of_a_sequence_stay_in_range(tmp_path):
    """Whatever row_start holds, a sequence's rows are rows of the call."""
    run(tmp_path, ROWS)
