"""Which steps of 32 tokens the attention over the paged 4-bit cache goes over and how the line of them is cut (csrc/kv4_steps.cuh, compiled for the host): no step lies behind
what a sequence has, also where a window lies behind all of it and the table's row is full, every token that a row sees is in one of them, every step is gone over once, and
every search ends."""
import subprocess

from tinygpt_b200 import build

MAIN = """
#include <algorithm>
#include <cstdio>
#include "kv4_steps.cuh"
using namespace b200;
// rows low ... high of a sequence, of whose steps a piece of `many` from `first` on is gone over as the kernels do
static bool fits(int pos, int rows, int last, int window, int max_pages, int columns) {
  const Kv4Steps all = kv4_seq_steps(pos, last, window);
  const int places = max_pages * 2;   // steps that the table's row has
  auto covers = [&](int low, int high, int from, int to) {
    for (int p = low; p <= high; ++p) {
      const int first = std::max(0, window > 0 ? p - window + 1 : 0), end = std::min(p + 1, last);
      if (first < end && (first / kStep < from || (end - 1) / kStep >= to)) return false;
    }
    return true;
  };
  if (all.first < 0 || all.n < 1 || all.first + all.n > std::max(places, 1)) return false;
  if (!covers(pos, pos + rows - 1, all.first, all.first + all.n)) return false;
  for (int low = pos; low < pos + rows; low += columns) {
    const int high = std::min(low + columns, pos + rows) - 1;
    // a warp's or a cluster's piece of all steps
    for (int first = 0; first < all.n; first += std::max(all.n / 3, 1)) {
      const int many = std::min(std::max(all.n / 3, 1), all.n - first), step0 = all.first + first, n = kv4_steps_end(high, last, step0, many);
      if (n > many || (n > 0 && (step0 < 0 || step0 + n > places))) return false;
    }
    // a block's own steps
    const Kv4Steps own = kv4_rows_steps(low, high, last, window, all);
    const int step0 = all.first + own.first, begin = kv4_steps_begin(low, window, step0), end = kv4_steps_end(high, last, step0, own.n);
    if (own.first < 0 || own.n < 1 || own.first + own.n > all.n || end > own.n) return false;
    if (begin < end && (step0 + begin < 0 || step0 + end > places)) return false;
    if (!covers(low, high, step0 + begin, step0 + end)) return false;
  }
  return true;
}
int main() {
  long n = 0;
  for (int max_pages : {1, 2, 3})
    for (int length = 0; length <= max_pages * 64; ++length)
      for (int pos : {0, 1, 30, 31, 32, 33, 63, 64, 65, 95, 96, 127, 128, 129, 160, 191, 192, 193, 500, 1 << 30, 2147483647 - 64 - 70})
        for (int rows : {1, 2, 33, 70})
          for (int window : {0, 1, 2, 10, 31, 32, 33, 64, 65, 150, 2147483647})
            for (int columns : {1, 8, 64}) {
              const int last = std::min(length, pos + rows);
              ++n;
              if (!fits(pos, rows, last, window, max_pages, columns))
                return printf("%d rows from %d on, %d tokens, window %d, %d pages, blocks of %d\\n", rows, pos, length, window, max_pages, columns), 1;
            }
  printf("%ld\\n", n);
  return 0;
}
"""


def test_steps_stay_within_the_table(tmp_path):
    (tmp_path / "main.cpp").write_text(MAIN)
    exe = tmp_path / "main"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(build.CSRC), str(tmp_path / "main.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and int(r.stdout) > 100000, r.stdout


def test_a_cluster_does_not_take_many_blocks_in_turn(built_lib):
    """A cluster goes over a sequence's blocks one after the other, so a call goes to clusters (no workspace) only where the one that may bring most rows has few."""
    import ctypes as C

    from tinygpt_b200._lib import KV4Desc, lib

    def clusters(heads, kv_heads, dim, max_pages, n, rows):
        cache = KV4Desc(None, None, None, None, 1, 4096, n, max_pages, kv_heads, dim)
        return lib().b200_kv4_attention_workspace_bytes(C.byref(cache), heads, n, rows) == 0

    # one token a sequence, small caches: as many columns as the group has
    assert clusters(14, 2, 64, 1, 2, 2) and clusters(4, 4, 128, 13, 32, 32) and clusters(24, 8, 128, 63, 1, 1) and clusters(32, 4, 64, 7, 18, 18)
    assert clusters(4, 2, 64, 6, 5, 8)
    # 32 tokens beside a piece of 800 rows, and of 500 beside four, whose average is few columns
    assert not clusters(4, 4, 128, 13, 33, 832) and not clusters(2, 2, 64, 13, 20, 519)
    # larger tables are cut evenly
    assert not clusters(24, 8, 128, 512, 1, 1)


CUT = """
#include <algorithm>
#include <cstdio>
#include <map>
#include <random>
#include <vector>
#include "kv4_steps.cuh"
using namespace b200;
struct Seq { int blocks, steps[2]; };   // steps as one reading or another finds them
#define NEED(cond) do { if (!(cond)) { printf("line %d: %s\\\\n", __LINE__, #cond); return 1; } } while (0)
static int walk(std::mt19937& rng, const std::vector<Seq>& seqs, int heads, int most, bool same) {
  const int n = (int)seqs.size();
  auto reading = [&] { return same ? 0 : (int)(rng() % 2); };
  std::map<long long, int> left;             // place of a part -> item
  std::map<int, std::vector<int>> covered;   // item -> how often each step
  std::map<int, int> many_left;
  struct Join { Kv4Pieces p; int item; };
  std::vector<Join> joins;
  auto id = [&](int i, int number) { int k = number; for (int j = 0; j < i; ++j) k += seqs[j].blocks * heads; return k; };
  for (int cta = 0; cta < kGrid; ++cta) {
    std::vector<int> ends(n);
    int line = 0;
    for (int i = 0; i < n; ++i) ends[i] = line += seqs[i].blocks * heads * (seqs[i].steps[reading()] + kAhead);
    const Kv4Cut cut(line, most);
    NEED(cut.each >= 1 && cut.each <= most && cut.start(0) == 0 && cut.start(cut.warps) == line);
    int here = 0, inside_item = -1;
    for (int warp = 0; warp < most; ++warp) {
      const int me = cta * cut.each + warp;
      int at = cut.start(me);
      const int stop = warp < cut.each ? cut.start(me + 1) : at;
      NEED(at <= stop && stop <= line);
      for (int i = 0; at < stop;) {
        while (ends[i] <= at) ++i;
        const int base = i > 0 ? ends[i - 1] : 0, steps = seqs[i].steps[reading()];
        const Kv4Item item = kv4_item(at, base, ends[i], steps);
        NEED(item.number >= 0 && item.end > at && item.end <= line);
        const int first = std::max(at - item.begin, 0), many = std::min(stop, item.end) - item.begin - first;
        at = std::min(stop, item.end);
        if (many <= 0) continue;
        NEED(first >= 0 && first + many <= steps);
        const int which = same ? id(i, item.number) : 0;
        if (same) {
          auto& c = covered[which];
          c.resize(steps);
          for (int s = first; s < first + many; ++s) ++c[s];
        }
        if (many == steps) continue;
        if (first == 0) {
          const Kv4Pieces p = kv4_pieces(cut, cta, me, item.begin, item.end);
          NEED(p.from >= 0 && p.from <= p.to && p.to < cut.warps && p.before >= 0 && p.whole >= 0 && p.parts >= 1 && p.parts <= cut.warps);
          for (int k = 0; k < p.parts; ++k) NEED(p.piece(k) >= p.from && p.piece(k) <= p.to && p.piece(k) / p.each < kGrid && p.piece(k) % p.each < most);
          joins.push_back({p, which});
        }
        if (!kv4_inside(cut, cta, item.begin, item.end)) {
          if (same) {
            const long long place = ((long long)cta * most + warp) * 2 + (first == 0);
            NEED(!left.count(place));
            left[place] = which;
            ++many_left[which];
          }
          continue;
        }
        NEED(at == stop);   // its last item
        ++here;
        if (same) {
          NEED(inside_item < 0 || inside_item == which);
          inside_item = which;
        }
      }
    }
    if (same) {
      NEED(here == 0 || here == cut.each);   // all of them meet or none
      if (here > 0) {
        left[(long long)cta * most * 2] = inside_item;
        ++many_left[inside_item];
      }
    }
  }
  if (!same) return 0;
  int items = 0;
  for (const Seq& s : seqs) items += s.blocks * heads;
  NEED((int)covered.size() == items);
  for (auto& c : covered)
    for (int v : c.second) NEED(v == 1);
  NEED(joins.size() == many_left.size());
  for (const Join& j : joins) {   // the parts that are joined are those that were left
    NEED(j.p.parts == many_left[j.item]);
    for (int k = 0; k < j.p.parts; ++k) {
      const int w = j.p.piece(k);
      const long long place = ((long long)(w / j.p.each) * most + w % j.p.each) * 2 + (k < j.p.before && k == 0);
      NEED(left.count(place) && left[place] == j.item);
      left.erase(place);
    }
  }
  NEED(left.empty());
  return 0;
}
int main() {
  std::mt19937 rng(1);
  for (int round = 0; round < 400; ++round) {
    const int n = 1 + rng() % (round % 3 ? 5 : 70), heads = 1 + rng() % 8, top = 1 << rng() % 11;
    std::vector<Seq> seqs(n);
    for (Seq& s : seqs) s = {(int)(rng() % (round % 4 ? 2 : 20) + (round % 5 > 0)), {(int)(1 + rng() % top), (int)(1 + rng() % top)}};
    for (int most : {1, 8}) {
      if (walk(rng, seqs, heads, most, true)) return printf("round %d, one reading\\\\n", round), 1;
      for (int k = 0; k < 3; ++k)
        if (walk(rng, seqs, heads, most, false)) return printf("round %d, changing lengths\\\\n", round), 1;
    }
  }
  return 0;
}
"""


def test_the_line_is_cut_and_joined(tmp_path):
    """Every step of every item is gone over once and every part that is left is joined, in one part a CTA or a warp; and where every reading of a sequence finds another
    length, as it may if another stream writes to it meanwhile, all searches end and all places lie where they may."""
    (tmp_path / "main.cpp").write_text(CUT.replace("\\\\n", "\\n"))
    exe = tmp_path / "main"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(build.CSRC), str(tmp_path / "main.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout
