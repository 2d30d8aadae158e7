"""Which steps of 32 tokens the attention over the paged 4-bit cache goes over (csrc/kv4_steps.cuh, compiled for the host): none lies behind what a sequence has, also
where a window lies behind all of it and the table's row is full, and every token that a row sees is in one of them."""
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
      for (int pos : {0, 1, 30, 31, 32, 33, 63, 64, 65, 95, 96, 127, 128, 129, 160, 191, 192, 193, 500, 1 << 30})
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
