"""How the paged attention cuts its list of key tiles: the runs are equal within a tile and cover the list, and the run of a tile, by
which the merge finds an item's last part, is the one that holds it."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r'''
#include <cstdio>
#include <initializer_list>
#include "heddle_b200/csrc/fa_paged_plan.h"
using namespace hb;
int main() {
  if (paged_tiles(0) != 1 || paged_tiles(-3) != 1 || paged_tiles(1) != 1 || paged_tiles(32) != 1 || paged_tiles(33) != 2) return printf("tiles\n"), 1;
  if (paged_row_tiles(0, 8, 16) != 0 || paged_row_tiles(1, 17, 16) != 2 || paged_row_tiles(2147483, 1000, 8) != 268435375) return printf("rows\n"), 1;
  for (int blocks : {1, 2, 5, 296})
    for (long long total : {1ll, 2ll, 3ll, 4ll, 5ll, 7ll, 64ll, 295ll, 296ll, 297ll, 1183ll, 1184ll, 1185ll, 100003ll, 1ll << 31, (1ll << 47) + 12345}) {
      const int runs = paged_runs(total, blocks);
      if (runs < 1 || runs > blocks || (runs > 1 && total < (runs - 1) * 4ll)) return printf("runs %lld %d\n", total, blocks), 1;
      if (paged_begin(total, runs, 0) != 0 || paged_begin(total, runs, runs) != total) return printf("ends %lld %d\n", total, blocks), 1;
      for (int w = 0; w < runs; ++w) {
        const long long a = paged_begin(total, runs, w), b = paged_begin(total, runs, w + 1);
        if (b - a < total / runs || b - a > total / runs + 1) return printf("length %lld %d %d\n", total, blocks, w), 1;
        for (long long t : {a, a + (b - a) / 2, b - 1})
          if (t >= a && t < b && paged_run_of(total, runs, t) != w) return printf("run %lld %d %lld\n", total, blocks, t), 1;
      }
    }
  printf("ok\n");
}
'''


def test_plan(tmp_path):
    src = tmp_path / "plan.cpp"
    src.write_text(PROGRAM)
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-std=c++17", "-O2", "-fwrapv", f"-I{ROOT}", str(src), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout.strip() == "ok", done.stdout
