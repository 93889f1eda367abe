"""What the kernels over 8-bit blocks and experts' weights may load: kernels/row_range.h, which holds the arithmetic of
their tiles, run on the host over every edge."""
import os
import subprocess

import __graft_entry__ as entry

EXPERTS = r"""
#include "row_range.h"
#include <cstdio>
int main() {
  for (int gated = 0; gated < 2; ++gated)
    for (int H = 1; H <= 130; ++H)
      for (int I = 1; I <= 130; ++I) {
        const int own = gated ? I : H, rows_of_matrix = gated ? 2 * I : H, unit = gated ? 16 : 32;
        int seen = 0;
        for (int n0 = 0; n0 < own; n0 += unit)
          for (int j = 0; j < 2; ++j) {
            const ohip::RowTile t = ohip::expert_rows(gated, n0, j, I, H);
            if (t.rows < 0 || t.rows > 16 || (t.rows > 0 && (t.row0 < 0 || t.row0 + t.rows > rows_of_matrix))) {
              printf("gated %d H %d I %d tile %d half %d: rows %d .. %d\n", gated, H, I, n0, j, t.row0, t.row0 + t.rows);
              return 1;
            }
            seen += t.rows;
          }
        if (seen != rows_of_matrix) { printf("gated %d H %d I %d: %d rows seen\n", gated, H, I, seen); return 1; }
      }
  return 0;
}
"""


def run_on_host(tmp_path, program):
    src, exe = tmp_path / "ranges.cc", tmp_path / "ranges"
    src.write_text(program)
    kernels = os.path.join(entry.PKG_DIR, "csrc", "kernels")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I" + kernels, str(src), "-o", str(exe)], check=True, timeout=120)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout


def test_tiles_of_experts_weights_end_with_the_matrix(tmp_path):
    """Every row of the matrix belongs to one tile, and no tile has others: H and I that no tile divides."""
    run_on_host(tmp_path, EXPERTS)
