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


# A request as the matrix of lanes sees it: `rows_of` rows of a tile, eight lanes a row, 16 bytes each.  What the range lets
# through has to be those 16 bytes of that row (or the row's last 16), inside the operand; what it does not is behind an end.
MODEL = r"""
#include "row_range.h"
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
typedef long long i64;
static const unsigned char* const kBase = (const unsigned char*)0x100000000ll;
static i64 bad(const char* what, int rows, int len, i64 row, int at) {
  printf("%s: %d rows of %d bytes: row %lld byte %d\n", what, rows, len, row, at);
  exit(1);
}
// the operand has `rows` rows of `len` bytes from kBase on; `tile_rows` of them from `row0` on are the tile's
static void request(const char* what, int rows, int len, bool whole, i64 row0, int tile_rows, bool in_vectors, int first, int most, int row, int at) {
  const ohip::RowRange r = ohip::row_range(kBase + row0 * len, in_vectors ? tile_rows : 0, first, most, len);
  const unsigned off = ohip::lane_offset((unsigned)row * len, at, len, whole);
  const bool wanted = in_vectors && first + row < tile_rows && at < len;
  const bool inside = off < r.size && (i64)off + 16 <= r.size;
  if (off < r.size && !inside) bad(what, rows, len, row0 + first + row, at);          // 16 bytes across the range's end
  if (inside != wanted) bad(what, rows, len, row0 + first + row, at);
  if (!inside) return;
  const i64 from = r.base - kBase + off, want = (row0 + first + row) * len + (whole || at + 16 <= len ? at : len - 16);
  if (from != want || from < 0 || from + 16 > (i64)rows * len) bad(what, rows, len, row0 + first + row, at);
}
"""

PRODUCT = MODEL + r"""
int main() {
  // tiles of 16, 32 or 64 rows, eight rows a request: rows that are no whole vectors
  for (int side = 16; side <= 64; side *= 2)
    for (int rows = 1; rows <= 130; ++rows)
      for (int len : {1, 7, 15, 16, 17, 31, 100, 127, 128, 129, 143, 144, 145, 271, 272, 300})
        for (int row0 = 0; row0 < rows; row0 += side) {
          const int tile = ohip::rows_within(rows - row0, side);
          for (int first = 0; first < side; first += 8)
            for (int row = 0; row < 8; ++row)
              for (int at = 0; at < (len + 127) / 128 * 128; at += 16) request("few tiles", rows, len, false, row0, tile, len >= 16, first, 8, row, at);
        }
  // tiles of 128 or 256 rows, whole vectors, 32 or 64 rows a request, one block of terms behind the last
  for (int waves : {4, 8})
    for (int rows = 1; rows <= 600; rows += rows < 40 || rows % 32 > 29 ? 1 : 3)
      for (int len : {16, 112, 128, 144, 256, 400})
        for (int row0 = 0; row0 < rows; row0 += 32 * waves) {
          const int tile = ohip::rows_within(rows - row0, 32 * waves);
          for (int i = 0; i < 4; ++i)
            for (int row = 0; row < 8 * waves; ++row)
              for (int at = 0; at < (len + 127) / 128 * 128 + 128; at += 16) request("many tiles", rows, len, true, row0, tile, true, i * 8 * waves, 8 * waves, row, at);
        }
  // the largest: 256 rows of 2^22 bytes, 64 of 2^24
  for (int row : {0, 63}) request("largest", 256, 1 << 22, true, 0, 256, true, 192, 64, row, (1 << 22) - 16);
  for (int row : {0, 7}) request("largest", 64, (1 << 24) - 1, false, 0, 64, true, 56, 8, row, (1 << 24) - 16);
  return 0;
}
"""

WEIGHTS = MODEL + r"""
int main() {
  for (int gated = 0; gated < 2; ++gated)
    for (int own = 1; own <= 130; ++own)                        // I of the first product, H of the second
      for (int len : {1, 15, 16, 24, 127, 128, 130, 712}) {
        const int rows = gated ? 2 * own : own;                 // (of the last expert: what lies behind it is not the operand's)
        for (int n0 = 0; n0 < own; n0 += gated ? 16 : 32)
          for (int j = 0; j < 2; ++j) {
            const ohip::RowTile t = ohip::expert_rows(gated, n0, j, own, own);
            for (int first = 0; first < 16; first += 8)
              for (int row = 0; row < 8; ++row)
                for (int at = 0; at < (len + 127) / 128 * 128; at += 16) request("weights", rows, len, len % 16 == 0, t.row0, t.rows, len >= 16, first, 8, row, at);
          }
      }
  return 0;
}
"""


def test_requests_of_a_product_stay_in_their_operand(tmp_path):
    run_on_host(tmp_path, PRODUCT)


def test_requests_of_experts_weights_stay_in_their_matrix(tmp_path):
    run_on_host(tmp_path, WEIGHTS)
