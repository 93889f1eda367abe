// Which rows of an operand a tile has, and which bytes its loads ask for.  Plain arithmetic for kernels and host
// alike: what a tile may load is checked on the host for every edge.
#ifndef ODLA_HIP_ROW_RANGE_H_
#define ODLA_HIP_ROW_RANGE_H_

#if defined(__HIPCC__)
#define OHIP_HD __host__ __device__ __forceinline__
#else
#define OHIP_HD inline
#endif

namespace ohip {

// `most` rows where `left` are left: none where the tile lies behind the operand's end.
OHIP_HD int rows_within(const int left, const int most) { return left < 0 ? 0 : left < most ? left : most; }

// Half j of the tile at n0 of an expert's matrix: sixteen of gate's I rows (0) or of up's behind them (1) in the
// first product, the first or second sixteen of 32 of down's H rows in the second.
struct RowTile { int row0, rows; };
OHIP_HD RowTile expert_rows(const bool gated, const int n0, const int j, const int I, const int H) {
  const int row0 = gated ? j * I + n0 : n0 + 16 * j;
  return {row0, rows_within(gated ? I - n0 : H - row0, 16)};
}

// One request of a wavefront: rows first .. first + most - 1 of a tile that starts at `tile` and has `rows` rows of
// `len` bytes.  Its buffer range is its own rows and nothing else, and every byte is asked for by a lane's offset
// from `base` alone: what a range check makes of a scalar offset beyond the size is not laid down anywhere.
struct RowRange { const unsigned char* base; unsigned size; };
OHIP_HD RowRange row_range(const unsigned char* tile, const int rows, const int first, const int most, const int len) {
  return {tile + (long long)first * len, (unsigned)rows_within(rows - first, most) * (unsigned)len};
}
// A lane's offset in such a request: its row's, `row`, and 16 bytes at `at` of it; outside every range behind the
// row's end.  Rows that are not whole vectors: 16 bytes that would pass the end are the last 16 (len >= 16).
constexpr unsigned kOutside = 0xfffffff0u;
OHIP_HD unsigned lane_offset(const unsigned row, const int at, const int len, const bool whole_vectors) {
  return at >= len ? kOutside : row + (unsigned)(whole_vectors || at + 16 <= len ? at : len - 16);
}

}  // namespace ohip
#endif
