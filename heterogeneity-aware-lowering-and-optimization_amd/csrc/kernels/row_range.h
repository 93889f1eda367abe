// Which rows of an operand a tile has.  Plain arithmetic for kernels and host alike: what a tile may load is
// checked on the host for every edge.
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

}  // namespace ohip
#endif
