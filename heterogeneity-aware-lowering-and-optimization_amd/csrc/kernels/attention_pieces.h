// Which keys a row of queries sees in a paged cache, where they lie, and how the work of a call is cut into pieces.
// Plain arithmetic for kernels and host alike: whatever the operands hold, what comes out stays inside them, and
// that is checked on the host.
#ifndef ODLA_HIP_ATTENTION_PIECES_H_
#define ODLA_HIP_ATTENTION_PIECES_H_

#include "row_range.h"

namespace ohip {

OHIP_HD int at_least(const int a, const int b) { return a > b ? a : b; }
OHIP_HD int at_most(const int a, const int b) { return a < b ? a : b; }

// A sequence: its new tokens first .. first + n - 1 of all, the tokens cached before, and how many places of it the
// page table reaches (`reach` places) once the new ones are there.
struct SeqSpan { int first, n, cached, len; };
OHIP_HD SeqSpan seq_span(const int start, const int next, const int cached, const int tokens, const int reach) {
  const int first = at_most(at_least(start, 0), tokens);
  const int n = at_least(at_most(at_least(next, 0), tokens) - first, 0);   // (both ends lie in 0 .. tokens: no difference passes 32 bits)
  const int before = at_most(at_least(cached, 0), reach);
  return {first, n, before, at_most(before + n, reach)};
}

// The places that rows r0 .. r0 + most - 1 of a sequence see between them (row r: query r % group of token r / group).
struct KeyRange { int lo, hi; };
OHIP_HD KeyRange keys_of_rows(const SeqSpan& s, const int r0, const int most, const int group, const int window) {
  const int last = at_most(r0 + most, s.n * group) - 1;
  const int hi = at_most(s.cached + last / group + 1, s.len);
  const int lo = window > 0 ? at_most(at_least(s.cached + r0 / group + 1 - window, 0), hi) : 0;
  return {lo, hi};
}
// At most so many tiles of `tile` places are seen by `most` rows of the sequence.
OHIP_HD int most_key_tiles(const SeqSpan& s, const int most, const int group, const int window, const int tile) {
  const int all = (s.len + tile - 1) / tile;
  if (window == 0) return all;
  const int tokens = (most - 1) / group + 2;     // whose rows share a tile of rows
  return at_most(all, (window + tokens + tile - 1) / tile + 1);
}

// Row of the cache (token of a page) where a place lies, or -1: not in the table, or a page that does not exist.
OHIP_HD int cache_row(const int page_index, const int in_page, const int page, const int pages) {
  return page_index >= 0 && page_index < pages ? page_index * page + in_page : -1;
}

// A call's pieces: the tiles of `rows` rows of every sequence, each with the keys cut into stretches of `stretch`
// tiles.  `target` stretches at most come from cutting: stretch >= work / target.
constexpr int kTargetPieces = 1024;
OHIP_HD int row_tiles(const SeqSpan& s, const int rows, const int group) { return (int)(((long long)s.n * group + rows - 1) / rows); }
OHIP_HD int stretch_of(const float work, const int least) { return at_least((int)(work / (float)kTargetPieces) + 1, least); }
OHIP_HD int stretches(const int tiles, const int stretch) { return tiles > 0 ? (tiles - 1) / stretch + 1 : 1; }
// Bounds over all calls of one size: pieces in all, and pieces of tiles that are cut (their parts have a slot each).
// (Cut: a tile of k > stretch key tiles gives at most 2 k / stretch parts.  An eighth on top: `work` is a sum in fp32.)
OHIP_HD long long most_units(const int tokens, const int seqs, const int heads, const int group, const int rows) {
  return (long long)heads * (at_most(seqs, tokens) + (long long)tokens * group / rows);
}
constexpr int kMostCutPieces = kTargetPieces + kTargetPieces / 8, kMostSlots = 2 * kMostCutPieces;

}  // namespace ohip
#endif
