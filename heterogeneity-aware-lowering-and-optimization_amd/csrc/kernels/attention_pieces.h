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

// A call's pieces.  A sequence is cut one of two ways, by how many rows a head of keys has in it: into tiles of `rows`
// rows, each with its keys in stretches of a number of key tiles of `keys` places that follows from the lengths of all
// sequences of its way: `target` pieces at most come from cutting (stretch >= work / target), none shorter than `least`.
struct Way { int rows, keys, least, target; };
OHIP_HD int row_tiles(const SeqSpan& s, const Way& w, const int group) { return (int)(((long long)s.n * group + w.rows - 1) / w.rows); }
OHIP_HD int key_tiles(const SeqSpan& s, const Way& w, const int group, const int window) { return most_key_tiles(s, w.rows, group, window, w.keys); }
OHIP_HD float work_of(const SeqSpan& s, const Way& w, const int group, const int heads, const int window) {
  return (float)row_tiles(s, w, group) * (float)heads * (float)key_tiles(s, w, group, window);
}
OHIP_HD int stretch_of(const float work, const Way& w) {
  const float each = work / (float)w.target;
  return at_least((int)(each < 0x1p30f ? each : 0x1p30f) + 1, w.least);      // (no row has more tiles than that)
}
OHIP_HD int stretches(const int tiles, const int stretch) { return tiles > 0 ? (tiles - 1) / stretch + 1 : 1; }
// Bounds over all calls of one size: pieces that come from cutting, and pieces of tiles that are cut (their parts have
// a slot each).  (Cut: a tile of k > stretch key tiles gives at most 2 k / stretch parts.  An eighth on top: the work
// is a sum in fp32.)
OHIP_HD int most_cut_pieces(const Way& w) { return w.target + w.target / 8; }
OHIP_HD int most_slots(const Way& w) { return 2 * most_cut_pieces(w); }

// Sequences of up to kFewRows rows go in tiles of 16, others in tiles of 128 (16-bit types; fp32: all in tiles of 16).
// Two tiles of 16 would read the keys twice.  bf16, 8 heads of 128, 24 and 32 rows each, two tiles of 16 against one of 128:
// 64 sequences of 8192 places 231 and 204 us against 203 and 176, of 512 places 44 and 45 against 30 and 32; 4 sequences of
// 8192 places 37 and 28 against 28 and 24, of 512 places 14 and 14.5 against 16 and 16.
// Stretches of at least 256 places: at 512 the last of these take 22 us, at 128 14.5, and the others no less.
// 512 pieces of 128 rows are two workgroups a CU, 1024 of 16 rows four.  256, 384, 512, 640 and 1024 pieces: a chunk of 509 tokens, 4 x 4
// heads of 96, behind 6000 places beside 16 single tokens 53, 50, 48, 54 and 52 us; four chunks of up to 300, 2 x 8 heads of 64, behind
// 8000 40, 33, 28, 32 and 33; 700 tokens, 8 x 4 heads of 128, behind 12000 beside 8 single ones 314, 251, 261, 237 and 241.
constexpr int kFewRows = 16;
constexpr Way kFew16 = {16, 32, 8, 1024}, kFew32 = {16, 16, 16, 1024}, kMany = {128, 64, 4, 512}, kManyWide = {128, 32, 8, 512};   // (wide: heads above 128)
OHIP_HD bool is_many(const SeqSpan& s, const int group) { return (long long)s.n * group > kFewRows; }
OHIP_HD long long most_few_units(const int tokens, const int seqs, const int heads, const int group, const bool all) {
  const long long each = at_most(seqs, tokens);
  return heads * (all ? each + (long long)tokens * group / 16 : each * (kFewRows / 16));
}
OHIP_HD long long most_many_units(const int tokens, const int seqs, const int heads, const int group) {
  const long long rows = (long long)tokens * group, each = at_most(seqs, tokens), with_many = rows / (kFewRows + 1);
  return heads * ((each < with_many ? each : with_many) + rows / 128);
}
// Both ways of 16-bit types together: a sequence has one tile more than whole ones of 128 rows at most.
OHIP_HD long long most_units(const int tokens, const int seqs, const int heads, const int group) {
  static_assert(kFewRows == 16, "a sequence of few rows is one tile");
  return heads * (at_most(seqs, tokens) + (long long)tokens * group / 128);
}

}  // namespace ohip
#endif
