"""How a call of the attention over a paged cache is cut into pieces, and which keys a piece reads: kernels/attention_pieces.h
run on the host over small sizes, odd lengths, and lengths and page numbers that make no sense."""
from test_row_ranges_cpu import run_on_host

KEYS = r"""
#include "attention_pieces.h"
#include <cstdio>
#include <initializer_list>
using namespace ohip;
int main() {
  const int odd[] = {-2147483647 - 1, -2147483647, -9, -1, 0, 1, 8, 9, 2147483646, 2147483647};
  for (int start : odd)
    for (int next : odd)
      for (int cached : odd)
        for (int tokens : {1, 8, (1 << 30) - 1})
          for (int reach : {1, 8, 1 << 30}) {
            const SeqSpan s = seq_span(start, next, cached, tokens, reach);
            if (s.first < 0 || s.n < 0 || s.first > tokens || s.n > tokens - s.first || s.cached < 0 || s.len < s.cached || s.len > reach) { printf("span %d %d %d %d %d\n", start, next, cached, tokens, reach); return 1; }
          }
  for (int tokens = 1; tokens <= 9; ++tokens)
    for (int start = -2; start <= 10; ++start)
      for (int next = -2; next <= 11; ++next)
        for (int cached = -1; cached <= 12; ++cached)
          for (int reach = 1; reach <= 11; reach += 2) {
            const SeqSpan s = seq_span(start, next, cached, tokens, reach);
            if (s.first < 0 || s.n < 0 || s.first + s.n > tokens || s.cached < 0 || s.len < s.cached || s.len > reach) { printf("span %d %d %d %d %d\n", start, next, cached, tokens, reach); return 1; }
            if (s.n == 0) continue;
            for (int group = 1; group <= 3; ++group)
              for (int window = 0; window <= 7; ++window)
                for (int most = 2; most <= 8; most += 3) {
                  const int tiles = row_tiles(s, Way{most, 4, 1, 1}, group);
                  if (tiles * most < s.n * group || (tiles - 1) * most >= s.n * group) { printf("tiles\n"); return 1; }
                  for (int tile = 0; tile < tiles; ++tile) {
                    const KeyRange k = keys_of_rows(s, tile * most, most, group, window);
                    int lo = 1 << 30, hi = 0;      // what the rows see, one by one
                    for (int r = tile * most; r < tile * most + most && r < s.n * group; ++r)
                      for (int place = 0; place < s.len; ++place) {
                        const int p = s.cached + r / group;
                        if (place > p || (window && place <= p - window)) continue;
                        if (place < lo) lo = place;
                        if (place + 1 > hi) hi = place + 1;
                      }
                    if (k.lo < 0 || k.hi > s.len || k.lo > k.hi || (hi > 0 && (k.lo > lo || k.hi < hi))) { printf("keys %d %d for %d %d\n", k.lo, k.hi, lo, hi); return 1; }
                    for (int kt = 2; kt <= 4; ++kt) {
                      const int of_tile = (k.hi + kt - 1) / kt - k.lo / kt;
                      if (of_tile > most_key_tiles(s, most, group, window, kt)) { printf("key tiles\n"); return 1; }
                    }
                  }
                }
          }
  for (int pages = 1; pages < 5; ++pages)
    for (int page = 1; page < 5; ++page)
      for (int index = -3; index < 8; ++index)
        for (int in = 0; in < page; ++in) {
          const int row = cache_row(index, in, page, pages);
          if (row >= pages * page || row < -1 || (row < 0) != (index < 0 || index >= pages)) { printf("row\n"); return 1; }
        }
  if (cache_row(2147483647, 0, 1, 2147483647) != -1 || cache_row(2147483646, 0, 1, 2147483647) != 2147483646) return 1;
  return 0;
}
"""

PIECES = r"""
#include "attention_pieces.h"
#include <cstdio>
#include <cstdlib>
using namespace ohip;
int main() {
  srand(1);
  for (int round = 0; round < 20000; ++round) {
    const int seqs = 1 + rand() % 40, heads = 1 + rand() % 8, group = 1 + rand() % 16, reach = 1 + rand() % 40000, window = rand() % 3 ? 0 : 1 + rand() % 5000;
    int starts[42] = {0};
    const int each = rand() % 3 == 0 ? 1 + rand() % 300 : 1;
    for (int b = 0; b < seqs; ++b) starts[b + 1] = starts[b] + rand() % (each + 1);
    const int tokens = starts[seqs] > 0 ? starts[seqs] : 1;
    const Way ways[] = {kFew16, kFew32, kMany, kManyWide};
    SeqSpan spans[42];
    for (int b = 0; b < seqs; ++b) spans[b] = seq_span(starts[b], starts[b + 1], rand() % (reach + 1), tokens, reach);
    long long both = 0;
    for (int b = 0; b < seqs; ++b) both += (long long)row_tiles(spans[b], is_many(spans[b], group) ? kMany : kFew16, group) * heads;
    if (both > most_units(tokens, seqs, heads, group)) { printf("%lld units of both ways\n", both); return 1; }
    for (int k = 0; k < 4; ++k) {
      const Way w = ways[k];
      auto mine = [&](int b) { return k == 1 || is_many(spans[b], group) == (k >= 2); };   // (fp32: all sequences one way)
      float work = 0.f;
      for (int b = 0; b < seqs; ++b) work += mine(b) ? work_of(spans[b], w, group, heads, window) : 0.f;
      const int stretch = stretch_of(work, w);
      long long pieces = 0, slots = 0, units = 0;
      for (int b = 0; b < seqs; ++b) {
        if (!mine(b)) continue;
        const int cuts = stretches(key_tiles(spans[b], w, group, window), stretch);
        const long long own = (long long)row_tiles(spans[b], w, group) * heads * cuts;
        pieces += own;
        units += (long long)row_tiles(spans[b], w, group) * heads;
        if (cuts > 1) slots += own;
        if ((cuts > 1) && stretch < w.least) { printf("stretch\n"); return 1; }
      }
      const long long most = k >= 2 ? most_many_units(tokens, seqs, heads, group) : most_few_units(tokens, seqs, heads, group, k == 1);
      if (units > most || pieces > most + most_cut_pieces(w) || slots > most_slots(w)) {
        printf("way %d: %lld units of %lld, %lld pieces, %lld slots\n", k, units, most, pieces, slots);
        return 1;
      }
    }
  }
  return 0;
}
"""

FAR = r"""
#include "attention_pieces.h"
#include <cstdio>
#include <initializer_list>
using namespace ohip;
int main() {
  // the longest sequences that can be: lengths that make no sense are clamped to them
  for (int tokens : {1, 1 << 10, 1 << 20, (1 << 25) - 1})
    for (int heads : {1, 8, 32})
      for (int seqs : {1, 3, 1000}) {
        const int reach = 1 << 30;
        const Way ways[] = {kFew16, kFew32, kMany, kManyWide};
        for (int k = 0; k < 4; ++k) {
          float work = 0.f;
          const SeqSpan s = seq_span(0, 2147483647, 2147483647, tokens, reach);     // (every sequence has all tokens)
          for (int b = 0; b < seqs; ++b) work += work_of(s, ways[k], 1, heads, 0);
          const int stretch = stretch_of(work, ways[k]), tiles = key_tiles(s, ways[k], 1, 0), cuts = stretches(tiles, stretch);
          const long long own = (long long)row_tiles(s, ways[k], 1) * heads, pieces = own * cuts * seqs;
          if (stretch < ways[k].least || cuts < 1 || (cuts > 1 && pieces > most_slots(ways[k])) || pieces > own * seqs + most_cut_pieces(ways[k])) {
            printf("way %d, %d x %d tokens, %d heads: stretch %d of %d tiles, %lld pieces\n", k, seqs, tokens, heads, stretch, tiles, pieces);
            return 1;
          }
        }
      }
  return 0;
}
"""

def test_what_rows_see(tmp_path):
    run_on_host(tmp_path, KEYS)


def test_pieces_and_slots_stay_within_their_bounds(tmp_path):
    run_on_host(tmp_path, PIECES)


def test_lengths_without_sense_cut_nothing_short(tmp_path):
    run_on_host(tmp_path, FAR)
