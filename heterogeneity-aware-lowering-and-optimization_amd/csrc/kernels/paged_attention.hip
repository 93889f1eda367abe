// Attention of new tokens over keys and values in the pages of a cache (formula and contract: odla_hip_PagedAttention).
//
// Rows are the queries that share a head of keys: row r of a sequence is query r % group of its token r / group, so that
// a tile of rows reads each key once for all of them.  Softmax in one pass: per row the running maximum m and
// the sum l of exp(s - m), and o = sum exp(s - m) v, rescaled when m grows.  m follows the true maximum only when that is 2^8
// times larger: the sums hold that, and o is seldom rescaled.  fp16 weights are 2^7 times as large (2^15 at most), l and o with them:
// what many distant keys add up to is not lost to the type's least number, which is 2^-32 of a row's largest weight then.
//
// Lengths are on the device, so the launch cannot be cut to them: every workgroup finds its piece - a tile of rows, a head
// and a stretch of the keys - from the lengths itself (attention_pieces.h).  Long sequences with few rows are cut
// into stretches, so that there are about a thousand pieces; a stretch leaves m, l and o in fp32, and
// a last launch joins them in the order of the stretches.
//
// Few rows are bound by reading the cache: 48 sequences of up to 16384 places, 8 heads of 128 for 8 queries each, bf16, 0.9 GB, 175 us
// and 6 for the join, 5.2 TB/s (a plain read of so much reaches 6.1 - 6.8); one of 4096 places 9.4 and 5.6 us, latency.  Many
// rows are bound by the matrix cores and by what is done between their products: a prompt of 8192 tokens, 32 heads of 128, bf16,
// 0.55 TFLOP, 0.66 ms, 840 TFLOP/s where a library product of 8192^3 reaches 1137.
#include "block_common.h"
#include "attention_pieces.h"

#include <algorithm>

namespace ohip {
namespace {

constexpr float kLog2e = 1.44269504f;
template <typename T> constexpr float kLift = std::is_same<T, f16_t>::value ? 7.f : 0.f;

struct Args : PagedAttentionParams {
  unsigned page_magic; int page_shift;
  int reach;          // places of a row of the page table
  int few_slots, many_slots;
  int writers, written;      // the first workgroups write the new tokens to their places, so many each
};

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_int(const int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
// Sum over the lanes up to one's own.
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_int<0x111, 0xf>(v);
  v += dpp_int<0x112, 0xf>(v);
  v += dpp_int<0x114, 0xf>(v);
  v += dpp_int<0x118, 0xf>(v);
  v += dpp_int<0x142, 0xa>(v);
  v += dpp_int<0x143, 0xc>(v);
  return v;
}
// op over the lanes l, l ^ 16, l ^ 32, l ^ 48: those that hold keys of one row.
template <typename Op>
__device__ __forceinline__ float over_row(float v, Op op) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uintx2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(a.x), __uint_as_float(a.y));
  const uintx2 b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(b.x), __uint_as_float(b.y));
#endif
  return v;
}

__device__ __forceinline__ SeqSpan span_of(const Args& a, const int b) {
  if (b >= a.seqs) return {0, 0, 0, 0};
  const int each = a.starts == nullptr ? a.tokens / a.seqs : 0;
  return seq_span(a.starts != nullptr ? a.starts[b] : b * each, a.starts != nullptr ? a.starts[b + 1] : (b + 1) * each, a.cached[b], a.tokens, a.reach);
}
// Spans of sequences b .. b + E - 1; all are requested before the first is looked at.
template <int E>
__device__ __forceinline__ void spans_of(const Args& a, const int b, SeqSpan (&s)[E]) {
  const int each = a.starts == nullptr ? a.tokens / a.seqs : 0;
  int start[E], next[E], cached[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = at_most(b + e, a.seqs - 1);
    start[e] = a.starts != nullptr ? a.starts[i] : i * each;
    next[e] = a.starts != nullptr ? a.starts[i + 1] : (i + 1) * each;
    cached[e] = a.cached[i];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s[e] = b + e < a.seqs ? seq_span(start[e], next[e], cached[e], a.tokens, a.reach) : SeqSpan{0, 0, 0, 0};
}
__device__ __forceinline__ SeqSpan span_from_lane(const SeqSpan& s, const int lane) {
  return {__builtin_amdgcn_readlane(s.first, lane), __builtin_amdgcn_readlane(s.n, lane), __builtin_amdgcn_readlane(s.cached, lane), __builtin_amdgcn_readlane(s.len, lane)};
}

// The two ways of a type (fp32 has one).
template <typename T, bool WIDE> struct Ways {
  static constexpr bool kTwo = sizeof(T) == 2;
  static constexpr Way few = kTwo ? kFew16 : kFew32, many = WIDE ? kManyWide : kMany;
};

// A sequence, how its tiles are cut, and where its pieces and the slots of its parts begin.
struct Found { int seq, cuts, stretch, tiles, piece0, slot0; bool many; SeqSpan span; };
constexpr Found kNowhere = {-1, 1, 0, 0, 0, 0, false, {0, 0, 0, 0}};
// The sequence with piece `key` (or, BY_TOKEN, with the new token `key`), by all lanes of a wavefront together; seq < 0: none.
// Pieces of the sequences with many rows, which take longest, come first.  E neighbouring sequences a lane.
template <typename T, bool WIDE, bool BY_TOKEN, int E>
__device__ __forceinline__ Found find_by(const Args& a, const int key) {
  using W = Ways<T, WIDE>;
  const int lane = threadIdx.x & 63;
  SeqSpan first[E], t[E];
  spans_of<E>(a, lane * E, first);      // (kept)
  float few = 0.f, many = 0.f;
#pragma unroll 1
  for (int b0 = 0; b0 < a.seqs; b0 += 64 * E) {
    if (b0 != 0) spans_of<E>(a, b0 + lane * E, t);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (b0 == 0) t[e] = first[e];
      if (W::kTwo && is_many(t[e], a.group)) many += work_of(t[e], W::many, a.group, a.kv_heads, a.window);
      else few += work_of(t[e], W::few, a.group, a.kv_heads, a.window);
    }
  }
  const float work[2] = {wave_sum(few), W::kTwo ? wave_sum(many) : 0.f};
  int piece0 = 0;
#pragma unroll
  for (int way = W::kTwo ? 1 : 0; way >= 0; --way) {
    if (work[way] == 0.f) continue;      // (every piece has a tile of keys at least)
    const Way w = way ? W::many : W::few;
    const int stretch = stretch_of(work[way], w);
    int slot0 = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < a.seqs; b0 += 64 * E) {
      if (b0 != 0) spans_of<E>(a, b0 + lane * E, t);
      bool mine[E];
      int cuts[E], pieces[E], slots[E], all_pieces = 0, all_slots = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (b0 == 0) t[e] = first[e];
        mine[e] = !W::kTwo || is_many(t[e], a.group) == (way == 1);
        cuts[e] = stretches(key_tiles(t[e], w, a.group, a.window), stretch);
        pieces[e] = mine[e] ? row_tiles(t[e], w, a.group) * a.kv_heads * cuts[e] : 0;
        slots[e] = cuts[e] > 1 ? pieces[e] : 0;
        all_pieces += pieces[e];
        all_slots += slots[e];
      }
      const int piece_end = piece0 + wave_scan(all_pieces), slot_end = slot0 + wave_scan(all_slots);
      // this lane's sequence with the key, if it has one
      int piece = piece_end - all_pieces, slot = slot_end - all_slots, which = -1, piece_of = 0, slot_of = 0, cuts_of = 0;
      SeqSpan span = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const bool is = which < 0 && (BY_TOKEN ? mine[e] && key >= t[e].first && key < t[e].first + t[e].n : key < piece + pieces[e]);
        which = is ? e : which;
        piece_of = is ? piece : piece_of;
        slot_of = is ? slot : slot_of;
        cuts_of = is ? cuts[e] : cuts_of;
        span = {is ? t[e].first : span.first, is ? t[e].n : span.n, is ? t[e].cached : span.cached, is ? t[e].len : span.len};
        piece += pieces[e];
        slot += slots[e];
      }
      const unsigned long long here = __ballot(which >= 0);
      if (here != 0) {
        const int at = __builtin_ctzll(here);
        Found f;
        f.seq = b0 + at * E + __builtin_amdgcn_readlane(which, at);
        f.many = way == 1;
        f.span = span_from_lane(span, at);
        f.cuts = __builtin_amdgcn_readlane(cuts_of, at);
        f.stretch = stretch;
        f.tiles = row_tiles(f.span, w, a.group);
        f.piece0 = __builtin_amdgcn_readlane(piece_of, at);
        f.slot0 = __builtin_amdgcn_readlane(slot_of, at);
        return f;
      }
      piece0 = __builtin_amdgcn_readlane(piece_end, 63);
      slot0 = __builtin_amdgcn_readlane(slot_end, 63);
    }
  }
  return kNowhere;
}
// (1024 sequences of up to 512 places, 8 heads: 326 us with two a lane, 343 with four, 460 with eight)
template <typename T, bool WIDE, bool BY_TOKEN>
__device__ __forceinline__ Found find(const Args& a, const int key) {
  return a.seqs <= 64 ? find_by<T, WIDE, BY_TOKEN, 1>(a, key) : find_by<T, WIDE, BY_TOKEN, 2>(a, key);
}
// Pieces of a sequence: heads side by side (their keys are neighbours in memory), then stretches, then tiles of rows from
// the last one on, which sees the most keys.  Neighbouring workgroups are on different XCDs, and a head's keys lie in few
// channels of an XCD's L2 (every heads * head size elements): from one stretch or tile to the next the heads move on by
// a place or two, so that each XCD has all of them.
struct Piece { int head, cut, tile, slot; };
__device__ __forceinline__ Piece piece_at(const Found& f, const int heads, const int in_seq) {
  const int rest = in_seq / heads, head = (int)((unsigned)(in_seq + f.seq + rest + (rest >> 1) + (rest >> 2) + (rest >> 3)) % (unsigned)heads);
  return {head, rest % f.cuts, f.tiles - 1 - rest / f.cuts, f.slot0 + rest * heads + head};
}
__device__ __forceinline__ int slot_of(const Found& f, const int heads, const int tile, const int head, const int cut) {
  return f.slot0 + ((f.tiles - 1 - tile) * f.cuts + cut) * heads + head;
}

// Work space: m and l of every row of every slot, then their o; slots of the one way, then those of the other.
struct Parts {
  float* base;
  int slots, rows, d;
  __host__ __device__ int64_t floats() const { return (int64_t)slots * rows * (d + 2); }
  __device__ float* sums(const int slot, const int row) const { return base + ((int64_t)slot * rows + row) * 2; }
  __device__ float* values(const int slot, const int row) const { return base + (int64_t)slots * rows * 2 + ((int64_t)slot * rows + row) * d; }
};
template <typename T, bool WIDE>
__host__ __device__ __forceinline__ Parts parts_of(const Args& a, const bool many) {
  using W = Ways<T, WIDE>;
  Parts p = {reinterpret_cast<float*>(a.work), a.few_slots, W::few.rows, a.d};
  if (many) p = {p.base + p.floats(), a.many_slots, W::many.rows, a.d};
  return p;
}
// Where a row's result goes.
template <typename T>
__device__ __forceinline__ T* result_row(const Args& a, const SeqSpan& s, const int head, const int row) {
  const int token = row / a.group;
  return reinterpret_cast<T*>(a.y) + ((int64_t)(s.first + token) * a.kv_heads * a.group + (int64_t)head * a.group + (row - token * a.group)) * a.d;
}

// ------------------------------------------------------------ the new tokens --
// The first workgroups of the launch write the new keys and values to their places; the others take them from where they
// are written from, so that nobody waits.  A wavefront writes one token after the other.
__device__ __forceinline__ void write_tokens(const Args& a, const int bytes) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int end = min((int)(blockIdx.x + 1) * a.written, a.tokens);
  int seq = -1;
  SeqSpan s = {0, 0, 0, 0};
#pragma unroll 1
  for (int token = blockIdx.x * a.written + wave; token < end; token += 4) {
    if (seq < 0 || token < s.first || token >= s.first + s.n) {
      // the last sequence that begins at the token or in front of it: among 64 ranges of all, then among those of one
      seq = -1;
      int lo = 0, some = a.seqs;
#pragma unroll 1
      while (some > 64) {
        const int step = (some + 63) / 64, at = lane * step;
        const bool before = at < some && (a.starts != nullptr ? a.starts[lo + at] : (lo + at) * (a.tokens / a.seqs)) <= token;
        const int skip = at_least(__builtin_popcountll(__ballot(before)) - 1, 0) * step;      // (less than `some`, whatever the starts are)
        lo += skip;
        some = at_most(step, some - skip);
      }
      const SeqSpan m = span_of(a, lo + lane);
      const unsigned long long here = __ballot(lane < some && token >= m.first && token < m.first + m.n);
      if (here != 0) {
        seq = lo + __builtin_ctzll(here);
        s = span_from_lane(m, __builtin_ctzll(here));
      }
      if (seq < 0) continue;
    }
    const int place = s.cached + (token - s.first);
    if (place >= s.len) continue;
    const int index = fast_div(place, a.page_magic, a.page_shift);
    const int row = cache_row(a.table[(int64_t)seq * a.table_width + index], place - index * a.page, a.page, a.pages);
    if (row < 0) continue;
    const uintx4* k = reinterpret_cast<const uintx4*>(reinterpret_cast<const char*>(a.k) + (int64_t)token * bytes);
    const uintx4* v = reinterpret_cast<const uintx4*>(reinterpret_cast<const char*>(a.v) + (int64_t)token * bytes);
    uintx4* kc = reinterpret_cast<uintx4*>(reinterpret_cast<char*>(a.k_cache) + (int64_t)row * bytes);
    uintx4* vc = reinterpret_cast<uintx4*>(reinterpret_cast<char*>(a.v_cache) + (int64_t)row * bytes);
    for (int i = lane; i < bytes / 16; i += 64) {
      const uintx4 x = k[i], y = v[i];
      kc[i] = x;
      vc[i] = y;
    }
  }
}
// Where the keys and values of one head of a sequence lie: in the caches up to the new tokens, which are read where they come from.
struct Source {
  const char *k_cache, *v_cache, *k_new, *v_new;      // (new: as if place 0 lay in front of the first new token)
  int64_t row_bytes;
  int fresh, end;      // the first new place, and the last one that is read
  __device__ __forceinline__ const char* at(const char* cache, const char* fresh_ones, const int place, const int row) const {
    const bool is = place >= fresh && place <= end;      // (row -1: any row of the cache)
    return (is ? fresh_ones : cache) + (int64_t)(is ? place : max(row, 0)) * row_bytes;
  }
  __device__ __forceinline__ const char* key(const int place, const int row) const { return at(k_cache, k_new, place, row); }
  __device__ __forceinline__ const char* value(const int place, const int row) const { return at(v_cache, v_new, place, row); }
};
template <typename T>
__device__ __forceinline__ Source source_of(const Args& a, const SeqSpan& s, const int head, const int hi) {
  Source o;
  o.row_bytes = (int64_t)a.kv_heads * a.d * (int)sizeof(T);
  const int64_t of_head = (int64_t)head * a.d * (int)sizeof(T), first = of_head + (int64_t)(s.first - s.cached) * o.row_bytes;
  o.k_cache = reinterpret_cast<const char*>(a.k_cache) + of_head;
  o.v_cache = reinterpret_cast<const char*>(a.v_cache) + of_head;
  o.k_new = reinterpret_cast<const char*>(a.k) + first;
  o.v_new = reinterpret_cast<const char*>(a.v) + first;
  o.end = at_least(hi, 1) - 1;       // (lookups stay in front of it)
  o.fresh = a.k != nullptr ? s.cached : INT32_MAX;
  return o;
}

// ------------------------------------------------------------------ few rows --
// Tiles of 16 rows; the four wavefronts take every fourth tile of KT keys each and meet in LDS at the end.  Nothing
// passes through LDS on the way: keys come from memory as operand fragments (lane l: key l % 16, 16 bytes of it), and the
// values as VE neighbouring elements of a key a lane (l % 16: which), which are operand fragments once the
// elements of eight keys have changed places inside the lane.  Which key a place of the product's inner axis has
// is free as long as weights and values agree: a lane's weights stay where the scores' product left them.
//   scores  C[key][row]: lane l has row l % 16, keys 4 (l / 16) + i of each block of 16
//   o       C[d][row]:   lane l has row l % 16, d = (4 (l / 16) + i) VE + e
template <typename T> struct Few {
  static constexpr int BLOCKS = sizeof(T) == 4 ? 1 : 2, KEYS = 4 * BLOCKS, KT = 16 * BLOCKS;   // blocks and keys a lane of a tile
};
template <typename T, int DP> struct FewShape {
  static constexpr int VE = DP / 16;                        // elements of a value that a lane has
  static constexpr int VW = VE * sizeof(T) / 4;             // in dwords
  static constexpr int KC = DP * sizeof(T) / 64;            // 16-byte vectors of a key that a lane has
};

// 16 bytes (or 8) of a row from element `at` on; behind its d elements any of it.  No branch: a load that is not taken by all
// lanes would be waited for where the lanes meet again, and everything requested before it.
template <typename T, int W, bool WHOLE>
__device__ __forceinline__ void load_part(const T* row, const int at, const int d, unsigned* to) {
  static_assert(W == 2 || W == 4, "8 or 16 bytes");
  const T* from = row + (WHOLE || at < d ? at : 0);
  if constexpr (W == 4) {
    const uintx4 v = *reinterpret_cast<const uintx4*>(from);
    to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
  } else {
    const uintx2 v = *reinterpret_cast<const uintx2*>(from);
    to[0] = v.x; to[1] = v.y;
  }
}

// A row's weight for a key that it does not see is zero, and zero times an infinite or missing value is none.  Where a
// tile has such weights, such values leave it; whoever found one looks at all values of its piece once more in the end and puts
// those into the sums of the rows that see them (what else a row's sum holds, and the weight, make no difference then).  So does
// whoever ends with a sum that is no number: a weight may be too small for its type, and so may the factor that makes up for a
// larger maximum, and a row gets what it would get from a weight that is not zero, wherever the tiles' edges lie.
template <typename T> constexpr unsigned kExponent = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, f16_t>::value ? 0x7c00u : 0x7f80u;
// The largest exponents of a dword's elements so far, and whether one says infinite or missing.
template <typename T> __device__ __forceinline__ unsigned with_exponents(const unsigned most, const unsigned w) {
  if constexpr (sizeof(T) == 4) {
    return max(most, w & kExponent<T>);
  } else {
    typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(ushortx2, most), __builtin_bit_cast(ushortx2, w & (kExponent<T> << 16 | kExponent<T>))));
  }
}
template <typename T> __device__ __forceinline__ bool not_finite(const unsigned most) {
  if constexpr (sizeof(T) == 4) return most == kExponent<T>;
  else return (most & 0xffffu) == kExponent<T> || most >> 16 == kExponent<T>;
}
template <typename T> __device__ __forceinline__ unsigned finite_part(const unsigned w) {
  constexpr unsigned m = kExponent<T>;
  if constexpr (sizeof(T) == 4) return (w & m) == m ? 0u : w;
  else return ((w & m) == m ? 0u : w & 0xffffu) | ((w >> 16 & m) == m ? 0u : w & 0xffff0000u);
}
// column(i): this lane's columns of its row, N times four; rows_of, row_at: as in the kernels, KT keys a tile; put(i, j, x,
// clear): the sum of column(i) + j is cleared, then has x added.
template <typename T, int KT, int N, typename RowsOf, typename RowAt, typename Column, typename Put>
__device__ __forceinline__ void put_odd_values(const Args& a, const Source& src, const int t_begin, const int t_end, const int step, const int last, RowsOf rows_of,
                                            RowAt row_at, Column column, Put put) {
#pragma unroll 1
  for (int clear = 1; clear >= 0; --clear) {
#pragma unroll 1
    for (int t = t_begin; t < t_end; t += step) {
      const auto rows_ = rows_of(t);
#pragma unroll 1
      for (int k = 0; k < KT; ++k) {
        const int row = row_at(rows_, t, k), place = t * KT + k;
        if (row < 0 || place > last || (a.window != 0 && place <= last - a.window)) continue;
        const T* v = reinterpret_cast<const T*>(src.value(place, row));
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = Store<T>::ld(v + (column(i) < a.d ? column(i) + j : 0));      // (behind the head: columns that are not stored)
            if (!__builtin_isfinite(x)) put(i, j, x, clear != 0);
          }
          asm volatile("" ::: "memory");      // (four at a time: this path is seldom taken and shall take no registers from the others)
        }
      }
    }
  }
}
// Whether a row's sums have one that is no number, although its weights' sum is (0 times it is 0 for numbers alone).
__device__ __forceinline__ bool lost_its_number(const float zeros, const float weights) { return zeros != zeros && weights == weights; }
// What a part's sums are joined with: its factor, but not zero (the exponential gives zero below 2^-126 in any case), so that what is no
// number in them remains.
constexpr float kLeastFactor = 0x1p-126f;

template <typename T, int DP> constexpr int kFewLds = (4 * 16 * (DP + 4) + 2 * 4 * 16) * (int)sizeof(float);
template <typename T, int DP, bool WHOLE, bool TWO>
__device__ __forceinline__ void attend_few(const Args& a, const Found& f, const Piece& piece, unsigned char* smem) {
  using F = Few<T>;
  using S = FewShape<T, DP>;
  constexpr bool WIDE = DP > 128;
  constexpr int R = 16, KEYS = F::KEYS, KT = F::KT, VE = S::VE, VW = S::VW, KC = S::KC, PER = 16 / (int)sizeof(T);
  static_assert(R == Ways<T, WIDE>::few.rows && KT == Ways<T, WIDE>::few.keys, "as the pieces are cut");
  auto part = reinterpret_cast<float (*)[16][DP + 4]>(smem);
  auto part_m = reinterpret_cast<float (*)[16]>(smem + sizeof(float) * 4 * 16 * (DP + 4));
  auto part_l = part_m + 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int head = piece.head, r0 = piece.tile * R, rows = min(R, f.span.n * a.group - r0);
  const KeyRange seen = keys_of_rows(f.span, r0, R, a.group, a.window);
  const int t_begin = seen.lo / KT + piece.cut * f.stretch, t_end = min((seen.hi + KT - 1) / KT, f.cuts > 1 ? t_begin + f.stretch : INT32_MAX);
  const Source src = source_of<T>(a, f.span, head, seen.hi);
  const int32_t* table = a.table + (int64_t)f.seq * a.table_width;

  // queries: this lane's row, and the last place that it sees
  uintx4 q[KC];
  const int r = min(r0 + l16, r0 + rows - 1), token = r / a.group, last = f.span.cached + token;
  {
    const T* row = reinterpret_cast<const T*>(a.q) + ((int64_t)(f.span.first + token) * a.kv_heads * a.group + (int64_t)head * a.group + (r - token * a.group)) * a.d;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      unsigned w[4];
      load_part<T, 4, WHOLE>(row, (4 * c + g) * PER, a.d, w);
      q[c] = WHOLE || (4 * c + g) * PER < a.d ? uintx4{w[0], w[1], w[2], w[3]} : uintx4{0u, 0u, 0u, 0u};
    }
  }
  // Where the keys of a tile lie.  TWO: in two pages at most, whose numbers come by scalar loads; otherwise lane l looks up key
  // l % KT.  A number is looked at one tile after it was requested: vector loads return in order, and whoever waits for one
  // waits for all keys and values requested before it.
  struct Where { int first, second, edge; };      // rows of place 0 of either page, if it went on that way, and where the second begins
  constexpr int kNone = INT32_MIN;
  auto look_up = [&](const int t) __attribute__((always_inline)) -> Where {
    if constexpr (TWO) {
      const int index = fast_div(at_most(t * KT, src.end), a.page_magic, a.page_shift), next = at_most(index + 1, fast_div(src.end, a.page_magic, a.page_shift));
      const auto numbers = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)table;
      return {numbers[index], numbers[next], (index + 1) * a.page};
    } else {
      return {table[fast_div(at_most(t * KT + (lane & (KT - 1)), src.end), a.page_magic, a.page_shift)], 0, 0};
    }
  };
  auto found = [&](const Where& w, const int t) __attribute__((always_inline)) -> Where {
    if constexpr (TWO) {
      const int p = t < t_end ? cache_row(w.first, 0, a.page, a.pages) : -1, q = t < t_end ? cache_row(w.second, 0, a.page, a.pages) : -1;
      return {p < 0 ? kNone : p - (w.edge - a.page), q < 0 ? kNone : q - w.edge, w.edge};
    } else {
      const int place = t * KT + (lane & (KT - 1));
      const int row = cache_row(w.first, place - fast_div(place, a.page_magic, a.page_shift) * a.page, a.page, a.pages);
      return {t < t_end && place < seen.hi ? row : -1, 0, 0};
    }
  };
  auto row_at = [&](const Where& w, const int t, const int key) __attribute__((always_inline)) -> int {      // -1: not there
    if constexpr (TWO) {
      const int place = t * KT + key, base = place < w.edge ? w.first : w.second;
      return place < seen.hi && base != kNone ? base + place : -1;
    } else {
      return __shfl(w.first, key);
    }
  };
  auto rows_of = [&](const int t) { return found(look_up(t), t); };
  auto key_of_slot = [&](const int j) { return (j >> 2) * 16 + g * 4 + (j & 3); };
  uintx4 kf[F::BLOCKS][KC];
  auto load_keys = [&](const Where& rows_, const int t) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < F::BLOCKS; ++b) {
      const T* row = reinterpret_cast<const T*>(src.key(t * KT + 16 * b + l16, row_at(rows_, t, 16 * b + l16)));
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        unsigned w[4];
        load_part<T, 4, WHOLE>(row, (4 * c + g) * PER, a.d, w);
        kf[b][c] = uintx4{w[0], w[1], w[2], w[3]};
      }
    }
  };
  unsigned vf[KEYS][VW];
  auto load_values = [&](const Where& rows_, const int t) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      const T* row = reinterpret_cast<const T*>(src.value(t * KT + key_of_slot(j), row_at(rows_, t, key_of_slot(j))));
      constexpr int W = VW < 4 ? 2 : 4;
#pragma unroll
      for (int w = 0; w < VW / W; ++w) load_part<T, W, WHOLE>(row, l16 * VE + w * (W * 4 / (int)sizeof(T)), a.d, &vf[j][w * W]);
    }
  };

  float m = -INFINITY, l = 0.f;
  bool odd = false;
  floatx4 o[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) o[e] = floatx4{0.f, 0.f, 0.f, 0.f};
  const float to_log2 = a.scale * kLog2e;
  const int window = a.window == 0 ? 1 << 30 : a.window;      // (no place lies further back)
  const int first_last = f.span.cached + r0 / a.group, last_last = f.span.cached + (r0 + rows - 1) / a.group;
  // A wavefront's requests are one tile ahead of their use (keys behind the scores' product, values behind the other), the
  // rows that they are for one more.  All are made, also those behind the last tile (of the cache's first row): where some paths
  // have fewer requests, waits are for all of them.
  Where here = found(look_up(t_begin + wave), t_begin + wave), ahead = look_up(t_begin + wave + 4);      // (ahead: numbers as they come)
  load_keys(here, t_begin + wave);
  load_values(here, t_begin + wave);
#pragma unroll 1
  for (int t = t_begin + wave; t < t_end; t += 4) {
    const Where next = found(ahead, t + 4);
    ahead = look_up(t + 8);
    floatx4 s[F::BLOCKS];
#pragma unroll
    for (int k = 0; k < F::BLOCKS; ++k) {
      s[k] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) s[k] = mma_vec<T>(WHOLE || (4 * c + g) * PER < a.d ? kf[k][c] : uintx4{0u, 0u, 0u, 0u}, q[c], s[k]);
    }
    load_keys(next, t + 4);
    // what all rows see needs no mask
    bool there = true;
    if constexpr (TWO) there = here.first != kNone && (here.second != kNone || here.edge >= t * KT + KT);
    else there = __all(here.first >= 0);
    const bool masked = !there || t * KT + KT > min(first_last + 1, seen.hi) || t * KT <= last_last - window;
    float p[KEYS], most = -INFINITY;
#pragma unroll
    for (int j = 0; j < KEYS; ++j) p[j] = s[j >> 2][j & 3] * to_log2;
    if (masked) {
#pragma unroll
      for (int j = 0; j < KEYS; ++j) {
        const int place = t * KT + key_of_slot(j);
        const bool sees = (row_at(here, t, key_of_slot(j)) >= 0) & (place <= last) & (place > last - window);
        p[j] = sees ? p[j] : -INFINITY;
      }
    }
#pragma unroll
    for (int j = 0; j < KEYS; ++j) most = fmaxf(most, p[j]);
    most = over_row(most, [](float x, float y) { return fmaxf(x, y); });
    const bool grows = most > m + 8.f;
    if (__any(grows)) {
      const float now = grows ? most : m, shrink = grows ? __builtin_amdgcn_exp2f(m - now) : 1.f;
      m = now;
      l *= shrink;
#pragma unroll
      for (int e = 0; e < VE; ++e) o[e] *= shrink;
    }
    const float base = (m == -INFINITY ? 0.f : m) - kLift<T>;
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      p[j] = __builtin_amdgcn_exp2f(p[j] - base);
      l += p[j];
    }
    // element e of this lane's keys, as an operand
    auto column = [&](const int e, unsigned (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = sizeof(T) == 4 ? vf[j][e] : __builtin_amdgcn_perm(vf[2 * j + 1 & KEYS - 1][e / 2], vf[2 * j & KEYS - 1][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
    };
    uintx4 weights;
    if constexpr (sizeof(T) == 4) weights = uintx4{__float_as_uint(p[0]), __float_as_uint(p[1]), __float_as_uint(p[2]), __float_as_uint(p[3])};
    else weights = pack8_rne<T>(p);
    if (masked) {
      unsigned most = 0;
#pragma unroll
      for (int j = 0; j < KEYS; ++j)
#pragma unroll
        for (int w = 0; w < VW; ++w) most = with_exponents<T>(most, vf[j][w]);
      if (__any(not_finite<T>(most))) {
        odd = true;
#pragma unroll
        for (int j = 0; j < KEYS; ++j)
#pragma unroll
          for (int w = 0; w < VW; ++w) vf[j][w] = finite_part<T>(vf[j][w]);
      }
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      unsigned v[4];
      column(e, v);
      o[e] = mma_vec<T>(uintx4{v[0], v[1], v[2], v[3]}, weights, o[e]);
    }
    load_values(next, t + 4);
    here = next;
  }

  const float own_sum = over_row(l, [](float x, float y) { return x + y; });
  float zeros = 0.f;
#pragma unroll
  for (int e = 0; e < VE; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) zeros = __builtin_fmaf(o[e][i], 0.f, zeros);
  if (odd || __any(lost_its_number(zeros, own_sum)))
    put_odd_values<T, KT, VE>(a, src, t_begin + wave, t_end, 4, last, rows_of, row_at, [&](const int n) { return 4 * (g * VE + n); },
                              [&](const int n, const int j, const float x, const bool clear) {
                                const int e = (4 * n + j) % VE, i = (4 * n + j) / VE;
                                o[e][i] = clear ? 0.f : o[e][i] + x;
                              });

  // ---- the wavefronts' parts
  const int mine = threadIdx.x >> 4, column0 = (threadIdx.x & 15) * VE;
  if (g == 0) { part_m[wave][l16] = m; part_l[wave][l16] = own_sum; }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < VE; ++e) part[wave][l16][(4 * g + i) * VE + e] = o[e][i];
  __syncthreads();
  const Parts parts = parts_of<T, WIDE>(a, false);
  const bool whole = f.cuts == 1;
  if (mine >= rows || (!whole && piece.slot >= parts.slots)) return;
  float most = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) most = fmaxf(most, part_m[w][mine]);
  float factor[4], sum = 0.f;      // (of a part without keys: 0; of one whose scores are all NaN: NaN)
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    factor[w] = part_m[w][mine] == -INFINITY ? part_l[w][mine] : __builtin_amdgcn_exp2f(part_m[w][mine] - most);
    sum = __builtin_fmaf(factor[w], part_l[w][mine], sum);
  }
  T* y = result_row<T>(a, f.span, head, r0 + mine);
  float* to = parts.values(piece.slot, mine);
  const float by = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < VE; e += 4) {
    if (column0 + e >= a.d) break;
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const floatx4 x = *reinterpret_cast<const floatx4*>(&part[w][mine][column0 + e]);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(fmaxf(factor[w], kLeastFactor), x[i], v[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = by == 0.f ? 0.f : v[i] * by;
    if (whole) store4<T>(y + column0 + e, v, 4, true);
    else *reinterpret_cast<floatx4*>(to + column0 + e) = v;
  }
  if (!whole && (threadIdx.x & 15) == 0) {
    float* ml = parts.sums(piece.slot, mine);
    ml[0] = most;
    ml[1] = sum;
  }
}

// ----------------------------------------------------------------- many rows --
// Tiles of 128 rows, 32 a wavefront, and of KT keys: keys and values come straight into LDS (one of two buffers, while the other
// is used) and are read from there by all four wavefronts.  The scores' product gives C[key][row], so that a lane
// holds, for ITS row, half of the tile's keys: maximum and sum are lane operations and one exchange with lane + 32, and the weights are the
// operand of the second product as they are (C[d][row], the order of its inner axis being free).  The values'
// operand has neighbouring keys in a lane: ds_read_b64_tr_b16 reads sixteen columns of four keys that way round.
// LDS rows keep their 16-byte chunks in other places (key_slot, value_slot), so that what is read at a time lies in different banks.
template <int DP> struct Big {
  static constexpr int KT = DP > 128 ? 32 : 64, BLOCKS = KT / 32;
  static constexpr int CHUNKS = DP / 8, ROW = DP * 2;                  // 16-byte chunks and bytes of a row
  static constexpr int TILE = KT * ROW, STAGE = 2 * TILE;              // keys, then values
  static constexpr int REQUESTS = TILE / 4096, PER = 64 / CHUNKS;      // of a wavefront for each, and rows of one
  static constexpr int LDS = 2 * STAGE;
};
template <int DP> __device__ __forceinline__ int key_slot(const int row, const int chunk) { return chunk ^ (DP == 64 ? row >> 1 & 7 : row & 15); }
template <int DP> __device__ __forceinline__ int value_slot(const int row, const int chunk) { return chunk ^ (DP == 64 ? (row & 2) << 1 : (row & 3) << 2); }

template <typename T>
__device__ __forceinline__ floatx16 mma32(const uintx4 a, const uintx4 b, const floatx16 c) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (std::is_same<T, f16_t>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
#else
  (void)a; (void)b;
  return c;
#endif
}
template <typename Op>
__device__ __forceinline__ float over_halves(const float v, Op op) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uintx2 a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(a.x), __uint_as_float(a.y));
#else
  return v;
#endif
}
// Four elements of one column, of the rows that the lanes of its sixteen point to.
__device__ __forceinline__ uintx2 read_column(const unsigned char* at) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef short shortx4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) shortx4* lds_vec;
  return __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec)(at)));
#else
  (void)at;
  return uintx2{0u, 0u};
#endif
}
__device__ __forceinline__ void request16(const char* from, unsigned char* to) {
#if defined(__HIP_DEVICE_COMPILE__)
  using lds_ptr = __attribute__((address_space(3))) void*;
  __builtin_amdgcn_global_load_lds(from, (lds_ptr)to, 16, 0, 0);
#else
  (void)from; (void)to;
#endif
}

// What a wavefront keeps of its 32 rows: lane l has row l % 32.
template <int DV> struct BigRows {
  uintx4 q[DV / 16];
  floatx16 o[DV / 32];
  float m, l;          // m in units of log 2
  int last;            // the last place that the row sees
  bool odd;            // infinite or missing values have left a tile
};

// Requests a tile of keys and values into LDS; rows: lane l, the cache's row of key l % KT.
template <int DP, int DV, bool WHOLE>
__device__ __forceinline__ void request_tile(const Args& a, const Source& src, unsigned char* to, const int rows, const int place0, const int lane, const int wave) {
  using B = Big<DP>;
#pragma unroll
  for (int i = 0; i < B::REQUESTS; ++i) {
    const int row = (wave * B::REQUESTS + i) * B::PER + lane / B::CHUNKS, slot = lane % B::CHUNKS, from = __shfl(rows, row);
    // (chunks behind the end of a head's row: any of it, they meet zeros of the query or leave columns that are not stored)
    const int k_chunk = key_slot<DP>(row, slot), v_chunk = value_slot<DP>(row, slot);
    unsigned char* at = to + (wave * B::REQUESTS + i) * 1024;
    if (DV == DP || k_chunk * 8 < DV) request16(src.key(place0 + row, from) + (WHOLE || k_chunk * 8 < a.d ? k_chunk * 16 : 0), at);
    if (DV == DP || v_chunk * 8 < DV) request16(src.value(place0 + row, from) + (WHOLE || v_chunk * 8 < a.d ? v_chunk * 16 : 0), at + B::TILE);
  }
}

// One tile of keys, out of `now`; the next one's rows of the cache are requested into `next` meanwhile (the two never
// overlap: without saying so, every read of LDS would wait for the requests).  valid: bit k, key k is there.
template <typename T, int DP, int DV, bool WHOLE>
__device__ __forceinline__ void big_tile(const Args& a, unsigned char* __restrict next, unsigned char* __restrict now, const int next_rows, const bool more, const Source& src,
                                         const int place0, const unsigned long long valid, const bool masked, const float mult, const int lane, const int wave,
                                         BigRows<DV>& w) {
  using B = Big<DP>;
  constexpr int BLOCKS = B::BLOCKS;
  const int l32 = lane & 31, h = lane >> 5;
  if (more) request_tile<DP, DV, WHOLE>(a, src, next, next_rows, place0 + B::KT, lane, wave);
  floatx16 s[BLOCKS];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    const unsigned char* row = now + (b * 32 + l32) * B::ROW;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
    for (int c = 0; c < DV / 16; ++c) {
      uintx4 k = *reinterpret_cast<const uintx4*>(row + key_slot<DP>(l32, 2 * c + h) * 16);
      if (!WHOLE && (2 * c + h) * 8 >= a.d) k = uintx4{0u, 0u, 0u, 0u};
      s[b] = mma32<T>(k, w.q[c], s[b]);
    }
  }
  // element i of block b: place place0 + 32 b + 8 (i / 4) + 4 h + i % 4
  if (masked) {
    const int from_place = a.window == 0 ? -1 : w.last - a.window;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      const unsigned there = (unsigned)(valid >> (32 * b)) >> (4 * h);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int in = 8 * (i >> 2) + (i & 3), place = place0 + 32 * b + 4 * h + in;
        const bool sees = ((there >> in & 1u) != 0) & (place <= w.last) & (place > from_place);
        s[b][i] = sees ? s[b][i] : -INFINITY;
      }
    }
  }
  float most = s[0][0];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) most = fmaxf(most, s[b][i]);
  most = over_halves(most, [](float x, float y) { return fmaxf(x, y); }) * mult;
  const bool grows = most > w.m + 8.f;
  if (__any(grows)) {
    const float m = grows ? most : w.m, shrink = grows ? __builtin_amdgcn_exp2f(w.m - m) : 1.f;
    w.m = m;
    w.l *= shrink;
#pragma unroll
    for (int d = 0; d < DV / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) w.o[d][i] *= shrink;
  }
  const float base = (w.m == -INFINITY ? 0.f : w.m) - kLift<T>;
  uintx4 p[BLOCKS][2];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][8 * c + i], mult, -base));
        w.l += e[i];
      }
      p[b][c] = pack8_rne<T>(e);
    }
  unsigned char* values = now + B::TILE;
  const int from = lane & 15, part = lane >> 4 & 1;
  // the operand of columns 32 d .. and of half c of block b
  auto column = [&](const int d, const int b, const int c, unsigned (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int k = 32 * b + 16 * c + 8 * half + 4 * h + (from >> 2), chunk = 4 * d + 2 * part + (from >> 1 & 1);
      const uintx2 x = read_column(values + k * B::ROW + value_slot<DP>(k, chunk) * 16 + (from & 1) * 8);
      v[2 * half] = x.x;
      v[2 * half + 1] = x.y;
    }
  };
  if (masked) {       // (for all four wavefronts, which look at the same values)
    unsigned most = 0;
#pragma unroll 4
    for (int c = lane; c < B::TILE / 16; c += 64) {
      const uintx4 v = reinterpret_cast<const uintx4*>(values)[c];
      const bool loaded = DV == DP || value_slot<DP>(c / B::CHUNKS, c % B::CHUNKS) * 8 < DV;
#pragma unroll
      for (int j = 0; j < 4; ++j) most = with_exponents<T>(most, loaded ? v[j] : 0u);
    }
    if (__any(not_finite<T>(most))) {
      w.odd = true;
      __syncthreads();
#pragma unroll 1
      for (int c = threadIdx.x; c < B::TILE / 16; c += 256) {
        const uintx4 v = reinterpret_cast<const uintx4*>(values)[c];
        reinterpret_cast<uintx4*>(values)[c] = uintx4{finite_part<T>(v.x), finite_part<T>(v.y), finite_part<T>(v.z), finite_part<T>(v.w)};
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int d = 0; d < DV / 32; ++d) {
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        unsigned v[4];
        column(d, b, c, v);
        w.o[d] = mma32<T>(uintx4{v[0], v[1], v[2], v[3]}, p[b][c], w.o[d]);
      }
  }
}

template <typename T, int DP, int DV, bool WHOLE>
__device__ __forceinline__ void attend_many(const Args& a, const Found& f, const Piece& piece, unsigned char* smem) {
  using B = Big<DP>;
  constexpr bool WIDE = DP > 128;
  constexpr int R = 128, KT = B::KT;
  static_assert(R == Ways<T, WIDE>::many.rows && KT == Ways<T, WIDE>::many.keys, "as the pieces are cut");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, h = lane >> 5;
  const int head = piece.head, r0 = piece.tile * R, rows = min(R, f.span.n * a.group - r0);
  const KeyRange seen = keys_of_rows(f.span, r0, R, a.group, a.window);
  const int t_begin = seen.lo / KT + piece.cut * f.stretch, t_end = min((seen.hi + KT - 1) / KT, f.cuts > 1 ? t_begin + f.stretch : INT32_MAX);
  const Source src = source_of<T>(a, f.span, head, seen.hi);
  const int32_t* table = a.table + (int64_t)f.seq * a.table_width;
  // The scale's sign goes to the queries, and so does a scale of zero: maxima are taken of the products as they are.
  const float mult = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
  BigRows<DV> w;
  const int r = min(wave * 32 + l32, rows - 1), token = (r0 + r) / a.group;
  {
    const T* row = reinterpret_cast<const T*>(a.q) + ((int64_t)(f.span.first + token) * a.kv_heads * a.group + (int64_t)head * a.group + (r0 + r - token * a.group)) * a.d;
    const unsigned flip = a.scale < 0.f ? 0x80008000u : 0u, keep = a.scale == 0.f ? 0u : 0xffffffffu;
#pragma unroll
    for (int c = 0; c < DV / 16; ++c) {
      unsigned x[4];
      load_part<T, 4, WHOLE>(row, 16 * c + 8 * h, a.d, x);
#pragma unroll
      for (int j = 0; j < 4; ++j) w.q[c][j] = WHOLE || 16 * c + 8 * h < a.d ? (x[j] & keep) ^ flip : 0u;
    }
  }
  w.last = f.span.cached + token;
  w.m = -INFINITY;
  w.l = 0.f;
  w.odd = false;
#pragma unroll
  for (int d = 0; d < DV / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) w.o[d][i] = 0.f;
  // what all rows of the tile see
  const int first_last = f.span.cached + r0 / a.group, last_last = f.span.cached + (r0 + rows - 1) / a.group;
  // (a number is looked at one tile after it was requested: what is on its way into LDS would be waited for with it)
  auto look_up = [&](const int t) __attribute__((always_inline)) -> int {
    return table[fast_div(at_most(t * KT + (lane & (KT - 1)), src.end), a.page_magic, a.page_shift)];
  };
  auto found = [&](const int number, const int t) __attribute__((always_inline)) -> int {
    const int place = t * KT + (lane & (KT - 1));
    const int row = cache_row(number, place - fast_div(place, a.page_magic, a.page_shift) * a.page, a.page, a.pages);
    return t < t_end && place < seen.hi ? row : -1;
  };
  auto rows_of = [&](const int t) { return found(look_up(t), t); };
  if (t_begin < t_end) {
    int here = rows_of(t_begin), number = look_up(t_begin + 1);
    request_tile<DP, DV, WHOLE>(a, src, smem, here, t_begin * KT, lane, wave);
#pragma unroll 1
    for (int t = t_begin; t < t_end; ++t) {
      // this tile has landed, and everybody has left the other buffer (the barrier alone does not wait for requests into LDS)
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __syncthreads();
      const unsigned long long valid = __ballot(here >= 0), all = KT == 64 ? ~0ull : 0xffffffffull;
      const bool masked = (valid & all) != all || t * KT + KT - 1 > first_last || (a.window != 0 && t * KT <= last_last - a.window);
      const int next = found(number, t + 1), at = (t - t_begin) & 1;
      number = look_up(t + 2);
      big_tile<T, DP, DV, WHOLE>(a, smem + (1 - at) * B::STAGE, smem + at * B::STAGE, next, t + 1 < t_end, src, t * KT, valid & all, masked, mult, lane, wave, w);
      here = next;
    }
  }
  const float sum = over_halves(w.l, [](float x, float y) { return x + y; });
  float zeros = 0.f;
#pragma unroll
  for (int d = 0; d < DV / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) zeros = __builtin_fmaf(w.o[d][i], 0.f, zeros);
  if (w.odd || __any(lost_its_number(zeros, sum)))
    put_odd_values<T, KT, DV / 8>(a, src, t_begin, t_end, 1, w.last, rows_of, [](const int rows_, int, const int k) { return __shfl(rows_, k); }, [&](const int n) { return 8 * n + 4 * h; },
                                  [&](const int n, const int j, const float x, const bool clear) { w.o[n / 4][n % 4 * 4 + j] = clear ? 0.f : w.o[n / 4][n % 4 * 4 + j] + x; });
  if (wave * 32 + l32 >= rows) return;
  if (f.cuts == 1) {
    T* y = result_row<T>(a, f.span, head, r0 + r);
    const float by = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int d = 0; d < DV / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = 32 * d + 8 * i + 4 * h;
        floatx4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = by == 0.f ? 0.f : w.o[d][4 * i + j] * by;
        if (WHOLE || col < a.d) store4<T>(y + col, v, 4, true);
      }
  } else {
    const Parts parts = parts_of<T, WIDE>(a, true);
    if (piece.slot >= parts.slots) return;
    float* to = parts.values(piece.slot, r);
#pragma unroll
    for (int d = 0; d < DV / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = 32 * d + 8 * i + 4 * h;
        if (WHOLE || col < a.d) *reinterpret_cast<floatx4*>(to + col) = floatx4{w.o[d][4 * i], w.o[d][4 * i + 1], w.o[d][4 * i + 2], w.o[d][4 * i + 3]};
      }
    if (h == 0) {
      float* ml = parts.sums(piece.slot, r);
      ml[0] = w.m;
      ml[1] = sum;
    }
  }
}

template <typename T, int DP> constexpr int kLds = sizeof(T) == 2 && Big<DP>::LDS > kFewLds<T, DP> ? Big<DP>::LDS : kFewLds<T, DP>;
// DV: the head size rounded up to what the tiles of many rows are multiplied for.
template <typename T, int DP, int DV, bool WHOLE>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) attend_kernel(const Args a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  if ((int)blockIdx.x < a.writers) {
    write_tokens(a, a.kv_heads * a.d * (int)sizeof(T));
    return;
  }
  const int number = blockIdx.x - a.writers;
  const Found f = find<T, (DP > 128), false>(a, number);
  if (f.seq < 0) return;
  const Piece piece = piece_at(f, a.kv_heads, number - f.piece0);
  if constexpr (sizeof(T) == 2) {
    if (f.many) {
      attend_many<T, DP, DV, WHOLE>(a, f, piece, smem);
      return;
    }
  }
  constexpr int KT = Few<T>::KT;
  constexpr bool FULL = WHOLE && DV == DP;
  // (48 x 16384 places, 4 queries a head, page numbers by scalar loads and by lanes: pages of 64 176 and 180 us, of 16 178 and 182)
  if (a.page >= KT || 2 * a.page == KT) attend_few<T, DP, FULL, true>(a, f, piece, smem);      // (tiles begin at multiples of KT)
  else attend_few<T, DP, FULL, false>(a, f, piece, smem);
}

// ------------------------------------------------------------------ the parts --
// A workgroup has `each` neighbouring rows of the result, its wavefronts one after the other.  Lanes first bring m and l of
// up to 64 parts at once, then, a group of lanes a part, their rows.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) attention_join_kernel(const Args a, const int each) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q_heads = a.kv_heads * a.group;
  const int end = min((int)(blockIdx.x + 1) * each, a.tokens * q_heads);
  const int lanes = a.d <= 64 ? 16 : a.d <= 128 ? 32 : 64, sub = lane / lanes, col = lane % lanes * 4, at_once = 64 / lanes;
  const bool mine = col < a.d;
  Found f = kNowhere;
#pragma unroll 1
  for (int at = blockIdx.x * each + wave; at < end; at += 4) {
    const int token = at / q_heads, q = at - token * q_heads, head = q / a.group;
    if (f.seq < 0 || token < f.span.first || token >= f.span.first + f.span.n) f = find<T, WIDE, true>(a, token);
    T* y = reinterpret_cast<T*>(a.y) + (int64_t)at * a.d;
    if (f.seq < 0) {       // no sequence's
      if (sub == 0 && mine) store4<T>(y + col, floatx4{0.f, 0.f, 0.f, 0.f}, 4, true);
      continue;
    }
    if (f.cuts == 1) {     // nothing of this sequence is in parts
      const int skip = min(end, (f.span.first + f.span.n) * q_heads) - at;
      at += (skip - 1) / 4 * 4;
      continue;
    }
    const Parts parts = parts_of<T, WIDE>(a, f.many);
    const int row = (token - f.span.first) * a.group + (q - head * a.group), tile = row / parts.rows, r = row - tile * parts.rows;
    float most = -INFINITY, sum = 0.f;
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int c0 = 0; c0 < f.cuts; c0 += 64) {
      const int n = min(f.cuts - c0, 64), slot = slot_of(f, a.kv_heads, tile, head, c0 + min(lane, n - 1));
      float m = -INFINITY, l = 0.f;
      if (lane < n && slot < parts.slots) {
        const float* ml = parts.sums(slot, r);
        m = ml[0];
        l = ml[1];
      }
      const float now = fmaxf(most, wave_max(m)), base = now == -INFINITY ? 0.f : now;
      const float shrink = __builtin_amdgcn_exp2f(most - base);
      // (a part without keys has l = 0 and counts nothing; one whose scores are all NaN has no m, and l is NaN)
      const float factor = l == 0.f ? 0.f : m == -INFINITY ? l : __builtin_amdgcn_exp2f(m - base);
      sum = sum * shrink + wave_sum(l == 0.f ? 0.f : factor * l);
      v *= fmaxf(shrink, kLeastFactor);
      most = now;
      const float least = fmaxf(factor, kLeastFactor);
#pragma unroll 1
      for (int j0 = 0; j0 < n; j0 += 4 * at_once) {
        floatx4 x[4];
        float by[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = j0 + k * at_once + sub, part = min(j, n - 1), from = slot_of(f, a.kv_heads, tile, head, c0 + part);
          by[k] = __shfl(least, part);
          if (j >= n || from >= parts.slots) by[k] = kLeastFactor;      // (the last part once more)
          x[k] = *reinterpret_cast<const floatx4*>(parts.values(min(from, parts.slots - 1), r) + (mine ? col : 0));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(by[k], x[k][i], v[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      for (int o = lanes; o < 64; o *= 2) v[i] += __shfl_xor(v[i], o);
      v[i] = sum == 0.f ? 0.f : v[i] / sum;
    }
    if (sub == 0 && mine) store4<T>(y + col, v, 4, true);
  }
}

// The most parts that the keys of one tile are cut into.
long long most_cuts(const PagedAttentionParams& p, const Way& w) {
  const SeqSpan longest = {0, p.tokens, 0, p.table_width * p.page};
  return stretches(key_tiles(longest, w, p.group, std::min(p.window, 1 << 30)), w.least);
}
int slots_of(const PagedAttentionParams& p, const Way& w, const long long units) {
  const long long cuts = most_cuts(p, w);
  return cuts == 1 ? 0 : (int)std::min((long long)most_slots(w), units * cuts);
}
long long pieces_of(const PagedAttentionParams& p, const Way& w, const long long units) { return std::min(units + most_cut_pieces(w), units * most_cuts(p, w)); }
template <typename T, bool WIDE> struct Units {
  using W = Ways<T, WIDE>;
  long long few, many;
  explicit Units(const PagedAttentionParams& p)
      : few(most_few_units(p.tokens, p.seqs, p.kv_heads, p.group, !W::kTwo)), many(W::kTwo ? most_many_units(p.tokens, p.seqs, p.kv_heads, p.group) : 0) {}
};
template <typename T, bool WIDE>
Args args_as(const PagedAttentionParams& p) {
  using W = Ways<T, WIDE>;
  const Units<T, WIDE> units(p);
  Args a;
  static_cast<PagedAttentionParams&>(a) = p;
  div_magic(p.page, &a.page_magic, &a.page_shift);
  a.reach = p.table_width * p.page;
  a.window = std::min(p.window, 1 << 30);   // (no place lies further back)
  a.few_slots = slots_of(p, W::few, units.few);
  a.many_slots = slots_of(p, W::many, units.many);
  a.written = std::max(4, (p.tokens + 127) / 128);      // (128 workgroups write a long prompt beside the others)
  a.writers = p.k != nullptr ? (p.tokens + a.written - 1) / a.written : 0;
  return a;
}
template <typename T> Args args_of(const PagedAttentionParams& p) { return p.d > 128 ? args_as<T, true>(p) : args_as<T, false>(p); }
template <typename T> size_t space_of(const PagedAttentionParams& p) {
  const Args a = args_of<T>(p);
  const bool wide = p.d > 128;
  const Parts few = wide ? parts_of<T, true>(a, false) : parts_of<T, false>(a, false);
  const Parts many = {nullptr, a.many_slots, kMany.rows, p.d};
  return (size_t)(few.floats() + many.floats() + 4) * sizeof(float);
}

// Workgroups of the launch.
template <typename T, bool WIDE>
long long grid_of(const Args& a) {
  using W = Ways<T, WIDE>;
  const Units<T, WIDE> units(a);
  const long long cuts = pieces_of(a, W::few, units.few) - units.few + pieces_of(a, W::many, units.many) - units.many;
  const long long tiles = W::kTwo ? std::min(units.few + units.many, most_units(a.tokens, a.seqs, a.kv_heads, a.group)) : units.few;
  return a.writers + tiles + cuts;
}

template <typename T, int DP, int DV, bool WHOLE>
hipError_t attend_with(const Args& a, hipStream_t stream) {
  const long long grid = grid_of<T, (DP > 128)>(a);
  static LdsLimit limit;
  if (kLds<T, DP> > 65536) {
    const hipError_t e = limit.raise(reinterpret_cast<const void*>(&attend_kernel<T, DP, DV, WHOLE>), kLds<T, DP>);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((attend_kernel<T, DP, DV, WHOLE>), dim3((unsigned)grid), dim3(256), (kLds<T, DP>), stream, a);
  return hipGetLastError();
}
template <typename T, int DP, int DV>
hipError_t attend_wide(const Args& a, hipStream_t stream) {
  return a.d == DV ? attend_with<T, DP, DV, true>(a, stream) : attend_with<T, DP, DV, false>(a, stream);
}
template <typename T>
hipError_t attend_as(const PagedAttentionParams& p, hipStream_t stream) {
  const Args a = args_of<T>(p);
  if (p.d <= 64) return attend_wide<T, 64, 64>(a, stream);
  if constexpr (sizeof(T) == 2) {
    if (p.d <= 96) return attend_wide<T, 128, 96>(a, stream);
    if (p.d > 128 && p.d <= 192) return attend_wide<T, 256, 192>(a, stream);
  }
  if (p.d <= 128) return attend_wide<T, 128, 128>(a, stream);
  return attend_wide<T, 256, 256>(a, stream);
}
template <typename T>
hipError_t join_as(const PagedAttentionParams& p, hipStream_t stream) {
  const Args a = args_of<T>(p);
  // A row a wavefront while the card holds them all, else about 2048 workgroups, most of which pass over rows that are in one part:
  // 8400 rows in parts 11.2 us, 12.4 with five a workgroup; 262144 rows, none in parts, 5.5 us, 9.3 with 64 a workgroup.
  const int rows = p.tokens * p.kv_heads * p.group, each = rows <= 16384 ? 4 : (rows + 8191) / 8192 * 4;
  const dim3 grid((unsigned)((rows + each - 1) / each));
  if (p.d > 128) hipLaunchKernelGGL((attention_join_kernel<T, true>), grid, dim3(256), 0, stream, a, each);
  else hipLaunchKernelGGL((attention_join_kernel<T, false>), grid, dim3(256), 0, stream, a, each);
  return hipGetLastError();
}

template <typename T> bool fits_as(const PagedAttentionParams& p) {
  const Args a = args_of<T>(p);
  return (p.d > 128 ? grid_of<T, true>(a) : grid_of<T, false>(a)) * 256 <= UINT32_MAX;
}

}  // namespace

bool paged_attention_fits(const PagedAttentionParams& p) { return p.dt == DT_F32 ? fits_as<float>(p) : fits_as<bf16_t>(p); }
size_t paged_attention_space(const PagedAttentionParams& p) { return p.dt == DT_F32 ? space_of<float>(p) : space_of<bf16_t>(p); }

hipError_t launch_paged_attention(const PagedAttentionParams& p, hipStream_t stream) {
  switch (p.dt) {
    case DT_F32: return attend_as<float>(p, stream);
    case DT_F16: return attend_as<f16_t>(p, stream);
    case DT_BF16: return attend_as<bf16_t>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_attention_join(const PagedAttentionParams& p, hipStream_t stream) {
  switch (p.dt) {
    case DT_F32: return join_as<float>(p, stream);
    case DT_F16: return join_as<f16_t>(p, stream);
    case DT_BF16: return join_as<bf16_t>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ohip
