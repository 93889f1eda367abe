// Attention of new tokens over keys and values in the pages of a cache (formula and contract: odla_hip_PagedAttention).
//
// Rows are the queries that share a head of keys: row r of a sequence is query r % group of its token r / group, so that
// a tile of rows reads each key once for all of them.  Softmax in one pass: per row the running maximum m and
// the sum l of exp(s - m), and o = sum exp(s - m) v rescaled when m grows.
//
// Lengths are on the device, so the launch cannot be cut to them: every workgroup finds its piece - a tile of rows, a head
// and a stretch of the keys - from the lengths itself (attention_pieces.h).  Long sequences with few rows are cut
// into stretches, so that there are about a thousand pieces; a stretch leaves m, l and o in fp32, and
// a last launch joins them in the order of the stretches.
#include "block_common.h"
#include "attention_pieces.h"

namespace ohip {
namespace {

constexpr float kLog2e = 1.44269504f;

struct Args : PagedAttentionParams {
  unsigned page_magic; int page_shift;
  int reach;          // places of a row of the page table
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
__device__ __forceinline__ SeqSpan span_from_lane(const SeqSpan& s, const int lane) {
  return {__builtin_amdgcn_readlane(s.first, lane), __builtin_amdgcn_readlane(s.n, lane), __builtin_amdgcn_readlane(s.cached, lane), __builtin_amdgcn_readlane(s.len, lane)};
}

// A sequence, how its tiles are cut, and where its pieces and the slots of its parts begin.
struct Found { int seq, cuts, stretch, tiles, piece0, slot0; SeqSpan span; };
// The sequence with piece `key` (or, BY_TOKEN, with the new token `key`), by all lanes of a wavefront together; seq < 0: none.
template <int R, int KT, int LEAST, bool BY_TOKEN>
__device__ __forceinline__ Found find(const Args& a, const int key) {
  const int lane = threadIdx.x & 63;
  float work = 0.f;
  for (int b0 = 0; b0 < a.seqs; b0 += 64) {
    const SeqSpan s = span_of(a, b0 + lane);
    work += wave_sum((float)row_tiles(s, R, a.group) * (float)a.kv_heads * (float)most_key_tiles(s, R, a.group, a.window, KT));
  }
  const int stretch = stretch_of(work, LEAST);
  int piece0 = 0, slot0 = 0;
  for (int b0 = 0; b0 < a.seqs; b0 += 64) {
    const SeqSpan s = span_of(a, b0 + lane);
    const int cuts = stretches(most_key_tiles(s, R, a.group, a.window, KT), stretch);
    const int pieces = row_tiles(s, R, a.group) * a.kv_heads * cuts, slots = cuts > 1 ? pieces : 0;
    const int piece_end = piece0 + wave_scan(pieces), slot_end = slot0 + wave_scan(slots);
    const unsigned long long here = BY_TOKEN ? __ballot(key >= s.first && key < s.first + s.n) : __ballot(key < piece_end);
    if (here != 0) {
      const int at = __builtin_ctzll(here);
      Found f;
      f.seq = b0 + at;
      f.span = span_from_lane(s, at);
      f.cuts = __builtin_amdgcn_readlane(cuts, at);
      f.stretch = stretch;
      f.tiles = row_tiles(f.span, R, a.group);
      f.piece0 = __builtin_amdgcn_readlane(piece_end - pieces, at);
      f.slot0 = __builtin_amdgcn_readlane(slot_end - slots, at);
      return f;
    }
    piece0 = __builtin_amdgcn_readlane(piece_end, 63);
    slot0 = __builtin_amdgcn_readlane(slot_end, 63);
  }
  return {-1, 1, stretch, 0, 0, 0, {0, 0, 0, 0}};
}
// Pieces of a sequence: heads side by side (their keys are neighbours in memory), then stretches, then tiles of rows from
// the last one on, which sees the most keys.
__device__ __forceinline__ int piece_of(const Found& f, const int heads, const int tile, const int head, const int cut) {
  return ((f.tiles - 1 - tile) * f.cuts + cut) * heads + head;
}

// Work space: m and l of every row of every slot, then their o.
template <int R> __device__ __forceinline__ float* slot_sums(const Args& a, const int slot, const int row) {
  return reinterpret_cast<float*>(a.work) + ((int64_t)slot * R + row) * 2;
}
template <int R> __device__ __forceinline__ float* slot_rows(const Args& a, const int slot, const int row) {
  return reinterpret_cast<float*>(a.work) + (int64_t)kMostSlots * R * 2 + ((int64_t)slot * R + row) * a.d;
}

// ------------------------------------------------------------ the new tokens --
// A workgroup takes four tokens, a wavefront each.
__global__ void __launch_bounds__(256) cache_write_kernel(const Args a, const int bytes) {
  const int token = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (token >= a.tokens) return;
  int seq = -1;
  SeqSpan s = {0, 0, 0, 0};
  if (a.starts == nullptr) {
    seq = token / (a.tokens / a.seqs);
    s = span_of(a, seq);
  } else {
    for (int b0 = 0; b0 < a.seqs && seq < 0; b0 += 64) {
      const SeqSpan m = span_of(a, b0 + lane);
      const unsigned long long here = __ballot(token >= m.first && token < m.first + m.n);
      if (here != 0) {
        seq = b0 + __builtin_ctzll(here);
        s = span_from_lane(m, __builtin_ctzll(here));
      }
    }
  }
  if (seq < 0) return;
  const int place = s.cached + (token - s.first);
  if (place >= s.len) return;
  const int index = fast_div(place, a.page_magic, a.page_shift);
  const int row = cache_row(a.table[(int64_t)seq * a.table_width + index], place - index * a.page, a.page, a.pages);
  if (row < 0) return;
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

// ------------------------------------------------------------------ few rows --
// Tiles of 16 RB rows; the four wavefronts take every fourth tile of KT keys each and meet in LDS at the end.  Nothing
// passes through LDS on the way: keys come from memory as operand fragments (lane l: key l % 16, 16 bytes of it), and the
// values as VE neighbouring elements of a key a lane (l % 16: which), which are operand fragments once the
// elements of eight keys have changed places inside the lane.  Which key a place of the product's inner axis has
// is free as long as weights and values agree: a lane's weights stay where the scores' product left them.
//   scores  C[key][row]: lane l has row l % 16, keys 4 (l / 16) + i of each block of 16
//   o       C[d][row]:   lane l has row l % 16, d = (4 (l / 16) + i) VE + e
template <typename T> struct Few {
  static constexpr int BLOCKS = sizeof(T) == 4 ? 1 : 2, KEYS = 4 * BLOCKS, KT = 16 * BLOCKS;   // blocks and keys a lane of a tile
  static constexpr int LEAST = 256 / KT;                    // tiles of the shortest stretch
};
template <typename T, int DP> struct FewShape {
  static constexpr int VE = DP / 16;                        // elements of a value that a lane has
  static constexpr int VW = VE * sizeof(T) / 4;             // in dwords
  static constexpr int KC = DP * sizeof(T) / 64;            // 16-byte vectors of a key that a lane has
};

// 16 bytes (or 8) of a row from element `at` on; zeros behind its d elements.
template <typename T, int W>
__device__ __forceinline__ void load_part(const T* row, const int at, const int d, unsigned* to) {
  constexpr int PER = W * 4 / (int)sizeof(T);
  static_assert(W == 2 || W == 4, "8 or 16 bytes");
  if (at + PER <= d) {
    if constexpr (W == 4) {
      const uintx4 v = *reinterpret_cast<const uintx4*>(row + at);
      to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
    } else {
      const uintx2 v = *reinterpret_cast<const uintx2*>(row + at);
      to[0] = v.x; to[1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) to[i] = 0u;
  }
}

// Whether one of the two 16-bit elements of a dword (or the fp32 element) is infinite or NaN.
template <typename T> __device__ __forceinline__ bool not_finite(const unsigned w) {
  if constexpr (sizeof(T) == 4) return (w & 0x7f800000u) == 0x7f800000u;
  constexpr unsigned m = std::is_same<T, f16_t>::value ? 0x7c00u : 0x7f80u;
  return (w & m) == m || (w >> 16 & m) == m;
}
template <typename T> __device__ __forceinline__ float element(const unsigned w, const int half) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w);
  else if constexpr (std::is_same<T, f16_t>::value) return f16_to_f32((uint16_t)(half ? w >> 16 : w));
  else return bf16_to_f32((uint16_t)(half ? w >> 16 : w));
}

template <typename T, int DP, int RB>
__global__ void __launch_bounds__(256, DP == 256 ? 1 : 2) attend_few_kernel(const Args a) {
  using F = Few<T>;
  using S = FewShape<T, DP>;
  constexpr int R = 16 * RB, KEYS = F::KEYS, KT = F::KT, VE = S::VE, VW = S::VW, KC = S::KC;
  __shared__ __attribute__((aligned(16))) float part[4][16][DP + 4];
  __shared__ float part_m[4][16], part_l[4][16];
  const Found f = find<R, KT, F::LEAST, false>(a, blockIdx.x);
  if (f.seq < 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int in_seq = blockIdx.x - f.piece0, rest = in_seq / a.kv_heads;
  const int head = in_seq - rest * a.kv_heads, cut = rest % f.cuts, tile = f.tiles - 1 - rest / f.cuts;
  const int r0 = tile * R, rows = min(R, f.span.n * a.group - r0);
  const KeyRange seen = keys_of_rows(f.span, r0, R, a.group, a.window);
  const int t_begin = seen.lo / KT + cut * f.stretch, t_end = min((seen.hi + KT - 1) / KT, f.cuts > 1 ? t_begin + f.stretch : INT32_MAX);
  const int64_t row_bytes = (int64_t)a.kv_heads * a.d * (int)sizeof(T);
  const char* kc = reinterpret_cast<const char*>(a.k_cache) + (int64_t)head * a.d * (int)sizeof(T);
  const char* vc = reinterpret_cast<const char*>(a.v_cache) + (int64_t)head * a.d * (int)sizeof(T);
  const int32_t* table = a.table + (int64_t)f.seq * a.table_width;

  // queries: this lane's row of each block, and the last place that it sees
  uintx4 q[RB][KC];
  int last[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const int r = min(r0 + 16 * b + l16, r0 + rows - 1), token = r / a.group;
    const T* row = reinterpret_cast<const T*>(a.q) + ((int64_t)(f.span.first + token) * a.kv_heads * a.group + (int64_t)head * a.group + (r - token * a.group)) * a.d;
    last[b] = f.span.cached + token;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      unsigned w[4];
      load_part<T, 4>(row, (4 * c + g) * (16 / (int)sizeof(T)), a.d, w);
      q[b][c] = uintx4{w[0], w[1], w[2], w[3]};
    }
  }
  // the rows of the cache that hold a tile's keys, lane l: key l % KT (-1: not there)
  auto rows_of = [&](const int t) __attribute__((always_inline)) -> int {
    const int place = t * KT + (lane & (KT - 1));
    if (t >= t_end || place >= seen.hi) return -1;
    const int index = fast_div(place, a.page_magic, a.page_shift);
    return cache_row(table[index], place - index * a.page, a.page, a.pages);
  };
  auto key_of_slot = [&](const int j) { return (j >> 2) * 16 + g * 4 + (j & 3); };
  uintx4 kf[F::BLOCKS][KC];
  auto load_keys = [&](const int rows_) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < F::BLOCKS; ++b) {
      const T* row = reinterpret_cast<const T*>(kc + max(__shfl(rows_, 16 * b + l16), 0) * row_bytes);
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        unsigned w[4];
        load_part<T, 4>(row, (4 * c + g) * (16 / (int)sizeof(T)), a.d, w);
        kf[b][c] = uintx4{w[0], w[1], w[2], w[3]};
      }
    }
  };
  unsigned vf[KEYS][VW];
  auto load_values = [&](const int rows_) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      const T* row = reinterpret_cast<const T*>(vc + max(__shfl(rows_, key_of_slot(j)), 0) * row_bytes);
      constexpr int W = VW < 4 ? 2 : 4, PER = W * 4 / (int)sizeof(T);
#pragma unroll
      for (int w = 0; w < VW / W; ++w) load_part<T, W>(row, l16 * VE + w * PER, a.d, &vf[j][w * W]);
    }
  };

  float m[RB], l[RB];
  floatx4 o[RB][VE];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    m[b] = -INFINITY;
    l[b] = 0.f;
#pragma unroll
    for (int e = 0; e < VE; ++e) o[b][e] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  const float to_log2 = a.scale * kLog2e;
  int here = rows_of(t_begin + wave), next = rows_of(t_begin + wave + 4);
  if (t_begin + wave < t_end) {
    load_keys(here);
    load_values(here);
  }
  // (a wavefront's requests for a tile are on their way while the one before is used)
#pragma unroll 1
  for (int t = t_begin + wave; t < t_end; t += 4) {
    floatx4 s[RB][F::BLOCKS];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int k = 0; k < F::BLOCKS; ++k) {
        s[b][k] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c) s[b][k] = mma_vec<T>(kf[k][c], q[b][c], s[b][k]);
      }
    if (t + 4 < t_end) load_keys(next);
    const int after = rows_of(t + 8);
    bool there[KEYS];
    bool all_there = true;
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      there[j] = __shfl(here, key_of_slot(j)) >= 0;
      all_there = all_there && there[j];
    }
    // values that are not there weigh nothing, whatever lies in their stead
    if (!__all(all_there)) {
#pragma unroll
      for (int j = 0; j < KEYS; ++j)
#pragma unroll
        for (int w = 0; w < VW; ++w) vf[j][w] = there[j] ? vf[j][w] : 0u;
    }
    float p[RB][KEYS];
    bool mixed = false;      // a key that one row sees and another does not
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      float most = -INFINITY;
#pragma unroll
      for (int j = 0; j < KEYS; ++j) {
        const int place = t * KT + key_of_slot(j);
        const bool sees = there[j] && place <= last[b] && (a.window == 0 || place > last[b] - a.window);
        mixed = mixed || sees != there[j];
        p[b][j] = sees ? s[b][j >> 2][j & 3] * to_log2 : -INFINITY;
        most = fmaxf(most, p[b][j]);
      }
      most = fmaxf(m[b], over_row(most, [](float x, float y) { return fmaxf(x, y); }));
      const float base = most == -INFINITY ? 0.f : most;
      const float shrink = __builtin_amdgcn_exp2f(m[b] - base);
      m[b] = most;
      l[b] *= shrink;
#pragma unroll
      for (int j = 0; j < KEYS; ++j) {
        p[b][j] = __builtin_amdgcn_exp2f(p[b][j] - base);
        l[b] += p[b][j];
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) o[b][e] *= shrink;
    }
    // A row's weight for a key that it does not see is zero, and zero times an infinite or missing value is none: such
    // values leave the product and are added to the rows that see them one by one.
    if (__any(mixed)) {
      bool odd = false;
#pragma unroll
      for (int j = 0; j < KEYS; ++j)
#pragma unroll
        for (int w = 0; w < VW; ++w) odd = odd || not_finite<T>(vf[j][w]);
      if (__any(odd)) {
#pragma unroll
        for (int j = 0; j < KEYS; ++j) {
#pragma unroll 1
          for (int from = 0; from < 4; ++from) {       // the key of slot j in group `from`
            const int place = t * KT + (j >> 2) * 16 + from * 4 + (j & 3);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int e = 0; e < VE; ++e) {
                const unsigned w = (unsigned)__shfl((int)vf[j][e * (int)sizeof(T) / 4], from * 16 + 4 * g + i);
                const float v = element<T>(w, e & 1);
                const bool finite = __builtin_isfinite(v);
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                  const float weight = __shfl(p[b][j], from * 16 + l16);
                  const bool sees = place <= last[b] && (a.window == 0 || place > last[b] - a.window);
                  if (!finite && sees) o[b][e][i] = __builtin_fmaf(weight, v, o[b][e][i]);
                }
              }
          }
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            if constexpr (sizeof(T) == 4) {
              vf[j][w] = not_finite<T>(vf[j][w]) ? 0u : vf[j][w];
            } else {
              const unsigned lo = __builtin_isfinite(element<T>(vf[j][w], 0)) ? 0xffffu : 0u, hi = __builtin_isfinite(element<T>(vf[j][w], 1)) ? 0xffff0000u : 0u;
              vf[j][w] &= lo | hi;
            }
          }
        }
      }
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int j = 0; j < KEYS; ++j) o[b][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vf[j][e]), p[b][j], o[b][e], 0, 0, 0);
    } else {
      uintx4 w[RB];
#pragma unroll
      for (int b = 0; b < RB; ++b) w[b] = pack8_rne<T>(p[b]);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        uintx4 column;       // element e of the eight keys
#pragma unroll
        for (int j = 0; j < 4; ++j)
          column[j] = __builtin_amdgcn_perm(vf[2 * j + 1][e / 2], vf[2 * j][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int b = 0; b < RB; ++b) o[b][e] = mma_vec<T>(column, w[b], o[b][e]);
      }
    }
    if (t + 4 < t_end) load_values(next);
    here = next;
    next = after;
  }

  // ---- the wavefronts' parts, 16 rows at a time
  const int mine = threadIdx.x >> 4, column = (threadIdx.x & 15) * VE;
#pragma unroll 1
  for (int b = 0; b < RB; ++b) {
    if (16 * b >= rows) break;
    if (b > 0) __syncthreads();
#pragma unroll
    for (int k = 0; k < RB; ++k) {
      if (k != b) continue;
      const float sum = over_row(l[k], [](float x, float y) { return x + y; });
      if (g == 0) { part_m[wave][l16] = m[k]; part_l[wave][l16] = sum; }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) part[wave][l16][(4 * g + i) * VE + e] = o[k][e][i];
    }
    __syncthreads();
    const int r = 16 * b + mine;
    if (r < rows) {
      float most = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) most = fmaxf(most, part_m[w][mine]);
      float factor[4], sum = 0.f;      // (of a part without keys: 0; of one whose scores are all NaN: NaN)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        factor[w] = part_m[w][mine] == -INFINITY ? part_l[w][mine] : __builtin_amdgcn_exp2f(part_m[w][mine] - most);
        sum = __builtin_fmaf(factor[w], part_l[w][mine], sum);
      }
      const int slot = f.slot0 + in_seq, token = (r0 + r) / a.group;
      const bool whole = f.cuts == 1;
      if (whole || slot < kMostSlots) {
        T* y = reinterpret_cast<T*>(a.y) + ((int64_t)(f.span.first + token) * a.kv_heads * a.group + (int64_t)head * a.group + (r0 + r - token * a.group)) * a.d;
        float* to = whole ? nullptr : slot_rows<R>(a, slot, r);
        const float by = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int e = 0; e < VE; e += 4) {
          if (column + e >= a.d) break;
          floatx4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const floatx4 x = *reinterpret_cast<const floatx4*>(&part[w][mine][column + e]);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = factor[w] != 0.f ? __builtin_fmaf(factor[w], x[i], v[i]) : v[i];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = by == 0.f ? 0.f : v[i] * by;
          if (whole) store4<T>(y + column + e, v, 4, true);
          else *reinterpret_cast<floatx4*>(to + column + e) = v;
        }
        if (!whole && (threadIdx.x & 15) == 0) {
          float* ml = slot_sums<R>(a, slot, r);
          ml[0] = most;
          ml[1] = sum;
        }
      }
    }
  }
}

// ------------------------------------------------------------------ the parts --
// A workgroup has a few neighbouring tokens of one head, a wavefront one row after the other.
template <typename T, int R, int KT, int LEAST>
__global__ void __launch_bounds__(256) attention_join_kernel(const Args a, const int tokens_each) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.x % (unsigned)a.kv_heads, token0 = blockIdx.x / (unsigned)a.kv_heads * tokens_each;
  Found f = {-1, 1, 0, 0, 0, 0, {0, 0, 0, 0}};
  for (int token = token0; token < min(token0 + tokens_each, a.tokens); ++token) {
    if (f.seq < 0 || token < f.span.first || token >= f.span.first + f.span.n) f = find<R, KT, LEAST, true>(a, token);
    if (f.seq >= 0 && f.cuts == 1) continue;
    for (int q = wave; q < a.group; q += 4) {
      T* y = reinterpret_cast<T*>(a.y) + ((int64_t)token * a.kv_heads * a.group + (int64_t)head * a.group + q) * a.d;
      if (f.seq < 0) {       // no sequence's
        for (int c = lane * 4; c < a.d; c += 256) store4<T>(y + c, floatx4{0.f, 0.f, 0.f, 0.f}, 4, true);
        continue;
      }
      const int row = (token - f.span.first) * a.group + q, tile = row / R, r = row - tile * R;
      float most = -INFINITY;
      for (int cut = 0; cut < f.cuts; ++cut) {
        const int slot = f.slot0 + piece_of(f, a.kv_heads, tile, head, cut);
        if (slot < kMostSlots) most = fmaxf(most, slot_sums<R>(a, slot, r)[0]);
      }
      float sum = 0.f;
      floatx4 v = {0.f, 0.f, 0.f, 0.f};
      for (int cut = 0; cut < f.cuts; ++cut) {
        const int slot = f.slot0 + piece_of(f, a.kv_heads, tile, head, cut);
        if (slot >= kMostSlots) continue;
        const float* ml = slot_sums<R>(a, slot, r);
        if (ml[1] == 0.f) continue;
        const float factor = ml[0] == -INFINITY ? ml[1] : __builtin_amdgcn_exp2f(ml[0] - most);
        sum = __builtin_fmaf(factor, ml[1], sum);
        if (lane * 4 < a.d) {
          const floatx4 x = *reinterpret_cast<const floatx4*>(slot_rows<R>(a, slot, r) + lane * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(factor, x[i], v[i]);
        }
      }
      if (lane * 4 < a.d) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = sum == 0.f ? 0.f : v[i] / sum;
        store4<T>(y + lane * 4, v, 4, true);
      }
    }
  }
}

Args args_of(const PagedAttentionParams& p) {
  Args a;
  static_cast<PagedAttentionParams&>(a) = p;
  div_magic(p.page, &a.page_magic, &a.page_shift);
  a.reach = p.table_width * p.page;
  a.window = p.window > (1 << 30) ? 1 << 30 : p.window;   // (no place lies further back)
  return a;
}
constexpr int kRowsFew = 16;

template <typename T, int DP>
void launch_few(const Args& a, hipStream_t stream) {
  const long long grid = most_units(a.tokens, a.seqs, a.kv_heads, a.group, kRowsFew) + kMostCutPieces;
  hipLaunchKernelGGL((attend_few_kernel<T, DP, kRowsFew / 16>), dim3((unsigned)grid), dim3(256), 0, stream, a);
}
template <typename T>
hipError_t attend_as(const PagedAttentionParams& p, hipStream_t stream) {
  const Args a = args_of(p);
  if (p.d <= 64) launch_few<T, 64>(a, stream);
  else if (p.d <= 128) launch_few<T, 128>(a, stream);
  else launch_few<T, 256>(a, stream);
  return hipGetLastError();
}
template <typename T>
hipError_t join_as(const PagedAttentionParams& p, hipStream_t stream) {
  const Args a = args_of(p);
  const int each = p.group >= 16 ? 1 : 16 / p.group;
  const unsigned grid = (unsigned)((p.tokens + each - 1) / each) * (unsigned)p.kv_heads;
  hipLaunchKernelGGL((attention_join_kernel<T, kRowsFew, Few<T>::KT, Few<T>::LEAST>), dim3(grid), dim3(256), 0, stream, a, each);
  return hipGetLastError();
}

}  // namespace

size_t paged_attention_space(const PagedAttentionParams& p) { return (size_t)kMostSlots * kRowsFew * (p.d + 2) * sizeof(float); }

hipError_t launch_cache_write(const PagedAttentionParams& p, hipStream_t stream) {
  hipLaunchKernelGGL(cache_write_kernel, dim3((unsigned)((p.tokens + 3) / 4)), dim3(256), 0, stream, args_of(p), p.kv_heads * p.d * dtype_size(p.dt));
  return hipGetLastError();
}

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
