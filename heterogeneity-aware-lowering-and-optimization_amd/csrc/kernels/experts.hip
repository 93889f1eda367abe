// A layer of experts for few tokens: the router's choice, the gated products of the chosen experts
// and the weighted sum of what they give.
//
//   l = router x, top k of l; w = softmax(l) of those (divided by their sum)
//   h = silu(gate_e x) * (up_e x),   y = sum_j w_j down_ej h_j
//
// Few tokens: bound by the weights of the experts that some token chose, which are read once: their rows are the
// rows of a matrix product, the tokens that chose the expert its columns.  Five launches (four where the first
// product makes the choice itself): logits, choice, first product, second product with its parts, sum.
//   64 experts of 2048 x 1024, 8 chosen, bf16: 1 token 5 + 17 (100 MB in all) + 8 + 4 us; 32 tokens 7 + 4 + 102 +
//   53 + 4 us, 5.2 TB/s in the products.  7 tokens, 128 experts of 2624 x 704, 8-bit weights 7 + 30 + 15 + 4 us,
//   4.6 TB/s; of 2600 x 712, rows that are no whole vectors, 33 + 17.
// Logits, softmax, sums and parts are fp32.  hidden is rounded to the input's type: it is an operand of the second
// product's matrix instructions, which take that type.
// The last of a token's parts adding them up instead of a launch was slower: making parts visible to the
// other chiplets costs more (a release of the whole L2 in every tile: 52 -> 240 us).
#include "block_common.h"
#include "lds_limit.h"

namespace ohip {
namespace {

// Where the choice stands in the work space: expert and weight of every (token, place), then the logits.
__host__ __device__ inline size_t route_weights(const int tokens, const int top_k) { return (size_t)tokens * top_k * 4; }
__host__ __device__ inline size_t route_logits(const int tokens, const int top_k) { return (size_t)tokens * top_k * 8; }

// ---- the router: 16 experts x 16 tokens a workgroup, the wavefronts split H ----
// A step is 128 bytes of every row, 32 of them a lane's; four steps are under way at a time.
template <typename X, bool ALIGNED>
__global__ void __launch_bounds__(512) experts_logits_kernel(const ExpertsParams p) {
  constexpr int P = 4;
  __shared__ floatx4 sums[8][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int e0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
  const int64_t len = (int64_t)p.H * sizeof(X);
  const unsigned char* wrow = (const unsigned char*)p.router + min(e0 + r, p.E - 1) * len;
  const unsigned char* xrow = (const unsigned char*)p.x + min(t0 + r, p.tokens - 1) * len;
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int64_t at = wave * 128 + g * 32; at - g * 32 < len; at += waves * 128 * P) {
    uintx4 w[P][2], x[P][2];
#pragma unroll
    for (int q = 0; q < P; ++q)
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        w[q][v] = load_row16<ALIGNED>(wrow, at + q * waves * 128 + v * 16, len);
        x[q][v] = load_row16<ALIGNED>(xrow, at + q * waves * 128 + v * 16, len);
      }
#pragma unroll
    for (int q = 0; q < P; ++q)
#pragma unroll
      for (int v = 0; v < 2; ++v) acc = mma_vec<X>(w[q][v], x[q][v], acc);
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave != 0) return;
  for (int w = 1; w < waves; ++w) acc += sums[w][lane];
  float* logits = (float*)((char*)p.route + route_logits(p.tokens, p.top_k));
  const int t = t0 + r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = e0 + 4 * g + i;
    if (t < p.tokens && e < p.E) logits[(int64_t)t * p.E + e] = acc[i];
  }
}

// Order of floats as unsigned numbers, and back: a NaN is 1 and comes before everything, 0 is no number.
__device__ __forceinline__ unsigned ordered(const float f) {
  const unsigned u = __float_as_uint(f);
  return f != f ? 1u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float number_of(const unsigned k) {
  return k == 1u ? __builtin_nanf("") : __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
// The largest of the wavefront's numbers (see group_allreduce).
template <int CTRL>
__device__ __forceinline__ unsigned larger_of_pair(const unsigned v) {
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ unsigned wave_largest(unsigned v) {
  v = larger_of_pair<0x140>(larger_of_pair<0x141>(larger_of_pair<0x4E>(larger_of_pair<0xB1>(v))));
  const unsigned a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
  const unsigned c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
  return max(max(a, b), max(c, d));
}

// The choice of token t, by one wavefront: expert and weight of place j in lane j.  `keys`: E words of LDS.
// Every lane knows the first of the largest of its experts lane, lane + 64, ...; a round finds the largest of
// those (the lowest expert among equals) and only its lane looks for another.  Nothing is loaded in a round:
// the number is made from its key.
__device__ __forceinline__ void choose(const ExpertsParams& p, const int t, const int lane, unsigned* keys, int* id, float* weight) {
  const float* logits = (const float*)((const char*)p.route + route_logits(p.tokens, p.top_k)) + (int64_t)t * p.E;
  float most = -__builtin_inff();
  for (int e = lane; e < p.E; e += 64) {
    const float l = logits[e];
    most = fmaxf(most, l);
    keys[e] = ordered(l);
  }
  most = wave_max(most);
  unsigned best = 0;
  int at = 0;
  float sum = 0.f;
  for (int e = lane; e < p.E; e += 64) {
    const unsigned k = keys[e];
    if (k > best) { best = k; at = e; }
    sum += expf(number_of(k) - most);
  }
  sum = wave_sum(sum);
  float chosen = 0.f, mine = 0.f;
  *id = 0;
  for (int j = 0; j < p.top_k; ++j) {
    const unsigned k = wave_largest(best);
    const unsigned long long some = __ballot(best == k);
    const int e = (some & (some - 1)) == 0 ? __builtin_amdgcn_readlane(at, __ffsll(some) - 1) : (int)~wave_largest(best == k ? ~(unsigned)at : 0u);
    const float v = expf(number_of(k) - most);
    chosen += v;
    if (lane == j) { mine = v; *id = e; }
    if (lane == (e & 63)) {
      keys[e] = 0;
      best = 0;
      if (p.E > 64)
        for (int o = lane; o < p.E; o += 64)
          if (keys[o] > best) { best = keys[o]; at = o; }
    }
  }
  // (a NaN among the logits reaches every weight through the whole sum)
  const float by = p.renormalize ? (sum == sum ? chosen : sum) : sum;
  *weight = mine / by * p.scaling;
}
__device__ __forceinline__ void keep_choice(const ExpertsParams& p, const int t, const int lane, const int id, const float weight) {
  if (lane >= p.top_k) return;
  ((int*)p.route)[t * p.top_k + lane] = id;
  ((float*)((char*)p.route + route_weights(p.tokens, p.top_k)))[t * p.top_k + lane] = weight;
}
__global__ void __launch_bounds__(64) experts_choice_kernel(const ExpertsParams p) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  int id;
  float weight;
  choose(p, blockIdx.x, threadIdx.x, (unsigned*)smem, &id, &weight);
  keep_choice(p, blockIdx.x, threadIdx.x, id, weight);
}

// The experts that some token chose (in ascending order), and for each the (token, place) pairs that chose it.
__host__ __device__ inline int slots_of(const int tokens, const int top_k, const int E) { return tokens * top_k < E ? tokens * top_k : E; }
struct Chosen {
  int* cursor;            // of every expert
  int* expert;            // of every slot
  int* first;             // pair of every slot, and behind the last
  unsigned short* pairs;
  int slots;
  __host__ __device__ static size_t bytes(const int tokens, const int top_k, const int E) {
    return ((size_t)E + 2 * slots_of(tokens, top_k, E) + 2) * 4 + ((size_t)tokens * top_k + 1) / 2 * 4;
  }
};
static_assert(kMaxExpertTokens * kMaxExpertTopK <= 65536, "pairs are numbered in 16 bits");
// `ids`: of every pair.  By the whole workgroup, with barriers.  The order of an expert's pairs is not settled: it
// is the order of columns of a matrix product, which do not touch each other.
__device__ __forceinline__ Chosen find_chosen(const ExpertsParams& p, const int* ids, unsigned char* lds) {
  const int n = p.tokens * p.top_k, most = slots_of(p.tokens, p.top_k, p.E);
  Chosen c;
  c.cursor = (int*)lds;
  c.expert = c.cursor + p.E;
  c.first = c.expert + most;
  int* const found = c.first + most + 1;
  c.pairs = (unsigned short*)(found + 1);
  for (int i = threadIdx.x; i < p.E; i += blockDim.x) c.cursor[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) atomicAdd(&c.cursor[ids[i]], 1);
  __syncthreads();
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int slot = 0, run = 0;
    for (int e0 = 0; e0 < p.E; e0 += 64) {
      const int here = e0 + lane < p.E ? c.cursor[e0 + lane] : 0;
      int upto = here;
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
      }
      const unsigned long long some = __ballot(here > 0);
      const int s = slot + __popcll(some & ((1ull << lane) - 1ull));
      if (here > 0) {
        c.expert[s] = e0 + lane;
        c.first[s] = run + upto - here;
        c.cursor[e0 + lane] = run + upto - here;
      }
      slot += __popcll(some);
      run += __builtin_amdgcn_readlane(upto, 63);
    }
    if (lane == 0) { c.first[slot] = run; *found = slot; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) c.pairs[atomicAdd(&c.cursor[ids[i]], 1)] = (unsigned short)i;
  __syncthreads();
  c.slots = __builtin_amdgcn_readfirstlane(*found);
  return c;
}

// ---- the two products ----
//   GATED:  hidden[pair][i] = silu(gate x) * (up x), sixteen i a tile (a tile of gate's rows, one of up's)
//   else:   parts[pair][n] = weight * down hidden, 32 n a tile
// A workgroup takes tiles of (expert, rows) in turn; its wavefronts share out the steps of 128 bytes of the
// weights' rows, and their sums meet in LDS in wavefront order.  Every wavefront has LDS of its own and no barrier
// inside the sum: eight lanes bring 128 neighbouring bytes of a row, P steps ahead, and the operand fragments
// (lane l: row l % 16) are read back from there.  The first steps of the next tile are under way while the sums of
// this one meet.  The columns are the pairs that chose the expert, C at a time (only as many as there are
// are loaded and multiplied).
template <typename X, typename W, int C>
struct Staging {
  static constexpr int PLANES = sizeof(X) / sizeof(W);            // 128-byte pieces of an x row in a step
  static constexpr int XR = C / 8 * PLANES;                       // requests of x in a step, of eight rows x 128 bytes
  static constexpr int BYTES = 4096 + XR * 1024;                  // of a wavefront
  static_assert(BYTES >= 2 * ((C + 15) / 16) * 1024, "the sums take the operands' place");
};
template <bool GATED>
__host__ __device__ inline int tile_rows(const ExpertsParams& p) { return GATED ? (p.I + 15) / 16 : (p.H + 31) / 32; }

template <typename X, typename W, int C, int P, bool ALIGNED, bool GATED>
__global__ void __launch_bounds__(512, C > 8 || sizeof(X) > 2 * sizeof(W) ? 1 : sizeof(X) == sizeof(W) || ALIGNED ? 4 : 3) experts_product_kernel(const ExpertsParams p, const bool choice) {
  using S = Staging<X, W, C>;
  constexpr int MT = (C + 15) / 16;    // (eight columns: the others of a tile repeat them)
  constexpr int PLANES = S::PLANES, XR = S::XR, NR = 4 + XR;
  constexpr bool SCALED = sizeof(W) == 1;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int r = lane & 15, g = lane >> 4, chunk = lane & 7, l8 = lane >> 3;
  unsigned char* const own = smem + wave * S::BYTES;
  const int* ids = (const int*)p.route;
  if (GATED && choice) {
    int* const mine = (int*)(smem + waves * S::BYTES + Chosen::bytes(p.tokens, p.top_k, p.E));
    for (int t = wave; t < p.tokens; t += waves) {
      int id;
      float weight;
      choose(p, t, lane, (unsigned*)own, &id, &weight);
      if (lane < p.top_k) mine[t * p.top_k + lane] = id;
      if (blockIdx.x == 0) keep_choice(p, t, lane, id, weight);
    }
    __syncthreads();
    ids = mine;
  }
  const Chosen c = find_chosen(p, ids, smem + waves * S::BYTES);

  const int K = GATED ? p.H : p.I, N = GATED ? 2 * p.I : p.H;      // of an expert's matrix
  const int wlen = K * (int)sizeof(W), steps = (wlen + 127) / 128;
  const int64_t xlen = (int64_t)K * sizeof(X);
  const int tiles_n = tile_rows<GATED>(p), tiles = tiles_n * c.slots;
  const float* weights = (const float*)((const char*)p.route + route_weights(p.tokens, p.top_k));
  const int SB = (N + kScaleBlock - 1) / kScaleBlock;               // rows of an expert's scales

  // the tile under way: columns c0 .. of slot `slot`, rows n0 ..
  int tile = blockIdx.x, slot = 0, n0 = 0, c0 = 0, here = 0;
  const unsigned char* w_tile[2] = {};
  int w_rows[2] = {};
  const float* w_scale[3] = {};        // of the first rows, of the second, and of the second from row `cut` on
  int cut = 16;
  unsigned x_row[C / 8] = {};
  float weight = 0.f;
  const unsigned char* const xs = (const unsigned char*)(GATED ? p.x : p.hidden);
  const unsigned xbytes = (unsigned)((GATED ? p.tokens : p.tokens * p.top_k) * xlen);      // (at most kOutside: see valid)
  const unsigned lane_row = (unsigned)l8 * wlen;
  const bool in_vectors = ALIGNED || wlen >= 16;     // (a row of fewer bytes: one step, byte by byte)
  uintx4 in[P][NR];
  float sc[3] = {};                    // lane l: of this wavefront's step l (of 64)
  auto fetch = [&](const int s, const int q) __attribute__((always_inline)) {
    if (s >= steps) return;
    const int at = s * 128 + chunk * 16;
    const unsigned lane_at = lane_offset(lane_row, at, wlen, ALIGNED);
#pragma unroll
    for (int i = 0; i < 4; ++i) in[q][i] = load_within(row_range(w_tile[i >> 1], in_vectors ? w_rows[i >> 1] : 0, 8 * (i & 1), 8, wlen), lane_at);
#pragma unroll
    for (int i = 0; i < XR; ++i) {
      const int from = s * (128 * PLANES) + i % PLANES * 128 + chunk * 16;
      if (8 * (i / PLANES) < here)
        in[q][4 + i] = load_within({xs, ALIGNED || xlen >= 16 ? xbytes : 0}, 8 * (i / PLANES) + l8 < here ? lane_offset(x_row[i / PLANES], from, (int)xlen, ALIGNED) : kOutside);
    }
  };
  auto scales_from = [&](const int s) __attribute__((always_inline)) {
    if constexpr (SCALED) {
#pragma unroll
      for (int i = 0; i < (GATED ? 3 : 1); ++i) sc[i] = w_scale[i][min(s + lane * waves, steps - 1)];
    }
  };
  auto start = [&]() __attribute__((always_inline)) {
    slot = tile / tiles_n;
    const int at = tile - slot * tiles_n;
    const int e = __builtin_amdgcn_readfirstlane(c.expert[slot]), pair0 = __builtin_amdgcn_readfirstlane(c.first[slot]) + c0;
    here = min(C, __builtin_amdgcn_readfirstlane(c.first[slot + 1]) - pair0);
    n0 = at * (GATED ? 16 : 32);
    const unsigned char* w = (const unsigned char*)(GATED ? p.gate_up : p.down) + (int64_t)e * N * wlen;
    int row0[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const RowTile half = expert_rows(GATED, n0, j, p.I, p.H);     // (the last tile's second half may have no rows)
      row0[j] = half.row0;
      w_rows[j] = half.rows;
      w_tile[j] = w + (int64_t)row0[j] * wlen;
    }
    if constexpr (SCALED) {
      const float* scales = (GATED ? p.gate_up_scale : p.down_scale) + (int64_t)e * SB * steps;
      w_scale[0] = scales + (int64_t)(row0[0] / kScaleBlock) * steps;
      if constexpr (GATED) {
        w_scale[1] = scales + (int64_t)(row0[1] / kScaleBlock) * steps;
        const int next = row0[1] / kScaleBlock + 1;
        w_scale[2] = scales + (int64_t)min(next, SB - 1) * steps;
        cut = next * kScaleBlock - row0[1];
      }
    }
#pragma unroll
    for (int i = 0; i < C / 8; ++i) {
      const int pair = 8 * i + l8 < here ? c.pairs[pair0 + 8 * i + l8] : 0;
      x_row[i] = (unsigned)((GATED ? pair / p.top_k : pair) * xlen);
    }
    if (!GATED) weight = 16 * wave + r < here ? weights[c.pairs[pair0 + 16 * wave + r]] : 0.f;
    scales_from(wave);
#pragma unroll
    for (int q = 0; q < P; ++q) fetch(wave + q * waves, q);
  };
  if (tile >= tiles) return;
  start();
  while (true) {
    floatx4 acc[2][MT];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[j][t] = floatx4{0.f, 0.f, 0.f, 0.f};
    static_assert(64 % P == 0, "a round of the loop has its scales in one load");
    int done = 0;
    for (int s0 = wave; s0 < steps; s0 += P * waves, done += P) {
      if (SCALED && done == 64) {
        scales_from(s0);
        done = 0;
      }
#pragma unroll
      for (int q = 0; q < P; ++q) {
        const int s = s0 + q * waves;
        if (s >= steps) break;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();     // (the fragments of the step before have been read: LDS keeps a wavefront's order)
        if (!ALIGNED && s == steps - 1) {
          // 16 bytes that would pass the row's end are its last 16: into place
          const int behind = s * 128 + chunk * 16 + 16 - wlen;
          if (in_vectors) {
            if (behind > 0 && behind < 16) {
#pragma unroll
              for (int i = 0; i < 4; ++i) in[q][i] = bytes_down(in[q][i], behind);
            }
          } else {
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
              uintx4 v = {0u, 0u, 0u, 0u};
              if (behind < 16 && 8 * (i & 1) + l8 < (i < 2 ? w_rows[0] : w_rows[1]))
                v = load_row16<false>((i < 2 ? w_tile[0] : w_tile[1]) + (int64_t)(8 * (i & 1) + l8) * wlen, chunk * 16, wlen);
              *reinterpret_cast<uintx4*>(own + (8 * i + l8) * 128 + ((chunk ^ ((8 * i + l8) >> 1 & 7)) << 4)) = v;
            }
          }
#pragma unroll
          for (int i = 0; i < XR; ++i) {
            const int64_t past = (int64_t)s * (128 * PLANES) + i % PLANES * 128 + chunk * 16 + 16 - xlen;
            if (past <= 0 || past >= 16) continue;
            if (xlen >= 16) in[q][4 + i] = bytes_down(in[q][4 + i], (int)past);
            else if (8 * (i / PLANES) + l8 < here) in[q][4 + i] = load_row16<false>(xs + x_row[i / PLANES], 0, xlen);
          }
        }
        if (in_vectors) {
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<uintx4*>(own + (8 * i + l8) * 128 + ((chunk ^ ((8 * i + l8) >> 1 & 7)) << 4)) = in[q][i];
        }
#pragma unroll
        for (int i = 0; i < XR; ++i) {
          // (chunk k of a row of x stands in plane k % PLANES, so that the chunks that belong to one of W have one place)
          const int row = 8 * (i / PLANES) + l8, k = i % PLANES * 8 + chunk;
          if (8 * (i / PLANES) < here)
            *reinterpret_cast<uintx4*>(own + 4096 + k % PLANES * (C * 128) + row * 128 + ((k / PLANES ^ (row >> 1 & 7)) << 4)) = in[q][4 + i];
        }
        float scale[3] = {1.f, 1.f, 1.f};
        if constexpr (SCALED) {
#pragma unroll
          for (int i = 0; i < (GATED ? 3 : 1); ++i) scale[i] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc[i]), done + q));
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        fetch(s + P * waves, q);
        // (8-bit weights: half a step at a time, or operands in 16 bits take the registers of steps under way)
        uintx4 w[2][2];
        if constexpr (!SCALED || MT > 1) {
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j >> 1][j & 1] = *reinterpret_cast<const uintx4*>(own + (16 * (j >> 1) + r) * 128 + ((g + 4 * (j & 1) ^ r >> 1) << 4));
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          if (16 * t >= here) break;
          floatx4 part[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) part[j] = SCALED ? floatx4{0.f, 0.f, 0.f, 0.f} : acc[j][t];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if constexpr (SCALED && MT == 1) {
              __builtin_amdgcn_sched_barrier(0);
#pragma unroll
              for (int j = 0; j < 2; ++j) w[j][h] = *reinterpret_cast<const uintx4*>(own + (16 * j + r) * 128 + ((g + 4 * h ^ r >> 1) << 4));
            }
#pragma unroll
            for (int v = 0; v < PLANES; ++v) {
              const int row = 16 * t + r & C - 1;
              const uintx4 x = *reinterpret_cast<const uintx4*>(own + 4096 + v * (C * 128) + row * 128 + ((g + 4 * h ^ (row >> 1 & 7)) << 4));
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                if constexpr (SCALED) part[j] = mma_vec<X>(values_of<X>(w[j][h], v), x, part[j]);
                else part[j] = mma_vec<X>(w[j][h], x, part[j]);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[j][t][i] = SCALED ? __builtin_fmaf(part[j][i], GATED && j == 1 ? (4 * g + i < cut ? scale[1] : scale[2]) : scale[0], acc[j][t][i]) : part[j][i];
        }
      }
    }
    // what the end of this tile needs, then the next tile's first steps
    const int rows_here = here, n_here = n0, pair_here = __builtin_amdgcn_readfirstlane(c.first[slot]) + c0;
    const float weight_here = weight;
    c0 += C;
    if (pair_here + C >= __builtin_amdgcn_readfirstlane(c.first[slot + 1])) { c0 = 0; tile += gridDim.x; }
    const bool more = tile < tiles;
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    floatx4* const sums = reinterpret_cast<floatx4*>(own);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int t = 0; t < MT; ++t) sums[(j * MT + t) * 64 + lane] = acc[j][t];
    if (more) start();
    __syncthreads();
    floatx4 v[2] = {};
    const int t = wave;
    if (16 * t < rows_here) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        for (int o = 0; o < waves; ++o) v[j] += reinterpret_cast<const floatx4*>(smem + o * S::BYTES)[(j * MT + t) * 64 + lane];
    }
    __syncthreads();
    if (16 * t + r < rows_here) {
      const int64_t pair = c.pairs[pair_here + 16 * t + r];
      if constexpr (GATED) {
        floatx4 h;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = v[0][i] / (1.f + expf(-v[0][i])) * v[1][i];
        const int n = n_here + 4 * g;
        if (n < p.I) store4((X*)p.hidden + pair * p.I + n, h, p.I - n, (p.I & 3) == 0);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int n = n_here + 16 * j + 4 * g;
          if (n < p.H) store4((float*)p.parts + pair * p.H + n, v[j] * weight_here, p.H - n, (p.H & 3) == 0);
        }
      }
    }
    if (!more) return;
  }
}

// ---- y[t][n] = sum of the parts of token t, in the order of its choices: a launch's 4 us and little else ----
template <typename X>
__global__ void __launch_bounds__(256) experts_sum_kernel(const ExpertsParams p) {
  const int64_t n = (int64_t)p.tokens * p.H;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / p.H;
    const float* part = (const float*)p.parts + t * p.top_k * p.H + (i - t * p.H);
    float v = part[0];
    for (int j = 1; j < p.top_k; ++j) v += part[(int64_t)j * p.H];
    Store<X>::st((X*)p.y + i, v);
  }
}

static_assert(kMaxExpertBytes <= kOutside, "what lies behind a row is asked for outside every range");
bool valid(const ExpertsParams& p) {
  return p.x != nullptr && p.router != nullptr && p.gate_up != nullptr && p.down != nullptr && p.y != nullptr && p.route != nullptr &&
         p.hidden != nullptr && p.parts != nullptr && p.tokens >= 1 && p.tokens <= kMaxExpertTokens && p.E >= 1 && p.E <= kMaxExperts &&
         p.H >= 1 && p.H <= (1 << 24) && p.I >= 1 && p.I <= (1 << 23) && p.top_k >= 1 && p.top_k <= p.E && p.top_k <= kMaxExpertTopK &&
         (int64_t)p.tokens * p.H * 4 <= kMaxExpertBytes && (int64_t)p.tokens * p.top_k * p.I * 4 <= kMaxExpertBytes && dtype_is_float(p.dt) && (p.w_dt == p.dt || (p.w_dt == DT_F8 && p.gate_up_scale != nullptr && p.down_scale != nullptr));
}
// rows of x, hidden and weights are whole 16-byte vectors
bool whole_vectors(const ExpertsParams& p, const int len) { return (int64_t)len * dtype_size(p.dt) % 16 == 0 && (int64_t)len * dtype_size(p.w_dt) % 16 == 0; }

// Eight columns at a time, unless experts get more than eight tokens on average (an expert with more is read again).
// 64 experts of 2048 x 1024, 8 chosen, both products in us, eight columns / 64 (bf16) or 32 (8-bit weights):
//   four tokens an expert 153 / 181, six 161 / 184, eight 179 / 186, twelve 226 / 194;  8-bit: eight 104 / 114, twelve 131 / 124.
bool few_columns(const ExpertsParams& p) { return p.tokens <= 8 || (int64_t)p.tokens * p.top_k <= 8 * (int64_t)p.E; }
// Two steps of 128 bytes a wavefront at least, and a wavefront for every sixteen columns.
template <int C>
int product_waves(const ExpertsParams& p, const int K) {
  const int steps = (K * (int)dtype_size(p.w_dt) + 127) / 128;
  return std::max((C + 15) / 16, std::min(C == 8 && p.w_dt != DT_F8 ? 8 : 4, (steps + 1) / 2));
}
// Few tokens: every workgroup of the first product makes the choice for itself, a wavefront for two tokens at most,
// which takes less than another launch.
bool choice_at_first_product(const ExpertsParams& p) { return few_columns(p) && p.tokens <= 2 * product_waves<8>(p, p.H); }

template <typename X>
hipError_t route_as(const ExpertsParams& p, hipStream_t stream) {
  const dim3 grid((p.E + 15) / 16, (p.tokens + 15) / 16);
  if ((int64_t)p.H * sizeof(X) % 16 == 0) hipLaunchKernelGGL((experts_logits_kernel<X, true>), grid, dim3(512), 0, stream, p);
  else hipLaunchKernelGGL((experts_logits_kernel<X, false>), grid, dim3(512), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (choice_at_first_product(p)) return hipSuccess;
  hipLaunchKernelGGL(experts_choice_kernel, dim3(p.tokens), dim3(64), p.E * 4, stream, p);
  return hipGetLastError();
}

constexpr int kComputeUnits = 256, kLdsOfUnit = 160 * 1024;
template <typename X, typename W, int C, int P, bool ALIGNED, bool GATED>
hipError_t product_one(const ExpertsParams& p, hipStream_t stream) {
  using S = Staging<X, W, C>;
  const bool choice = GATED && choice_at_first_product(p);
  const int waves = product_waves<C>(p, GATED ? p.H : p.I);
  const size_t lds = (size_t)waves * S::BYTES + Chosen::bytes(p.tokens, p.top_k, p.E) + (choice ? (size_t)p.tokens * p.top_k * 4 : 0);
  static LdsLimit limit;
  hipError_t e = limit.raise(reinterpret_cast<const void*>(&experts_product_kernel<X, W, C, P, ALIGNED, GATED>), kLdsOfUnit);
  if (e != hipSuccess) return e;
  const int64_t tiles = (int64_t)slots_of(p.tokens, p.top_k, p.E) * tile_rows<GATED>(p);
  const int64_t resident = kComputeUnits * std::max<int64_t>(1, std::min<int64_t>((sizeof(X) == sizeof(W) || ALIGNED ? 16 : 12) / waves, kLdsOfUnit / lds));
  hipLaunchKernelGGL((experts_product_kernel<X, W, C, P, ALIGNED, GATED>), dim3((unsigned)std::min(tiles, resident)), dim3(64 * waves), lds, stream, p, choice);
  return hipGetLastError();
}
template <typename X, typename W, bool GATED>
hipError_t product_as(const ExpertsParams& p, hipStream_t stream) {
  constexpr int MANY = 64 * sizeof(W) / sizeof(X);      // (two steps under way within registers)
  const bool a = whole_vectors(p, GATED ? p.H : p.I);
  if (few_columns(p)) return a ? product_one<X, W, 8, 2, true, GATED>(p, stream) : product_one<X, W, 8, 2, false, GATED>(p, stream);
  return a ? product_one<X, W, MANY, 2, true, GATED>(p, stream) : product_one<X, W, MANY, 2, false, GATED>(p, stream);
}
template <typename X, typename W>
hipError_t gate_up_as(const ExpertsParams& p, hipStream_t stream) { return product_as<X, W, true>(p, stream); }
template <typename X, typename W>
hipError_t down_as(const ExpertsParams& p, hipStream_t stream) {
  hipError_t e = product_as<X, W, false>(p, stream);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((experts_sum_kernel<X>), dim3(grid_for((int64_t)p.tokens * p.H, 256)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

ExpertsSpace experts_space(const ExpertsParams& p) {
  const size_t places = (size_t)p.tokens * p.top_k;
  return {route_logits(p.tokens, p.top_k) + (size_t)p.tokens * p.E * 4, places * p.I * dtype_size(p.dt), places * p.H * 4};
}

hipError_t launch_experts_route(const ExpertsParams& p, hipStream_t stream) {
  if (!valid(p)) return hipErrorInvalidValue;
  switch (p.dt) {
    case DT_F32: return route_as<float>(p, stream);
    case DT_F16: return route_as<f16_t>(p, stream);
    default: return route_as<bf16_t>(p, stream);
  }
}
hipError_t launch_experts_gate_up(const ExpertsParams& p, hipStream_t stream) {
  if (!valid(p)) return hipErrorInvalidValue;
  const bool f8 = p.w_dt == DT_F8;
  switch (p.dt) {
    case DT_F32: return f8 ? gate_up_as<float, f8_t>(p, stream) : gate_up_as<float, float>(p, stream);
    case DT_F16: return f8 ? gate_up_as<f16_t, f8_t>(p, stream) : gate_up_as<f16_t, f16_t>(p, stream);
    default: return f8 ? gate_up_as<bf16_t, f8_t>(p, stream) : gate_up_as<bf16_t, bf16_t>(p, stream);
  }
}
hipError_t launch_experts_down(const ExpertsParams& p, hipStream_t stream) {
  if (!valid(p)) return hipErrorInvalidValue;
  const bool f8 = p.w_dt == DT_F8;
  switch (p.dt) {
    case DT_F32: return f8 ? down_as<float, f8_t>(p, stream) : down_as<float, float>(p, stream);
    case DT_F16: return f8 ? down_as<f16_t, f8_t>(p, stream) : down_as<f16_t, f16_t>(p, stream);
    default: return f8 ? down_as<bf16_t, f8_t>(p, stream) : down_as<bf16_t, bf16_t>(p, stream);
  }
}

}  // namespace ohip
