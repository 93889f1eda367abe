// The next token of every row of logits: temperature, top-k, top-p, min-p and one given random number.
//
//   w_i = exp((l_i - max l) / T);  ranking by l, ties by ascending index
//   kept = the first of the ranking as far as top-k, top-p and min-p all go
//   token = lowest kept i with  sum of kept w up to i  >  u * sum of kept w
//
// A token is a whole number: whether a sum passes a border must not hang on the order of additions or
// on the last bits of an exponential.  Weights are exponentials in 64 bits, rounded to whole multiples
// of 2^-44 of the largest; up to 2^19 of them add up exactly in 64-bit integers, in any order.
//
// One workgroup per row.  A pass over the row reads it from L2 or the last-level cache (the first from memory),
// but what it costs is instructions: one per element is four cycles of a SIMD for 64 of them, a weight twenty of
// them in 64 bits, and a wavefront's additions to counters in LDS 36 cycles (32 bits) or 100 (64).  Kernel times
// of 256 x 128256 fp32 (24 us to read once) and 1 x 32000 fp32: the largest 25 and 6 us, temperature alone 62 and
// 17, top-k of 50 48 and 15, top-p 117 and 30.  So:
//   1  the largest logit of every thread (half an instruction per element), and of all;
//   2  where the ranking is cut, by bins of equal width in (max - l) / T (the logits' leading bits would
//      put most of a row into a few bins, whose counters then take turns).  Top-k: the k-th of the
//      threads' largest is a bound, found among those 1024.  Top-p: weights are added by bins, but only of
//      elements in front of the place behind which too little weight is left;
//   3  top-k: everything from the bound on goes to a list in LDS (not many more than k), where the cut,
//      top-p, min-p and the draw are settled; top-p alone: the elements of the one bin, which give the cut;
//   4  without a list: the kept weights, added by parts of 256 vectors; the part where the sum passes u is
//      looked at once more by one wavefront.
// Rows whose cut is not found that way (thousands of equal logits, top-k in the thousands) take a
// radix descent over the logits' bits as ordered 32-bit keys, a pass for each of three digits.
#include "block_common.h"

namespace ohip {
namespace {

constexpr int kThreads = 1024, kWavesPerRow = kThreads / 64, kBins = 2048;
constexpr int kList = 4096;     // candidates that are settled in LDS
constexpr int kBorder = 1024;   // elements of one bin that are ranked against each other: n / 1024 n steps
constexpr double kOne = 17592186044416.0;   // 2^44: the largest weight
constexpr int kPowers = 1024;
static_assert(kPowers == kThreads, "a thread makes one of the powers");
typedef unsigned long long u64;

// Order of floats as unsigned numbers: -inf and NaN give 0x007fffff, everything that can be drawn more.
constexpr unsigned kKeyOfMinusInf = 0x007fffffu;
__device__ __forceinline__ unsigned key_of(const float l) {
  const unsigned u = __float_as_uint(l);
  if (l != l) return kKeyOfMinusInf;
  if (l == 0.f) return 0x80000000u;   // (-0 and 0 are one logit)
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(const unsigned k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
// a before b in the ranking
__device__ __forceinline__ bool before(const float la, const int ia, const float lb, const int ib) { return la > lb || (la == lb && ia < ib); }

struct Shared {
  u64 sum[kBins];
  unsigned count[kBins];
  float logit[kList];
  int index[kList];
  int border[kBorder];
  double power[kPowers];       // 2^(44 + j / kPowers)
  u64 wave_a[kWavesPerRow], wave_b[kWavesPerRow];
  float wave_f[kWavesPerRow];
  int listed, bordered;
  int bin;                     // results of find()
  u64 front;
  float cut_l;
  int cut_at;
};

struct Row {
  float most;         // the largest logit
  float per_f;        // log2(e) / temperature
  float per_bin;      // bins per unit of (max - l)
  double most_d, per; // kPowers of the exponent's units per unit of (l - max), in 64 bits
  double floor;       // (so many of those units that a weight rounds to nothing)
  const double* power;
};
// 2^44 exp((l - max) / T) = 2^n 2^(44 + j / 1024) 2^f with |f| <= 1 / 2048, the last as its series, whose terms
// from f^4 on are below 2^-50.  1024 y is rounded by adding 1.5 * 2^52, which leaves it in the sum's low
// word; 2^n goes straight into the exponent of the power from the table.  The product and its rounding to a whole
// number are one fused operation: the sum with 2^52 has it in its low bits, nearest even.  Nineteen instructions
// and no branch.  NaN weighs what `floor` does: nothing, but all of it in a row with infinite logits, where `floor` is 0
// and everything weighs the same: there the cut leaves out what is not infinite.
struct Factors { double series, power; };
__device__ __forceinline__ Factors factors(const Row& r, const float l) {
  const double y = __builtin_fmax(((double)l - r.most_d) * r.per, r.floor);
  const double t = y + 6755399441055744.0;
  const double f = y - (t - 6755399441055744.0);
  const int k = (int)(unsigned)(u64)__double_as_longlong(t);
  double p = __builtin_fma(f, 5.169222938345892e-11, 2.290978498068816e-7);   // (ln(2) / 1024)^3 / 3!, ^2 / 2!
  p = __builtin_fma(p, f, 6.769015435155716e-4);
  p = __builtin_fma(p, f, 1.0);
  const u64 power = (u64)__double_as_longlong(r.power[k & (kPowers - 1)]);
  const unsigned hi = (unsigned)(power >> 32) + ((unsigned)(k & -kPowers) << 10);
  return {p, __longlong_as_double((long long)((u64)hi << 32 | (unsigned)power))};
}
__device__ __forceinline__ double weight(const Row& r, const float l) {      // before it is rounded
  const Factors f = factors(r, l);
  return f.series * f.power;
}
__device__ __forceinline__ u64 whole_weight(const Row& r, const float l) {
  const Factors f = factors(r, l);
  return (u64)__double_as_longlong(__builtin_fma(f.series, f.power, 4503599627370496.0)) & 0xfffffffffffffull;
}
// The histogram's bin, not decreasing as l falls; 0 for the largest, kBins for what lies behind the last.
__device__ __forceinline__ int bin_of(const Row& r, const float l) {
  const float x = (r.most - l) * r.per_bin;       // NaN (infinite logits or temperatures) counts as far away
  return l == r.most ? 0 : (int)fminf(x, (float)kBins);
}

// What bin_of gives may lie behind the last bin and still have a weight: max - l beyond fp32, or so low a
// temperature that log2(e) / T is.  Nothing is added then; a cut that the bins do not hold is found by descent.
template <typename N>
__device__ __forceinline__ void add_to_bin(N* bins, const int b, const N n) {
  if (b < kBins) atomicAdd(&bins[b], n);
}

// Sums over the lanes up to one's own, by DPP (no trip through LDS): the shifts inside rows of 16,
// then the last lane of a row to the next row, and of the first half to the second.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_u64(const u64 v) {
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xf, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xf, false);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 scan(u64 v) {
  v += dpp_u64<0x111, 0xf>(v);
  v += dpp_u64<0x112, 0xf>(v);
  v += dpp_u64<0x114, 0xf>(v);
  v += dpp_u64<0x118, 0xf>(v);
  v += dpp_u64<0x142, 0xa>(v);
  v += dpp_u64<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ u64 last_lane(const u64 v) {
  const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, 63), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), 63);
  return (u64)hi << 32 | lo;
}
// Sum over the workgroup; `room` may be in use until the call.
__device__ __forceinline__ u64 block_sum_u64(u64 v, u64* room) {
  v = scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) room[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < kWavesPerRow; ++i) v += room[i];
  return v;
}

// s->bin = the first bin whose value together with those in front of it reaches `need` (>= 1), s->front
// = what stands in front.  Returns the sum of all; where that is less than `need` there is no such bin.
template <typename N>
__device__ __forceinline__ u64 find(Shared* s, const N* bins, const u64 need) {
  const int tid = threadIdx.x, wave = tid >> 6;
  const u64 a = bins[2 * tid], b = bins[2 * tid + 1];
  u64 v = scan(a + b);
  if ((tid & 63) == 63) s->wave_b[wave] = v;
  __syncthreads();
  u64 all = 0;
#pragma unroll
  for (int i = 0; i < kWavesPerRow; ++i) {
    const u64 w = s->wave_b[i];
    v += i < wave ? w : 0;
    all += w;
  }
  const u64 front = v - a - b;
  if (front < need && v >= need) {
    const bool first = front + a >= need;
    s->bin = 2 * tid + (first ? 0 : 1);
    s->front = front + (first ? 0 : a);
  }
  __syncthreads();
  return all;
}

__device__ __forceinline__ void clear(u64* sum) {
  sum[threadIdx.x] = 0ull;
  sum[threadIdx.x + kThreads] = 0ull;
}
__device__ __forceinline__ void clear(unsigned* count) {
  count[threadIdx.x] = 0u;
  count[threadIdx.x + kThreads] = 0u;
}

// ---- the row in vectors of 16 bytes ----
template <typename T>
struct RowReader {
  static constexpr int PER = 16 / sizeof(T);
  const T* row;
  int V;
  __device__ __forceinline__ Vec16<T> whole_vector(const int v) const {
    Vec16<T> x;
    x.raw = reinterpret_cast<const Bytes16*>(row + (int64_t)v * PER)->v;
    return x;
  }
  __device__ __forceinline__ Vec16<T> vector(const int v) const {   // -inf behind the row's end
    if ((v + 1) * PER <= V) return whole_vector(v);
    Vec16<T> x;
#pragma unroll
    for (int e = 0; e < PER; ++e) x.set(e, v * PER + e < V ? Store<T>::ld(row + v * PER + e) : -__builtin_inff());
    return x;
  }
  // f(vector's number, vector, 0 .. 3) for all of the row, four vectors of a thread requested at a time
  template <typename F>
  __device__ __forceinline__ void each_vector(F f) const {
    const int full = V / PER;
    for (int v0 = threadIdx.x; v0 < full; v0 += 4 * kThreads) {
      Vec16<T> x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v0 + j * kThreads < full) x[j] = whole_vector(v0 + j * kThreads);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v0 + j * kThreads < full) f(v0 + j * kThreads, x[j], j);
    }
    if (full * PER < V && threadIdx.x == 0) f(full, vector(full), 0);
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {    // f(index, logit)
    each_vector([&](const int v, const Vec16<T>& x, const int) {
#pragma unroll
      for (int e = 0; e < PER; ++e) f(v * PER + e, x.get(e));
    });
  }
  // f(index, logit) for every element of the vectors where some lane has one with test(logit)
  template <typename P, typename F>
  __device__ __forceinline__ void each_in(P test, F f) const {
    each_vector([&](const int v, const Vec16<T>& x, const int) {
      bool any = false;
#pragma unroll
      for (int e = 0; e < PER; ++e) any = any || test(x.get(e));
      if (any)
        for (int e = 0; e < PER; ++e) {
          const float l = x.get(e);
          if (test(l)) f(v * PER + e, l);
        }
    });
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  __shared__ Shared s;
  constexpr int PER = RowReader<T>::PER, MINE = kList / kThreads;
  const int row_i = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const RowReader<T> row{(const T*)p.logits + (int64_t)row_i * p.V, p.V};
  const int V = p.V;
  const float temperature = p.temperature ? p.temperature[(int64_t)row_i * p.step_t] : 1.f;
  const int top_k = p.top_k ? p.top_k[(int64_t)row_i * p.step_k] : 0;
  const float top_p = p.top_p ? p.top_p[(int64_t)row_i * p.step_p] : 1.f;
  const float min_p = p.min_p ? p.min_p[(int64_t)row_i * p.step_m] : 0.f;
  const float u = p.uniform[(int64_t)row_i * p.step_u];

  // ---- 1: the largest logit, and the vector where it first stands ----
  // (each_vector's four vectors of a turn apart: four samples of a thread's elements)
  float own[4] = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
  int own_v[4] = {0, 0, 0, 0};
  row.each_vector([&](const int v, const Vec16<T>& x, const int j) {
    float m = x.get(0);
#pragma unroll
    for (int e = 1; e < PER; ++e) m = fmaxf(m, x.get(e));     // (a NaN is passed over)
    if (m > own[j]) { own[j] = m; own_v[j] = v; }
  });
  float best = own[0];
  int best_v = own_v[0];
#pragma unroll
  for (int j = 1; j < 4; ++j)
    if (own[j] > best || (own[j] == best && own_v[j] < best_v)) { best = own[j]; best_v = own_v[j]; }
  u64 pair = (u64)key_of(best) << 32 | (unsigned)~best_v;
  for (int d = 32; d > 0; d >>= 1) {
    const u64 o = __shfl_xor(pair, d);
    pair = o > pair ? o : pair;
  }
  if (lane == 0) s.wave_a[wave] = pair;
  s.power[tid] = exp2(44.0 + tid * 0.0009765625);
  if (tid == 0) s.listed = s.bordered = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWavesPerRow; ++i) pair = s.wave_a[i] > pair ? s.wave_a[i] : pair;
  const unsigned top_key = (unsigned)(pair >> 32);
  Row r;
  r.most = logit_of(top_key);
  if (top_key <= kKeyOfMinusInf || !(temperature > 0.f) || top_k == 1 || min_p > 1.f) {   // nothing to draw from, or one token left
    if (tid == 0) {
      const int v = (int)~(unsigned)pair;
      const Vec16<T> x = row.vector(v);
      int at = -1;
#pragma unroll
      for (int e = PER - 1; e >= 0; --e) at = x.get(e) == r.most ? v * PER + e : at;
      p.token[row_i] = top_key <= kKeyOfMinusInf ? -1 : at;
    }
    return;
  }
  r.per_f = 1.4426950408889634f / temperature;
  // (infinite logits: those alone are kept, and all weigh the same)
  const bool infinite = r.most == __builtin_inff();
  r.most_d = infinite ? 0.0 : (double)r.most;
  r.per = infinite ? 0.0 : 1024.0 * 1.4426950408889634 / (double)temperature;
  r.floor = infinite ? 0.0 : -60.0 * 1024.0;
  r.per_bin = (float)kBins / 45.1f * r.per_f;   // (weights round to nothing behind 2^-45)
  r.power = s.power;
  const double least = (double)min_p * kOne;    // (NaN: nothing is below)

  // The elements up to (cut_l, cut_at) in the ranking are kept.
  float cut_l = infinite ? r.most : -3.402823466e38f;
  int cut_at = V;
  auto in_cut = [&](const float l, const int i) { return (bool)((int)(l > cut_l) | ((int)(l == cut_l) & (int)(i <= cut_at))); };

  // Radix descent among the elements kept so far: the last that a cut at `need` (elements, or weight) keeps
  // becomes the new cut.  That much must be there.
  auto descend = [&](const bool by_sum, u64 need) {
    unsigned prefix = 0, known = 0;
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
      const unsigned mask = level == 2 ? 1023u : 2047u;
      clear(s.count);
      clear(s.sum);
      __syncthreads();
      row.each([&](const int i, const float l) {
        if (!in_cut(l, i)) return;
        const unsigned k = key_of(l);
        if ((k & known) != prefix) return;
        const unsigned b = mask - ((k >> shift) & mask);    // (the highest digit first)
        if (by_sum) atomicAdd(&s.sum[b], whole_weight(r, l));
        else atomicAdd(&s.count[b], 1u);
      });
      __syncthreads();
      if (by_sum) find(&s, s.sum, need);
      else find(&s, s.count, need);
      need -= s.front;
      prefix |= (mask - (unsigned)s.bin) << shift;
      known |= mask << shift;
      __syncthreads();
    }
    // `need` is what the elements equal to the key still have to give: the first `ties` of them,
    // counted by parts of the row
    const float l0 = logit_of(prefix);
    const u64 w = whole_weight(r, l0);
    const u64 ties = by_sum ? (w ? (need + w - 1) / w : 1) : need;
    const int part = (V + kBins - 1) / kBins;
    clear(s.count);
    __syncthreads();
    row.each([&](const int i, const float l) {
      if (l == l0 && in_cut(l, i)) atomicAdd(&s.count[i / part], 1u);
    });
    __syncthreads();
    find(&s, s.count, ties);
    if (tid == 0) {
      u64 seen = s.front;
      int i = s.bin * part;
      for (; i < V; ++i)
        if (Store<T>::ld(row.row + i) == l0 && in_cut(l0, i) && ++seen == ties) break;
      s.cut_at = i;
    }
    __syncthreads();
    cut_l = l0;
    cut_at = s.cut_at;
    __syncthreads();
  };

  bool listed = false;      // the candidates are in s.logit / s.index
  // of them this thread's, strided; weight 0, bin kBins + 1: not kept
  u64 kept_w[MINE];
  float kept_l[MINE];
  int kept_i[MINE], kept_bin[MINE];

  bool cut_k = top_k > 0 && top_k < V;
  if (cut_k && top_k <= kList / 2) {
    // ---- 2: a bound that at least top_k elements reach.  The bin of the top_k-th of the threads' largest, and the
    // least of those up to it (fewer than that exist, or it lies behind the bins: the descent); any, where the
    // list holds the row ----
    float bound = -3.402823466e38f;
    bool bounded = V <= kList;
    if (!bounded) {
      clear(s.count);
      __syncthreads();
      int own_bin[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        own_bin[j] = own[j] > -__builtin_inff() ? bin_of(r, own[j]) : kBins;
        add_to_bin(s.count, own_bin[j], 1u);
      }
      __syncthreads();
      bounded = find(&s, s.count, (u64)top_k) >= (u64)top_k;
      if (bounded) {
        float least_own = r.most;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (own_bin[j] <= s.bin) least_own = fminf(least_own, own[j]);
        bound = -block_max<kThreads>(-least_own, s.wave_f);
      }
    }
    if (bounded) {
      // ---- 3: the candidates, and their bins ----
      clear(s.count);
      __syncthreads();
      row.each_in([&](const float l) { return l >= bound; }, [&](const int i, const float l) {
        const int n = atomicAdd(&s.listed, 1);
        if (n < kList) {
          s.logit[n] = l;
          s.index[n] = i;
          add_to_bin(s.count, bin_of(r, l), 1u);
        }
      });
      __syncthreads();
      const int n = s.listed;
      const bool cut = n >= top_k;     // (the list may hold a row with fewer)
      if (n <= kList && (!cut || find(&s, s.count, (u64)top_k) >= (u64)top_k)) {
        const int edge = cut ? s.bin : kBins + 1;
        const unsigned front = (unsigned)s.front;
        if (!cut || s.count[edge] <= kBorder) {
          listed = true;
#pragma unroll
          for (int j = 0; j < MINE; ++j) {
            const int c = tid + j * kThreads;
            kept_l[j] = c < n ? s.logit[c] : 0.f;
            kept_i[j] = c < n ? s.index[c] : 0;
            kept_bin[j] = c < n ? bin_of(r, kept_l[j]) : kBins + 1;
            if (cut && kept_bin[j] == edge) s.border[atomicAdd(&s.bordered, 1)] = c;
          }
          __syncthreads();
          const int m = s.bordered;
          if (tid == 0 && !cut) { s.cut_l = cut_l; s.cut_at = cut_at; }
          if (tid < m) {     // the elements of that bin against each other
            const int c = s.border[tid];
            const float l = s.logit[c];
            const int i = s.index[c];
            unsigned rank = front;
            for (int j = 0; j < m; ++j) rank += before(s.logit[s.border[j]], s.index[s.border[j]], l, i);
            if (rank + 1 == (unsigned)top_k) { s.cut_l = l; s.cut_at = i; }
          }
          __syncthreads();
          cut_l = s.cut_l;
          cut_at = s.cut_at;
          if (infinite && cut_l != r.most) { cut_l = r.most; cut_at = V; }
#pragma unroll
          for (int j = 0; j < MINE; ++j) {
            const bool in = kept_bin[j] <= kBins && in_cut(kept_l[j], kept_i[j]);
            kept_w[j] = in ? whole_weight(r, kept_l[j]) : 0;
            if (!in) kept_bin[j] = kBins + 1;
          }
        }
      }
    }
  }
  if (cut_k && !listed) {
    u64 live = 0;
    row.each([&](const int i, const float l) { live += in_cut(l, i); });
    cut_k = block_sum_u64(live, s.wave_a) > (u64)top_k;
    if (cut_k) descend(false, (u64)top_k);
  }

  if (top_p < 1.f) {
    // ---- 2 and 3 of a cut by weight ----
    u64 total = 0;
    clear(s.sum);
    if (tid == 0) s.bordered = 0;
    if (listed) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < MINE; ++j)
        if (kept_w[j] != 0) {
          total += kept_w[j];
          add_to_bin(s.sum, kept_bin[j], kept_w[j]);
        }
    } else {
      // Behind 2^-e of the largest weight, e = log2(V / ((1 - p) S)) + 1, all elements together weigh at most half
      // of (1 - p) S: the cut is in front of it.  For S, the sum of all weights, serves that of the threads' largest.
      // (After a cut by number that may be too much: the bins then end where weights round to nothing.)
      float e = 45.1f;
      if (!cut_k) {
        float w = __builtin_amdgcn_exp2f((best - r.most) * r.per_f);
        w = block_sum<kThreads>(w >= 0.f && w <= 1.f ? w : 0.f, s.wave_f);
        e = fmaxf(1.f, fminf(e, __log2f((float)V / ((1.f - top_p) * fmaxf(w, 1.f))) + 1.01f));
      }
      r.per_bin = (float)kBins / e * r.per_f;
      const bool whole_row = !cut_k && !infinite;
      __syncthreads();
      row.each_vector([&](const int v, const Vec16<T>& x, const int) {
        u64 w[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const float l = x.get(e);
          w[e] = whole_weight(r, l) & ((int)whole_row | (int)in_cut(l, v * PER + e) ? ~0ull : 0ull);
          total += w[e];
        }
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const int b = bin_of(r, x.get(e));
          if (w[e] != 0) add_to_bin(s.sum, b, w[e]);
        }
      });
    }
    total = block_sum_u64(total, s.wave_a);
    const double want = ceil((double)top_p * (double)total);
    const u64 need = want > 1.0 ? (u64)want : 1ull;
    if (need < total) {
      const bool binned = find(&s, s.sum, need) >= need;
      const int edge = s.bin;
      const u64 front = s.front;
      // the elements of that bin, ranked against each other (their logits and indices in s.logit / s.index;
      // s.sum is done with and takes their weights)
      if (binned && listed) {
#pragma unroll
        for (int j = 0; j < MINE; ++j)
          if (kept_bin[j] == edge) {
            const int n = atomicAdd(&s.bordered, 1);
            if (n < kBorder) { s.border[n] = tid + j * kThreads; s.sum[n] = kept_w[j]; }
          }
      } else if (binned) {
        // (logits beside the middle of the bin by more than half of its width, and a little, are not in it)
        const float middle = r.most - ((float)edge + 0.5f) / r.per_bin;
        const float half = 0.5f / r.per_bin + 1e-5f * (fabsf(r.most) + fabsf(middle));
        row.each_in([&](const float l) { return !(fabsf(l - middle) > half); }, [&](const int i, const float l) {
          if (l > -__builtin_inff() && bin_of(r, l) == edge && in_cut(l, i)) {
            const int n = atomicAdd(&s.bordered, 1);
            if (n < kBorder) { s.border[n] = n; s.logit[n] = l; s.index[n] = i; s.sum[n] = whole_weight(r, l); }
          }
        });
      }
      __syncthreads();
      const int m = s.bordered;
      if (binned && m <= kBorder) {
        if (tid < m) {
          const int c = s.border[tid];
          const float l = s.logit[c];
          const int i = s.index[c];
          u64 ahead = front;
          for (int j = 0; j < m; ++j) ahead += before(s.logit[s.border[j]], s.index[s.border[j]], l, i) ? s.sum[j] : 0;
          if (ahead < need && ahead + s.sum[tid] >= need) { s.cut_l = l; s.cut_at = i; }
        }
        __syncthreads();
        cut_l = s.cut_l;
        cut_at = s.cut_at;
        __syncthreads();
      } else {
        __syncthreads();
        descend(true, need);
        listed = false;
      }
    }
  }

  // ---- 4: the draw ----
  if (listed) {
    // by parts of the row's indices: the part where the sum passes, then its elements against each other
    const int part = (V + kBins - 1) / kBins;
    clear(s.sum);
    if (tid == 0) s.bordered = 0;
    __syncthreads();
    u64 all = 0;
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      if (kept_w[j] == 0 || !in_cut(kept_l[j], kept_i[j]) || weight(r, kept_l[j]) < least) kept_w[j] = 0;
      if (kept_w[j] != 0) { all += kept_w[j]; atomicAdd(&s.sum[kept_i[j] / part], kept_w[j]); }
    }
    all = block_sum_u64(all, s.wave_a);
    const double want = floor((double)u * (double)all);
    u64 target = want > 0.0 ? (u64)want : 0ull;   // the first sum above it
    if (target >= all) target = all - 1;
    find(&s, s.sum, target + 1);
    const int b = s.bin;
    const u64 front = s.front;
    // (at most `part` <= 256 elements; s.sum is done with and takes their weights)
#pragma unroll
    for (int j = 0; j < MINE; ++j)
      if (kept_w[j] != 0 && kept_i[j] / part == b) {
        const int n = atomicAdd(&s.bordered, 1);
        s.border[n] = kept_i[j];
        s.sum[n] = kept_w[j];
      }
    __syncthreads();
    const int m = s.bordered;
    if (tid < m) {
      u64 ahead = front;
      for (int j = 0; j < m; ++j) ahead += s.border[j] < s.border[tid] ? s.sum[j] : 0;
      if (ahead <= target && ahead + s.sum[tid] > target) p.token[row_i] = s.border[tid];
    }
    return;
  }
  auto kept = [&](const int i, const float l) -> u64 {
    const Factors f = factors(r, l);
    const u64 w = (u64)__double_as_longlong(__builtin_fma(f.series, f.power, 4503599627370496.0)) & 0xfffffffffffffull;
    bool in = in_cut(l, i);
    if (least > 0.0) in = (int)in & (int)!(f.series * f.power < least);
    return w & (in ? ~0ull : 0ull);
  };
  // a part is 256 neighbouring vectors of the row, four per lane of a wavefront
  const int vectors = (V + PER - 1) / PER, parts = (vectors + 255) / 256;
  clear(s.sum);
  __syncthreads();
  u64 all = 0;
  for (int part = wave; part < parts; part += kWavesPerRow) {
    Vec16<T> x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = row.vector(part * 256 + j * 64 + lane);
    u64 sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bool any = false;
#pragma unroll
      for (int e = 0; e < PER; ++e) any = any || x[j].get(e) >= cut_l;
      if (any)
#pragma unroll
        for (int e = 0; e < PER; ++e) sum += kept((part * 256 + j * 64 + lane) * PER + e, x[j].get(e));
    }
    sum = scan(sum);
    if (lane == 63) { s.sum[part] = sum; all += sum; }
  }
  all = block_sum_u64(all, s.wave_a);
  const double want = floor((double)u * (double)all);
  u64 target = want > 0.0 ? (u64)want : 0ull;
  if (target >= all) target = all - 1;
  find(&s, s.sum, target + 1);
  if (wave == 0) {
    u64 ahead = s.front;
    Vec16<T> x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = row.vector(s.bin * 256 + j * 64 + lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int v = s.bin * 256 + j * 64 + lane;
      u64 w[PER], sum = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) sum += w[e] = kept(v * PER + e, x[j].get(e));
      const u64 upto = scan(sum);
      u64 at = ahead + upto - sum;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        if (at <= target && at + w[e] > target) p.token[row_i] = v * PER + e;
        at += w[e];
      }
      ahead += last_lane(upto);
    }
  }
}

}  // namespace

hipError_t launch_sample(const SampleParams& p, hipStream_t stream) {
  if (p.logits == nullptr || p.uniform == nullptr || p.token == nullptr || p.rows < 1 || p.V < 1 || p.V > kMaxVocabulary) return hipErrorInvalidValue;
  switch (p.dt) {
    case DT_F32: hipLaunchKernelGGL((sample_kernel<float>), dim3(p.rows), dim3(kThreads), 0, stream, p); break;
    case DT_F16: hipLaunchKernelGGL((sample_kernel<f16_t>), dim3(p.rows), dim3(kThreads), 0, stream, p); break;
    case DT_BF16: hipLaunchKernelGGL((sample_kernel<bf16_t>), dim3(p.rows), dim3(kThreads), 0, stream, p); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace ohip
