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
// One workgroup per row.  A pass over the row reads it from L2 (the first from memory); what a row
// costs is its passes and the exponentials in them, so that there are few of either:
//   1  the largest logit and its index (a greedy row ends here);
//   2  a histogram over 2048 bins of equal width in (max - l) / T - equal width and not the logits'
//      leading bits, because those put most of a row into a few bins, whose counters then take turns.
//      With top-k it counts (no exponentials), otherwise it adds weights; it names the bin where the
//      ranking is cut;
//   3  top-k: everything up to that bin goes to a list in LDS (a few more than k elements), where
//      top-p, min-p and the draw are settled; top-p alone: the elements of the one bin, which give the cut;
//   4  without a list: the kept weights, added by 64 x 16 bytes of the row (a wavefront's vectors of one
//      iteration); the part where the sum passes u is looked at once more by one wavefront.
// Rows whose cut is not found that way (thousands of equal logits, top-k in the thousands) take a
// radix descent over the logits' bits as ordered 32-bit keys, a pass for each of three digits.
#include "block_common.h"

namespace ohip {
namespace {

constexpr int kThreads = 1024, kWavesPerRow = kThreads / 64, kBins = 2048;
constexpr int kList = 4096;     // candidates that are settled in LDS
constexpr int kBorder = 1024;   // elements of one bin that are ranked against each other: n / 1024 n steps
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

struct Shared {
  u64 sum[kBins];
  unsigned count[kBins];
  unsigned key[kList];
  int index[kList];
  int border[kBorder];
  double power[64];            // 2^(j / 64)
  u64 wave_a[kWavesPerRow], wave_b[kWavesPerRow];
  int listed, bordered, found;
  // result of find()
  int bin;
  u64 before;
  unsigned cut_key;
  int cut_at;
};

struct Row {
  float most;         // the largest logit
  float per_bin;      // bins per unit of (max - l)
  double per;         // log2(e) / temperature
  const double* power;
};
// 2^44 exp((l - max) / T) in 64 bits: 2^y = 2^n 2^(j / 64) 2^f with |f| <= 1 / 128, the last as its
// series, whose terms from f^6 on are below 2^-55.
__device__ __forceinline__ double weight(const Row& r, const float l) {
  const double y = ((double)l - (double)r.most) * r.per;
  if (!(y >= -64.0)) return l == r.most ? 17592186044416.0 : 0.0;   // (NaN: infinite logits or temperatures)
  const double k = rint(y * 64.0), f = y - k * 0.015625;
  const int i = (int)k;
  double p = 1.3333558146428443e-3;               // ln(2)^5 / 5!
  p = __builtin_fma(p, f, 9.6181291076284770e-3);
  p = __builtin_fma(p, f, 5.5504108664821580e-2);
  p = __builtin_fma(p, f, 2.4022650695910072e-1);
  p = __builtin_fma(p, f, 6.9314718055994531e-1);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p * r.power[i & 63], (i >> 6) + 44);
}
// ... as a whole number: the sum with 2^52 has it in its low bits, rounded to nearest even.
__device__ __forceinline__ u64 whole(const double w) {
  return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
}
// The histogram's bin, not decreasing as l falls; 0 for the largest.
__device__ __forceinline__ int bin_of(const Row& r, const float l) {
  const float x = (r.most - l) * r.per_bin;       // NaN (infinite logits or temperatures) counts as far away
  return l == r.most ? 0 : (int)fminf(x, (float)(kBins - 1));
}

__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ u64 block_sum_u64(u64 v, u64* room) {
  v = wave_sum_u64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < kWavesPerRow; ++i) v += room[i];
  return v;
}

// s->bin = the first bin whose value together with those in front of it reaches `need` (>= 1), s->before
// = what stands in front.  Some bin must.
template <typename N>
__device__ __forceinline__ void find(Shared* s, const N* bins, const u64 need) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const u64 a = bins[2 * tid], b = bins[2 * tid + 1];
  u64 v = a + b;
  for (int d = 1; d < 64; d <<= 1) {
    const u64 o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  if (lane == 63) s->wave_b[wave] = v;
  __syncthreads();
  for (int i = 0; i < kWavesPerRow; ++i) v += i < wave ? s->wave_b[i] : 0;
  const u64 front = v - a - b;
  if (front < need && v >= need) {
    const bool first = front + a >= need;
    s->bin = 2 * tid + (first ? 0 : 1);
    s->before = front + (first ? 0 : a);
  }
  __syncthreads();
}

__device__ __forceinline__ void clear(u64* sum) {
  sum[threadIdx.x] = 0ull;
  sum[threadIdx.x + kThreads] = 0ull;
}
__device__ __forceinline__ void clear(unsigned* count) {
  count[threadIdx.x] = 0u;
  count[threadIdx.x + kThreads] = 0u;
}

// ---- the row in vectors of 16 bytes: vector j * 1024 + tid in iteration j ----
template <typename T>
struct RowReader {
  static constexpr int PER = 16 / sizeof(T);
  const T* row;
  int V;
  // f(index, logit) for every element, four vectors of a thread requested at a time
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const int full = V / PER;
    for (int v0 = threadIdx.x; v0 < full; v0 += 4 * kThreads) {
      Vec16<T> x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v0 + j * kThreads < full) x[j].raw = reinterpret_cast<const Bytes16*>(row + (int64_t)(v0 + j * kThreads) * PER)->v;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v0 + j * kThreads < full)
#pragma unroll
          for (int e = 0; e < PER; ++e) f((v0 + j * kThreads) * PER + e, x[j].get(e));
    }
    const int rest = full * PER + (int)threadIdx.x;
    if (rest < V) f(rest, Store<T>::ld(row + rest));
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  __shared__ Shared s;
  const int row_i = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const RowReader<T> row{(const T*)p.logits + (int64_t)row_i * p.V, p.V};
  const int V = p.V;
  const float temperature = p.temperature ? p.temperature[(int64_t)row_i * p.step_t] : 1.f;
  const int top_k = p.top_k ? p.top_k[(int64_t)row_i * p.step_k] : 0;
  const float top_p = p.top_p ? p.top_p[(int64_t)row_i * p.step_p] : 1.f;
  const float min_p = p.min_p ? p.min_p[(int64_t)row_i * p.step_m] : 0.f;
  const float u = p.uniform[(int64_t)row_i * p.step_u];
  if (tid < 64) s.power[tid] = exp2(tid * 0.015625);
  if (tid == 0) s.listed = s.bordered = 0;

  // ---- 1: the largest logit, its lowest index, and how many can be drawn ----
  unsigned best = 0;
  int at = V;
  unsigned live = 0;
  row.each([&](const int i, const float l) {
    const unsigned k = key_of(l);
    if (k > best || (k == best && i < at)) { best = k; at = i; }
    live += k > kKeyOfMinusInf;
  });
  u64 pair = (u64)best << 32 | (unsigned)~at;
  for (int d = 32; d > 0; d >>= 1) {
    const u64 o = __shfl_xor(pair, d);
    pair = o > pair ? o : pair;
  }
  if (lane == 0) s.wave_a[wave] = pair;
  __syncthreads();
  for (int i = 0; i < kWavesPerRow; ++i) pair = s.wave_a[i] > pair ? s.wave_a[i] : pair;
  const unsigned top_key = (unsigned)(pair >> 32);
  const int first = (int)~(unsigned)pair;
  if (top_key <= kKeyOfMinusInf || !(temperature > 0.f) || top_k == 1 || min_p > 1.f) {   // nothing to draw from, or one token left
    if (tid == 0) p.token[row_i] = top_key <= kKeyOfMinusInf ? -1 : first;
    return;
  }
  const u64 live_all = block_sum_u64(live, s.wave_b);
  Row r;
  r.most = logit_of(top_key);
  r.per = 1.4426950408889634 / (double)temperature;
  // (a weight rounds to nothing from (max - l) / T = 45 ln 2 = 31.2 on: the last bin takes all of those)
  r.per_bin = (float)kBins / 31.25f / temperature;
  r.power = s.power;
  const double least = (double)min_p * 17592186044416.0;   // (NaN: nothing is below)

  // Of everything at or above the first cut: the elements before and at (cut_key, cut_at) in the ranking are kept.
  unsigned cut_key = kKeyOfMinusInf + 1;
  int cut_at = V;
  auto in_cut = [&](const unsigned k, const int i) { return k > cut_key || (k == cut_key && i <= cut_at); };

  // Radix descent among the elements kept so far: the last that a cut at `need` (elements, or weight) keeps
  // becomes the new cut; the weight of all that remain is returned.
  auto descend = [&](const bool by_sum, u64 need) -> u64 {
    unsigned prefix = 0, known = 0;
    u64 sum_front = 0;
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
      const unsigned mask = level == 2 ? 1023u : 2047u;
      clear(s.count);
      clear(s.sum);
      __syncthreads();
      row.each([&](const int i, const float l) {
        const unsigned k = key_of(l);
        if ((k & known) != prefix || !in_cut(k, i)) return;
        const unsigned b = mask - ((k >> shift) & mask);    // (the highest digit first)
        atomicAdd(&s.count[b], 1u);
        const u64 w = whole(weight(r, l));
        if (w != 0) atomicAdd(&s.sum[b], w);
      });
      __syncthreads();
      if (by_sum) find(&s, s.sum, need); else find(&s, s.count, need);
      const int b = s.bin;
      need -= s.before;
      u64 front = 0;      // weight of the digits in front
      for (int i = tid; i < b; i += kThreads) front += s.sum[i];
      sum_front += block_sum_u64(front, s.wave_a);
      prefix |= (mask - (unsigned)b) << shift;
      known |= mask << shift;
      __syncthreads();
    }
    // `need` is what the elements equal to the key still have to give: the first `ties` of them
    const u64 w = whole(weight(r, logit_of(prefix)));
    const u64 ties = by_sum ? (w ? (need + w - 1) / w : 1) : need;
    // the index of the last of them: ties counted by parts of 2048 / V of the row
    const int part = (V + kBins - 1) / kBins;
    clear(s.count);
    __syncthreads();
    row.each([&](const int i, const float l) {
      if (key_of(l) == prefix && in_cut(prefix, i)) atomicAdd(&s.count[i / part], 1u);
    });
    __syncthreads();
    find(&s, s.count, ties);
    if (tid == 0) {
      u64 seen = s.before;
      int i = s.bin * part;
      for (; i < V; ++i)
        if (key_of(Store<T>::ld(row.row + i)) == prefix && in_cut(prefix, i) && ++seen == ties) break;
      s.cut_at = i;
    }
    __syncthreads();
    cut_key = prefix;
    cut_at = s.cut_at;
    __syncthreads();
    return sum_front + ties * w;
  };

  bool listed = false;      // the candidates are in s.key / s.index
  // of them this thread's, strided; weight 0, bin kBins: not kept
  u64 kept_w[kList / kThreads];
  unsigned kept_key[kList / kThreads];
  int kept_i[kList / kThreads], kept_bin[kList / kThreads];

  const bool cut_k = top_k > 0 && (u64)top_k < live_all;
  if (cut_k) {
    // ---- 2: where the k-th element stands ----
    clear(s.count);
    __syncthreads();
    row.each([&](const int i, const float l) {
      if (key_of(l) > kKeyOfMinusInf) atomicAdd(&s.count[bin_of(r, l)], 1u);
    });
    __syncthreads();
    find(&s, s.count, (u64)top_k);
    const int last = s.bin;
    const unsigned front = (unsigned)s.before, in_bin = s.count[last];
    if (front + in_bin <= kList && in_bin <= kBorder) {
      // ---- 3: those up to its bin, and the elements of the bin against each other ----
      listed = true;
      row.each([&](const int i, const float l) {
        const unsigned k = key_of(l);
        if (k <= kKeyOfMinusInf) return;
        const int b = bin_of(r, l);
        if (b > last) return;
        const int n = atomicAdd(&s.listed, 1);
        s.key[n] = k;
        s.index[n] = i;
        if (b == last) s.border[atomicAdd(&s.bordered, 1)] = n;
      });
      __syncthreads();
      const int n = s.listed, m = s.bordered;
      if (tid < m) {
        const int c = s.border[tid];
        const unsigned k = s.key[c];
        const int i = s.index[c];
        unsigned rank = front;
        for (int j = 0; j < m; ++j) {
          const int o = s.border[j];
          rank += s.key[o] > k || (s.key[o] == k && s.index[o] < i);
        }
        if (rank + 1 == (unsigned)top_k) { s.cut_key = k; s.cut_at = i; }
      }
      __syncthreads();
      cut_key = s.cut_key;
      cut_at = s.cut_at;
#pragma unroll
      for (int j = 0; j < kList / kThreads; ++j) {
        const int c = tid + j * kThreads;
        kept_w[j] = 0;
        kept_key[j] = 0;
        kept_i[j] = 0;
        kept_bin[j] = kBins;
        if (c < n && in_cut(s.key[c], s.index[c])) {
          kept_key[j] = s.key[c];
          kept_i[j] = s.index[c];
          const float l = logit_of(s.key[c]);
          kept_bin[j] = bin_of(r, l);
          kept_w[j] = whole(weight(r, l));
        }
      }
    }
  }

  u64 total = 0;     // weight of what top-k keeps, where top-p asks for it
  if (cut_k && !listed) total = descend(false, (u64)top_k);

  if (top_p < 1.f) {
    // ---- 2 and 3 of a cut by weight ----
    clear(s.sum);
    if (tid == 0) s.bordered = 0;
    __syncthreads();
    if (listed) {
#pragma unroll
      for (int j = 0; j < kList / kThreads; ++j)
        if (kept_w[j] != 0) { total += kept_w[j]; atomicAdd(&s.sum[kept_bin[j]], kept_w[j]); }
    } else {
      total = 0;
      row.each([&](const int i, const float l) {
        const unsigned k = key_of(l);
        if (!in_cut(k, i)) return;
        const u64 w = whole(weight(r, l));
        if (w != 0) { total += w; atomicAdd(&s.sum[bin_of(r, l)], w); }
      });
    }
    total = block_sum_u64(total, s.wave_a);
    const double want = ceil((double)top_p * (double)total);
    const u64 need = want > 1.0 ? (u64)want : 1ull;
    if (need < total) {
      find(&s, s.sum, need);
      const int last = s.bin;
      const u64 front = s.before;
      // the elements of that bin, ranked against each other (their keys and indices in s.key / s.index;
      // s.sum is done with and takes their weights)
      if (listed) {
        // (the list itself: positions of its elements)
#pragma unroll
        for (int j = 0; j < kList / kThreads; ++j)
          if (kept_bin[j] == last) {
            const int n = atomicAdd(&s.bordered, 1);
            if (n < kBorder) { s.border[n] = tid + j * kThreads; s.sum[n] = kept_w[j]; }
          }
      } else {
        row.each([&](const int i, const float l) {
          const unsigned k = key_of(l);
          if (!in_cut(k, i) || bin_of(r, l) != last) return;
          const int n = atomicAdd(&s.bordered, 1);
          if (n < kBorder) { s.border[n] = n; s.key[n] = k; s.index[n] = i; s.sum[n] = whole(weight(r, l)); }
        });
      }
      __syncthreads();
      const int m = s.bordered;
      if (m <= kBorder) {
        if (tid < m) {
          const int c = s.border[tid];
          const unsigned k = s.key[c];
          const int i = s.index[c];
          u64 before = front;
          for (int j = 0; j < m; ++j) {
            const int o = s.border[j];
            before += s.key[o] > k || (s.key[o] == k && s.index[o] < i) ? s.sum[j] : 0;
          }
          if (before < need && before + s.sum[tid] >= need) { s.cut_key = k; s.cut_at = i; }
        }
        __syncthreads();
        cut_key = s.cut_key;
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
    for (int j = 0; j < kList / kThreads; ++j) {
      if (kept_w[j] == 0 || !in_cut(kept_key[j], kept_i[j]) || weight(r, logit_of(kept_key[j])) < least) kept_w[j] = 0;
      if (kept_w[j] != 0) { all += kept_w[j]; atomicAdd(&s.sum[kept_i[j] / part], kept_w[j]); }
    }
    all = block_sum_u64(all, s.wave_a);
    const double want = floor((double)u * (double)all);
    u64 target = want > 0.0 ? (u64)want : 0ull;   // the first sum above it
    if (target >= all) target = all - 1;
    find(&s, s.sum, target + 1);
    const int b = s.bin;
    const u64 front = s.before;
    // (at most `part` <= 256 elements; s.sum is done with and takes their weights)
#pragma unroll
    for (int j = 0; j < kList / kThreads; ++j)
      if (kept_w[j] != 0 && kept_i[j] / part == b) {
        const int n = atomicAdd(&s.bordered, 1);
        s.border[n] = kept_i[j];
        s.sum[n] = kept_w[j];
      }
    __syncthreads();
    const int m = s.bordered;
    if (tid < m) {
      u64 before = front;
      for (int j = 0; j < m; ++j) before += s.border[j] < s.border[tid] ? s.sum[j] : 0;
      if (before <= target && before + s.sum[tid] > target) p.token[row_i] = s.border[tid];
    }
    return;
  }
  constexpr int PER = RowReader<T>::PER;
  auto kept = [&](const int i, const float l) -> u64 {
    if (!in_cut(key_of(l), i)) return 0;
    const double w = weight(r, l);
    return w < least ? 0 : whole(w);
  };
  // a wavefront's vectors of iteration j are part 16 j + wave of the row, 64 x PER elements
  const int vectors = (V + PER - 1) / PER, parts = (vectors + 63) / 64;
  clear(s.sum);
  __syncthreads();
  u64 all = 0;
  auto vector_sum = [&](const int v, u64 (&w)[PER]) {   // of vector v, and its weights
    u64 sum = 0;
    if ((v + 1) * PER <= V) {
      Vec16<T> x;
      x.raw = reinterpret_cast<const Bytes16*>(row.row + (int64_t)v * PER)->v;
#pragma unroll
      for (int e = 0; e < PER; ++e) sum += w[e] = kept(v * PER + e, x.get(e));
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e) sum += w[e] = v * PER + e < V ? kept(v * PER + e, Store<T>::ld(row.row + v * PER + e)) : 0;
    }
    return sum;
  };
  for (int part = wave; part < parts; part += kWavesPerRow) {
    u64 w[PER];
    const u64 sum = wave_sum_u64(vector_sum(part * 64 + lane, w));
    all += sum;
    if (lane == 0) s.sum[part] = sum;
  }
  all = block_sum_u64(lane == 0 ? all : 0, s.wave_a);
  const double want = floor((double)u * (double)all);
  u64 target = want > 0.0 ? (u64)want : 0ull;
  if (target >= all) target = all - 1;
  find(&s, s.sum, target + 1);
  if (wave == 0) {
    u64 w[PER];
    const u64 sum = vector_sum(s.bin * 64 + lane, w);
    u64 upto = sum;
    for (int d = 1; d < 64; d <<= 1) {
      const u64 o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    u64 before = s.before + upto - sum;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (before <= target && before + w[e] > target) p.token[row_i] = (s.bin * 64 + lane) * PER + e;
      before += w[e];
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
