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
// One workgroup per row; the row is read again by every pass, from L2.  The cut of the ranking is a
// radix descent over the logits' bits as ordered 32-bit keys (11 + 11 + 10 bits): a pass counts the
// elements and adds the weights of every digit among those that share the digits found so far.
#include "device_utils.h"

namespace ohip {
namespace {

constexpr int kThreads = 1024, kWavesPerRow = kThreads / 64, kBins = 2048;
typedef unsigned long long u64;

// Order of floats as unsigned numbers: -inf gives 0x007fffff, everything that can be drawn more.
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

struct Row {
  float most;         // the largest logit
  double per;         // 1 / temperature
};
__device__ __forceinline__ double weight(const Row& r, const float l) {
  if (l == r.most) return 1.0;
  const double x = ((double)l - (double)r.most) * r.per;
  return x == x ? exp(x) : 0.0;   // (an infinite temperature below an infinite logit)
}
__device__ __forceinline__ u64 fixed(const double w) { return (u64)__double2ull_rn(w * 17592186044416.0); }   // 2^44

__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// The digit of the ranking where a border falls: walking the bins from the highest, the first whose
// elements (BY_SUM: whose weights) reach `need` together with those above it.  cnt / sum: what stands
// above that bin on return.  The border must be reached.
struct Cut { int bin; unsigned above; u64 above_sum; };

struct Shared {
  unsigned count[kBins];
  u64 sum[kBins];
  u64 wave_a[kWavesPerRow];
  u64 wave_b[kWavesPerRow];
  float wave_f[kWavesPerRow];
  int wave_i[kWavesPerRow];
  Cut cut;
  int found;
};

template <typename T>
__device__ __forceinline__ float logit_at(const T* row, const int i) { return Store<T>::ld(row + i); }

// Every thread holds two neighbouring bins of the descending order; the border is found by a scan over the threads.
template <bool BY_SUM>
__device__ void find_cut(Shared* s, const u64 need) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b0 = kBins - 1 - 2 * tid, b1 = b0 - 1;   // b0 ranks before b1
  const u64 v0 = BY_SUM ? s->sum[b0] : s->count[b0], v1 = BY_SUM ? s->sum[b1] : s->count[b1];
  const unsigned c0 = s->count[b0], c1 = s->count[b1];
  const u64 w0 = s->sum[b0], w1 = s->sum[b1];
  u64 v = v0 + v1, c = c0 + c1, w = w0 + w1;
  for (int d = 1; d < 64; d <<= 1) {
    const u64 ov = __shfl_up(v, d), oc = __shfl_up(c, d), ow = __shfl_up(w, d);
    if (lane >= d) { v += ov; c += oc; w += ow; }
  }
  __shared__ u64 tv[kWavesPerRow], tc[kWavesPerRow], tw[kWavesPerRow];
  if (lane == 63) { tv[wave] = v; tc[wave] = c; tw[wave] = w; }
  __syncthreads();
  u64 bv = 0, bc = 0, bw = 0;
  for (int i = 0; i < wave; ++i) { bv += tv[i]; bc += tc[i]; bw += tw[i]; }
  v += bv; c += bc; w += bw;          // inclusive of both bins
  const u64 before = v - v0 - v1;
  if (before < need && v >= need) {
    const bool first = before + v0 >= need;
    s->cut.bin = first ? b0 : b1;
    s->cut.above = (unsigned)(c - c0 - c1 + (first ? 0 : c0));
    s->cut.above_sum = w - w0 - w1 + (first ? 0 : w0);
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  __shared__ Shared s;
  const int row_i = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* row = (const T*)p.logits + (int64_t)row_i * p.V;
  const int V = p.V;
  const float temperature = p.temperature ? p.temperature[(int64_t)row_i * p.step_t] : 1.f;
  const int top_k = p.top_k ? p.top_k[(int64_t)row_i * p.step_k] : 0;
  const float top_p = p.top_p ? p.top_p[(int64_t)row_i * p.step_p] : 1.f;
  const float min_p = p.min_p ? p.min_p[(int64_t)row_i * p.step_m] : 0.f;
  const float u = p.uniform[(int64_t)row_i * p.step_u];

  // ---- the largest logit and its lowest index ----
  unsigned best = 0;
  int at = V;
  for (int i = tid; i < V; i += kThreads) {
    const unsigned k = key_of(logit_at(row, i));
    if (k > best) { best = k; at = i; }
  }
  u64 pair = (u64)best << 32 | (unsigned)~at;
  for (int d = 32; d > 0; d >>= 1) {
    const u64 o = __shfl_xor(pair, d);
    pair = o > pair ? o : pair;
  }
  if (lane == 0) s.wave_a[wave] = pair;
  __syncthreads();
  for (int i = 0; i < kWavesPerRow; ++i) pair = s.wave_a[i] > pair ? s.wave_a[i] : pair;
  __syncthreads();
  const unsigned top_key = (unsigned)(pair >> 32);
  const int first = (int)~(unsigned)pair;
  if (top_key <= kKeyOfMinusInf || !(temperature > 0.f) || top_k == 1 || min_p > 1.f) {   // nothing to draw from, or one token left
    if (tid == 0) p.token[row_i] = top_key <= kKeyOfMinusInf ? -1 : first;
    return;
  }
  Row r;
  r.most = logit_of(top_key);
  r.per = 1.0 / (double)temperature;

  // ---- the cut: everything above cut_key, and of those equal to it the ones up to index cut_at ----
  unsigned cut_key = kKeyOfMinusInf + 1;
  int cut_at = V;
  auto descend = [&](auto by_sum, u64 need, const unsigned floor_key, const int floor_at, u64* reached) {
    constexpr bool BY_SUM = decltype(by_sum)::value;
    // among elements with key > floor_key, or key == floor_key and index <= floor_at
    unsigned prefix = 0, fixed_bits = 0;
    u64 sum_above = 0;
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
      const unsigned bins_mask = level == 2 ? 1023u : 2047u;
      for (int i = tid; i < kBins; i += kThreads) { s.count[i] = 0u; s.sum[i] = 0ull; }
      __syncthreads();
      for (int i = tid; i < V; i += kThreads) {
        const float l = logit_at(row, i);
        const unsigned k = key_of(l);
        if ((k & fixed_bits) != prefix || k < floor_key || (k == floor_key && i > floor_at)) continue;
        const unsigned b = (k >> shift) & bins_mask;
        atomicAdd(&s.count[b], 1u);
        const u64 w = fixed(weight(r, l));
        if (w != 0) atomicAdd(&s.sum[b], w);
      }
      __syncthreads();
      find_cut<BY_SUM>(&s, need);
      const Cut c = s.cut;
      need -= BY_SUM ? c.above_sum : c.above;
      sum_above += c.above_sum;
      prefix |= (unsigned)c.bin << shift;
      fixed_bits |= bins_mask << shift;
      __syncthreads();
    }
    // `need` is what the elements equal to the key still have to give: the first `ties` of them
    const u64 w = fixed(weight(r, logit_of(prefix)));
    const u64 ties = BY_SUM ? (w ? (need + w - 1) / w : 1) : need;
    cut_key = prefix;
    *reached = sum_above + ties * w;
    // the index of the last tie kept: wavefronts own neighbouring segments
    const int per = (V + kWavesPerRow - 1) / kWavesPerRow;
    const int lo = wave * per, hi = min(V, lo + per);
    unsigned mine = 0;
    for (int i = lo; i < hi; i += 64) {
      const bool tie = i + lane < hi && key_of(logit_at(row, i + lane)) == prefix && !(prefix == floor_key && i + lane > floor_at);
      mine += (unsigned)__popcll(__ballot(tie));
    }
    if (lane == 0) s.wave_i[wave] = (int)mine;
    if (tid == 0) s.found = V;
    __syncthreads();
    u64 before = 0;
    for (int i = 0; i < wave; ++i) before += (u64)s.wave_i[i];
    if (before < ties && before + mine >= ties) {
      u64 seen = before;
      for (int i = lo; i < hi; i += 64) {
        const bool tie = i + lane < hi && key_of(logit_at(row, i + lane)) == prefix && !(prefix == floor_key && i + lane > floor_at);
        const u64 votes = __ballot(tie);
        const unsigned here = (unsigned)__popcll(votes);
        if (seen + here >= ties) {
          const unsigned rank = (unsigned)__popcll(votes & ((1ull << lane) - 1ull));
          if (tie && seen + rank + 1 == ties) s.found = i + lane;
          break;
        }
        seen += here;
      }
    }
    __syncthreads();
    cut_at = s.found;
    __syncthreads();
  };

  // how many can be drawn at all, and their weights together
  unsigned live = 0;
  u64 total = 0;
  for (int i = tid; i < V; i += kThreads) {
    const float l = logit_at(row, i);
    if (key_of(l) <= kKeyOfMinusInf) continue;
    ++live;
    total += fixed(weight(r, l));
  }
  total = wave_sum_u64(total);
  u64 live64 = wave_sum_u64(live);
  if (lane == 0) { s.wave_a[wave] = total; s.wave_b[wave] = live64; }
  __syncthreads();
  total = 0; live64 = 0;
  for (int i = 0; i < kWavesPerRow; ++i) { total += s.wave_a[i]; live64 += s.wave_b[i]; }
  __syncthreads();

  if (top_k > 0 && (u64)top_k < live64) descend(std::false_type(), (u64)top_k, cut_key, cut_at, &total);
  if (top_p < 1.f) {
    const double want = ceil((double)top_p * (double)total);
    u64 need = want > 1.0 ? (u64)want : 1ull;
    if (need < total) {
      u64 dropped;
      descend(std::true_type(), need, cut_key, cut_at, &dropped);
    }
  }

  // ---- the draw: wavefronts own neighbouring segments of the row ----
  auto kept = [&](const int i, u64* w) {
    const float l = logit_at(row, i);
    const unsigned k = key_of(l);
    if (k < cut_key || (k == cut_key && i > cut_at)) return false;
    const double d = weight(r, l);
    if (d < (double)min_p) return false;
    *w = fixed(d);
    return true;
  };
  const int per = ((V + kWavesPerRow - 1) / kWavesPerRow + 63) / 64 * 64;
  const int lo = min(V, wave * per), hi = min(V, lo + per);
  u64 mine = 0;
  for (int i = lo + lane; i < hi; i += 64) {
    u64 w;
    if (kept(i, &w)) mine += w;
  }
  mine = wave_sum_u64(mine);
  if (lane == 0) s.wave_a[wave] = mine;
  if (tid == 0) s.found = -1;
  __syncthreads();
  u64 all = 0, before = 0;
  for (int i = 0; i < kWavesPerRow; ++i) { if (i < wave) before += s.wave_a[i]; all += s.wave_a[i]; }
  const double want = floor((double)u * (double)all);
  u64 target = want > 0.0 ? (u64)want : 0ull;   // the first sum above it
  if (target >= all) target = all - 1;
  if (before <= target && before + mine > target) {
    u64 seen = before;
    for (int i = lo; i < hi; i += 64) {
      u64 w = 0;
      if (i + lane < hi && !kept(i + lane, &w)) w = 0;
      u64 upto = w;
      for (int d = 1; d < 64; d <<= 1) {
        const u64 o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
      }
      const u64 here = __shfl(upto, 63);
      if (seen + here > target) {
        if (seen + upto > target && seen + upto - w <= target) s.found = i + lane;
        break;
      }
      seen += here;
    }
  }
  __syncthreads();
  if (tid == 0) p.token[row_i] = s.found;
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
