// Log probabilities of given tokens, the entropy and the best alternatives of rows of logits:
//
//   M = max l,  rest = sum exp(l - M) without one largest term,  log p_i = (l_i - M) - log1p(rest)
//   entropy = log1p(rest) + (sum exp(l - M) (M - l)) / (1 + rest)
//
// (no term of either cancels another, and a nearly certain token keeps its digits).
//
// Bound by reading the logits once: a workgroup holds its part of a row - up to 32768 logits - in registers, 32 a thread,
// and takes from there the largest, the sums and the alternatives.  Longer rows are several workgroups', whose parts a
// second launch joins.
//
// The alternatives: of 64 groups of threads the top-th largest maximum bounds them from below; what reaches the bound
// (for scattered logits hardly more than `top`) goes to a list in LDS, where every entry counts the entries in front of it.
// Rows with more than 1024 such logits (equal ones, in the main) take the largest of the rest `top` times instead.
#include "block_common.h"

namespace ohip {
namespace {

constexpr int kEach = 32, kGroups = 64, kList = 1024, kWide = 1024, kNarrow = 256;
constexpr float kLog2e = 1.44269504f;
typedef unsigned long long u64;

// Logit and index as one number: larger logits first, equal ones by ascending index; 0 is below all.
__device__ __forceinline__ u64 key_of(const float l, const int i) {
  const unsigned u = __float_as_uint(l + 0.f);      // (-0 and 0 are one logit)
  return (u64)((u & 0x80000000u) ? ~u : u | 0x80000000u) << 32 | (unsigned)~i;
}
__device__ __forceinline__ float logit_of(const u64 k) {
  const unsigned u = (unsigned)(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

// What a part of a row, or all of it, adds up to.
struct Sums {
  float most;    // the largest logit
  float count;   // how often
  float low;     // sum of exp(l - most) over the others
  float away;    // sum of exp(l - most) (most - l)
};
struct RowResult { float most, log_sum; };
// log p of logit l (NaN counts as -inf)
__device__ __forceinline__ float log_prob_of(const RowResult& r, const float l) {
  if (!(l > -INFINITY)) return -INFINITY;
  return (l == r.most ? 0.f : l - r.most) - r.log_sum;
}
__device__ __forceinline__ RowResult finish_row(const LogProbsParams& p, const int row, const Sums& s) {
  const bool any = s.most > -INFINITY;
  const float rest = (s.count - 1.f) + s.low;
  const RowResult r = {s.most, any ? log1pf(rest) : 0.f};
  if (threadIdx.x == 0) p.entropy[row] = any ? r.log_sum + s.away / (1.f + rest) : 0.f;
  if ((int)threadIdx.x < p.per_row) {
    const int64_t at = (int64_t)row * p.per_row + threadIdx.x;
    const int t = p.tokens[at];
    float l = -INFINITY;
    if (t >= 0 && t < p.V) {
      const int64_t i = (int64_t)row * p.V + t;
      l = p.dt == DT_F32 ? reinterpret_cast<const float*>(p.logits)[i] : p.dt == DT_F16 ? Store<f16_t>::ld(reinterpret_cast<const f16_t*>(p.logits) + i)
                                                                                        : Store<bf16_t>::ld(reinterpret_cast<const bf16_t*>(p.logits) + i);
    }
    p.log_prob[at] = log_prob_of(r, l);
  }
  return r;
}
__device__ __forceinline__ void put_alternative(const LogProbsParams& p, const int64_t row, const int place, const u64 key, const RowResult& r) {
  p.top_log_prob[row * p.top + place] = key == 0 ? -INFINITY : log_prob_of(r, logit_of(key));
  p.top_token[row * p.top + place] = key == 0 ? -1 : (int)~(unsigned)key;
}

// Work space: the Sums of every part of every row, then `top` keys for each.
__host__ __device__ inline int64_t keys_at(const LogProbsParams& p, const int parts) { return (int64_t)p.rows * parts * (int64_t)sizeof(Sums); }

template <int NT> struct Room {
  float wave[4][NT / 64];
  float group[kGroups];
  float bound;
  int listed;
  u64 best[NT / 64];
  u64 list[kList];
};

template <typename T, int NT, bool VECTOR>
__global__ void __launch_bounds__(NT, 4) log_probs_kernel(const LogProbsParams p, const int parts, const int each) {
  constexpr int WAVES = NT / 64, LPG = NT / kGroups;
  __shared__ Room<NT> room;
  const int part = blockIdx.x % (unsigned)parts, row = blockIdx.x / (unsigned)parts;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int first = part * each, end = min(p.V, first + each);
  const T* logits = reinterpret_cast<const T*>(p.logits) + (int64_t)row * p.V;
  // logit e of group i: index first + (i NT + tid) 8 + e
  float l[kEach / 8][8];
#pragma unroll
  for (int i = 0; i < kEach / 8; ++i) load8<T, VECTOR>(logits, first + (i * NT + tid) * 8, end, l[i]);
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < kEach / 8; ++i) {
    const int at = first + (i * NT + tid) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      l[i][e] = l[i][e] > -INFINITY && at + e < end ? l[i][e] : -INFINITY;      // (NaN too)
      most = fmaxf(most, l[i][e]);
    }
  }
  const float mine = most;
  const float group = group_allreduce<LPG>(mine, [](float a, float b) { return fmaxf(a, b); });
  if ((tid & (LPG - 1)) == 0) room.group[tid / LPG] = group;
  if (tid == 0) room.listed = 0;
  __syncthreads();
  const float of_group = room.group[lane];
  most = wave_max(of_group);
  if (p.top > 0) {
    // the group whose maximum has top - 1 others in front of it
#pragma unroll 1
    for (int j = wave; j < kGroups; j += WAVES) {
      const float g = room.group[j];
      const int rank = __popcll(__ballot(of_group > g || (of_group == g && lane < j)));
      if (rank == p.top - 1 && lane == 0) room.bound = g;
    }
  }
  Sums s = {most, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // (a distance of 10^4 weighs nothing; -inf, and everything beside infinite logits, is as far)
      const float d = fminf(most - l[i][e], 1e4f);
      const bool top = l[i][e] == most;
      const float w = top ? 0.f : __builtin_amdgcn_exp2f(d * -kLog2e);
      s.count += top ? 1.f : 0.f;
      s.low += w;
      s.away = __builtin_fmaf(w, d, s.away);
    }
  s.count = wave_sum(s.count);
  s.low = wave_sum(s.low);
  s.away = wave_sum(s.away);
  if (lane == 0) { room.wave[0][wave] = s.count; room.wave[1][wave] = s.low; room.wave[2][wave] = s.away; }
  __syncthreads();
  s.count = s.low = s.away = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) { s.count += room.wave[0][w]; s.low += room.wave[1][w]; s.away += room.wave[2][w]; }
  RowResult r = {0.f, 0.f};
  Sums* sums = reinterpret_cast<Sums*>(p.work) + (int64_t)row * parts + part;
  if (parts == 1) r = finish_row(p, row, s);
  else if (tid == 0) *sums = s;
  if (p.top == 0) return;

  u64* keys = reinterpret_cast<u64*>(reinterpret_cast<char*>(p.work) + keys_at(p, parts)) + ((int64_t)row * parts + part) * p.top;
  auto put = [&](const int place, const u64 key) {
    if (parts == 1) put_alternative(p, row, place, key, r);
    else keys[place] = key;
  };
  const float bound = room.bound;
  if (mine >= bound && mine > -INFINITY) {
#pragma unroll
    for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (l[i][e] >= bound && l[i][e] > -INFINITY) {
          const int at = atomicAdd(&room.listed, 1);
          if (at < kList) room.list[at] = key_of(l[i][e], first + (i * NT + tid) * 8 + e);
        }
  }
  __syncthreads();
  const int n = room.listed;
  if (n <= kList) {
    for (int c = tid; c < n; c += NT) {
      const u64 key = room.list[c];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += room.list[j] > key;
      if (rank < p.top) put(rank, key);
    }
    for (int place = n + tid; place < p.top; place += NT) put(place, 0);
    return;
  }
  u64 last = ~0ull;
#pragma unroll 1
  for (int place = 0; place < p.top; ++place) {
    u64 best = 0;
#pragma unroll
    for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const u64 key = key_of(l[i][e], first + (i * NT + tid) * 8 + e);
        if (l[i][e] > -INFINITY && key < last && key > best) best = key;
      }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const u64 other = __shfl_xor(best, o);
      best = other > best ? other : best;
    }
    __syncthreads();      // (the last round's have been read)
    if (lane == 0) room.best[wave] = best;
    __syncthreads();
    best = room.best[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) best = room.best[w] > best ? room.best[w] : best;
    if (tid == 0) put(place, best);
    last = best;
  }
}

// One workgroup a row: its parts' sums in their order, and the best of their alternatives.
constexpr int kMostParts = (kMaxVocabulary + kWide * kEach - 1) / (kWide * kEach);
__global__ void __launch_bounds__(256) log_probs_join_kernel(const LogProbsParams p, const int parts) {
  __shared__ u64 list[kMostParts * kMaxAlternatives];
  const int row = blockIdx.x, n = parts * p.top;
  const u64* keys = reinterpret_cast<const u64*>(reinterpret_cast<const char*>(p.work) + keys_at(p, parts)) + (int64_t)row * n;
  for (int c = threadIdx.x; c < n; c += 256) list[c] = keys[c];
  const Sums* sums = reinterpret_cast<const Sums*>(p.work) + (int64_t)row * parts;
  Sums s = {-INFINITY, 0.f, 0.f, 0.f};
  for (int k = 0; k < parts; ++k) s.most = fmaxf(s.most, sums[k].most);
  for (int k = 0; k < parts; ++k) {
    const Sums a = sums[k];
    if (!(a.most > -INFINITY)) continue;
    if (a.most == s.most) {
      s.count += a.count;
      s.low += a.low;
      s.away += a.away;
    } else {
      const float d = fminf(s.most - a.most, 1e4f), f = __builtin_amdgcn_exp2f(d * -kLog2e), w = a.count + a.low;
      s.low = __builtin_fmaf(f, w, s.low);
      s.away = __builtin_fmaf(f, __builtin_fmaf(d, w, a.away), s.away);
    }
  }
  __syncthreads();
  const RowResult r = finish_row(p, row, s);
  for (int c = threadIdx.x; c < n; c += 256) {
    const u64 key = list[c];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > key || (list[j] == key && j < c);      // (places without a logit are alike)
    if (rank < p.top) put_alternative(p, row, rank, key, r);
  }
}

template <typename T>
hipError_t log_probs_as(const LogProbsParams& p, const int parts, hipStream_t stream) {
  // (parts begin at whole groups of eight, so at 16-byte boundaries where rows do)
  const int each = ((p.V + parts - 1) / parts + 7) / 8 * 8;
  const dim3 grid((unsigned)p.rows * parts);
  if (p.V <= kNarrow * kEach) {
    if (p.V % 8 == 0) hipLaunchKernelGGL((log_probs_kernel<T, kNarrow, true>), grid, dim3(kNarrow), 0, stream, p, parts, each);
    else hipLaunchKernelGGL((log_probs_kernel<T, kNarrow, false>), grid, dim3(kNarrow), 0, stream, p, parts, each);
  } else {
    if (p.V % 8 == 0) hipLaunchKernelGGL((log_probs_kernel<T, kWide, true>), grid, dim3(kWide), 0, stream, p, parts, each);
    else hipLaunchKernelGGL((log_probs_kernel<T, kWide, false>), grid, dim3(kWide), 0, stream, p, parts, each);
  }
  return hipGetLastError();
}

}  // namespace

int log_probs_parts(const LogProbsParams& p) { return (p.V + kWide * kEach - 1) / (kWide * kEach); }
size_t log_probs_space(const LogProbsParams& p) {
  const int parts = log_probs_parts(p);
  return (size_t)(keys_at(p, parts) + (int64_t)p.rows * parts * p.top * (int64_t)sizeof(u64));
}

hipError_t launch_log_probs(const LogProbsParams& p, hipStream_t stream) {
  const int parts = log_probs_parts(p);
  switch (p.dt) {
    case DT_F32: return log_probs_as<float>(p, parts, stream);
    case DT_F16: return log_probs_as<f16_t>(p, parts, stream);
    case DT_BF16: return log_probs_as<bf16_t>(p, parts, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_log_probs_join(const LogProbsParams& p, hipStream_t stream) {
  hipLaunchKernelGGL(log_probs_join_kernel, dim3((unsigned)p.rows), dim3(256), 0, stream, p, log_probs_parts(p));
  return hipGetLastError();
}

}  // namespace ohip
