// Log probabilities of given tokens, the entropy and the best alternatives of rows of logits:
//
//   M = max l,  rest = sum exp(l - M) without one largest term,  log p_i = (l_i - M) - log1p(rest)
//   entropy = log1p(rest) + (sum exp(l - M) (M - l)) / (1 + rest)
//
// (no term of either cancels another, and a nearly certain token keeps its digits).
//
// Bound by reading the logits once: 256 x 128256 fp32 with 20 alternatives, 131 MB, 30 us and 5 for the join; 4001 x 32000 bf16 without
// any, 256 MB, 49 us, 5.2 TB/s.  One row of 32000 fp32 logits is one compute unit's: 9 us, two memory latencies and the alternatives.
// A workgroup holds its part of a row - up to 32768 logits - in registers, 32 a thread,
// and takes from there the largest, the sums and the alternatives.  Longer rows are several workgroups', whose parts a
// second launch joins.
//
// The alternatives: of 64 groups of threads the top-th largest maximum bounds them from below; what reaches the bound
// (for scattered logits hardly more than `top`) goes to a list in LDS, where every entry counts the entries in front of it.
// Rows with more than 1024 such logits (equal ones, or the largest side by side) take the largest of the rest `top` times instead: 1 x 32000 and
// 256 x 128256 fp32 logits sorted by size, 20 alternatives, 120 and 556 us for 9 and 30.
#include "block_common.h"

namespace ohip {
namespace {

constexpr int kEach = 32, kGroups = 64, kList = 1024, kWide = 1024, kNarrow = 256, kManyRows = 1024;
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
  float rest;    // sum of exp(l - most) over the others
  float away;    // sum of exp(l - most) (most - l)
};
struct RowResult { float most, log_sum; };
// log p of logit l (NaN counts as -inf)
__device__ __forceinline__ float log_prob_of(const RowResult& r, const float l) {
  if (!(l > -INFINITY)) return -INFINITY;
  return (l == r.most ? 0.f : l - r.most) - r.log_sum;
}
// (by the first wavefront of a row's; me: thread of those)
__device__ __forceinline__ RowResult finish_row(const LogProbsParams& p, const int row, const Sums& s, const int me) {
  const bool any = s.most > -INFINITY;
  const RowResult r = {s.most, any ? log1pf(s.rest) : 0.f};
  if (me == 0) p.entropy[row] = any ? r.log_sum + s.away / (1.f + s.rest) : 0.f;
  if (me < p.per_row) {
    const int64_t at = (int64_t)row * p.per_row + me;
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
__host__ __device__ inline int64_t keys_at(const LogProbsParams& p, const int parts) { return ((int64_t)p.rows * parts * (int64_t)sizeof(Sums) + 7) / 8 * 8; }

// A thread's 32 logits as they are in memory: group i are those from index first + (i NT + tid) 8 on; -inf behind the end.
template <typename T> struct Group { unsigned w[2 * sizeof(T)]; };
template <typename T> __device__ __forceinline__ float logit_at(const Group<T>& g, const int e) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(g.w[e]);
  else if constexpr (std::is_same<T, f16_t>::value) return f16_to_f32((uint16_t)(g.w[e >> 1] >> (16 * (e & 1))));
  else return __uint_as_float(e & 1 ? g.w[e >> 1] & 0xffff0000u : g.w[e >> 1] << 16);
}
template <typename T, bool VECTOR>
__device__ __forceinline__ Group<T> load_whole_group(const T* from) {
  Group<T> g;
#pragma unroll
  for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
    uintx4 v;
    if constexpr (VECTOR) v = *reinterpret_cast<const uintx4*>(from + h * (16 / (int)sizeof(T)));
    else v = reinterpret_cast<const Bytes16*>(from + h * (16 / (int)sizeof(T)))->v;
#pragma unroll
    for (int j = 0; j < 4; ++j) g.w[4 * h + j] = v[j];
  }
  return g;
}
template <typename T, bool VECTOR>
__device__ __forceinline__ Group<T> load_group(const T* row, const int at, const int end) {
  Group<T> g;
  if (at + 8 <= end) {
    g = load_whole_group<T, VECTOR>(row + at);
  } else {
    constexpr unsigned out = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, f16_t>::value ? 0xfc00u : 0xff80u;
#pragma unroll
    for (int j = 0; j < 2 * (int)sizeof(T); ++j) {
      if constexpr (sizeof(T) == 4) {
        g.w[j] = at + j < end ? reinterpret_cast<const unsigned*>(row)[at + j] : out;
      } else {
        const unsigned lo = at + 2 * j < end ? row[at + 2 * j].bits : out, hi = at + 2 * j + 1 < end ? row[at + 2 * j + 1].bits : out;
        g.w[j] = lo | hi << 16;
      }
    }
  }
  return g;
}

template <int NT> struct Room {
  Sums wave[NT / 64];
  float group[kGroups];
  float bound;
  int listed;
  u64 best[NT / 64];
  u64 list[kList];
};

// Sums of parts (lane l has one; `n` of them, the first lanes), in every lane.
__device__ __forceinline__ Sums joined(Sums s, const bool have) {
  if (!have) s = {-INFINITY, 0.f, 0.f};
  const float most = wave_max(s.most);
  const bool top = s.most == most;
  const float d = fminf(most - s.most, 1e4f), f = top ? 1.f : __builtin_amdgcn_exp2f(d * -kLog2e), all = 1.f + s.rest;
  const int first = __builtin_ctzll(__ballot(top));      // (the others' largest are terms like any other)
  return {most, wave_sum((int)(threadIdx.x & 63) == first ? s.rest : f * all), wave_sum(top ? s.away : f * __builtin_fmaf(d, all, s.away))};
}

// The `top` best of a part whose logits reach the bound too often: the largest behind the last one, again and again.
template <typename T, int NT>
__device__ __noinline__ void best_by_rounds(const T* logits, const int first, const int end, const int top, Room<NT>& room, u64* keys) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 last = ~0ull;
#pragma unroll 1
  for (int place = 0; place < top; ++place) {
    u64 best = 0;
#pragma unroll 1
    for (int i = first + (int)threadIdx.x; i < end; i += NT) {
      const float l = Store<T>::ld(logits + i);
      const u64 key = key_of(l, i);
      if (l > -INFINITY && key < last && key > best) best = key;
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
#pragma unroll 1
    for (int w = 1; w < NT / 64; ++w) best = room.best[w] > best ? room.best[w] : best;
    if (threadIdx.x == 0) keys[place] = best;
    last = best;
  }
}

// Sums are of a wavefront's logits around its own largest, so that nothing is waited for before they are complete.
// Per logit: widen, maximum (half an instruction), difference, its bound, exponent, exponential (as long as four others),
// two sums.
template <typename T, int NT, bool VECTOR, bool TOP>
__global__ void __launch_bounds__(NT, NT == kWide ? 8 : 6) log_probs_kernel(const LogProbsParams p, const int parts, const int each) {
  constexpr int WAVES = NT / 64, LPG = NT / kGroups;
  __shared__ Room<NT> room;
  const int part = blockIdx.x % (unsigned)parts, row = blockIdx.x / (unsigned)parts;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int first = part * each, end = min(p.V, first + each);
  const T* logits = reinterpret_cast<const T*>(p.logits) + (int64_t)row * p.V;
  Group<T> l[kEach / 8];
#pragma unroll
  for (int i = 0; i < kEach / 8; ++i) l[i] = load_group<T, VECTOR>(logits, first + (i * NT + tid) * 8, end);
  float mine = -INFINITY;       // (NaN is no maximum)
#pragma unroll
  for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) mine = fmaxf(mine, logit_at<T>(l[i], e));
  if constexpr (TOP) {
    const float group = group_allreduce<LPG>(mine, [](float a, float b) { return fmaxf(a, b); });
    if ((tid & (LPG - 1)) == 0) room.group[tid / LPG] = group;
    if (tid == 0) room.listed = 0;
  }
  const float most = wave_max(mine);
  float sum = 0.f, away = 0.f;
#pragma unroll
  for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // (a distance of 10^4 weighs nothing; -inf, NaN, and everything beside infinite logits, is as far)
      const float d = fminf(most - logit_at<T>(l[i], e), 1e4f), w = __builtin_amdgcn_exp2f(d * -kLog2e);
      sum += w;
      away = __builtin_fmaf(w, d, away);
    }
  Sums s = {most, wave_sum(sum) - 1.f, wave_sum(away)};
  // What little is left beside the largest has lost digits to it: it is added once more without.  (A wavefront whose logits
  // are all -inf comes here too; one with infinities has no weight of its own for them.)
  if (!(s.rest > 3.f)) {
    sum = 0.f;
    int equal = 0;
    float again = most;      // (hidden from the compiler, which would keep all 32 differences for this)
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("" : "+v"(again));
#endif
#pragma unroll
    for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = logit_at<T>(l[i], e);
        const bool top = x == again;
        equal += __popcll(__ballot(top));
        sum += top ? 0.f : __builtin_amdgcn_exp2f(fminf(again - x, 1e4f) * -kLog2e);
      }
    s.rest = wave_sum(sum) + (float)(equal - 1);
  }
  if (lane == 0) room.wave[wave] = s;
  __syncthreads();
  const Sums of_row = joined(room.wave[lane & (WAVES - 1)], lane < WAVES);
  if constexpr (TOP) {
    // the group whose maximum has top - 1 others in front of it
    const float of_group = room.group[lane];
#pragma unroll 1
    for (int j = wave; j < kGroups; j += WAVES) {
      const float g = room.group[j];
      const int rank = __popcll(__ballot(of_group > g || (of_group == g && lane < j)));
      if (rank == p.top - 1 && lane == 0) room.bound = g;
    }
  }
  RowResult r = {0.f, 0.f};
  if (parts == 1) r = finish_row(p, row, of_row, tid);
  else if (tid == 0) reinterpret_cast<Sums*>(p.work)[(int64_t)row * parts + part] = of_row;
  if constexpr (TOP) {
    u64* keys = reinterpret_cast<u64*>(reinterpret_cast<char*>(p.work) + keys_at(p, parts)) + ((int64_t)row * parts + part) * p.top;
    auto put = [&](const int place, const u64 key) {
      if (parts == 1) put_alternative(p, row, place, key, r);
      else keys[place] = key;
    };
    __syncthreads();
    const float bound = room.bound;
    if (mine >= bound && mine > -INFINITY) {
#pragma unroll
      for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = logit_at<T>(l[i], e);
          if (x >= bound && x > -INFINITY) {
            const int at = atomicAdd(&room.listed, 1);
            if (at < kList) room.list[at] = key_of(x, first + (i * NT + tid) * 8 + e);
          }
        }
    }
    __syncthreads();
    int n = room.listed;
    if (n > kList) {
      best_by_rounds<T, NT>(logits, first, end, p.top, room, room.list);
      __syncthreads();
      n = p.top;
    }
    for (int c = tid; c < n; c += NT) {
      const u64 key = room.list[c];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += room.list[j] > key || (room.list[j] == key && j < c);      // (places without a logit are alike)
      if (rank < p.top) put(rank, key);
    }
    for (int place = n + tid; place < p.top; place += NT) put(place, 0);
  }
}

// Many rows without alternatives: a wavefront each, which streams its row with a running maximum a lane and waits for
// nobody.  What the lane of the largest has added to that one's 1 has lost digits: its logits are added once more
// by all lanes, without it.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(256) log_probs_stream_kernel(const LogProbsParams p) {
  constexpr int N = 4, STEP = 64 * 8 * N;      // groups of eight a lane at a time
  const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= p.rows) return;
  const T* logits = reinterpret_cast<const T*>(p.logits) + (int64_t)row * p.V;
  float m = -INFINITY, sum = 0.f, away = 0.f;
  Group<T> next[N];
#pragma unroll
  for (int i = 0; i < N; ++i) next[i] = load_group<T, VECTOR>(logits, (i * 64 + lane) * 8, p.V);
#pragma unroll 1
  for (int at = 0; at < p.V; at += STEP) {
    Group<T> l[N];
#pragma unroll
    for (int i = 0; i < N; ++i) l[i] = next[i];
    if (at + 2 * STEP <= p.V) {
#pragma unroll
      for (int i = 0; i < N; ++i) next[i] = load_whole_group<T, VECTOR>(logits + at + STEP + (i * 64 + lane) * 8);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) next[i] = load_group<T, VECTOR>(logits, at + STEP + (i * 64 + lane) * 8, p.V);
    }
    float most = m;       // (NaN is no maximum)
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, logit_at<T>(l[i], e));
    // (a distance of 10^4 weighs nothing; -inf, NaN, and everything beside infinite logits, is as far)
    const float up = fminf(most - m, 1e4f), f = most == m ? 1.f : __builtin_amdgcn_exp2f(up * -kLog2e);
    away = most == m ? away : f * __builtin_fmaf(up, sum, away);
    sum *= f;
    m = most;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = fminf(most - logit_at<T>(l[i], e), 1e4f), w = __builtin_amdgcn_exp2f(d * -kLog2e);
        sum += w;
        away = __builtin_fmaf(w, d, away);
      }
  }
  const float most = wave_max(m), d = fminf(most - m, 1e4f), f = m == most ? 1.f : __builtin_amdgcn_exp2f(d * -kLog2e);
  const int owner = __builtin_ctzll(__ballot(m == most));
  Sums s = {most, wave_sum(lane == owner ? 0.f : f * sum), wave_sum(m == most ? away : f * __builtin_fmaf(d, sum, away))};
  // the owner's groups, or all where infinite logits share the row
  const bool whole = most == INFINITY;
  const int stride = whole ? 1 : 64, first = whole ? 0 : owner;
  float again = 0.f, equal = 0.f;
  for (int k = lane; (k * stride + first) * 8 < p.V; k += 64) {
    const Group<T> l = load_group<T, VECTOR>(logits, (k * stride + first) * 8, p.V);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = logit_at<T>(l, e);
      again += x == most ? 0.f : __builtin_amdgcn_exp2f(fminf(most - x, 1e4f) * -kLog2e);
      equal += x == most ? 1.f : 0.f;
    }
  }
  s.rest += wave_sum(again) + (wave_sum(equal) - 1.f);
  finish_row(p, row, s, lane);
}

// One workgroup a row: its parts' sums in their order, and the best of their alternatives.
constexpr int kMostParts = (kMaxVocabulary + kWide * kEach - 1) / (kWide * kEach);
__global__ void __launch_bounds__(256) log_probs_join_kernel(const LogProbsParams p, const int parts) {
  __shared__ u64 list[kMostParts * kMaxAlternatives];
  const int row = blockIdx.x, n = parts * p.top;
  const u64* keys = reinterpret_cast<const u64*>(reinterpret_cast<const char*>(p.work) + keys_at(p, parts)) + (int64_t)row * n;
  for (int c = threadIdx.x; c < n; c += 256) list[c] = keys[c];
  const Sums* sums = reinterpret_cast<const Sums*>(p.work) + (int64_t)row * parts;
  const int lane = threadIdx.x & 63;
  const Sums s = joined(sums[min(lane, parts - 1)], lane < parts);
  __syncthreads();
  const RowResult r = finish_row(p, row, s, threadIdx.x);
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
  // From 1024 rows on every SIMD has one to stream.  bf16, a wavefront a row against a workgroup a row: 512 rows of 4096 logits
  // 6.2 and 6.7 us, of 32000 18.7 and 12.7, of 128256 58 and 37; 1024 rows 6.1 and 9.1, 20 and 22, 63 and 63; 2048 rows 7.5
  // and 13.4, 29 and 39, 105 and 123; 4001 rows of 32000 49 and 119.
  if (p.top == 0 && p.rows >= kManyRows) {
    const dim3 waves((unsigned)(p.rows + 3) / 4);
    if (p.V % 8 == 0) hipLaunchKernelGGL((log_probs_stream_kernel<T, true>), waves, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((log_probs_stream_kernel<T, false>), waves, dim3(256), 0, stream, p);
    return hipGetLastError();
  }
#define OHIP_LOG_PROBS(NT, VECTOR)                                                                                                   \
  do {                                                                                                                             \
    if (p.top > 0) hipLaunchKernelGGL((log_probs_kernel<T, NT, VECTOR, true>), grid, dim3(NT), 0, stream, p, parts, each);          \
    else hipLaunchKernelGGL((log_probs_kernel<T, NT, VECTOR, false>), grid, dim3(NT), 0, stream, p, parts, each);                   \
  } while (0)
  // Short rows by 256 threads, of which a compute unit has several workgroups at once.  bf16, 5 alternatives, against 1024 threads: 8192
  // logits 7.3 and 9.0 us for a row, 8.7 and 11 for 256, 18 and 48 for 2048; 2048 logits 8.0 and 9.4, 9.2 and 11, 20 and 50.
  if (p.V <= kNarrow * kEach) {
    if (p.V % 8 == 0) OHIP_LOG_PROBS(kNarrow, true);
    else OHIP_LOG_PROBS(kNarrow, false);
  } else {
    if (p.V % 8 == 0) OHIP_LOG_PROBS(kWide, true);
    else OHIP_LOG_PROBS(kWide, false);
  }
#undef OHIP_LOG_PROBS
  return hipGetLastError();
}

}  // namespace

int log_probs_parts(const LogProbsParams& p) { return p.top == 0 && p.rows >= kManyRows ? 1 : (p.V + kWide * kEach - 1) / (kWide * kEach); }
bool log_probs_fits(const LogProbsParams& p) { return p.V <= kNarrow * kEach || (p.top == 0 && p.rows >= kManyRows) || (int64_t)p.rows * log_probs_parts(p) * kWide <= UINT32_MAX; }
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
