// A layer of experts for few tokens: the router's choice, the gated products of the chosen experts
// and the weighted sum of what they give.
//
//   l = router x, top k of l; w = softmax(l) of those (divided by their sum)
//   h = silu(gate_e x) * (up_e x),   y = sum_j w_j down_ej h_j
//
// Few tokens: bound by the weights of the experts that some token chose, which are read once.  Their
// rows go straight into operand registers of the matrix instructions, sixteen rows a tile; the
// tokens that chose the expert are the columns (up to sixteen at no further cost).
#include "block_common.h"

namespace ohip {
namespace {

// A step of the reduction: 32 bytes of weights per lane, 128 of a row.
template <typename X, typename W>
struct Step {
  static constexpr int ELEMS = 128 / sizeof(W);                  // of a row
  static constexpr int XV = 32 / sizeof(W) * sizeof(X) / 16;     // vectors of x per lane
  template <bool ALIGNED>
  __device__ static __forceinline__ void load_x(const X* row, const int step, const int g, const int len, uintx4 (&x)[XV]) {
    const int64_t at = ((int64_t)step * ELEMS + g * (ELEMS / 4)) * (int64_t)sizeof(X);
#pragma unroll
    for (int v = 0; v < XV; ++v) x[v] = load_row16<ALIGNED>((const unsigned char*)row, at + 16 * v, (int64_t)len * sizeof(X));
  }
  template <bool ALIGNED>
  __device__ static __forceinline__ void load_w(const W* row, const int step, const int g, const int len, uintx4 (&w)[2]) {
    const int64_t at = (int64_t)step * 128 + g * 32;
#pragma unroll
    for (int v = 0; v < 2; ++v) w[v] = load_row16<ALIGNED>((const unsigned char*)row, at + 16 * v, (int64_t)len * sizeof(W));
  }
  __device__ static __forceinline__ floatx4 mma(const uintx4 (&w)[2], const uintx4 (&x)[XV], floatx4 c) {
    if constexpr (sizeof(W) == 1) {
      const unsigned b[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
      for (int v = 0; v < XV; ++v) c = mma_vec<X>(values_of<X>(b, v), x[v], c);
    } else {
      c = mma_vec<X>(w[0], x[0], c);
      c = mma_vec<X>(w[1], x[1], c);
    }
    return c;
  }
};

// Where the choice stands in the work space: expert and weight of every (token, place), then the logits.
__host__ __device__ inline size_t route_weights(const int tokens, const int top_k) { return (size_t)tokens * top_k * 4; }
__host__ __device__ inline size_t route_logits(const int tokens, const int top_k) { return (size_t)tokens * top_k * 8; }

// ---- the router: 16 experts x 16 tokens a workgroup, the wavefronts split H ----
template <typename X, bool ALIGNED>
__global__ void __launch_bounds__(512) experts_logits_kernel(const ExpertsParams p) {
  using S = Step<X, X>;
  __shared__ floatx4 sums[8][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int e0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
  const X* wrow = (const X*)p.router + (int64_t)min(e0 + r, p.E - 1) * p.H;
  const X* xrow = (const X*)p.x + (int64_t)min(t0 + r, p.tokens - 1) * p.H;
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  const int steps = (p.H + S::ELEMS - 1) / S::ELEMS;
#pragma unroll 2
  for (int s = wave; s < steps; s += waves) {
    uintx4 w[2], x[S::XV];
    S::template load_w<ALIGNED>(wrow, s, g, p.H, w);
    S::template load_x<ALIGNED>(xrow, s, g, p.H, x);
    acc = S::mma(w, x, acc);
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

// Order of floats as unsigned numbers; a NaN comes before everything.
__device__ __forceinline__ unsigned ordered(const float f) {
  const unsigned u = __float_as_uint(f);
  return f != f ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// ---- the choice: a wavefront per token ----
__global__ void __launch_bounds__(64) experts_choice_kernel(const ExpertsParams p) {
  constexpr int PER = kMaxExperts / 64;
  const int t = blockIdx.x, lane = threadIdx.x;
  const float* logits = (const float*)((const char*)p.route + route_logits(p.tokens, p.top_k)) + (int64_t)t * p.E;
  int* ids = (int*)p.route + (int64_t)t * p.top_k;
  float* weights = (float*)((char*)p.route + route_weights(p.tokens, p.top_k)) + (int64_t)t * p.top_k;
  unsigned long long key[PER];   // value, then the lower index first; 0: taken or none
  float most = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 64 * i;
    key[i] = 0;
    if (e < p.E) {
      const float l = logits[e];
      most = fmaxf(most, l);
      key[i] = (unsigned long long)ordered(l) << 32 | (unsigned)~e;
    }
  }
  most = wave_max(most);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 64 * i < p.E) sum += expf(logits[lane + 64 * i] - most);
  sum = wave_sum(sum);
  float chosen = 0.f, mine = 0.f;   // sum over the chosen; lane j: exponential of choice j
  for (int j = 0; j < p.top_k; ++j) {
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) best = key[i] > best ? key[i] : best;
    for (int d = 32; d > 0; d >>= 1) {
      const unsigned long long o = __shfl_xor(best, d);
      best = o > best ? o : best;
    }
    const int e = (int)~(unsigned)best;
    const float v = expf(logits[e] - most);
    chosen += v;
    if (lane == j) { mine = v; ids[j] = e; }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (key[i] == best) key[i] = 0;
  }
  // (a NaN among the logits reaches every weight through the whole sum)
  const float by = p.renormalize ? (sum == sum ? chosen : sum) : sum;
  if (lane < p.top_k) weights[lane] = mine / by * p.scaling;
}

// The expert of slot blockIdx.y (experts that some token chose, in ascending order) and the
// (token, place) pairs that chose it; false: there are fewer experts.
struct Chosen {
  unsigned mask[kMaxExperts / 32];
  int list[kMaxExpertTokens];
  int count;
};
__device__ __forceinline__ bool find_expert(const ExpertsParams& p, Chosen* c, int* expert) {
  const int* ids = (const int*)p.route;
  const int n = p.tokens * p.top_k, words = (p.E + 31) / 32;
  for (int i = threadIdx.x; i < words; i += blockDim.x) c->mask[i] = 0u;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) atomicOr(&c->mask[ids[i] >> 5], 1u << (ids[i] & 31));
  __syncthreads();
  int left = blockIdx.y, e = -1;
  for (int w = 0; w < words && e < 0; ++w) {
    unsigned m = c->mask[w];
    const int here = __popc(m);
    if (left >= here) { left -= here; continue; }
    for (; left > 0; --left) m &= m - 1u;
    e = 32 * w + __ffs((int)m) - 1;
  }
  if (e < 0) return false;
  if (threadIdx.x < 64) {
    int at = 0;
    for (int i = 0; i < n; i += 64) {
      const bool hit = i + (int)threadIdx.x < n && ids[i + threadIdx.x] == e;
      const unsigned long long votes = __ballot(hit);
      if (hit) c->list[at + __popcll(votes & ((1ull << threadIdx.x) - 1ull))] = i + threadIdx.x;
      at += __popcll(votes);
    }
    if (threadIdx.x == 0) c->count = at;
  }
  __syncthreads();
  *expert = e;
  return true;
}

// Scales of the four rows row .. row + 3 of a matrix for one block of terms.
__device__ __forceinline__ floatx4 row_scales(const float* s, const int row, const int rows, const int KB, const int kb) {
  floatx4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = s[(int64_t)(min(row + i, rows - 1) / kScaleBlock) * KB + kb];
  return v;
}

constexpr int kWaves = 4;

// ---- hidden[slot][i] = silu(gate x) * (up x): sixteen i of one expert a workgroup, the wavefronts split H ----
template <typename X, typename W, int MT, bool ALIGNED>
__global__ void __launch_bounds__(64 * kWaves) experts_gate_up_kernel(const ExpertsParams p) {
  using S = Step<X, W>;
  __shared__ Chosen chosen;
  __shared__ floatx4 sums[kWaves][2][MT][64];
  int e;
  if (!find_expert(p, &chosen, &e)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int i0 = blockIdx.x * 16;
  const W* base = (const W*)p.gate_up + (int64_t)e * 2 * p.I * p.H;
  const W* rows[2] = {base + (int64_t)min(i0 + r, p.I - 1) * p.H, base + (int64_t)(p.I + min(i0 + r, p.I - 1)) * p.H};
  const int steps = (p.H + S::ELEMS - 1) / S::ELEMS;
  const int RB = (2 * p.I + kScaleBlock - 1) / kScaleBlock;
  const float* scales = sizeof(W) == 1 ? p.gate_up_scale + (int64_t)e * RB * steps : nullptr;
  for (int c0 = 0; c0 < chosen.count; c0 += 16 * MT) {
    const X* xrow[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xrow[t] = (const X*)p.x + (int64_t)(chosen.list[min(c0 + 16 * t + r, chosen.count - 1)] / p.top_k) * p.H;
    floatx4 acc[2][MT];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[h][t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int s = wave; s < steps; s += kWaves) {
      uintx4 w[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) S::template load_w<ALIGNED>(rows[h], s, g, p.H, w[h]);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        uintx4 x[S::XV];
        S::template load_x<ALIGNED>(xrow[t], s, g, p.H, x);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (sizeof(W) == 1) {
            const floatx4 part = S::mma(w[h], x, floatx4{0.f, 0.f, 0.f, 0.f});
            const floatx4 sc = row_scales(scales, h * p.I + i0 + 4 * g, 2 * p.I, steps, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[h][t][i] = __builtin_fmaf(part[i], sc[i], acc[h][t][i]);
          } else {
            acc[h][t] = S::mma(w[h], x, acc[h][t]);
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < MT; ++t) sums[wave][h][t][lane] = acc[h][t];
    __syncthreads();
    for (int t = wave; t < MT; t += kWaves) {
      floatx4 gate = sums[0][0][t][lane], up = sums[0][1][t][lane];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) { gate += sums[w][0][t][lane]; up += sums[w][1][t][lane]; }
      floatx4 h;
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = gate[i] / (1.f + expf(-gate[i])) * up[i];
      const int c = c0 + 16 * t + r, n = i0 + 4 * g;
      if (c < chosen.count && n < p.I) store4((X*)p.hidden + (int64_t)chosen.list[c] * p.I + n, h, p.I - n, (p.I & 3) == 0);
    }
  }
}

// ---- parts[slot][n] = weight * down hidden: sixteen n of one expert a workgroup, the wavefronts split I ----
template <typename X, typename W, int MT, bool ALIGNED>
__global__ void __launch_bounds__(64 * kWaves) experts_down_kernel(const ExpertsParams p) {
  using S = Step<X, W>;
  __shared__ Chosen chosen;
  __shared__ floatx4 sums[kWaves][MT][64];
  int e;
  if (!find_expert(p, &chosen, &e)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const W* row = (const W*)p.down + ((int64_t)e * p.H + min(n0 + r, p.H - 1)) * p.I;
  const int steps = (p.I + S::ELEMS - 1) / S::ELEMS;
  const int RB = (p.H + kScaleBlock - 1) / kScaleBlock;
  const float* scales = sizeof(W) == 1 ? p.down_scale + ((int64_t)e * RB + n0 / kScaleBlock) * steps : nullptr;
  const float* weights = (const float*)((const char*)p.route + route_weights(p.tokens, p.top_k));
  for (int c0 = 0; c0 < chosen.count; c0 += 16 * MT) {
    const X* xrow[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xrow[t] = (const X*)p.hidden + (int64_t)chosen.list[min(c0 + 16 * t + r, chosen.count - 1)] * p.I;
    floatx4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int s = wave; s < steps; s += kWaves) {
      uintx4 w[2];
      S::template load_w<ALIGNED>(row, s, g, p.I, w);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        uintx4 x[S::XV];
        S::template load_x<ALIGNED>(xrow[t], s, g, p.I, x);
        if constexpr (sizeof(W) == 1) {
          const floatx4 part = S::mma(w, x, floatx4{0.f, 0.f, 0.f, 0.f});
          const float sc = scales[s];
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][i] = __builtin_fmaf(part[i], sc, acc[t][i]);
        } else {
          acc[t] = S::mma(w, x, acc[t]);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < MT; ++t) sums[wave][t][lane] = acc[t];
    __syncthreads();
    for (int t = wave; t < MT; t += kWaves) {
      floatx4 v = sums[0][t][lane];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v += sums[w][t][lane];
      const int c = c0 + 16 * t + r, n = n0 + 4 * g;
      if (c < chosen.count && n < p.H) {
        const int slot = chosen.list[c];
        store4((float*)p.parts + (int64_t)slot * p.H + n, v * weights[slot], p.H - n, (p.H & 3) == 0);
      }
    }
  }
}

// ---- y[t][n] = sum of the parts of token t, in the order of its choices ----
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

bool valid(const ExpertsParams& p) {
  return p.x != nullptr && p.router != nullptr && p.gate_up != nullptr && p.down != nullptr && p.y != nullptr && p.route != nullptr &&
         p.hidden != nullptr && p.parts != nullptr && p.tokens >= 1 && p.tokens <= kMaxExpertTokens && p.E >= 1 && p.E <= kMaxExperts &&
         p.H >= 1 && p.H <= (1 << 24) && p.I >= 1 && p.I <= (1 << 23) && p.top_k >= 1 && p.top_k <= p.E && p.top_k <= kMaxExpertTopK &&
         dtype_is_float(p.dt) && (p.w_dt == p.dt || (p.w_dt == DT_F8 && p.gate_up_scale != nullptr && p.down_scale != nullptr));
}
int slots(const ExpertsParams& p) { return p.tokens * p.top_k < p.E ? p.tokens * p.top_k : p.E; }
// rows of x, hidden and weights are whole 16-byte vectors
bool whole_vectors(const ExpertsParams& p, const int len) { return (int64_t)len * dtype_size(p.dt) % 16 == 0 && (int64_t)len * dtype_size(p.w_dt) % 16 == 0; }

template <typename X>
hipError_t route_as(const ExpertsParams& p, hipStream_t stream) {
  const dim3 grid((p.E + 15) / 16, (p.tokens + 15) / 16);
  if ((int64_t)p.H * sizeof(X) % 16 == 0) hipLaunchKernelGGL((experts_logits_kernel<X, true>), grid, dim3(512), 0, stream, p);
  else hipLaunchKernelGGL((experts_logits_kernel<X, false>), grid, dim3(512), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(experts_choice_kernel, dim3(p.tokens), dim3(64), 0, stream, p);
  return hipGetLastError();
}

template <typename X, typename W, int MT, bool ALIGNED>
hipError_t gate_up_one(const ExpertsParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((experts_gate_up_kernel<X, W, MT, ALIGNED>), dim3((p.I + 15) / 16, slots(p)), dim3(64 * kWaves), 0, stream, p);
  return hipGetLastError();
}
template <typename X, typename W>
hipError_t gate_up_as(const ExpertsParams& p, hipStream_t stream) {
  const bool a = whole_vectors(p, p.H);
  if (p.tokens <= 16) return a ? gate_up_one<X, W, 1, true>(p, stream) : gate_up_one<X, W, 1, false>(p, stream);
  return a ? gate_up_one<X, W, 2, true>(p, stream) : gate_up_one<X, W, 2, false>(p, stream);
}
template <typename X, typename W, int MT, bool ALIGNED>
hipError_t down_one(const ExpertsParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((experts_down_kernel<X, W, MT, ALIGNED>), dim3((p.H + 15) / 16, slots(p)), dim3(64 * kWaves), 0, stream, p);
  return hipGetLastError();
}
template <typename X, typename W>
hipError_t down_as(const ExpertsParams& p, hipStream_t stream) {
  const bool a = whole_vectors(p, p.I);
  hipError_t e = p.tokens <= 16 ? (a ? down_one<X, W, 1, true>(p, stream) : down_one<X, W, 1, false>(p, stream))
                                : (a ? down_one<X, W, 2, true>(p, stream) : down_one<X, W, 2, false>(p, stream));
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
