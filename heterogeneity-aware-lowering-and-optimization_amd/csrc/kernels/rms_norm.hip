// Rows normalised by their root mean square, with the residual's addition in front and, if asked for, 8-bit results
// with a scale for each block of 128 behind:
//
//   s = x + r,   y = s / sqrt(mean s^2 + eps) * w,   q = e4m3(y / scale),  scale = max(max |y| / 448, 2^-126)
//
// Bound by memory: every operand is read and every result written once.  bf16, residual, 8-bit result: 8192 rows of 7168 values, 415 MB,
// 86 us, 4.8 TB/s (a copy of 1 GiB 5.1); one row of 4096 values 3 us, of which a launch is 2.  A row stays in its workgroup's registers
// between the sum of its squares and its results, eight neighbouring values a lane, so that sixteen lanes hold a block.
// Squares, their sum and y are fp32; s is rounded on its way out alone, so that y is not twice rounded.
#include "block_common.h"

namespace ohip {
namespace {

// WAVES wavefronts a row and NV groups of eight values a lane; LONG: rows of any length, which are read twice.
// ROWS rows a workgroup (short rows are a wavefront's each, and nothing is waited for).
template <typename T, int WAVES, int NV, int ROWS, bool QUANTIZE, bool VECTOR, bool LONG>
__global__ void __launch_bounds__(64 * WAVES * ROWS) rms_norm_kernel(const RmsNormParams p) {
  constexpr int NT = 64 * WAVES;
  static_assert(WAVES == 1 || ROWS == 1, "rows of several wavefronts meet in LDS");
  __shared__ float room[WAVES];
  const int tid = ROWS > 1 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * ROWS + (ROWS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
  if (row >= p.rows) return;
  const int len = p.len, blocks = (len + kScaleBlock - 1) / kScaleBlock;
  const T* x = reinterpret_cast<const T*>(p.x) + row * len;
  const T* r = reinterpret_cast<const T*>(p.residual) + row * len;
  T* sum = reinterpret_cast<T*>(p.sum) + row * len;
  const bool joined = p.residual != nullptr, kept = p.sum != nullptr;
  auto fetch = [&](const int at, float (&v)[8]) __attribute__((always_inline)) {
    load8<T, VECTOR>(x, at, len, v);
    if (joined) {
      float a[8];
      load8<T, VECTOR>(r, at, len, a);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += a[e];
    }
  };
  float v[LONG ? 1 : NV][8];
  float squares = 0.f;
  if constexpr (LONG) {
    for (int at = tid * 8; at < len; at += NT * 8) {
      fetch(at, v[0]);
#pragma unroll
      for (int e = 0; e < 8; ++e) squares = __builtin_fmaf(v[0][e], v[0][e], squares);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) fetch((i * NT + tid) * 8, v[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) squares = __builtin_fmaf(v[i][e], v[i][e], squares);
  }
  squares = block_sum<NT>(squares, room);
  const float by = 1.f / sqrtf(squares / (float)len + p.eps);
  auto finish = [&](const int at, float (&a)[8]) __attribute__((always_inline)) {
    if (kept) store8<T, VECTOR>(sum, at, len, a);
    float w[8];
    if (p.weight == nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.f;
    } else if (p.w_dt == DT_F32) {
      load8<float, VECTOR>(reinterpret_cast<const float*>(p.weight), at, len, w);
    } else {
      load8<T, VECTOR>(reinterpret_cast<const T*>(p.weight), at, len, w);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = a[e] * by * w[e];
    if constexpr (QUANTIZE) {
      float most = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, at + e < len ? fabsf(a[e]) : 0.f);
      most = group_allreduce<16>(most, [](float c, float d) { return fmaxf(c, d); });
      const float s = e4m3_scale(most);
      const uintx2 codes = e4m3_of(a, s);
      uint8_t* q = reinterpret_cast<uint8_t*>(p.y) + row * len;
      if (at + 8 <= len) {
        if constexpr (VECTOR) *reinterpret_cast<uintx2*>(q + at) = codes;
        else reinterpret_cast<Bytes8*>(q + at)->v = codes;
      } else if (!VECTOR) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (at + e < len) q[at + e] = (uint8_t)(codes[e >> 2] >> (8 * (e & 3)));
      }
      if ((tid & 15) == 0 && at < len) p.scale[row * blocks + at / kScaleBlock] = s;
    } else {
      store8<T, VECTOR>(reinterpret_cast<T*>(p.y) + row * len, at, len, a);
    }
  };
  if constexpr (LONG) {
    // (whole wavefronts walk on together: the lanes of a block exchange their largest values)
    for (int base = 0; base < len; base += NT * 8) {
      const int at = base + tid * 8;
      fetch(at, v[0]);
      finish(at, v[0]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) finish((i * NT + tid) * 8, v[i]);
  }
}

template <typename T, bool QUANTIZE, bool VECTOR>
hipError_t norm_as(const RmsNormParams& p, hipStream_t stream) {
#define OHIP_NORM(WAVES, NV, ROWS, LONG) \
  hipLaunchKernelGGL((rms_norm_kernel<T, WAVES, NV, ROWS, QUANTIZE, VECTOR, LONG>), dim3((unsigned)((p.rows + ROWS - 1) / ROWS)), dim3(64 * WAVES * ROWS), 0, stream, p)
  // By the length alone, so that a row's bits do not depend on how many there are.  As many wavefronts as there are groups of eight
  // values a lane, up to sixteen: what one lane would hold more waits longer.  bf16, residual, 8-bit result, 1 and 8192 rows, us: 512 values
  // a wavefront 2.4 and 7.6, four (three idle) 2.4 and 16; 1024 values by two 2.4 and 13.5, by one 3.2 and 13.7, by four 2.4 and 17.8; 2048 by
  // four 2.5 and 21, by one 5 and 24; 4096 by eight 3.0 and 39, by four 3.7 and 39; 8192 by sixteen 3.4 and 89, by four 5.6 and 96;
  // 16384 by sixteen with two groups 4.9 and 167, with four 7.2 and 268.  Held rather than read twice up to 32768: that length 8.1
  // against 11.6 for one row, 434 for 8192 either way (20000 values 7.2 and 7.1, 321 and 294).
  if (p.len <= 512) OHIP_NORM(1, 1, 4, false);
  else if (p.len <= 1024) OHIP_NORM(2, 1, 1, false);
  else if (p.len <= 2048) OHIP_NORM(4, 1, 1, false);
  else if (p.len <= 4096) OHIP_NORM(8, 1, 1, false);
  else if (p.len <= 8192) OHIP_NORM(16, 1, 1, false);
  else if (p.len <= 16384) OHIP_NORM(16, 2, 1, false);
  else if (p.len <= 32768) OHIP_NORM(16, 4, 1, false);
  else OHIP_NORM(16, 1, 1, true);
#undef OHIP_NORM
  return hipGetLastError();
}
template <typename T>
hipError_t norm_of(const RmsNormParams& p, hipStream_t stream) {
  if (p.len % 8 == 0) return p.quantize ? norm_as<T, true, true>(p, stream) : norm_as<T, false, true>(p, stream);
  return p.quantize ? norm_as<T, true, false>(p, stream) : norm_as<T, false, false>(p, stream);
}

}  // namespace

bool rms_norm_fits(const RmsNormParams& p) { return p.rows * (p.len <= 4096 ? 512 : 1024) <= UINT32_MAX; }

hipError_t launch_rms_norm(const RmsNormParams& p, hipStream_t stream) {
  switch (p.dt) {
    case DT_F32: return norm_of<float>(p, stream);
    case DT_F16: return norm_of<f16_t>(p, stream);
    case DT_BF16: return norm_of<bf16_t>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ohip
