// 8-bit floating point with a scale for each block of 128: rows quantised on the way to a product,
// and the product itself.
#include "block_common.h"

namespace ohip {
namespace {

constexpr float kMostE4m3 = 448.f;
constexpr float kLeastScale = 1.17549435e-38f;   // 2^-126: x / scale stays finite for blocks of subnormals and zeros

// ------------------------------------------------------------- quantisation --
// scale = max(max |x| / 448, 2^-126), q = e4m3(x / scale).  Bound by memory: es + 1 bytes per value.
// Sixteen lanes hold a block, eight values each.  8192 x 7168 bf16: 32 us, 5.5 TB/s read and written (with a
// division per value 40); 1 x 4096: 2.1 us, a launch.  Rows whose length is no multiple of 8 go element by element:
// 8192 x 7001 50 us.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(256) block_quantize_kernel(const T* x, uint8_t* q, float* scale, const int64_t rows, const int len, const int blocks) {
  const int l16 = threadIdx.x & 15;
  const int64_t total = rows * blocks, per_pass = (int64_t)gridDim.x * 16;
  // (whole wavefronts walk on together: group_allreduce reads lanes whatever their EXEC bit)
  for (int64_t base = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 6 << 2); base < total; base += per_pass) {
    const int64_t unit = base + (threadIdx.x >> 4 & 3);
    const bool live = unit < total;
    const int64_t row = live ? unit / blocks : 0;
    const int b = live ? (int)(unit - row * blocks) : 0;
    const int n = live ? min(kScaleBlock, len - b * kScaleBlock) : 0;
    const int64_t at = row * len + (int64_t)b * kScaleBlock;
    float v[8];
    if constexpr (VECTOR) {   // len is a multiple of 8: a lane's eight values are all there or none is
      const bool in = l16 * 8 < n;
      constexpr int PER = Vec16<T>::N;
#pragma unroll
      for (int h = 0; h < 8 / PER; ++h) {
        Vec16<T> w;
        if (in) w.load(x + at + l16 * 8 + h * PER);
        else w.raw = uintx4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int e = 0; e < PER; ++e) v[h * PER + e] = w.get(e);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = l16 + 16 * e < n ? Store<T>::ld(x + at + l16 + 16 * e) : 0.f;
    }
    float most = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
    most = group_allreduce<16>(most, [](float a, float c) { return fmaxf(a, c); });
    const float s = fmaxf(most / kMostE4m3, kLeastScale);
    // v / s, correctly rounded: from the correctly rounded 1 / s, two steps of quotient += remainder / s with exact
    // remainders give what the division gives in half of its instructions.  Where a remainder that matters could
    // underflow, or s is infinite, the division itself.  (The sign is v's: a zero's would be lost.)
    if (s >= 0x1p-70f && s <= 0x1p120f) {
      const float by = 1.f / s;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float u = v[e] * by;
        u = __builtin_fmaf(__builtin_fmaf(-u, s, v[e]), by, u);
        u = __builtin_fmaf(__builtin_fmaf(-u, s, v[e]), by, u);
        v[e] = __builtin_copysignf(u, v[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] /= s;
    }
    int w0 = 0, w1 = 0;
#if defined(__HIP_DEVICE_COMPILE__)
    w0 = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], w0, false);
    w0 = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w0, true);
    w1 = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], w1, false);
    w1 = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], w1, true);
#endif
    if constexpr (VECTOR) {
      if (l16 * 8 < n) *reinterpret_cast<uintx2*>(q + at + l16 * 8) = uintx2{(unsigned)w0, (unsigned)w1};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (l16 + 16 * e < n) q[at + l16 + 16 * e] = (uint8_t)((unsigned)(e < 4 ? w0 : w1) >> (8 * (e & 3)));
    }
    if (live && l16 == 0) scale[unit] = s;
  }
}

template <typename T>
hipError_t quantize_as(const void* x, void* q, float* scale, int64_t rows, int64_t len, hipStream_t stream) {
  const int blocks = (int)((len + kScaleBlock - 1) / kScaleBlock);
  const int grid = grid_for(rows * blocks, 16);
  if (len % 8 == 0)
    hipLaunchKernelGGL((block_quantize_kernel<T, true>), dim3(grid), dim3(256), 0, stream, (const T*)x, (uint8_t*)q, scale, rows, (int)len, blocks);
  else
    hipLaunchKernelGGL((block_quantize_kernel<T, false>), dim3(grid), dim3(256), 0, stream, (const T*)x, (uint8_t*)q, scale, rows, (int)len, blocks);
  return hipGetLastError();
}

// ------------------------------------------------------------------ product --
// Few tiles: a workgroup owns 16 NT columns n x 16 MT rows m, and its wavefronts share out the blocks of 128
// terms; their sums meet in LDS in wavefront order.  Every wavefront has LDS of its own and no barrier:
// eight lanes bring 128 neighbouring bytes of a row, P blocks ahead, and the operand fragments (lane l: row
// l % 16) are read back from there.  Straight from memory a fragment's neighbouring lanes are rows apart, and
// a compute unit gets 36 KB/us out of L2 instead of 120 (measured; from memory 26 either way).
// A block's sum is scaled on its way into the accumulator: the scale of row m belongs to a lane (column of
// the matrix result), that of B to the whole tile.  EXACT: through bf16 (see mma_exact).
// K = 4096: 1 row x 4096 columns 5.3 us, 64 rows 11.0, 128 rows 11.3, 256 rows 14.4; 48 x 7168 x 2048 6.9 us;
// 100 x 1000 x 8000 13.5; 509 x 2500 x 1400 (rows that are no whole vectors) 11.4.  A call's first bytes from memory and
// the meeting of the sums are 4 to 5 us of that.
template <typename TOut, int NT, int MT, int P, bool EXACT, bool ALIGNED>
__global__ void __launch_bounds__(512) block_gemm_split_kernel(const BlockGemmParams p) {
  constexpr int ROWS = 16 * (NT + MT);     // of B, then of A
  constexpr int OWN = ROWS * kScaleBlock;  // bytes of a wavefront's LDS
  constexpr int NR = ROWS / 8;             // requests of a block: eight rows each
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (16 * NT), m0 = blockIdx.y * (16 * MT);
  const int KB = (p.K + kScaleBlock - 1) / kScaleBlock;
  unsigned char* const own = smem + wave * OWN;
  // what this lane brings: 16 bytes at chunk lane % 8 of rows 8 i + lane / 8, of B and then of A (rows
  // behind the operand's end: nothing); addresses are a wavefront's base and 32 bits of a lane's own
  const int chunk = lane & 7, l8 = lane >> 3;
  const unsigned char *const b_tile = p.b + (int64_t)n0 * p.K, *const a_tile = p.a + (int64_t)m0 * p.K;
  const int b_rows = min(16 * NT, p.N - n0), a_rows = min(16 * MT, p.M - m0);
  const unsigned lane_row = (unsigned)l8 * p.K;
  const float* as[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) as[t] = p.a_scale + (int64_t)min(m0 + 16 * t + r, p.M - 1) * KB;
  const float* bs = p.b_scale + (int64_t)(n0 / kScaleBlock) * KB;
  floatx4 acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[j][t] = floatx4{0.f, 0.f, 0.f, 0.f};

  uintx4 in[P][NR];
  float sa[P][MT], sb[P];
  // Unaligned rows: 16 bytes that would pass the row's end are its last 16 (moved into place on their way to LDS),
  // and a row of fewer is read by bytes, one step for the whole product.
  const bool in_vectors = ALIGNED || p.K >= 16;
  auto fetch = [&](const int kb, const int q) __attribute__((always_inline)) {
    if (kb >= KB) return;
    const int at = kb * kScaleBlock + chunk * 16;
    const unsigned lane_at = ALIGNED ? lane_row + at : lane_offset(lane_row, at, p.K, false);
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const bool is_b = i < 2 * NT;
      const int first = 8 * (is_b ? i : i - 2 * NT), rows = is_b ? b_rows : a_rows;
      const unsigned char* const tile = is_b ? b_tile : a_tile;
      if constexpr (ALIGNED) {
        in[q][i] = uintx4{0u, 0u, 0u, 0u};
        if (first + l8 < rows && at < p.K) in[q][i] = *reinterpret_cast<const uintx4*>(tile + (int64_t)first * p.K + lane_at);
      } else {            // (a load with a range: fewer registers)
        in[q][i] = load_within(row_range(tile, in_vectors ? rows : 0, first, 8, p.K), lane_at);
      }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) sa[q][t] = as[t][kb];
    sb[q] = bs[kb];
  };
#pragma unroll
  for (int q = 0; q < P; ++q) fetch(wave + q * waves, q);
  for (int kb0 = wave; kb0 < KB; kb0 += P * waves) {
#pragma unroll
    for (int q = 0; q < P; ++q) {
      const int kb = kb0 + q * waves;
      if (kb >= KB) break;
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();     // (the fragments of the block before have been read: LDS keeps a wavefront's order)
      auto place = [&](const int i) { return reinterpret_cast<uintx4*>(own + (8 * i + l8) * kScaleBlock + ((chunk ^ ((8 * i + l8) >> 1 & 7)) << 4)); };
      if (!ALIGNED && (kb + 1) * kScaleBlock > p.K) {
        const int behind = kb * kScaleBlock + chunk * 16 + 16 - p.K;     // bytes of this lane's 16 that are not the row's
        if (in_vectors) {
          if (behind > 0 && behind < 16) {
#pragma unroll
            for (int i = 0; i < NR; ++i) in[q][i] = bytes_down(in[q][i], behind);
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < NR; ++i) {
            const bool is_b = i < 2 * NT;
            const int row = 8 * (is_b ? i : i - 2 * NT) + l8;
            uintx4 v = {0u, 0u, 0u, 0u};
            if (behind < 16 && row < (is_b ? b_rows : a_rows)) v = load_row16<false>((is_b ? b_tile : a_tile) + (int64_t)row * p.K, chunk * 16, p.K);
            *place(i) = v;
          }
        }
      }
      if (in_vectors) {
#pragma unroll
        for (int i = 0; i < NR; ++i) *place(i) = in[q][i];
      }
      float scale[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) scale[t] = sa[q][t] * sb[q];
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      fetch(kb + P * waves, q);
      const int c0 = (g ^ (r >> 1)) << 4, c1 = ((g + 4) ^ (r >> 1)) << 4;
      uintx4 w[NT][2], wv[EXACT ? NT : 1][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const unsigned char* at = own + (16 * j + r) * kScaleBlock;
        w[j][0] = *reinterpret_cast<const uintx4*>(at + c0);
        w[j][1] = *reinterpret_cast<const uintx4*>(at + c1);
        if constexpr (EXACT) bf16_of_e4m3(w[j][0], w[j][1], wv[j]);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const unsigned char* at = own + (16 * (NT + t) + r) * kScaleBlock;
        const uintx4 x0 = *reinterpret_cast<const uintx4*>(at + c0), x1 = *reinterpret_cast<const uintx4*>(at + c1);
        uintx4 xv[4];
        if constexpr (EXACT) bf16_of_e4m3(x0, x1, xv);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          floatx4 part;
          if constexpr (EXACT) part = mma_exact(wv[j], xv);
          else part = mma_e4m3(w[j][0], w[j][1], x0, x1, floatx4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[j][t][i] = __builtin_fmaf(part[i], scale[t], acc[j][t][i]);
        }
      }
    }
  }
  // the sums: NT x MT x 64 quads of every wavefront
  floatx4* const sums = reinterpret_cast<floatx4*>(smem);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) sums[(wave * NT * MT + j * MT + t) * 64 + lane] = acc[j][t];
  __syncthreads();
  for (int q = wave; q < NT * MT; q += waves) {
    floatx4 v = sums[q * 64 + lane];
    for (int w = 1; w < waves; ++w) v += sums[(w * NT * MT + q) * 64 + lane];
    const int m = m0 + 16 * (q % MT) + r, n = n0 + 16 * (q / MT) + 4 * g;
    if (m < p.M && n < p.N) store4((TOut*)p.y + (int64_t)m * p.N + n, v, p.N - n, (p.N & 3) == 0);
  }
}

// Many tiles that the kernel below does not take: a workgroup of four wavefronts owns BN columns n x BM rows m;
// both operands pass through LDS, 128 terms at a time, the next 128 on their way in registers.
// 8192 x 8192 x 4096 with fp32 results (bf16 matrix instructions) 614 us, x 4090 with bf16 results 573; 2048 x 4096 x
// 4096 82 and 83.
template <typename TOut, int BM, int BN, bool ALIGNED>
__global__ void __launch_bounds__(256) block_gemm_tile_kernel(const BlockGemmParams p) {
  constexpr bool EXACT = sizeof(TOut) == 4;
  constexpr int PITCH = kScaleBlock + 16;   // (16 bytes more: sixteen rows start in different banks)
  constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16;
  constexpr int NB = BN * 8 / 256, NA = BM * 8 / 256;  // 16-byte chunks a thread brings of either
  __shared__ __attribute__((aligned(16))) unsigned char lds[(BM + BN) * PITCH];
  __shared__ float sc[BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * BN, m0 = blockIdx.y * BM;
  const int wn = (wave & 1) * WN, wm = (wave >> 1) * WM;
  const int KB = (p.K + kScaleBlock - 1) / kScaleBlock;
  floatx4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  const unsigned char *arow[NA], *brow[NB];
#pragma unroll
  for (int i = 0; i < NA; ++i) arow[i] = p.a + (int64_t)min(m0 + (tid >> 3) + 32 * i, p.M - 1) * p.K;
#pragma unroll
  for (int i = 0; i < NB; ++i) brow[i] = p.b + (int64_t)min(n0 + (tid >> 3) + 32 * i, p.N - 1) * p.K;
  const float* as = p.a_scale + (int64_t)min(m0 + tid % BM, p.M - 1) * KB;
  const float* bs = p.b_scale + (int64_t)(n0 / kScaleBlock) * KB;
  uintx4 ra[NA], rb[NB];
  float rs, rt;
  auto fetch = [&](const int kb) __attribute__((always_inline)) {
    const int64_t k = (int64_t)kb * kScaleBlock + (tid & 7) * 16;
    if (ALIGNED || kb + 1 < KB) {      // (a row's last block may end inside a vector)
#pragma unroll
      for (int i = 0; i < NA; ++i) ra[i] = ALIGNED ? load_row16<ALIGNED>(arow[i], k, p.K) : reinterpret_cast<const Bytes16*>(arow[i] + k)->v;
#pragma unroll
      for (int i = 0; i < NB; ++i) rb[i] = ALIGNED ? load_row16<ALIGNED>(brow[i], k, p.K) : reinterpret_cast<const Bytes16*>(brow[i] + k)->v;
    } else {
#pragma unroll
      for (int i = 0; i < NA; ++i) ra[i] = load_row16<ALIGNED>(arow[i], k, p.K);
#pragma unroll
      for (int i = 0; i < NB; ++i) rb[i] = load_row16<ALIGNED>(brow[i], k, p.K);
    }
    rs = as[kb];
    rt = bs[kb];     // (multiplied where they are stored: here that would wait for the whole request)
  };
  unsigned char *const sa = lds, *const sb = lds + BM * PITCH;
  fetch(0);
  for (int kb = 0; kb < KB; ++kb) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NA; ++i) *reinterpret_cast<uintx4*>(sa + ((tid >> 3) + 32 * i) * PITCH + (tid & 7) * 16) = ra[i];
#pragma unroll
    for (int i = 0; i < NB; ++i) *reinterpret_cast<uintx4*>(sb + ((tid >> 3) + 32 * i) * PITCH + (tid & 7) * 16) = rb[i];
    if (tid < BM) sc[tid] = rs * rt;
    __syncthreads();
    if (kb + 1 < KB) fetch(kb + 1);
    uintx4 w0[TN], w1[TN], wv[EXACT ? TN : 1][4];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const unsigned char* at = sb + (wn + 16 * j + r) * PITCH + g * 32;
      w0[j] = *reinterpret_cast<const uintx4*>(at);
      w1[j] = *reinterpret_cast<const uintx4*>(at + 16);
      if constexpr (EXACT) bf16_of_e4m3(w0[j], w1[j], wv[j]);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const unsigned char* at = sa + (wm + 16 * i + r) * PITCH + g * 32;
      const uintx4 x0 = *reinterpret_cast<const uintx4*>(at), x1 = *reinterpret_cast<const uintx4*>(at + 16);
      const float s = sc[wm + 16 * i + r];
      uintx4 xv[4];
      if constexpr (EXACT) bf16_of_e4m3(x0, x1, xv);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        floatx4 part;
        if constexpr (EXACT) part = mma_exact(wv[j], xv);
        else part = mma_e4m3(w0[j], w1[j], x0, x1, floatx4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(part[e], s, acc[i][j][e]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int m = m0 + wm + 16 * i + r, n = n0 + wn + 16 * j + 4 * g;
      if (m < p.M && n < p.N) store4((TOut*)p.y + (int64_t)m * p.N + n, acc[i][j], p.N - n, (p.N & 3) == 0);
    }
}

// Many rows and columns: 256 x 256 results a workgroup of eight wavefronts, 128 rows m x 64 columns n each, or
// 128 x 128 of four, 64 x 64 each, two workgroups a compute unit.
// Both operands come by direct-to-LDS loads, 128 terms (64 or 32 KiB) at a time into one of two buffers while
// the other is multiplied: one barrier per block of terms, and every fragment of B stays in registers
// through those of A.  LDS rows are 128 bytes, 16-byte chunk c of row r in slot c ^ (r / 2 & 7), and a
// quarter g of a wavefront takes chunks g and g + 4 (which terms a lane holds does not matter as long as A
// and B agree): no two of the sixteen lanes that LDS serves at a time share a bank.  With chunks 2 g and
// 2 g + 1 half of LDS's busy cycles are conflicts (counters: 25 M of 55 M at 8192 x 8192 x 4096).
template <int WAVES>
struct Big {
  static constexpr int SIDE = 32 * WAVES;                            // rows of A, of B
  static constexpr int FM = WAVES;                                   // fragments of a wavefront's rows, of its columns
  static constexpr int FN = 4;
  static constexpr int STAGE = 2 * SIDE * kScaleBlock;               // bytes of a buffer
  static constexpr int LDS = 2 * STAGE + 2 * 64 * WAVES * 4;         // and the scales of the rows of A (twice: every thread stores one)
};
// A wavefront's request i is of rows 8 WAVES i + 8 wave .. + 7; what lies behind the operand's end, or in the last
// block behind the row's, is out of the request's range and arrives as zeros.
struct BigSource {
  const unsigned char *a, *b;   // the tile's rows
  int a_rows, b_rows, len;
  unsigned row;                 // this lane's row of a request, in bytes
  int chunk;                    // and its bytes of a block
};
template <int WAVES>
__device__ __forceinline__ void big_request(const BigSource& f, const int kb, unsigned char* to) {
  using lds_ptr = __attribute__((address_space(3))) void*;
#if defined(__HIP_DEVICE_COMPILE__)
  const unsigned at = lane_offset(f.row, kb * kScaleBlock + f.chunk, f.len, true);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const RowRange r = i < 4 ? row_range(f.a, f.a_rows, i * 8 * WAVES, 8 * WAVES, f.len) : row_range(f.b, f.b_rows, (i - 4) * 8 * WAVES, 8 * WAVES, f.len);
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(r.base), 0, r.size, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(to + i * 1024 * WAVES), 16, at, 0, 0, 0);
  }
#else
  (void)f; (void)kb; (void)to;
#endif
}

// One block of terms: the next one is requested into `next`, the one in `now` multiplied.  The two
// never overlap (without saying so, every read of LDS would wait for the requests).
template <int WAVES>
__device__ __forceinline__ void big_block(const BigSource& from, const int kb, unsigned char* __restrict next, const unsigned char* __restrict now,
                                          const float* __restrict scales, const float sb, const int wm, const int wn, const int lane, const int wave,
                                          floatx4 (&acc)[Big<WAVES>::FM][Big<WAVES>::FN]) {
  constexpr int FM = Big<WAVES>::FM, FN = Big<WAVES>::FN, PRODUCTS = FM * FN;
  big_request<WAVES>(from, kb + 1, next + wave * 1024);   // (behind the last block: zeros)
  const int r = lane & 15, g = lane >> 4;
  const int sw = r >> 1;      // (rows of a fragment start at multiples of 16)
  const int c0 = (g ^ sw) * 16, c1 = ((g + 4) ^ sw) * 16;
  uintx4 w0[FN], w1[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const unsigned char* at = now + (Big<WAVES>::SIDE + wn + 16 * j + r) * kScaleBlock;
    w0[j] = *reinterpret_cast<const uintx4*>(at + c0);
    w1[j] = *reinterpret_cast<const uintx4*>(at + c1);
  }
  // Product n (fragment n / 4 of A with n % 4 of B) is issued, and while the matrix cores are at it the vector
  // units scale product n - LAG; the next fragment of A is on its way.  The order is kept as written: left to
  // itself the compiler issues all products of the block first and spills them, or scales right behind the
  // products it then waits for.
  constexpr int LAG = 3;
  uintx4 x[2][2];
  floatx4 part[LAG + 1];
  float s[2], by[2];
  auto fetch = [&](const int i) __attribute__((always_inline)) {
    const unsigned char* at = now + (wm + 16 * i + r) * kScaleBlock;
    x[i & 1][0] = *reinterpret_cast<const uintx4*>(at + c0);
    x[i & 1][1] = *reinterpret_cast<const uintx4*>(at + c1);
    s[i & 1] = scales[wm + 16 * i + r];
  };
  auto scale = [&](const int n) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n >> 2][n & 3][e] = __builtin_fmaf(part[n % (LAG + 1)][e], by[n >> 2 & 1], acc[n >> 2][n & 3][e]);
  };
  fetch(0);
#pragma unroll
  for (int n = 0; n < PRODUCTS; ++n) {
    const int i = n >> 2, j = n & 3;
    if (j == 0) by[i & 1] = s[i & 1] * sb;
    part[n % (LAG + 1)] = mma_e4m3(w0[j], w1[j], x[i & 1][0], x[i & 1][1], floatx4{0.f, 0.f, 0.f, 0.f});
    if (j == 0 && i + 1 < FM) fetch(i + 1);
    if (n >= LAG) scale(n - LAG);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int n = PRODUCTS - LAG; n < PRODUCTS; ++n) scale(n);
}

template <typename TOut, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, 2) block_gemm_big_kernel(const BlockGemmParams p, const int tiles_m, const int tiles_n) {
  constexpr int SIDE = Big<WAVES>::SIDE, FM = Big<WAVES>::FM, FN = Big<WAVES>::FN, STAGE = Big<WAVES>::STAGE;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  float* const scales = reinterpret_cast<float*>(smem + 2 * STAGE);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Workgroups are dealt round-robin to the 8 XCDs: an XCD takes neighbours of a walk through groups of
  // eight tiles of rows, so that its workgroups share both operands in its L2.
  int t = blockIdx.x;
  {
    const int per = gridDim.x >> 3;
    if (t < per << 3) t = (t & 7) * per + (t >> 3);
  }
  const int group = t / (8 * tiles_n), rows = min(8, tiles_m - 8 * group), in = t - group * 8 * tiles_n;
  const int m0 = (8 * group + in % rows) * SIDE, n0 = in / rows * SIDE;
  const int KB = (p.K + kScaleBlock - 1) / kScaleBlock;
  const int chunk = ((lane & 7) ^ (((8 * wave + (lane >> 3)) >> 1) & 7)) * 16;
  BigSource from;
  from.a = p.a + (int64_t)m0 * p.K;
  from.b = p.b + (int64_t)n0 * p.K;
  from.a_rows = rows_within(p.M - m0, SIDE);
  from.b_rows = rows_within(p.N - n0, SIDE);
  from.len = p.K;
  from.row = (unsigned)(8 * wave + (lane >> 3)) * p.K;
  from.chunk = chunk;
  const float* arow_scale = p.a_scale + (int64_t)min(m0 + (tid & (SIDE - 1)), p.M - 1) * KB;
  const int wm = (wave & 1) * 16 * FM, wn = (wave >> 1) * 16 * FN;
  const float* bs = p.b_scale + (int64_t)min((n0 + wn) / kScaleBlock, (p.N - 1) / kScaleBlock) * KB;
  floatx4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  scales[tid] = arow_scale[0];
  float sb = bs[0];
  big_request<WAVES>(from, 0, smem + wave * 1024);
  for (int kb = 0; kb < KB; ++kb) {
    // This block's operands have landed, and everybody has left the other buffer.  The scales stored below in the turn
    // before are waited for here: the barrier comes without a wait for LDS (the compiler takes it away in this loop).
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();
    // (both scales of the next block ahead of its operands: a wait for them would wait for those too)
    const float next_scale = arow_scale[min(kb + 1, KB - 1)], next_sb = bs[min(kb + 1, KB - 1)];
    __builtin_amdgcn_sched_barrier(0);
    big_block<WAVES>(from, kb, smem + (~kb & 1) * STAGE, smem + (kb & 1) * STAGE, scales + (kb & 1) * 64 * WAVES, sb, wm, wn, lane, wave, acc);
    scales[(~kb & 1) * 64 * WAVES + tid] = next_scale;
    sb = next_sb;
  }
  __syncthreads();       // (nothing is under way into LDS when the workgroup ends)
  const int r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int m = m0 + wm + 16 * i + r, n = n0 + wn + 16 * j + 4 * g;
      if (m < p.M && n < p.N) store4((TOut*)p.y + (int64_t)m * p.N + n, acc[i][j], p.N - n, (p.N & 3) == 0);
    }
}

template <typename TOut, int NT, int MT, int P, bool ALIGNED>
hipError_t gemm_split(const BlockGemmParams& p, hipStream_t stream) {
  constexpr bool EXACT = sizeof(TOut) == 4 || MT == 1;
  constexpr int kOwn = 16 * (NT + MT) * kScaleBlock, kSums = NT * MT * 64 * 16;   // bytes of a wavefront: operands, sums
  const int KB = (p.K + kScaleBlock - 1) / kScaleBlock;
  // Eight wavefronts, but four where eight fill a compute unit's LDS and there are more tiles than units: two tiles a
  // unit then run side by side.  N = K = 4096, 512 rows: 24.4 us (eight: 26.9); 509 x 2500 x 1400, before its loads had a range, 13.5 (18.0).
  const int64_t tiles = (int64_t)((p.N + 16 * NT - 1) / (16 * NT)) * ((p.M + 16 * MT - 1) / (16 * MT));
  const int most = tiles > 256 && 8 * kOwn > 80 * 1024 ? 4 : 8;
  const int waves = KB < most ? KB : most, lds = waves * (kOwn > kSums ? kOwn : kSums);
  static LdsLimit limit;
  hipError_t e = limit.raise(reinterpret_cast<const void*>(&block_gemm_split_kernel<TOut, NT, MT, P, EXACT, ALIGNED>), 8 * (kOwn > kSums ? kOwn : kSums));
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((block_gemm_split_kernel<TOut, NT, MT, P, EXACT, ALIGNED>), dim3((p.N + 16 * NT - 1) / (16 * NT), (p.M + 16 * MT - 1) / (16 * MT)),
                     dim3(64 * waves), lds, stream, p);
  return hipGetLastError();
}
// From here on 128 x 128 results a workgroup, loaded straight into LDS, beat 64 x 64 with the terms shared out.
// N = K = 4096: 512 rows (128 tiles) 26.6 us against 24.4, 1024 rows 33 against 47 (four times 256 rows' 14.4).
constexpr int kMiddleTiles = 144;
template <typename TOut, int WAVES>
hipError_t gemm_big(const BlockGemmParams& p, hipStream_t stream) {
  constexpr int SIDE = Big<WAVES>::SIDE, LDS = Big<WAVES>::LDS;
  const int64_t tm = (p.M + SIDE - 1) / SIDE, tn = (p.N + SIDE - 1) / SIDE;
  static LdsLimit limit;
  hipError_t e = limit.raise(reinterpret_cast<const void*>(&block_gemm_big_kernel<TOut, WAVES>), LDS);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((block_gemm_big_kernel<TOut, WAVES>), dim3((unsigned)(tm * tn)), dim3(64 * WAVES), LDS, stream, p, (int)tm, (int)tn);
  return hipGetLastError();
}
template <typename TOut, bool ALIGNED>
hipError_t gemm_as(const BlockGemmParams& p, hipStream_t stream) {
  // Two tiles of columns a workgroup where that still leaves one for most of the compute units.
  if (p.M <= 16) return gemm_split<TOut, 1, 1, 4, ALIGNED>(p, stream);
  if (p.M <= 32) return p.N > 32 * 192 ? gemm_split<TOut, 2, 2, 2, ALIGNED>(p, stream) : gemm_split<TOut, 1, 2, 2, ALIGNED>(p, stream);
  if (p.M <= 64) return p.N > 32 * 192 ? gemm_split<TOut, 2, 4, 1, ALIGNED>(p, stream) : gemm_split<TOut, 1, 4, 2, ALIGNED>(p, stream);
  if constexpr (ALIGNED && sizeof(TOut) == 2) {
    // 256 x 256 for three quarters of the compute units at least: 3000 x 4096 x 4096 73 us; 2048 rows in 128 x 128 50 us.
    if (p.K <= 1 << 22) {   // (256 rows of an operand within 2^30 bytes of buffer range)
      if ((int64_t)((p.M + 255) / 256) * ((p.N + 255) / 256) >= 192) return gemm_big<TOut, 8>(p, stream);
      if ((int64_t)((p.M + 127) / 128) * ((p.N + 127) / 128) >= kMiddleTiles) return gemm_big<TOut, 4>(p, stream);
    }
  }
  // Too few of the tiles below for every compute unit: 64 x 64 results (64 rows x 32 columns where even those are
  // few).  N = K = 4096: a tile below takes 47 us however few there are; here 512 rows take 24 us, 256 14.5.
  if ((int64_t)((p.M + 127) / 128) * ((p.N + 127) / 128) < 256) {
    if ((int64_t)((p.M + 63) / 64) * ((p.N + 31) / 32) <= 320) return gemm_split<TOut, 2, 4, 1, ALIGNED>(p, stream);
    if constexpr (sizeof(TOut) == 2) return gemm_split<TOut, 4, 4, 1, ALIGNED>(p, stream);
    else return gemm_split<TOut, 2, 4, 1, ALIGNED>(p, stream);      // (bf16 copies of four tiles do not fit in registers)
  }
  hipLaunchKernelGGL((block_gemm_tile_kernel<TOut, 128, 128, ALIGNED>), dim3((p.N + 127) / 128, (p.M + 127) / 128), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_block_quantize(const void* x, DType dt, void* q, float* scale, int64_t rows, int64_t len, hipStream_t stream) {
  if (x == nullptr || q == nullptr || scale == nullptr || rows < 1 || len < 1 || len > (1 << 24)) return hipErrorInvalidValue;
  switch (dt) {
    case DT_F32: return quantize_as<float>(x, q, scale, rows, len, stream);
    case DT_F16: return quantize_as<f16_t>(x, q, scale, rows, len, stream);
    case DT_BF16: return quantize_as<bf16_t>(x, q, scale, rows, len, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_block_gemm(const BlockGemmParams& p, hipStream_t stream) {
  if (p.a == nullptr || p.b == nullptr || p.a_scale == nullptr || p.b_scale == nullptr || p.y == nullptr) return hipErrorInvalidValue;
  if (p.M < 1 || p.N < 1 || p.K < 1 || p.N > (1 << 24) || p.K > (1 << 24)) return hipErrorInvalidValue;
  if (p.M > 65535 * 128) return hipErrorInvalidValue;   // (rows of tiles in one launch)
  const bool aligned = p.K % 16 == 0;
  switch (p.out_dt) {
    case DT_F32: return aligned ? gemm_as<float, true>(p, stream) : gemm_as<float, false>(p, stream);
    case DT_F16: return aligned ? gemm_as<f16_t, true>(p, stream) : gemm_as<f16_t, false>(p, stream);
    case DT_BF16: return aligned ? gemm_as<bf16_t, true>(p, stream) : gemm_as<bf16_t, false>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ohip
