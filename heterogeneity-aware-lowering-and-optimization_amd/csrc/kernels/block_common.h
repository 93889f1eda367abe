// Device code shared by the kernels over 8-bit floating-point blocks (block_fp8.hip) and over the
// experts' weights (experts.hip).
#ifndef ODLA_HIP_BLOCK_COMMON_H_
#define ODLA_HIP_BLOCK_COMMON_H_

#include "device_utils.h"
#include "row_range.h"

#include <type_traits>

namespace ohip {

typedef int intx8 __attribute__((ext_vector_type(8)));

// 16 bytes from an address of any alignment (one global_load_dwordx4: gfx950 takes them unaligned).
struct __attribute__((packed, aligned(1))) Bytes16 { uintx4 v; };

// The bytes n .. 15 (0 < n < 16) moved to the front, zeros behind them.
__device__ __forceinline__ uintx4 bytes_down(const uintx4 v, const int n) {
  const unsigned long long lo = (unsigned long long)v.y << 32 | v.x, hi = (unsigned long long)v.w << 32 | v.z;
  const int bits = 8 * n;
  const unsigned long long l = bits >= 64 ? hi >> (bits - 64) : lo >> bits | hi << (63 - bits) << 1, h = bits >= 64 ? 0ull : hi >> bits;
  return uintx4{(unsigned)l, (unsigned)(l >> 32), (unsigned)h, (unsigned)(h >> 32)};
}

// Bytes at .. at + 15 of a row of `len` bytes; zero behind its end.  Never reads outside the row.
// ALIGNED: rows start on 16-byte boundaries and are whole 16-byte vectors.
template <bool ALIGNED>
__device__ __forceinline__ uintx4 load_row16(const unsigned char* row, const int64_t at, const int64_t len) {
  if constexpr (ALIGNED) {
    return at < len ? *reinterpret_cast<const uintx4*>(row + at) : uintx4{0u, 0u, 0u, 0u};
  } else {
    if (len >= 16) {      // (16 bytes that would pass the end are the last 16)
      const int64_t from = at + 16 <= len ? at : len - 16;
      const uintx4 v = reinterpret_cast<const Bytes16*>(row + from)->v;
      return at == from ? v : at >= len ? uintx4{0u, 0u, 0u, 0u} : bytes_down(v, (int)(at - from));
    }
    unsigned long long lo = 0, hi = 0;
#pragma unroll 1
    for (int i = 0; at + i < len; ++i) {
      const unsigned long long b = row[at + i];
      if (i < 8) lo |= b << 8 * i;
      else hi |= b << 8 * (i - 8);
    }
    return uintx4{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
  }
}

// 16 bytes at range.base + at (any alignment); zeros where that is not within the range.
__device__ __forceinline__ uintx4 load_within(const RowRange range, const unsigned at) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(range.base), 0, range.size, 0x00020000);
  return __builtin_bit_cast(uintx4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
#else
  (void)range; (void)at;
  return uintx4{0u, 0u, 0u, 0u};
#endif
}

// c + A B^T for 16 rows of A and 16 of B over 128 e4m3 values: lane l supplies 32 values of row
// l % 16 of either, those of quarter l / 16 of the 128 (which quarter holds which values does not
// matter as long as A and B agree).  Result element i of lane l: row 4 * (l / 16) + i of A, row
// l % 16 of B.  No block exponents (the two zero scales select the plain form).
__device__ __forceinline__ floatx4 mma_e4m3(const uintx4 a0, const uintx4 a1, const uintx4 b0, const uintx4 b1, const floatx4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
  const intx8 a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w, (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
  const intx8 b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w, (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
#else
  (void)a0; (void)a1; (void)b0; (void)b1;
  return c;
#endif
}

struct f8_t { uint8_t bits; };

// c + W X^T over the elements of one 16-byte vector of X per lane (16 rows of either).
template <typename X>
__device__ __forceinline__ floatx4 mma_vec(const uintx4 w, const uintx4 x, floatx4 c) {
  if constexpr (std::is_same<X, float>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[i]), __uint_as_float(x[i]), c, 0, 0, 0);
    return c;
  } else {
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (std::is_same<X, f16_t>::value)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, w), __builtin_bit_cast(halfx8, x), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), c, 0, 0, 0);
#else
    return c;
#endif
  }
}

// e4m3 values as X, exactly: vector `v` of the 16 values in w (16 / sizeof(X) of them).
template <typename X>
__device__ __forceinline__ uintx4 values_of(const uintx4 w, const int v) {
  uintx4 o = {0u, 0u, 0u, 0u};
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (std::is_same<X, float>::value) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[v], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[v], true);
    o = uintx4{__float_as_uint(lo[0]), __float_as_uint(lo[1]), __float_as_uint(hi[0]), __float_as_uint(hi[1])};
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int src = (int)w[2 * v + i];
      if constexpr (std::is_same<X, f16_t>::value) {
        o[2 * i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(src, 1.0f, false));
        o[2 * i + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(src, 1.0f, true));
      } else {
        o[2 * i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, 1.0f, false));
        o[2 * i + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, 1.0f, true));
      }
    }
  }
#endif
  return o;
}

// Sum of 128 products of e4m3 values in fp32 (operands as in mma_e4m3): as bf16, which holds them
// exactly, through the 16-bit matrix instructions.  The 8-bit ones align the products of eight
// neighbouring terms to the largest of them and drop what lies below 2^-13 of it.
__device__ __forceinline__ void bf16_of_e4m3(const uintx4 w0, const uintx4 w1, uintx4 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = values_of<bf16_t>(i < 2 ? w0 : w1, i & 1);
}
__device__ __forceinline__ floatx4 mma_exact(const uintx4 (&a)[4], const uintx4 (&b)[4]) {
  floatx4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) c = mma_vec<bf16_t>(a[i], b[i], c);
  return c;
}

// Four neighbouring results from fp32 sums, `n` of them inside the row; vector: the address allows one store.
template <typename T>
__device__ __forceinline__ void store4(T* y, const floatx4 v, const int n, const bool vector) {
  if (vector && n >= 4) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<floatx4*>(y) = v;
    else *reinterpret_cast<uintx2*>(y) = uintx2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) Store<T>::st(y + i, v[i]);
  }
}

}  // namespace ohip
#endif
