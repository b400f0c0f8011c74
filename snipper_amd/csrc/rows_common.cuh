// rows_common.cuh -- element types, 8-element row accesses and the 8-bit block format shared by the kernels of fp8_capi.hip (gfx950).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace snipper {
namespace rows {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;

constexpr int kBlock = 128;                       // elements behind one scale

enum { kF32 = 0, kBF16 = 1, kF16 = 3 };           // type codes of the C ABI

// Eight consecutive elements of a row as float.  The address needs no more than the element's own alignment: memory instructions
// take any on this hardware (a piece that straddles a cache line costs one more access), so odd widths and strides run the same
// code as even ones.  `n` elements exist (n >= 8: all); the others read as 0.
template <typename T>
__device__ __forceinline__ void load8(const T *p, int n, float (&v)[8]) {
  if (n >= 8) {
    T t[8];
    __builtin_memcpy(t, p, 8 * sizeof(T));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)t[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)p[j] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, int n, const float (&v)[8]) {
  T t[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = (T)v[j];     // to nearest, ties to even
  if (n >= 8) {
    __builtin_memcpy(p, t, 8 * sizeof(T));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = t[j];
  }
}
// the same for parameters, whose type is known at run time only; a null pointer reads as `none`
__device__ __forceinline__ void load_param8(const void *p, int dtype, long long at, int n, float none, float (&v)[8]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = none;
  } else if (dtype == kF32) {
    load8((const float *)p + at, n, v);
  } else if (dtype == kBF16) {
    load8((const bf16_t *)p + at, n, v);
  } else {
    load8((const f16_t *)p + at, n, v);
  }
}
__device__ __forceinline__ float load_param(const void *p, int dtype, long long at) {
  return dtype == kF32 ? ((const float *)p)[at] : dtype == kBF16 ? (float)((const bf16_t *)p)[at] : (float)((const f16_t *)p)[at];
}
__device__ __forceinline__ void store_param(void *p, int dtype, long long at, float v) {
  if (dtype == kF32) ((float *)p)[at] = v;
  else if (dtype == kBF16) ((bf16_t *)p)[at] = (bf16_t)v;
  else ((f16_t *)p)[at] = (f16_t)v;
}

// ---- the scale of a block -------------------------------------------------------------------------------------------
// Magnitude that counts for the scale: |x| of a finite x, 0 of an infinity or NaN.  As bits, so that a maximum is one of integers.
__device__ __forceinline__ unsigned mag(float x) {
  const unsigned b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// Biased exponent of the smallest 2^e, e >= -127, with max / 2^e <= largest value = 1.75 * 2^8 (e4m3) or 1.75 * 2^15 (e5m2): the
// exponent of max less 8 or 15, one more where max's significand is above 1.75; 2^0 for a block of zeros.
template <int FMT>
__device__ __forceinline__ int scale_byte(unsigned max_bits) {
  if (max_bits == 0) return 127;
  const int e = (int)(max_bits >> 23) - (FMT == 0 ? 8 : 15) + ((max_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e > 0 ? e : 0;
}
// 2^-(byte - 127): the factor of the elements.  byte <= 247, so the exponent 254 - byte is a normal one.
__device__ __forceinline__ float inv_scale(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }

// four floats, in range by the choice of the scale, to 8 bits: nearest, ties to even (NaN stays; an infinity is the type's own or NaN)
template <int FMT>
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d) {
  int r = 0;
  if constexpr (FMT == 0) {
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  } else {
    r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true);
  }
  return (unsigned)r;
}

__device__ __forceinline__ unsigned max16(unsigned v) {        // over the 16 lanes of a row of the wave
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const unsigned t = (unsigned)__shfl_xor((int)v, o, 64);
    v = v > t ? v : t;
  }
  return v;
}

}  // namespace rows
}  // namespace snipper
