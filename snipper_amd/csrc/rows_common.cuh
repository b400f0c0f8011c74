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

enum { kF32 = 0, kBF16 = 1, kF16 = 3 };           // type codes of the C ABI

// W consecutive elements of a row as float.  The address needs no more than the element's own alignment: memory instructions take any
// on this hardware (a piece that straddles a cache line costs one more access), so odd widths and strides run the same code as even
// ones.  `n` elements exist (n >= W: all); the others read as 0.
template <int W, bool NT = false, typename T>
__device__ __forceinline__ void load_w(const T *p, int n, float (&v)[W]) {
  if (n >= W) {
    T t[W];
    if constexpr (NT) {
      typedef unsigned U __attribute__((ext_vector_type(W * sizeof(T) / 4), aligned(sizeof(T))));
      const U u = __builtin_nontemporal_load((const U *)p);
      __builtin_memcpy(t, &u, sizeof(u));
    } else {
      __builtin_memcpy(t, p, W * sizeof(T));
    }
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = (float)t[j];
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = j < n ? (float)p[j] : 0.f;
  }
}
template <int W, typename T>
__device__ __forceinline__ void store_w(T *p, int n, const float (&v)[W]) {
  T t[W];
#pragma unroll
  for (int j = 0; j < W; ++j) t[j] = (T)v[j];     // to nearest, ties to even
  if (n >= W) {
    __builtin_memcpy(p, t, W * sizeof(T));
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (j < n) p[j] = t[j];
  }
}
// past the caches
template <int W, typename T>
__device__ __forceinline__ void store_nt(T *p, int n, const float (&v)[W]) {
  if (n >= W) {
    typedef unsigned V __attribute__((ext_vector_type(W * sizeof(T) / 4), aligned(sizeof(T))));
    T t[W];
#pragma unroll
    for (int j = 0; j < W; ++j) t[j] = (T)v[j];
    V u;
    __builtin_memcpy(&u, t, sizeof(u));
    __builtin_nontemporal_store(u, (V *)p);
  } else {
    store_w<W>(p, n, v);
  }
}
template <typename T>
__device__ __forceinline__ void load8(const T *p, int n, float (&v)[8]) { load_w<8>(p, n, v); }
template <typename T>
__device__ __forceinline__ void store8(T *p, int n, const float (&v)[8]) { store_w<8>(p, n, v); }
// load_w in two halves, so that a loop can have the next row's elements on the way: what it reads, in the element's own type
template <typename T, int W>
struct Raw {
  typedef T V __attribute__((ext_vector_type(W)));
  V v;
  template <bool NT = false>                      // NT: read for the last time, past the caches
  __device__ __forceinline__ void load(const T *p, int n) {
    if (n >= W) {
      if constexpr (NT) {
        typedef unsigned U __attribute__((ext_vector_type(W * sizeof(T) / 4), aligned(sizeof(T))));
        const U u = __builtin_nontemporal_load((const U *)p);
        __builtin_memcpy(&v, &u, sizeof(u));
      } else {
        __builtin_memcpy(&v, p, W * sizeof(T));
      }
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = j < n ? p[j] : (T)0.f;
    }
  }
  __device__ __forceinline__ void get(float (&f)[W]) const {
#pragma unroll
    for (int j = 0; j < W; ++j) f[j] = (float)v[j];
  }
};
// the same for parameters, whose type is known at run time only; a null pointer reads as `none`
template <int W>
__device__ __forceinline__ void load_param_w(const void *p, int dtype, long long at, int n, float none, float (&v)[W]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = none;
  } else if (dtype == kF32) {
    load_w<W>((const float *)p + at, n, v);
  } else if (dtype == kBF16) {
    load_w<W>((const bf16_t *)p + at, n, v);
  } else {
    load_w<W>((const f16_t *)p + at, n, v);
  }
}
__device__ __forceinline__ void load_param8(const void *p, int dtype, long long at, int n, float none, float (&v)[8]) {
  load_param_w<8>(p, dtype, at, n, none, v);
}
__device__ __forceinline__ float load_param(const void *p, int dtype, long long at) {
  return dtype == kF32 ? ((const float *)p)[at] : dtype == kBF16 ? (float)((const bf16_t *)p)[at] : (float)((const f16_t *)p)[at];
}
__device__ __forceinline__ void store_param(void *p, int dtype, long long at, float v) {
  if (dtype == kF32) ((float *)p)[at] = v;
  else if (dtype == kBF16) ((bf16_t *)p)[at] = (bf16_t)v;
  else ((f16_t *)p)[at] = (f16_t)v;
}

// sum_b part[b][e] of nparts rows of `width`, for threads 0 .. 31 of a workgroup of 1024, each an element e: 32 elements (a line of 128
// bytes) x 32 slices of b that meet in LDS, in a fixed order
__device__ __forceinline__ float sum_parts(const float *part, int nparts, int width, int e) {
  __shared__ float red[32][33];
  const int i = threadIdx.x & 31, slice = threadIdx.x >> 5;
  float s = 0.f;
  if (e < width) {
#pragma unroll 8
    for (int b = slice; b < nparts; b += 32) s += part[(long long)b * width + e];
  }
  red[slice][i] = s;
  __syncthreads();
  s = 0.f;
  if (slice == 0) {
#pragma unroll
    for (int k = 0; k < 32; ++k) s += red[k][i];
  }
  return s;
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

template <int L>
__device__ __forceinline__ unsigned max_over(unsigned v) {     // over L neighbouring lanes
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    const unsigned t = (unsigned)__shfl_xor((int)v, o, 64);
    v = v > t ? v : t;
  }
  return v;
}
__device__ __forceinline__ unsigned max16(unsigned v) { return max_over<16>(v); }

}  // namespace rows
}  // namespace snipper
