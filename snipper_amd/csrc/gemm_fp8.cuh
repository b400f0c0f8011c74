// gemm_fp8.cuh -- out [M][N] = act(A [M][K] . B [N][K]^T + bias) of two matrices in 8-bit blocks (gfx950; format: include/snipper_fp8.h).
//
//   out[m][n] = sum_b 2^(ea[m][b] + eb[n][b]) sum_{k in block b} a[m][k] b[n][k]
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 elements with a power-of-two scale for each 32 of a lane's
// elements: a block of 128 is one instruction whose four scales are the same byte, so scaling costs no instruction at all and any
// order of the 128 elements within the operands is right as long as both have the same one.  The unit adds the products of an
// instruction after aligning them to the largest and drops what lies 2^13 or more below it (measured: 1.5e-5 of the result's norm at K
// = 128 .. 65 536; the sum over blocks is float32): far inside half a step of a bfloat16 (2^-9) or float16 (2^-12) result, but not
// of a float32 one.  EXACT kernels therefore widen the operands to bfloat16 with their scales -- 4 bits and a power of two fit
// exactly -- and use v_mfma_f32_16x16x32_bf16 (1e-7), at a quarter of the rate.
//
// Rows of n are the first operand and rows of m the second, so that a lane holds four consecutive columns of one row of the result.
#pragma once
#include "rows_common.cuh"

namespace snipper {
namespace rows {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

struct MmArgs {
  const uint8_t *A, *sA, *B, *sB;            // [M][P], [M][Q], [N][P], [N][Q]
  int M, N;
  int steps;                                 // P / 128
  const void *bias; int bias_dt; int relu;
  void *out; int out_dt;
  float *part;                               // [splits][M][N] or null
  int splits, per_split;                     // K steps of a split (a multiple of 4)
};

// four elements of a row of the result: columns n .. n + 3
__device__ __forceinline__ void mm_store4(const MmArgs &a, long long m, int n, f32x4 v) {
  const int cnt = a.N - n;
  if (cnt <= 0) return;
  if (a.bias) {
#pragma unroll
    for (int t = 0; t < 4; ++t) v[t] += t < cnt ? load_param(a.bias, a.bias_dt, n + t) : 0.f;
  }
  if (a.relu) {
#pragma unroll
    for (int t = 0; t < 4; ++t) v[t] = v[t] < 0.f ? 0.f : v[t];      // (a NaN stays one)
  }
  const long long at = m * a.N + n;
  if (a.out_dt == kF32) {
    float *p = (float *)a.out + at;
    if (cnt >= 4) __builtin_memcpy(p, &v, 16);
    else for (int t = 0; t < cnt; ++t) p[t] = v[t];
  } else {
    uint16_t h[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
      h[t] = a.out_dt == kBF16 ? __builtin_bit_cast(uint16_t, (bf16_t)v[t]) : __builtin_bit_cast(uint16_t, (f16_t)v[t]);
    uint16_t *p = (uint16_t *)a.out + at;
    if (cnt >= 4) __builtin_memcpy(p, h, 8);
    else for (int t = 0; t < cnt; ++t) p[t] = h[t];
  }
}

// 8 bytes -> 8 bfloat16, times 2^(byte - 127)
template <int FMT>
__device__ __forceinline__ bf16x8 widen8(int lo, int hi, float scale) {
  bf16x2 p[4];
  if constexpr (FMT == 0) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, scale, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, scale, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, scale, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, scale, true);
  }
  bf16x8 r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
__device__ __forceinline__ float scale_of(int word, int sel) {
  const unsigned byte = ((unsigned)word >> (8 * sel)) & 255u;
  return __uint_as_float(byte ? byte << 23 : 0x400000u);
}

// the operand of a 16-row tile: 32 elements of a row in a lane
template <int FMT, bool EXACT>
struct Operand {
  i32x8 raw;
  __device__ __forceinline__ void set(i32x4 lo, i32x4 hi, int, int) { raw = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
};
template <int FMT>
struct Operand<FMT, true> {
  bf16x8 w[4];
  __device__ __forceinline__ void set(i32x4 lo, i32x4 hi, int word, int sel) {
    const float s = scale_of(word, sel);
    w[0] = widen8<FMT>(lo[0], lo[1], s); w[1] = widen8<FMT>(lo[2], lo[3], s);
    w[2] = widen8<FMT>(hi[0], hi[1], s); w[3] = widen8<FMT>(hi[2], hi[3], s);
  }
};
// SEL: which byte of the scale words (0 .. 3) is this step's
template <int FB, int FA, int SEL>
__device__ __forceinline__ f32x4 mm_step(const Operand<FB, false> &b, const Operand<FA, false> &x, f32x4 acc, int sb, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.raw, x.raw, acc, FB, FA, SEL, sb, SEL, sa);
}
template <int FB, int FA, int SEL>
__device__ __forceinline__ f32x4 mm_step(const Operand<FB, true> &b, const Operand<FA, true> &x, f32x4 acc, int, int) {
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.w[j], x.w[j], acc, 0, 0, 0);
  return acc;
}

// ---- tiles -----------------------------------------------------------------------------------------------------------
// A workgroup of WM x WN waves makes a (16 TM WM) x (16 TN WN) tile; a K step of 128 is one byte-row of 128 per row of either side.
// Rows go to LDS by DMA in 16-byte pieces, piece c of row r at place c ^ (r & 7), so that the 16 rows of an operand are read without
// bank conflicts; two buffers, one barrier a step.  The scale words of four K steps come the same way (plain loads of them would make
// the compiler wait for the DMAs issued after them).
template <int FA, int FB, bool EXACT, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(64 * WM * WN) void mm_tile_kernel(MmArgs a) {
  constexpr int kWaves = WM * WN, BM = 16 * TM * WM, BN = 16 * TN * WN, kBuf = (BM + BN) * 128, kScl = (BM + BN) * 4;
  static_assert((BM + BN) % (8 * kWaves) == 0 && BM % 8 == 0, "whole DMA instructions of 8 rows");
  constexpr int kDma = (BM + BN) / (8 * kWaves);                // 1 KB instructions of a wave and step
  static_assert((BM + BN) % 64 == 0 && BM % 64 == 0 && (BM + BN) / 64 <= kWaves, "one DMA instruction of 64 scale words a wave");
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * kBuf + 2 * kScl];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave - wm * WN;
  const int r = lane & 15, g = lane >> 4;

  // workgroup -> tile: each XCD (ids modulo 8) walks a contiguous run of tiles, column tiles of eight row tiles at a time
  const int tm_n = (a.M + BM - 1) / BM, tn_n = (a.N + BN - 1) / BN, tiles = tm_n * tn_n;
  const int id = blockIdx.x, per = tiles >> 3, rem = tiles & 7, xcd = id & 7;
  const int t = xcd * per + (xcd < rem ? xcd : rem) + (id >> 3);
  const int band = t / (8 * tn_n), in_band = t - band * 8 * tn_n, bh = min(8, tm_n - band * 8);
  const int m0 = (band * 8 + in_band % bh) * BM, n0 = (in_band / bh) * BN;

  const long long P = (long long)a.steps * 128, Q = (long long)((a.steps + 3) >> 2) * 4;
  const int k_begin = blockIdx.y * a.per_split, k_end = min(a.steps, k_begin + a.per_split);

  const int rows_a = min(BM, a.M - m0), rows_b = min(BN, a.N - n0);
  const __amdgpu_buffer_rsrc_t asrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.A + m0 * P), 0, (int)(rows_a * P), 0x00020000);
  const __amdgpu_buffer_rsrc_t bsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.B + n0 * P), 0, (int)(rows_b * P), 0x00020000);
  auto issue = [&](int kt, int buf) {
#pragma unroll
    for (int d = 0; d < kDma; ++d) {
      const int q = wave + kWaves * d;                          // rows 8 q .. 8 q + 7 of the buffer: first A's, then B's
      const bool is_a = q < BM / 8;
      const int row = (is_a ? q : q - BM / 8) * 8 + (lane >> 3);
      const unsigned voff = (unsigned)row * (unsigned)P + (unsigned)(((lane & 7) ^ (lane >> 3)) * 16);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(is_a ? asrc : bsrc, (__attribute__((address_space(3))) void *)(smem + buf * kBuf + q * 1024), 16,
                                               voff, kt * 128, 0, 0);
    }
  };
  // scale words of K steps 4 kg .. 4 kg + 3, rows as above
  const __amdgpu_buffer_rsrc_t asc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.sA + m0 * Q), 0, (int)(rows_a * Q), 0x00020000);
  const __amdgpu_buffer_rsrc_t bsc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.sB + n0 * Q), 0, (int)(rows_b * Q), 0x00020000);
  auto issue_scales = [&](int kg) {
    if (wave < (BM + BN) / 64) {
      const bool is_a = wave < BM / 64;
      const int row = (is_a ? wave : wave - BM / 64) * 64 + lane;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(is_a ? asc : bsc, (__attribute__((address_space(3))) void *)(smem + 2 * kBuf + (kg & 1) * kScl + wave * 256),
                                               4, (unsigned)row * (unsigned)Q, kg * 4, 0, 0);
    }
  };
  int sa[TM], sb[TN];
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto read_frag = [&](const unsigned char *rowp, i32x4 &lo, i32x4 &hi) {
    lo = *(const i32x4 *)(rowp + (((2 * g) ^ (r & 7)) * 16));
    hi = *(const i32x4 *)(rowp + (((2 * g + 1) ^ (r & 7)) * 16));
  };
  auto step = [&](auto sel_c, int kt) {
    constexpr int SEL = decltype(sel_c)::value;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (kt + 1 < k_end) {
      issue(kt + 1, (kt + 1) & 1);
      if (SEL == 3) issue_scales((kt + 1) >> 2);
    }
    if constexpr (SEL == 0) {
      const int *sc = (const int *)(smem + 2 * kBuf + ((kt >> 2) & 1) * kScl);
#pragma unroll
      for (int i = 0; i < TM; ++i) sa[i] = sc[(wm * TM + i) * 16 + r];
#pragma unroll
      for (int j = 0; j < TN; ++j) sb[j] = sc[BM + (wn * TN + j) * 16 + r];
    }
    const unsigned char *base = smem + (kt & 1) * kBuf;
    Operand<FB, EXACT> b[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      i32x4 lo, hi;
      read_frag(base + (BM + (wn * TN + j) * 16 + r) * 128, lo, hi);
      b[j].set(lo, hi, sb[j], SEL);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      i32x4 lo, hi;
      read_frag(base + ((wm * TM + i) * 16 + r) * 128, lo, hi);
      Operand<FA, EXACT> x;
      x.set(lo, hi, sa[i], SEL);
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mm_step<FB, FA, SEL>(b[j], x, acc[i][j], sb[j], sa[i]);
    }
  };
  if (k_begin < k_end) {
    issue(k_begin, k_begin & 1);
    issue_scales(k_begin >> 2);
  }
  for (int kt = k_begin; kt < k_end; kt += 4) {
    step(std::integral_constant<int, 0>{}, kt);
    if (kt + 1 < k_end) step(std::integral_constant<int, 1>{}, kt + 1);
    if (kt + 2 < k_end) step(std::integral_constant<int, 2>{}, kt + 2);
    if (kt + 3 < k_end) step(std::integral_constant<int, 3>{}, kt + 3);
  }

  // a lane's four consecutive columns of row (l & 15) of each 16 x 16 piece
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const long long m = m0 + (wm * TM + i) * 16 + r;
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + (wn * TN + j) * 16 + 4 * g;
      if (a.part) {
        float *p = a.part + ((long long)blockIdx.y * a.M + m) * a.N + n;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + q < a.N) p[q] = acc[i][j][q];
      } else {
        mm_store4(a, m, n, acc[i][j]);
      }
    }
  }
}

// the splits' sums in a fixed order, then the epilogue; four columns per thread
__global__ __launch_bounds__(256) void mm_join_kernel(MmArgs a) {
  const int n4 = (a.N + 3) >> 2;
  const long long total = (long long)a.M * n4;
  for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < total; u += (long long)gridDim.x * 256) {
    const long long m = u / n4;
    const int n = (int)(u - m * n4) * 4, cnt = min(4, a.N - n);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; ++s) {
      const float *p = a.part + ((long long)s * a.M + m) * a.N + n;
      f32x4 w = {0.f, 0.f, 0.f, 0.f};
      if (cnt == 4) __builtin_memcpy(&w, p, 16);
      else for (int t = 0; t < cnt; ++t) w[t] = p[t];
      v += w;
    }
    mm_store4(a, m, n, v);
  }
}

// ---- few rows -----------------------------------------------------------------------------------------------------------
// At most 16 T rows of A: B's bytes count, and they are read once, straight into registers.  A workgroup of W waves makes 16 columns;
// the waves take every W-th K step and add their sums through LDS in a fixed order.
template <int FA, int FB, bool EXACT, int T>
__global__ __launch_bounds__(1024) void mm_rows_kernel(MmArgs a) {
  extern __shared__ f32x4 red[];                                // [W][T][64]
  const int lane = threadIdx.x & 63, W = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * T;
  const long long P = (long long)a.steps * 128, Q = (long long)((a.steps + 3) >> 2) * 4;
  const long long nb = min(n0 + r, a.N - 1);
  const uint8_t *bp = a.B + nb * P + g * 32, *sbp = a.sB + nb * Q;
  const uint8_t *ap[T], *sap[T];
  f32x4 acc[T];
#pragma unroll
  for (int i = 0; i < T; ++i) {
    const long long m = min(m0 + 16 * i + r, a.M - 1);
    ap[i] = a.A + m * P + g * 32;
    sap[i] = a.sA + m * Q;
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int kt = wave; kt < a.steps; kt += W) {
    const long long at = (long long)kt * 128;
    Operand<FB, EXACT> b;
    const int sb = sbp[kt];
    b.set(*(const i32x4 *)(bp + at), *(const i32x4 *)(bp + at + 16), sb, 0);
#pragma unroll
    for (int i = 0; i < T; ++i) {
      Operand<FA, EXACT> x;
      const int sa = sap[i][kt];
      x.set(*(const i32x4 *)(ap[i] + at), *(const i32x4 *)(ap[i] + at + 16), sa, 0);
      acc[i] = mm_step<FB, FA, 0>(b, x, acc[i], sb, sa);
    }
  }
#pragma unroll
  for (int i = 0; i < T; ++i) red[(wave * T + i) * 64 + lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < T; i += W) {
    f32x4 v = red[i * 64 + lane];
    for (int w = 1; w < W; ++w) v += red[(w * T + i) * 64 + lane];
    const long long m = m0 + 16 * i + r;
    if (m < a.M) mm_store4(a, m, n0 + 4 * g, v);
  }
}

}  // namespace rows
}  // namespace snipper
