// gemm_fp8.cuh -- out [M][N] = act(A [M][K] . B [N][K]^T + bias) of two matrices in 8-bit blocks (gfx950; format: include/snipper_fp8.h).
//
//   out[m][n] = sum_b 2^(ea[m][b] + eb[n][b]) sum_{k in block b} a[m][k] b[n][k]
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 elements with a power-of-two scale for each 32 of a lane's
// elements: a block of 128 is one instruction whose four scales are the same byte, so scaling costs no instruction at all and any
// order of the 128 elements within the operands is right as long as both have the same one.  Its sums: the products of eight neighbours
// (bytes 8 i .. 8 i + 7 of a lane's operand, here of a row) are aligned to the largest of the eight and cut off at 2^-13 of it, towards
// zero; the groups and the accumulator are added in float32.  (Found with single products over and under a larger one, every
// distance, place and sign; the unscaled 16 x 16 x 32 instruction does the same.)  So a group loses less than 7 * 2^-13 = 8.5e-4 of its largest
// product, an element less than that of sum |a b|, in the worst case: under a quarter of half a step of a bfloat16 (2^-8) of that size, 1.75 half
// steps of a float16 (2^-11).  On random data 1.5e-5 of the result's norm at K = 128 .. 65 536.  That is the rounding to fewer bits that 16-bit
// results take for the rate: beside the operands' own, up to 2^-4 of every product, it is small; a caller whose operands are exact can ask
// for float32 sums (SNIPPER_FP8_FULL_SUMS), and float32 results always have them.  Those EXACT kernels widen the operands to bfloat16
// with their scales -- 4 bits and a power of two fit exactly -- and use v_mfma_f32_16x16x32_bf16 (1e-7), at a quarter of the rate (4096^3
// 66 us with the 8-bit instructions, 119 so; 384 x 1024 x 79 000 62 and 73; 480 x 1024 x 384 4.7 and 5.2).
//
// Rows of n are the first operand and rows of m the second, so that a lane holds consecutive columns of one row of the result.
#pragma once
#include <utility>
#include "rows_common.cuh"

namespace snipper {
namespace rows {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

constexpr int kPastCaches = 2;               // (non-temporal, of buffer accesses)

struct MmArgs {
  const uint8_t *A, *sA, *B, *sB;            // [M][P], [M][Q], [N][P], [N][Q]
  int M, N;
  int steps;                                 // P / 128
  const void *bias; int bias_dt; int relu;
  void *out; int out_dt;
  float *part;                               // [splits][M][N] or null
  int splits, per_split;                     // K steps of a split (a multiple of 4)
};

__device__ __forceinline__ uint16_t mm_half(float v, int dt) {
  return dt == kBF16 ? __builtin_bit_cast(uint16_t, (bf16_t)v) : __builtin_bit_cast(uint16_t, (f16_t)v);
}
template <int W>
__device__ __forceinline__ void mm_bias(const MmArgs &a, int n, float (&v)[W]) {       // of columns n .. n + W - 1, 0 where there is none
#pragma unroll
  for (int t = 0; t < W; ++t) v[t] = a.bias && n + t < a.N ? load_param(a.bias, a.bias_dt, n + t) : 0.f;
}
// W elements of a row of the result: columns n .. n + W - 1
template <int W>
__device__ __forceinline__ void mm_store(const MmArgs &a, long long m, int n, const float (&acc)[W], const float (&bias)[W]) {
  const int cnt = a.N - n;
  if (cnt <= 0) return;
  float v[W];
#pragma unroll
  for (int t = 0; t < W; ++t) {
    v[t] = acc[t] + bias[t];
    v[t] = a.relu && v[t] < 0.f ? 0.f : v[t];                         // (a NaN stays one)
  }
  const long long at = m * a.N + n;
  if (a.out_dt == kF32) {
    float *p = (float *)a.out + at;
    if (cnt >= W) __builtin_memcpy(p, v, 4 * W);
    else {
#pragma unroll
      for (int t = 0; t < W; ++t) if (t < cnt) p[t] = v[t];
    }
  } else {
    uint16_t h[W];
#pragma unroll
    for (int t = 0; t < W; ++t) h[t] = mm_half(v[t], a.out_dt);
    uint16_t *p = (uint16_t *)a.out + at;
    if (cnt >= W) __builtin_memcpy(p, h, 2 * W);
    else {
#pragma unroll
      for (int t = 0; t < W; ++t) if (t < cnt) p[t] = h[t];
    }
  }
}
// Which row of B a lane holds in operand j of a pair (j even, j + 1): with these the two 16 x 16 results of a pair give a lane eight
// consecutive columns of a row, 16 bytes of a 16-bit result, and a wave's store whole 64-byte pieces.
__device__ __forceinline__ int mm_pair_row(int j, int r) { return 32 * (j >> 1) + 8 * (r >> 2) + 4 * (j & 1) + (r & 3); }

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

// Widened with their scales, elements are exact bfloat16 values and sums of their products float32 ones as long as the scales of both
// sides lie in 2^-95 .. 2^96 (bytes 32 .. 223: the upper three bits not all alike).  Others (a caller's, or those of magnitudes above
// 2^104 or below 2^-86) would overflow or vanish in bfloat16 where the product's own scale 2^(ea + eb) need not: there the widened
// elements stay without their scales, and each block's sum takes both at once (mm_add_scaled).  A workgroup of the tile kernel decides
// that once, before its loop (1024^3 7.2 -> 7.6 us, 384 x 1024 x 79 000 72 -> 73), the kernel for few
// rows for each group of steps; a tile of such scales takes 1.8 times as long.
constexpr unsigned kEachByte = 0x80808080u;
__device__ __forceinline__ unsigned ordinary_scales(int word) {        // the top bits of the bytes that are ordinary
  const unsigned w = (unsigned)word, t = w ^ (w << 1);
  return t | (t << 1) | (((w & ~kEachByte) + 0x01010101u) & w);       // (255, which stands for NaN, is one of them)
}
template <int SEL>
__device__ __forceinline__ f32x4 mm_add_scaled(f32x4 acc, f32x4 part, int sa, i32x4 sb) {
  const int ea = (int)(((unsigned)sa >> (8 * SEL)) & 255u);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int eb = (int)(((unsigned)sb[q] >> (8 * SEL)) & 255u);
    acc[q] += ea == 255 || eb == 255 ? __builtin_nanf("") : __builtin_ldexpf(part[q], ea + eb - 254);
  }
  return acc;
}
constexpr int kScaleOne = 0x7f7f7f7f;

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

// a value that has been loaded: the wait for its load is placed here
template <typename T>
__device__ __forceinline__ void settle(T &x) { asm volatile("" : "+v"(x)); }
// 16 (4) bytes per lane from base + voff + soff to LDS, lane after lane; for offsets voff >= range zeros
__device__ __forceinline__ void dma16(const uint8_t *base, int range, unsigned char *lds, unsigned voff, unsigned soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, range, 0x00020000),
                                           (__attribute__((address_space(3))) void *)lds, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void dma4(const uint8_t *base, int range, unsigned char *lds, unsigned voff, unsigned soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, range, 0x00020000),
                                           (__attribute__((address_space(3))) void *)lds, 4, voff, soff, 0, 0);
}
// all but the last N vector memory instructions of this wave are done
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// f(0), f(1), ... with constants
template <typename F, int... K>
__device__ __forceinline__ void each_step(F &&f, std::integer_sequence<int, K...>) { (f(std::integral_constant<int, K>{}), ...); }

// ---- tiles -----------------------------------------------------------------------------------------------------------
// A workgroup of WM x WN waves makes a (16 TM WM) x (16 TN WN) tile; a K step of 128 is one byte-row of 128 per row of either side.
// Rows go to LDS by DMA in 16-byte pieces, piece c of row r at place c ^ key(r), and a lane takes pieces g and g + 4 of its row (both
// sides alike), so that reads are free of bank conflicts: a 16-byte read serves lanes 0-3, 12-15, 20-27, then 4-11, 16-19, 28-31, then
// the same of the upper half, 256 bytes each (counted; keys that suit groups of 8 or 16 neighbours cost twice the clocks).  A:
// consecutive rows, key = r & 7; B: rows of mm_pair_row, key = bits 0, 1 and 3 of r; two buffers, one barrier a step.  The scale words
// of four K steps come the same way (plain loads of them would make the compiler wait for the DMAs issued after them).
// 8192^3 in tiles of 256 x 256 by eight waves of 128 x 64: 458 us, 2.4 PFLOP/s, where the instructions alone reach 3.65 .. 4.45 on such
// data and a large library product 2.98.  A K step takes 64 KB from the L2 into LDS for 16.8 MFLOP a CU, and the LDS reads of its waves
// and that fill share the LDS; four waves of 128 x 128, which read less, hold half the rows in flight (510 .. 568 us), operands
// straight from the L2 735, steps of half a block with the 32 x 32 x 64 instruction 558, touching lines a step ahead 491.  EXACT: 79 000
// x 1024 x 384's weight gradient 72 us = 0.86 PFLOP/s; the bfloat16 instructions' own limit is 43 us, the rest is widening.
// INWARD (M >= BM, N >= BN): the last tile of an edge is moved inwards, and two workgroups store the same values; rows need no range
// checks then, and their addresses one register a side instead of one for each load.
template <int FA, int FB, bool EXACT, int WM, int WN, int TM, int TN, bool INWARD>
__global__ __launch_bounds__(64 * WM * WN) void mm_tile_kernel(MmArgs a) {
  constexpr int kWaves = WM * WN, BM = 16 * TM * WM, BN = 16 * TN * WN, kBuf = (BM + BN) * 128, kScl = (BM + BN) * 4;
  static_assert((BM + BN) % (8 * kWaves) == 0 && BM % 8 == 0, "whole DMA instructions of 8 rows");
  constexpr int kDma = (BM + BN) / (8 * kWaves);                // 1 KB instructions of a wave and step
  static_assert((BM + BN) % 64 == 0 && BM % 64 == 0 && (BM + BN) / 64 <= kWaves, "one DMA instruction of 64 scale words a wave");
  // (one object: with another beside it the compiler waits for the DMA into this one before every read, 73 -> 84 us)
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * kBuf + 2 * kScl + (EXACT ? 16 : 0)];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave - wm * WN;
  const int r = lane & 15, g = lane >> 4;

  // workgroup -> piece of the K axis and tile: each XCD (ids modulo 8) walks a contiguous run, so that the tiles of a piece, which share
  // its rows' bytes, are on one XCD; within a piece column tiles of eight row tiles at a time
  const int tm_n = (a.M + BM - 1) / BM, tn_n = (a.N + BN - 1) / BN, tiles = tm_n * tn_n;
  const int id = blockIdx.x, all = tiles * a.splits, per = all >> 3, rem = all & 7, xcd = id & 7;
  const int at = xcd * per + (xcd < rem ? xcd : rem) + (id >> 3);
  const int split = at / tiles, t = at - split * tiles;
  const int band = t / (8 * tn_n), in_band = t - band * 8 * tn_n, bh = min(8, tm_n - band * 8);
  int m0 = (band * 8 + in_band % bh) * BM, n0 = (in_band / bh) * BN;
  if constexpr (INWARD) { m0 = min(m0, a.M - BM); n0 = min(n0, a.N - BN); }

  const long long P = (long long)a.steps * 128, Q = (long long)((a.steps + 3) >> 2) * 4;
  const int k_begin = split * a.per_split, k_end = min(a.steps, k_begin + a.per_split);

  const int rows_a = min(BM, a.M - m0), rows_b = min(BN, a.N - n0);
  static_assert((BM / 8) % kWaves == 0 && kWaves % 2 == 0, "an instruction's side is known at compile time, its parity the wave's");
  const unsigned key_a = lane >> 3, key_w = ((lane >> 3) & 3) | ((wave & 1) << 2);
  const unsigned va = (8 * wave + (lane >> 3)) * (unsigned)P + ((lane & 7) ^ key_a) * 16, vb = (8 * wave + (lane >> 3)) * (unsigned)P + ((lane & 7) ^ key_w) * 16;
  auto issue = [&](int kt, int buf) {
#pragma unroll
    for (int d = 0; d < kDma; ++d) {
      constexpr int kA = BM / 8 / kWaves;
      const bool is_a = d < kA;                                 // 8 rows of A, or of B, behind them
      const unsigned rows_on = (unsigned)(is_a ? d : d - kA) * (8u * kWaves) * (unsigned)P;
      dma16(is_a ? a.A + m0 * P : a.B + n0 * P, (int)((is_a ? rows_a : rows_b) * P), smem + buf * kBuf + (wave + kWaves * d) * 1024,
            (is_a ? va : vb) + (INWARD ? 0u : rows_on), kt * 128u + (INWARD ? rows_on : 0u));
    }
  };
  // scale words of K steps 4 kg .. 4 kg + 3, rows as above
  auto issue_scales = [&](int kg) {
    if (wave < (BM + BN) / 64) {
      const bool is_a = wave < BM / 64;
      const int row = (is_a ? wave : wave - BM / 64) * 64 + lane;
      dma4(is_a ? a.sA + m0 * Q : a.sB + n0 * Q, (int)((is_a ? rows_a : rows_b) * Q), smem + 2 * kBuf + (kg & 1) * kScl + wave * 256,
           (unsigned)row * (unsigned)Q, kg * 4);
    }
  };
  auto read_frag = [&](const unsigned char *rowp, int key, i32x4 &lo, i32x4 &hi) {
    lo = *(const i32x4 *)(rowp + ((g ^ key) * 16));
    hi = *(const i32x4 *)(rowp + (((g + 4) ^ key) * 16));
  };
  const int key_b = (r & 3) | (r & 4);                          // bit 3 of mm_pair_row(., r) is bit 2 of r
  auto step = [&](auto far_c, auto sel_c, int kt, int (&sa)[TM], int (&sb)[TN], f32x4 (&acc)[TM][TN]) {
    constexpr bool FAR = decltype(far_c)::value;
    constexpr int SEL = decltype(sel_c)::value;
    wait_loads<0>();
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
      for (int j = 0; j < TN; ++j) sb[j] = sc[BM + wn * TN * 16 + mm_pair_row(j, r)];
    }
    const unsigned char *base = smem + (kt & 1) * kBuf;
    if constexpr (FAR) {
      const int *sc = (const int *)(smem + 2 * kBuf + ((kt >> 2) & 1) * kScl);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        i32x4 lo, hi;
        read_frag(base + (BM + wn * TN * 16 + mm_pair_row(j, r)) * 128, key_b, lo, hi);
        Operand<FB, true> o;
        o.set(lo, hi, kScaleOne, SEL);
        const i32x4 eb = *(const i32x4 *)(sc + BM + wn * TN * 16 + mm_pair_row(j, 4 * g));        // rows 4 g .. 4 g + 3 of the pair: neighbours
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          read_frag(base + ((wm * TM + i) * 16 + r) * 128, r & 7, lo, hi);
          Operand<FA, true> x;
          x.set(lo, hi, kScaleOne, SEL);
          acc[i][j] = mm_add_scaled<SEL>(acc[i][j], mm_step<FB, FA, SEL>(o, x, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0), sa[i], eb);
          __builtin_amdgcn_sched_barrier(0);                    // (one piece at a time: registers)
        }
      }
      return;
    }
    Operand<FB, EXACT> b[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      i32x4 lo, hi;
      read_frag(base + (BM + wn * TN * 16 + mm_pair_row(j, r)) * 128, key_b, lo, hi);
      b[j].set(lo, hi, sb[j], SEL);
    }
    if constexpr (EXACT) __builtin_amdgcn_s_setprio(1);         // (the wave beside this one widens meanwhile: 274 -> 269 us of a training step)
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      i32x4 lo, hi;
      read_frag(base + ((wm * TM + i) * 16 + r) * 128, r & 7, lo, hi);
      Operand<FA, EXACT> x;
      x.set(lo, hi, sa[i], SEL);
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mm_step<FB, FA, SEL>(b[j], x, acc[i][j], sb[j], sa[i]);
    }
    if constexpr (EXACT) __builtin_amdgcn_s_setprio(0);
  };
  auto sums = [&](auto far_c) {
    int sa[TM], sb[TN];
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int kt = k_begin; kt < k_end; kt += 4) {
      step(far_c, std::integral_constant<int, 0>{}, kt, sa, sb, acc);
      if (kt + 1 < k_end) step(far_c, std::integral_constant<int, 1>{}, kt + 1, sa, sb, acc);
      if (kt + 2 < k_end) step(far_c, std::integral_constant<int, 2>{}, kt + 2, sa, sb, acc);
      if (kt + 3 < k_end) step(far_c, std::integral_constant<int, 3>{}, kt + 3, sa, sb, acc);
    }
    // a lane's eight consecutive columns of row (l & 15) of each pair of 16 x 16 pieces
#pragma unroll
    for (int j = 0; j < TN; j += 2) {
      const int n = n0 + wn * TN * 16 + j * 16 + 8 * g;
      float bias[8];
      if (!a.part) mm_bias(a, n, bias);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const long long m = m0 + (wm * TM + i) * 16 + r;
        if (m >= a.M) continue;
        float v[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) { v[q] = acc[i][j][q]; v[4 + q] = acc[i][j + 1][q]; }
        if (a.part) store8(a.part + ((long long)split * a.M + m) * a.N + n, a.N - n, v);
        else mm_store(a, m, n, v, bias);
      }
    }
  };
  // EXACT: are the scales of the tile's rows, one row a thread, all ordinary ones?  Eight words a time, the first of them on their way
  // before the first step's rows.  (A choice for each group of steps inside the loop: 384 x 1024 x 79 000 73 -> 81 us, in registers.)
  const int n_words = ((k_end + 3) >> 2) - (k_begin >> 2);
  const int *words = nullptr;
  int w[8];
  auto look = [&](int at) {                                     // (the last one again behind it: no branches)
#pragma unroll
    for (int q = 0; q < 8; ++q) w[q] = words[min(at + q, n_words - 1)];
  };
  if constexpr (EXACT) {
    static_assert(BM + BN <= 64 * kWaves, "a thread for each row");
    const int row = threadIdx.x % (BM + BN);
    // (the tile's last row again behind it)
    words = (const int *)(row < BM ? a.sA + (m0 + min(row, rows_a - 1)) * Q : a.sB + (n0 + min(row - BM, rows_b - 1)) * Q) + (k_begin >> 2);
    look(0);
  }
  if (k_begin < k_end) {
    issue(k_begin, k_begin & 1);
    issue_scales(k_begin >> 2);
  }
  bool far = false;
  if constexpr (EXACT) {
    unsigned usual = kEachByte;
    for (int at = 0;;) {
#pragma unroll
      for (int q = 0; q < 8; ++q) usual &= ordinary_scales(w[q]);
      at += 8;
      if (at >= n_words) break;
      look(at);
    }
    static_assert(kWaves == 4, "a word of flags each");
    int *flags = (int *)(smem + 2 * kBuf + 2 * kScl);
    if (lane == 0) flags[wave] = 0;
    if (usual != kEachByte) flags[wave] = 1;
    __syncthreads();
    const i32x4 any = *(const i32x4 *)flags;
    far = (any[0] | any[1] | any[2] | any[3]) != 0;
  }
  if (EXACT && far) sums(std::integral_constant<bool, EXACT>{});
  else sums(std::false_type{});
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
    const float o[4] = {v[0], v[1], v[2], v[3]};
    float bias[4];
    mm_bias(a, n, bias);
    mm_store(a, m, n, o, bias);
  }
}

// the loads of a chunk of 64 rows and of its scale words, KS + ceil(KS / 4) instructions of every wave; behind the last chunk the range
// is empty: zeros for a slot that nobody reads
template <int KS>
__device__ __forceinline__ void issue_chunk(const MmArgs &a, unsigned char *slot, const unsigned *voff, int chunk, int wave, int lane) {
  constexpr int PB = KS * 128, QB = (KS + 3) / 4 * 4;
  const int rows = max(0, min(64, a.M - chunk * 64));
  const long long first = rows > 0 ? (long long)chunk * 64 : 0;
#pragma unroll
  for (int d = 0; d < KS; ++d) dma16(a.A + first * PB, rows * PB, slot + (wave * KS + d) * 1024, voff[d], 0);
#pragma unroll
  for (int d = 0; d < QB / 4; ++d)                              // (every wave the same words: the counts stay equal)
    dma4(a.sA + first * QB, rows * QB, slot + 64 * PB + d * 256, (unsigned)(d * 64 + lane) * 4, 0);
}

// ---- short rows, many of them ----------------------------------------------------------------------------------------
// K <= 128 KS: B stays in registers.  Each of the eight waves holds 32 columns (two operands of KS steps, 16 KS registers), a workgroup
// 256; the rows of A stream past in chunks of 64 through an LDS ring filled by DMA, and one persistent workgroup per CU walks over
// chunks.  A tile kernel of such shapes spends its time filling and draining: its two or three K steps do not cover the latency of
// their loads, nor the stores of the tile before.  Here loads run S - 1 chunks ahead across the stores; the counted waits rely on every
// wave issuing the same number of memory instructions per chunk, so rows and columns past the end go through the buffers' range
// checks.  The workgroups that share a chunk sit on one XCD: A comes from HBM once.  Results go past the caches where the 64 bytes
// that a wave writes of a row are whole ones in memory (WHOLE: N a multiple of 32): 79 000 x 1024 x 384 54 -> 49 us (tiles of 128 x 128: 90), 193 MB at 3.9 TB/s, nearly
// all of them stores; elsewhere two waves' pieces meet in the L2 first: N = 1000 101 -> 46 us, 520 48 -> 36 (264 24 -> 25).
template <int FA, int FB, int KS, bool WHOLE>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void mm_stationary_kernel(MmArgs a, int n_series) {
  constexpr int ROWS = 64, PB = KS * 128, S = KS <= 4 ? 4 : KS <= 6 ? 3 : 2, QW = (KS + 3) / 4, kChunk = ROWS * PB, kScl = ROWS * QW * 4;
  constexpr int kLoads = KS + QW, kStores = 4;
  __shared__ __attribute__((aligned(16))) unsigned char smem[S * (kChunk + kScl)];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int ncb = (a.N + 255) >> 8, per_group = 8 * ncb;
  const int grp = blockIdx.x / per_group, within = blockIdx.x - grp * per_group;
  const int series = grp * 8 + (within & 7), n0 = (within >> 3) * 256 + wave * 32;
  const int chunks = (a.M + ROWS - 1) / ROWS;
  const int iters = series < chunks ? (chunks - series + n_series - 1) / n_series : 0;
  if (iters == 0) return;                                       // (the whole workgroup)

  // piece c of row `row` of a chunk lies at place c ^ (row & 7) of its 128 bytes, and where a row is a multiple of 256 bytes the odd
  // ones have neighbouring 128s swapped (see mm_tile_kernel on bank conflicts); a wave's instruction moves 64 pieces
  unsigned voff[KS];
#pragma unroll
  for (int d = 0; d < KS; ++d) {
    const int p = (wave * KS + d) * 64 + lane, row = p / (8 * KS), c = p - row * (8 * KS);
    voff[d] = row * PB + ((((c >> 3) ^ (KS % 2 ? 0 : row & 1)) << 3) | ((c ^ row) & 7)) * 16;
  }
  i32x8 b[2][KS];
  int sb[2][QW];
  float bias[8];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const long long n = min(n0 + mm_pair_row(j, r), a.N - 1);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const i32x4 lo = *(const i32x4 *)(a.B + n * PB + k * 128 + g * 16), hi = *(const i32x4 *)(a.B + n * PB + k * 128 + g * 16 + 64);
      b[j][k] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
#pragma unroll
    for (int q = 0; q < QW; ++q) sb[j][q] = *(const int *)(a.sB + n * QW * 4 + q * 4);
  }
  load_param8(a.bias, a.bias_dt, n0 + 8 * g, a.N - (n0 + 8 * g), 0.f, bias);
  // the loads above are waited for here, not at their first use in the loop (where the wait would drain the ring every time)
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int k = 0; k < KS; ++k) settle(b[j][k]);
#pragma unroll
    for (int q = 0; q < QW; ++q) settle(sb[j][q]);
  }
#pragma unroll
  for (int t = 0; t < 8; ++t) settle(bias[t]);
#pragma unroll
  for (int it = 0; it < S - 1; ++it) issue_chunk<KS>(a, smem + it * (kChunk + kScl), voff, it < iters ? series + it * n_series : chunks, wave, lane);

  for (int it = 0; it < iters; ++it) {
    // chunk `it` has come when all but the instructions behind its loads are done: S - 2 chunks of loads and (once the pipe is
    // full) S - 1 chunks of stores
    if (it < S - 1) wait_loads<(S - 2) * kLoads>();
    else wait_loads<(S - 2) * kLoads + (S - 1) * kStores>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const int ahead = it + S - 1;                               // into the slot that every wave has left
    issue_chunk<KS>(a, smem + (ahead % S) * (kChunk + kScl), voff, ahead < iters ? series + ahead * n_series : chunks, wave, lane);
    const unsigned char *slot = smem + (it % S) * (kChunk + kScl);
    const int *scl = (const int *)(slot + kChunk);
    const int chunk = series + it * n_series;
    const int rows = min(ROWS, a.M - chunk * ROWS);
    const __amdgpu_buffer_rsrc_t dst = __builtin_amdgcn_make_buffer_rsrc((uint16_t *)a.out + (long long)chunk * ROWS * a.N, 0, rows * a.N * 2, 0x00020000);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * i + r;
      f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
      int sa[QW];
#pragma unroll
      for (int q = 0; q < QW; ++q) sa[q] = scl[row * QW + q];
      each_step([&](auto step) {
        constexpr int K = decltype(step)::value;
        const unsigned char *at = slot + row * PB + (KS % 2 ? K : K ^ (r & 1)) * 128;
        Operand<FA, false> x;
        x.set(*(const i32x4 *)(at + ((g ^ (r & 7)) * 16)), *(const i32x4 *)(at + (((g + 4) ^ (r & 7)) * 16)), 0, 0);
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[j] = mm_step<FB, FA, K & 3>(Operand<FB, false>{b[j][K]}, x, acc[j], sb[j][K >> 2], sa[K >> 2]);
      }, std::make_integer_sequence<int, KS>{});
      uint16_t h[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        float v = acc[t >> 2][t & 3] + bias[t];
        v = a.relu && v < 0.f ? 0.f : v;
        h[t] = mm_half(v, a.out_dt);
      }
      u32x4 w;
      __builtin_memcpy(&w, h, 16);
      const int n = n0 + 8 * g;
      const unsigned to = n < a.N ? (unsigned)row * (unsigned)a.N * 2u + (unsigned)n * 2u : 0x80000000u;
      __builtin_amdgcn_raw_buffer_store_b128(w, dst, to, 0, WHOLE ? kPastCaches : 0);
    }
  }
  wait_loads<0>();                                              // (the empty loads behind the last chunk)
}

// ---- few rows -----------------------------------------------------------------------------------------------------------
// At most 16 rows of A: B's bytes count, and they are read once, straight into registers; the sums are full ones for every type of result,
// since widening costs nothing beside the loads (1 x 8192 x 8192 15.7 us with the 8-bit instructions, 15.0 so).  A workgroup of W waves makes 16 columns; the
// waves take every W-th group of four K steps (a word of scales; all of a group's loads are on the way before its first product) and
// add their sums through LDS in a fixed order.  Bound by latency and HBM: 1 x 4096 x 4096 6.6 us (17 MB, 2.5 TB/s), 1 x 8192 x 8192 15 us
// (67 MB, 4.5 TB/s).
template <int FA, int FB>
__global__ __launch_bounds__(512) void mm_rows_kernel(MmArgs a) {
  __shared__ f32x4 red[8][64];
  const int lane = threadIdx.x & 63, W = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const long long P = (long long)a.steps * 128, Q = (long long)((a.steps + 3) >> 2) * 4;
  const long long nb = min(n0 + r, a.N - 1), m = min(r, a.M - 1);
  const uint8_t *bp = a.B + nb * P + g * 32, *sbp = a.sB + nb * Q, *ap = a.A + m * P + g * 32, *sap = a.sA + m * Q;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int kg = wave; kg < (a.steps + 3) >> 2; kg += W) {
    const int sb = *(const int *)(sbp + kg * 4), sa = *(const int *)(sap + kg * 4);
    i32x4 b[4][2], x[4][2];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const long long at = min(kg * 4 + q, a.steps - 1) * 128ll;        // (a step behind the last one: loaded, not used)
      b[q][0] = *(const i32x4 *)(bp + at);
      b[q][1] = *(const i32x4 *)(bp + at + 16);
      x[q][0] = *(const i32x4 *)(ap + at);
      x[q][1] = *(const i32x4 *)(ap + at + 16);
    }
    if (!__all((ordinary_scales(sa) & ordinary_scales(sb) & kEachByte) == kEachByte)) {
      i32x4 eb;
#pragma unroll
      for (int q = 0; q < 4; ++q) eb[q] = __shfl(sb, 4 * g + q, 64);
      each_step([&](auto step) {
        constexpr int S = decltype(step)::value;
        if (kg * 4 + S < a.steps) {
          Operand<FB, true> o;
          Operand<FA, true> i;
          o.set(b[S][0], b[S][1], kScaleOne, S);
          i.set(x[S][0], x[S][1], kScaleOne, S);
          acc = mm_add_scaled<S>(acc, mm_step<FB, FA, S>(o, i, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0), sa, eb);
        }
      }, std::make_integer_sequence<int, 4>{});
      continue;
    }
    each_step([&](auto step) {
      constexpr int S = decltype(step)::value;
      if (kg * 4 + S < a.steps) {
        Operand<FB, true> o;
        Operand<FA, true> i;
        o.set(b[S][0], b[S][1], sb, S);
        i.set(x[S][0], x[S][1], sa, S);
        acc = mm_step<FB, FA, S>(o, i, acc, sb, sa);
      }
    }, std::make_integer_sequence<int, 4>{});
  }
  red[wave][lane] = acc;
  __syncthreads();
  if (wave == 0) {
    for (int w = 1; w < W; ++w) acc += red[w][lane];
    const float o[4] = {acc[0], acc[1], acc[2], acc[3]};
    float bias[4];
    mm_bias(a, n0 + 4 * g, bias);
    if (r < a.M) mm_store(a, r, n0 + 4 * g, o, bias);
  }
}

}  // namespace rows
}  // namespace snipper
