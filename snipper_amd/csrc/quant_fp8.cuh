// quant_fp8.cuh -- matrices into 8-bit blocks with a power-of-two scale for each 128 elements (gfx950); format: include/snipper_fp8.h.
//
//   q = round(x / 2^e),   e = smallest exponent with max|x| / 2^e <= largest value of the type,   over 128 elements of a row, of a
//   column, or of a 128 x 128 tile.
//
// Powers of two make the division exact, so a result is the input rounded once, and they are what the block-scaled matrix
// instructions of gemm_fp8.cuh take as they are.  The scale's exponent comes from the bits of the maximum, not from a logarithm.
// Bound by HBM: one read of x, one byte written per element and form.
#pragma once
#include "rows_common.cuh"

namespace snipper {
namespace rows {

struct QuantArgs {
  const void *x; long long ldx;
  int R, C;                                  // rows, columns
  const float *mean, *rstd;                  // [R] or null: normalise first
  const void *gamma, *beta; int p_dtype;     // [C] or null
  uint8_t *data, *scale;                     // [R][P], [R][Q] or null
  uint8_t *data_t, *scale_t;                 // [C][Pt], [C][Qt] or null
  float *part;                               // [ceil(R / 128)][C] or null: sums over the rows of a tile
};

__host__ __device__ __forceinline__ long long pitch_of(int cols) { return (long long)((cols + 127) / 128) * 128; }
__host__ __device__ __forceinline__ long long scales_of(int cols) { return (long long)((cols + 511) / 512) * 4; }

// ---- rows only.  A wave takes 512 consecutive elements of a row, 8 per lane: four blocks, so that it writes a whole 32-bit word of
// scales; 16 lanes share a block.  79 000 x 1024 bf16 43.5 us (5.6 TB/s), 79 000 x 384 float32 28.6 (5.3 TB/s), 16 384 x 8192 bf16 77.6 (5.2
// TB/s).  A row's last piece leaves lanes idle: 131 072 x 100 bf16 42 us (0.9 TB/s).
template <typename T, int FMT>
__global__ __launch_bounds__(256) void quant_rows_kernel(QuantArgs a) {
  const int lane = threadIdx.x & 63;
  const int groups = (a.C + 511) >> 9;
  const long long units = (long long)a.R * groups;
  const long long P = pitch_of(a.C), Q = scales_of(a.C);
  for (long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); u < units; u += (long long)gridDim.x * 4) {
    const long long row = u / groups;
    const int g = (int)(u - row * groups), c = g * 512 + lane * 8;
    float v[8];
    load8((const T *)a.x + row * a.ldx + c, a.C - c, v);
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, mag(v[j]));
    const int byte = scale_byte<FMT>(max16(m));
    const float f = inv_scale(byte);
    if (c < P) {
      const u32x2 w = {pack4<FMT>(v[0] * f, v[1] * f, v[2] * f, v[3] * f), pack4<FMT>(v[4] * f, v[5] * f, v[6] * f, v[7] * f)};
      *(u32x2 *)(a.data + row * P + c) = w;
    }
    const unsigned b0 = __shfl(byte, 0, 64), b1 = __shfl(byte, 16, 64), b2 = __shfl(byte, 32, 64), b3 = __shfl(byte, 48, 64);
    if (lane == 0) *(unsigned *)(a.scale + row * Q + g * 4) = b0 | (b1 << 8) | (b2 << 16) | (b3 << 24);
  }
}

// ---- both forms from one read.  A workgroup of eight waves holds a 128 x 128 tile in registers: lane (i, l) = (lane >> 4, lane & 15)
// of wave w the columns 8 l .. 8 l + 7 of rows 16 w + 4 i + k (k < 4); with four waves and twice the rows a lane the kernel took 192
// registers and ran at two waves a SIMD.  Four consecutive rows in one lane make a 32-bit word of the transposed form, which crosses
// LDS once (16-byte pieces XORed by the column's octet: reads are free of bank conflicts, writes two-way) and is written as whole
// 128-byte lines.  79 000 x 1024 bf16 with the columns' sums 67 us (4.8 TB/s), 79 000 x 384 float32 40 us (4.6 TB/s).
// Waves a SIMD: 6 without the normalisation (5: 72 us instead of 63 at 79 000 x 1024; 8 spills: 127), 5 with it (8192 x 4096: 37, with 6 45).
template <typename T, int FMT, bool TILE, bool NORM>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(NORM ? 5 : 6))) void quant_tile_kernel(QuantArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned img[128 * 32];
  __shared__ unsigned cmax[8][128];
  __shared__ __attribute__((aligned(16))) unsigned cfin[128];
  __shared__ float csum[8][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, i4 = lane >> 4;
  const int c0 = blockIdx.x * 128, c = c0 + 8 * l;
  const int rb = blockIdx.y + (int)blockIdx.z * 32768;
  const long long r0 = (long long)rb * 128;
  if (r0 >= a.R) return;                                   // (the whole workgroup)
  float v[4][8];
  float gm[8], bt[8];
  if constexpr (NORM) {
    load_param8(a.gamma, a.p_dtype, c, a.C - c, 1.f, gm);
    load_param8(a.beta, a.p_dtype, c, a.C - c, 0.f, bt);
  }
  const int n = a.C - c;                                     // columns this lane has (8 of them unless the matrix ends)
  const long long rl = r0 + 16 * wave + 4 * i4;
  auto row_of = [&](int k) { return rl + k; };
  if (n >= 8) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long long r = row_of(k) < a.R ? row_of(k) : a.R - 1;
      load_w<8, true>((const T *)a.x + r * a.ldx + c, 8, v[k]);        // (past the caches: what comes out is what is read again)
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long r = row_of(k) < a.R ? row_of(k) : a.R - 1;
        v[k][j] = j < n ? (float)((const T *)a.x)[r * a.ldx + c + j] : 0.f;
      }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const bool in = row_of(k) < a.R;
    if constexpr (NORM) {
      const float mu = in ? a.mean[row_of(k)] : 0.f, rs = in ? a.rstd[row_of(k)] : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = j < n ? (v[k][j] - mu) * rs * gm[j] + bt[j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[k][j] = in ? v[k][j] : 0.f;
  }
  const long long P = pitch_of(a.C), Q = scales_of(a.C), Pt = pitch_of(a.R), Qt = scales_of(a.R);
  const int kb = blockIdx.x, last_kb = (int)((P >> 7) - 1), last_rb = (int)((Pt >> 7) - 1);

  // largest magnitude of each column over the tile (and the columns' sums)
  unsigned cm[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    unsigned m = 0;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) { m = max(m, mag(v[k][j])); s += v[k][j]; }
#pragma unroll
    for (int o = 16; o <= 32; o <<= 1) {
      m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
      if (a.part) s += __shfl_xor(s, o, 64);
    }
    if (i4 == 0) { cmax[wave][8 * l + j] = m; if (a.part) csum[wave][8 * l + j] = s; }
  }
  __syncthreads();
  if (threadIdx.x < 128) {
    const int t = threadIdx.x;
    unsigned m = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, cmax[w][t]);
    cfin[t] = m;
    if (a.part && c0 + t < a.C) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += csum[w][t];
      a.part[(long long)rb * a.C + c0 + t] = s;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; j += 4) {
    const u32x4 m = *(const u32x4 *)(cfin + 8 * l + j);
    cm[j] = m[0]; cm[j + 1] = m[1]; cm[j + 2] = m[2]; cm[j + 3] = m[3];
  }
  unsigned all = 0;
  if constexpr (TILE) {
#pragma unroll
    for (int j = 0; j < 8; ++j) all = max(all, cm[j]);
    all = max16(all);
  }

  // rows
  if (a.data) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      unsigned m = all;
      if constexpr (!TILE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, mag(v[k][j]));
        m = max16(m);
      }
      const int byte = scale_byte<FMT>(m);
      const float f = inv_scale(byte);
      const float (&x)[8] = v[k];
      const long long r = row_of(k);
      if (r < a.R) {
        const u32x2 w = {pack4<FMT>(x[0] * f, x[1] * f, x[2] * f, x[3] * f), pack4<FMT>(x[4] * f, x[5] * f, x[6] * f, x[7] * f)};
        *(u32x2 *)(a.data + r * P + c) = w;
        if (l == 0) a.scale[r * Q + kb] = (uint8_t)byte;
        if (kb == last_kb && l > 0 && kb + l < Q) a.scale[r * Q + kb + l] = 127;
      }
    }
  }
  if (!a.data_t) return;
  // columns
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int byte = scale_byte<FMT>(TILE ? all : cm[j]);
    const float f = inv_scale(byte);
    const int cl = 8 * l + j;
    const int piece = wave ^ (l & 7);                             // 16-byte piece of the column's line; (cl >> 3) & 7 = l & 7
    img[cl * 32 + piece * 4 + i4] = pack4<FMT>(v[0][j] * f, v[1][j] * f, v[2][j] * f, v[3][j] * f);
    if (wave == 0 && i4 == 0 && c + j < a.C) {
      uint8_t *s = a.scale_t + (long long)(c + j) * Qt;
      s[rb] = (uint8_t)byte;
      if (rb == last_rb)
        for (int t = rb + 1; t < Qt; ++t) s[t] = 127;
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int idx = threadIdx.x + 512 * q, cl = idx >> 3, piece = idx & 7;
    if (c0 + cl < a.C)
      *(u32x4 *)(a.data_t + (long long)(c0 + cl) * Pt + r0 + piece * 16) = *(const u32x4 *)(img + cl * 32 + (piece ^ ((cl >> 3) & 7)) * 4);
  }
}

// out[c] = sum_b part[b][c]
__global__ __launch_bounds__(1024) void colsum_parts_kernel(const float *part, int nparts, int C, void *out, int out_dt) {
  const int c = blockIdx.x * 32 + (threadIdx.x & 31);
  const float s = sum_parts(part, nparts, C, c);
  if (threadIdx.x < 32 && c < C) store_param(out, out_dt, c, s);
}

}  // namespace rows
}  // namespace snipper
