// layernorm_rows.cuh -- layer norm of rows of any width up to 16 384, forward and backward (gfx950).
//
//   y = h gamma + beta,  h = (x - mean) rstd,  rstd = 1 / sqrt(var + eps)                     (statistics of a row, in float32)
//   dx = rstd (t - mean(t) - h mean(t h)),  t = g gamma;      dgamma = sum_rows g h,  dbeta = sum_rows g
//
// csrc/ln_fused.cuh has the residual + dropout form for widths that are multiples of 4 up to 1024, in float32 and bfloat16; this one
// takes any width, stride and alignment, float16 too, and can write its result as 8-bit blocks (format: include/snipper_fp8.h).
// Bound by HBM.  A row stays in the registers of LPR lanes, 8 consecutive elements per lane and chunk, from its one load to its
// store: the mean first, then the sum of squared deviations from it, so nothing cancels.  Workgroups walk over rows, so gamma, beta
// and the column sums of the backward pass live in registers too; the sums meet in LDS, then in one row of a partial buffer per
// workgroup, which a second kernel adds in a fixed order.
#pragma once
#include "rows_common.cuh"

namespace snipper {
namespace rows {

struct LnRowsArgs {
  const void *x; long long ldx;
  const void *gamma, *beta; int p_dtype;
  int R, C;
  float eps;
  void *y;
  float *mean, *rstd;
  uint8_t *data, *scale;
  // backward
  const void *g; void *dx; float *part;      // part [gridDim.x][2][C] or null
};

// sum over the LPR lanes that share a row (LPR = 16: a quarter of a wave; 64: a wave; more: whole workgroup, through LDS)
template <int LPR>
__device__ __forceinline__ float ln_row_sum(float v, float *red) {
#pragma unroll
  for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    __syncthreads();                                   // (the last call's values have been read)
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) v += red[w];
  }
  return v;
}

constexpr int ln_threads(int lpr) { return lpr > 256 ? lpr : 256; }

// FMT < 0: no blocks
template <typename T, int LPR, int NIT, int FMT>
__global__ __launch_bounds__(ln_threads(LPR)) void ln_rows_fwd_kernel(LnRowsArgs a) {
  constexpr int RPW = ln_threads(LPR) / LPR;           // rows of a workgroup at a time
  __shared__ float red[16];
  const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  float gm[NIT][8], bt[NIT][8];
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    const int c = (l + LPR * it) * 8;
    load_param8(a.gamma, a.p_dtype, c, a.C - c, 1.f, gm[it]);
    load_param8(a.beta, a.p_dtype, c, a.C - c, 0.f, bt[it]);
  }
  const float inv = 1.f / (float)a.C;
  const long long P = (long long)((a.C + 127) / 128) * 128, Q = (long long)((a.C + 511) / 512) * 4;
  // every thread of a workgroup makes the same number of rounds (there are barriers inside where LPR > 64)
  for (long long r0 = (long long)blockIdx.x * RPW; r0 < a.R; r0 += (long long)gridDim.x * RPW) {
    const long long row = r0 + sub;
    const bool in = row < a.R;
    float v[NIT][8];
    float s = 0.f;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int c = (l + LPR * it) * 8;
      load8((const T *)a.x + (in ? row * a.ldx + c : 0), in ? a.C - c : 0, v[it]);
      s += ((v[it][0] + v[it][1]) + (v[it][2] + v[it][3])) + ((v[it][4] + v[it][5]) + (v[it][6] + v[it][7]));
    }
    const float mean = ln_row_sum<LPR>(s, red) * inv;
    float q = 0.f;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int n = a.C - (l + LPR * it) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = v[it][j] - mean;
        v[it][j] = d;
        q += j < n ? d * d : 0.f;
      }
    }
    const float rstd = 1.f / sqrtf(ln_row_sum<LPR>(q, red) * inv + a.eps);
    if (a.mean && in && l == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int c = (l + LPR * it) * 8, n = in ? a.C - c : 0;
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = j < n ? v[it][j] * rstd * gm[it][j] + bt[it][j] : 0.f;
      if (a.y && n > 0) store8((T *)a.y + row * a.C + c, n, y);
      if constexpr (FMT >= 0) {
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, mag(y[j]));
        const int byte = scale_byte<FMT>(max16(m));
        const float f = inv_scale(byte);
        if (in && c < P) {
          const u32x2 w = {pack4<FMT>(y[0] * f, y[1] * f, y[2] * f, y[3] * f), pack4<FMT>(y[4] * f, y[5] * f, y[6] * f, y[7] * f)};
          *(u32x2 *)(a.data + row * P + c) = w;
        }
        // 16 lanes share a block: the first of them writes its byte (127 behind the last block: those blocks are zeros)
        if (in && (l & 15) == 0 && (c >> 7) < Q) a.scale[row * Q + (c >> 7)] = (uint8_t)byte;
        if (LPR == 16 && in && l > 0 && l < 4) a.scale[row * Q + l] = 127;      // (one block: the lanes of the other three are not here)
      }
    }
  }
}

template <typename T, int LPR, int NIT>
__global__ __launch_bounds__(ln_threads(LPR)) void ln_rows_bwd_kernel(LnRowsArgs a) {
  constexpr int TH = ln_threads(LPR), RPW = TH / LPR;
  __shared__ float red[16];
  const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  float gm[NIT][8], dg[NIT][8], db[NIT][8];
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    const int c = (l + LPR * it) * 8;
    load_param8(a.gamma, a.p_dtype, c, a.C - c, 1.f, gm[it]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dg[it][j] = db[it][j] = 0.f;
  }
  const float inv = 1.f / (float)a.C;
  for (long long r0 = (long long)blockIdx.x * RPW; r0 < a.R; r0 += (long long)gridDim.x * RPW) {
    const long long row = r0 + sub;
    const bool in = row < a.R;
    const float mean = in ? a.mean[row] : 0.f, rstd = in ? a.rstd[row] : 0.f;
    float t[NIT][8], h[NIT][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int c = (l + LPR * it) * 8, n = in ? a.C - c : 0;
      load8((const T *)a.x + (in ? row * a.ldx + c : 0), n, h[it]);
      load8((const T *)a.g + (in ? row * a.C + c : 0), n, t[it]);
    }
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int n = in ? a.C - (l + LPR * it) * 8 : 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[it][j] = j < n ? (h[it][j] - mean) * rstd : 0.f;
        dg[it][j] += t[it][j] * h[it][j];
        db[it][j] += t[it][j];
        t[it][j] *= gm[it][j];
        s1 += t[it][j];
        s2 += t[it][j] * h[it][j];
      }
    }
    if (a.dx) {
      const float m1 = ln_row_sum<LPR>(s1, red) * inv, m2 = ln_row_sum<LPR>(s2, red) * inv;
#pragma unroll
      for (int it = 0; it < NIT; ++it) {
        const int c = (l + LPR * it) * 8, n = in ? a.C - c : 0;
        float d[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = rstd * (t[it][j] - m1 - h[it][j] * m2);
        if (n > 0) store8((T *)a.dx + row * a.C + c, n, d);
      }
    }
  }
  if (!a.part) return;
  // the workgroup's sums: one row of the partial buffer; lanes of different rows (LPR < threads) meet in LDS, a chunk at a time
  float *out = a.part + (long long)blockIdx.x * 2 * a.C;
  if constexpr (RPW == 1) {
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int c = (l + LPR * it) * 8;
      if (a.C - c > 0) { store8(out + c, a.C - c, dg[it]); store8(out + a.C + c, a.C - c, db[it]); }
    }
  } else {
    __shared__ float meet[RPW][LPR * 8 + 8];
#pragma unroll
    for (int it = 0; it < NIT; ++it)
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) meet[sub][l * 8 + j] = which ? db[it][j] : dg[it][j];
        __syncthreads();
        for (int e = threadIdx.x; e < LPR * 8; e += TH) {
          const int c = LPR * it * 8 + e;
          float s = 0.f;
#pragma unroll
          for (int k = 0; k < RPW; ++k) s += meet[k][e];
          if (c < a.C) out[which * a.C + c] = s;
        }
      }
  }
}

// dgamma[c] = sum_b part[b][0][c], dbeta[c] = sum_b part[b][1][c]: 8 columns x 32 slices of b per workgroup, a fixed order
__global__ __launch_bounds__(256) void ln_rows_join_kernel(const float *part, int nparts, int C, void *dgamma, void *dbeta, int p_dtype) {
  __shared__ float red[32][9];
  const int ci = threadIdx.x & 7, slice = threadIdx.x >> 3, e = blockIdx.x * 8 + ci;           // over 2 C
  float s = 0.f;
  if (e < 2 * C) {
#pragma unroll 8
    for (int b = slice; b < nparts; b += 32) s += part[(long long)b * 2 * C + e];
  }
  red[slice][ci] = s;
  __syncthreads();
  if (slice == 0 && e < 2 * C) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) s += red[k][ci];
    store_param(e < C ? dgamma : dbeta, p_dtype, e < C ? e : e - C, s);
  }
}

}  // namespace rows
}  // namespace snipper
