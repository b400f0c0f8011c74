// layernorm_rows.cuh -- layer norm of rows of any width up to 16 384, forward and backward (gfx950).
//
//   y = h gamma + beta,  h = (x - mean) rstd,  rstd = 1 / sqrt(var + eps)                     (statistics of a row, in float32)
//   dx = rstd (t - mean(t) - h mean(t h)),  t = g gamma;      dgamma = sum_rows g h,  dbeta = sum_rows g
//
// csrc/ln_fused.cuh has the residual + dropout form for widths that are multiples of 4 up to 1024, in float32 and bfloat16; this one
// takes any width, stride and alignment, float16 too, and can write its result as 8-bit blocks (format: include/snipper_fp8.h).
// Bound by HBM: 79 000 x 384 float32 forward 44 us (5.6 TB/s), backward 56 + 4 us (6.5 TB/s); 16 384 x 8192 bf16 104 and 152 + 7 us (5.2 and
// 5.3 TB/s).  What is written once and what the backward pass reads for the last time goes past the caches (non-temporal: the first
// pair of those 136 -> 105 us); x of the forward pass does not, the backward pass reads it again.  A row stays in the registers of LPR
// lanes, 16 bytes per lane and piece, from its one load to its store: the mean first, then the sum of squared deviations from it, so
// nothing cancels; the next row's loads run meanwhile (not two rows ahead: 75 -> 102 us backward at 79 000 x 384).  Workgroups walk over
// rows, so gamma, beta and the column sums of the backward pass live in registers too; the sums meet in LDS, then in one row of a
// partial buffer per workgroup, which a second kernel adds in a fixed order.
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

// Sums over the LPR lanes that share a row (LPR = 16: a quarter of a wave; 64: a wave; more: the whole workgroup, through LDS).  Calls
// in turn use `red` with turn 0, 1, 0, ...: what the last call but one left there has been read by everybody, so one barrier does.
template <int LPR, int K>
__device__ __forceinline__ void ln_row_sums(float (&v)[K], float (*red)[K][16], int turn) {
#pragma unroll
  for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], o, 64);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) red[turn][k][threadIdx.x >> 6] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) v[k] += red[turn][k][w];
    }
  }
}

constexpr int ln_threads(int lpr) { return lpr > 256 ? lpr : 256; }

// A lane's elements of a row: 8 NIT of them, in pieces of W neighbours that make 16 bytes (float32: 4, so that a wave's load is one run
// of 1 KB; 16 lanes a row: 8 always, so that they share one block of 128).  Piece p begins at column (p LPR + lane) W.
template <typename T, int LPR, int NIT>
struct LnShape {
  static constexpr int W = sizeof(T) == 4 && LPR > 16 ? 4 : 8, PIECES = 8 * NIT / W;
  static constexpr int RPW = ln_threads(LPR) / LPR;    // rows of a workgroup at a time
};

// FMT < 0: no blocks
template <typename T, int LPR, int NIT, int FMT>
__global__ __launch_bounds__(ln_threads(LPR)) void ln_rows_fwd_kernel(LnRowsArgs a) {
  using S = LnShape<T, LPR, NIT>;
  constexpr int W = S::W, NP = S::PIECES, RPW = S::RPW;
  __shared__ float red[2][1][16];
  const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  float gm[NP][W], bt[NP][W];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int c = (p * LPR + l) * W;
    load_param_w<W>(a.gamma, a.p_dtype, c, a.C - c, 1.f, gm[p]);
    load_param_w<W>(a.beta, a.p_dtype, c, a.C - c, 0.f, bt[p]);
  }
  const float inv = 1.f / (float)a.C;
  const long long P = (long long)((a.C + 127) / 128) * 128, Q = (long long)((a.C + 511) / 512) * 4;
  Raw<T, W> raw[NP];
  auto fetch = [&](long long row) {
    const bool in = row < a.R;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int c = (p * LPR + l) * W;
      raw[p].load((const T *)a.x + (in ? row * a.ldx + c : 0), in ? a.C - c : 0);
    }
  };
  constexpr bool AHEAD = NIT == 1;                      // (with more the registers cost more waves than the early loads gain)
  if (AHEAD) fetch((long long)blockIdx.x * RPW + sub);
  // every thread of a workgroup makes the same number of rounds (there are barriers inside where LPR > 64)
  for (long long r0 = (long long)blockIdx.x * RPW; r0 < a.R; r0 += (long long)gridDim.x * RPW) {
    const long long row = r0 + sub;
    const bool in = row < a.R;
    if (!AHEAD) fetch(row);
    float v[NP][W];
    float s[1] = {0.f};
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      raw[p].get(v[p]);
#pragma unroll
      for (int j = 0; j < W; j += 4) s[0] += (v[p][j] + v[p][j + 1]) + (v[p][j + 2] + v[p][j + 3]);
    }
    if (AHEAD) fetch(row + (long long)gridDim.x * RPW); // the next row, while this one is worked on
    ln_row_sums<LPR, 1>(s, red, 0);
    const float mean = s[0] * inv;
    float q[1] = {0.f};
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int n = a.C - (p * LPR + l) * W;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float d = v[p][j] - mean;
        v[p][j] = d;
        q[0] += j < n ? d * d : 0.f;
      }
    }
    ln_row_sums<LPR, 1>(q, red, 1);
    const float rstd = 1.f / sqrtf(q[0] * inv + a.eps);
    if (a.mean && in && l == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int c = (p * LPR + l) * W, n = in ? a.C - c : 0;
      float y[W];
#pragma unroll
      for (int j = 0; j < W; ++j) y[j] = j < n ? v[p][j] * rstd * gm[p][j] + bt[p][j] : 0.f;
      if (a.y && n > 0) store_nt<W>((T *)a.y + row * a.C + c, n, y);
      if constexpr (FMT >= 0) {
        constexpr int LPB = 128 / W;                    // lanes that share a block
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < W; ++j) m = max(m, mag(y[j]));
        const int byte = scale_byte<FMT>(max_over<LPB>(m));
        const float f = inv_scale(byte);
        if (in && c < P) {
          unsigned w[W / 4];
#pragma unroll
          for (int j = 0; j < W; j += 4) w[j / 4] = pack4<FMT>(y[j] * f, y[j + 1] * f, y[j + 2] * f, y[j + 3] * f);
          __builtin_memcpy(a.data + row * P + c, w, W);
        }
        // the first of a block's lanes writes its byte (127 behind the last block: those blocks are zeros)
        if (in && l % LPB == 0 && (c >> 7) < Q) a.scale[row * Q + (c >> 7)] = (uint8_t)byte;
        if (LPR == 16 && p == 0 && in && l >= NIT && l < 4) a.scale[row * Q + l] = 127;      // (behind the last block: no lanes there)
      }
    }
  }
}

template <typename T, int LPR, int NIT>
__global__ __launch_bounds__(ln_threads(LPR)) void ln_rows_bwd_kernel(LnRowsArgs a) {
  using S = LnShape<T, LPR, NIT>;
  constexpr int W = S::W, NP = S::PIECES, RPW = S::RPW, TH = ln_threads(LPR);
  __shared__ float red[2][2][16];
  const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  float gm[NP][W], dg[NP][W], db[NP][W];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int c = (p * LPR + l) * W;
    load_param_w<W>(a.gamma, a.p_dtype, c, a.C - c, 1.f, gm[p]);
#pragma unroll
    for (int j = 0; j < W; ++j) dg[p][j] = db[p][j] = 0.f;
  }
  const float inv = 1.f / (float)a.C;
  Raw<T, W> rx[NP], rg[NP];
  float mean_next, rstd_next;
  auto fetch = [&](long long row) {
    const bool in = row < a.R;
    mean_next = in ? a.mean[row] : 0.f;
    rstd_next = in ? a.rstd[row] : 0.f;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int c = (p * LPR + l) * W, n = in ? a.C - c : 0;
      rx[p].template load<true>((const T *)a.x + (in ? row * a.ldx + c : 0), n);
      rg[p].template load<true>((const T *)a.g + (in ? row * a.C + c : 0), n);
    }
  };
  constexpr bool AHEAD = NIT == 1;
  if (AHEAD) fetch((long long)blockIdx.x * RPW + sub);
  int turn = 0;
  for (long long r0 = (long long)blockIdx.x * RPW; r0 < a.R; r0 += (long long)gridDim.x * RPW, turn ^= 1) {
    const long long row = r0 + sub;
    const bool in = row < a.R;
    if (!AHEAD) fetch(row);
    const float mean = mean_next, rstd = rstd_next;
    float t[NP][W], h[NP][W];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      rx[p].get(h[p]);
      rg[p].get(t[p]);
    }
    if (AHEAD) fetch(row + (long long)gridDim.x * RPW); // the next row, while this one is worked on
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int n = in ? a.C - (p * LPR + l) * W : 0;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        h[p][j] = j < n ? (h[p][j] - mean) * rstd : 0.f;
        dg[p][j] += t[p][j] * h[p][j];
        db[p][j] += t[p][j];
        t[p][j] *= gm[p][j];
        s[0] += t[p][j];
        s[1] += t[p][j] * h[p][j];
      }
    }
    if (a.dx) {
      ln_row_sums<LPR, 2>(s, red, turn);
      const float m1 = s[0] * inv, m2 = s[1] * inv;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int c = (p * LPR + l) * W, n = in ? a.C - c : 0;
        float d[W];
#pragma unroll
        for (int j = 0; j < W; ++j) d[j] = rstd * (t[p][j] - m1 - h[p][j] * m2);
        if (n > 0) store_nt<W>((T *)a.dx + row * a.C + c, n, d);
      }
    }
  }
  if (!a.part) return;
  // the workgroup's sums: one row of the partial buffer; lanes of different rows (LPR < threads) meet in LDS, a piece at a time
  float *out = a.part + (long long)blockIdx.x * 2 * a.C;
  if constexpr (RPW == 1) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int c = (p * LPR + l) * W;
      if (a.C - c > 0) { store_w<W>(out + c, a.C - c, dg[p]); store_w<W>(out + a.C + c, a.C - c, db[p]); }
    }
  } else {
    __shared__ float meet[RPW][LPR * W + 8];
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < W; ++j) meet[sub][l * W + j] = which ? db[p][j] : dg[p][j];
        __syncthreads();
        for (int e = threadIdx.x; e < LPR * W; e += TH) {
          const int c = LPR * W * p + e;
          float s = 0.f;
#pragma unroll
          for (int k = 0; k < RPW; ++k) s += meet[k][e];
          if (c < a.C) out[which * a.C + c] = s;
        }
      }
  }
}

// dgamma[c] = sum_b part[b][0][c], dbeta[c] = sum_b part[b][1][c]
__global__ __launch_bounds__(1024) void ln_rows_join_kernel(const float *part, int nparts, int C, void *dgamma, void *dbeta, int p_dtype) {
  const int e = blockIdx.x * 32 + (threadIdx.x & 31);          // over 2 C
  const float s = sum_parts(part, nparts, 2 * C, e);
  if (threadIdx.x < 32 && e < 2 * C) store_param(e < C ? dgamma : dbeta, p_dtype, e < C ? e : e - C, s);
}

}  // namespace rows
}  // namespace snipper
