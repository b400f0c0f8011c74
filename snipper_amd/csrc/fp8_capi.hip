// fp8_capi.hip -- extern "C" entry points of include/snipper_fp8.h: 8-bit block quantizers, the product of two such matrices, layer
// norm of rows of any width.  As in msda_capi.hip: validate, pick a kernel, launch on the caller's stream, report errors; no
// allocation, no synchronisation, no state.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/snipper_fp8.h"
#include "gemm_fp8.cuh"
#include "layernorm_rows.cuh"
#include "quant_fp8.cuh"

using namespace snipper::rows;

namespace {

constexpr int kMaxDim = 1 << 23;
constexpr int kCUs = 256;
constexpr int kLnMaxCols = 16384;

int launch_status() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SNIPPER_OK : (int)e;
}
bool type_ok(int t) { return t == kF32 || t == kBF16 || t == kF16; }
bool fmt_ok(int f) { return f == 0 || f == 1; }
bool dim_ok(int n) { return n > 0 && n <= kMaxDim; }
bool full_sums(int out_dtype) { return out_dtype == kF32 || (out_dtype & SNIPPER_FP8_FULL_SUMS); }
int element_type(int out_dtype) { return out_dtype & ~SNIPPER_FP8_FULL_SUMS; }
bool result_ok(int M, int N) { return (long long)M * N < (1ll << 40); }       // (tiles are counted in 32 bits)
int ceil_div(int a, int b) { return a / b + (a % b != 0); }

// f(T{}) for the element type of a code
template <typename F>
void with_type(int t, F &&f) {
  if (t == kF32) f(float{});
  else if (t == kBF16) f(bf16_t{});
  else f(f16_t{});
}
template <typename F>
void with_fmt(int fmt, F &&f) {
  if (fmt == 0) f(std::integral_constant<int, 0>{});
  else f(std::integral_constant<int, 1>{});
}

// ---- layer norm: lanes of a row and how often eight elements of a lane.  Times in us, forward / backward, of 2^27 bytes (cols x type):
// 16 lanes share a block of 128 and four rows a wave, one wave a row needs no barrier, four waves a row only one number from each.
//   256 x 16 bits: 16 lanes 82 / 135, a wave 141 / 231; 384 x 16 bits: 83 / 137 against 104 / 205; but 384 x float32, whose pieces of 16
//   bytes fill a wave, 89 / 158 against 80 / 133, and 512 x 16 bits 84 / 133 against 86 / 137
//   2048: four waves 79 / 135 (float32), 83 / 141 (16 bits), a wave 78 / 138, 82 / 137; 4096: four waves 79 / 132, 79 / 140, eight 80 / 131,
//   86 / 150; 8192: four 79 / 141, 79 / 139, eight 79 / 149, 80 / 173, sixteen 79 / 147, 116 / 171; 16 384: sixteen 84 / 155, 91 / 150,
//   eight (with all their registers) 91 / 158, 87 / 162
template <typename T, typename F>
void with_ln_shape(int cols, F &&f) {
  using std::integral_constant;
  if (cols <= 128) return f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  if constexpr (sizeof(T) == 2) {
    if (cols <= 256) return f(integral_constant<int, 16>{}, integral_constant<int, 2>{});
    if (cols <= 384) return f(integral_constant<int, 16>{}, integral_constant<int, 3>{});
  }
  if (cols <= 512) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (cols <= 1024) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (cols <= 2048) f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (cols <= 4096) f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (cols <= 8192) f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
}
// Forward: short runs of rows (more workgroups than are resident even out the card's ends: 8 of four waves per CU 84 .. 93, 32 77 .. 83),
// except that with sixteen waves a row the parameters' loads weigh (2 per CU 91, 8 98).  Backward: every workgroup leaves a row of sums
// behind, so no more than are resident; fewer for the widest (8192: 4 per CU 147 / 150, 2 141 / 139; 16 384: 2 158, 1 152).
int ln_fwd_blocks(int rows, int rows_per_wg, int cols) { return std::min(ceil_div(rows, rows_per_wg), (cols <= 8192 ? 32 : 2) * kCUs); }
int ln_bwd_most(int cols) { return (cols <= 2048 ? 4 : cols <= 8192 ? 2 : 1) * kCUs; }
int ln_bwd_blocks(int rows, int rows_per_wg, int cols) { return std::min(ceil_div(rows, rows_per_wg), ln_bwd_most(cols)); }

// ---- product: which kernel, and how many pieces the K axis is cut into (times in us of bfloat16 results, M x N x K, 256 CUs)
struct MmPlan {
  int kind;                  // 0 few rows, 1 tiles of 128 x 128, 2 tiles of 256 x 256, 3 B in registers, 4 tiles of 64 x 64
  int tiles, splits, per_split, waves;
};
MmPlan mm_plan(int M, int N, int K, bool exact) {
  MmPlan p{};
  const int steps = ceil_div(K, 128);
  p.splits = 1;
  p.per_split = steps;
  // one operand of rows: 16 x 4096 x 4096 7.8 against 8.3 in tiles; 33 rows 12.1 (a second and third pass over A's operands) against 9.4
  if (M <= 16) {
    p.waves = std::max(1, std::min(8, ceil_div(steps, 4)));
    return p;
  }
  // K <= 1024: loads and stores bound such products, and the kernel with B in registers overlaps them.  Whole 16-byte pieces of rows
  // only (N = 1001 goes to tiles: 79 000 x 1001 x 384 94, N = 1000 46), at least as many chunks of 64 rows as there are CUs, and no more
  // than 32 column blocks of 256: chunk lists come in multiples of 8 (one an XCD), and with 33 blocks 8 workgroups are left for a second
  // round.  Here against the better tile: 79 000 x 1024 x 384 45 / 85, 79 000 x 384 x 1024 44 / 54, 16 384 x 1024 x 1024 24 / 27, 4096 x 4096 x 512
  // 15 / 21; wide N at K = 1024, 8192 rows: N = 1024 17.7 / 16.9, 2048 24 / 27, 2816 (176 workgroups) 35 / 40, 4096 37 / 50, 4104 (136) 61 / 59, at
  // K = 384 34 / 40; 8200: 123 / 118 (K = 384: 106 / 86); with fewer chunks 1024^3 13 / 6
  if (!exact && steps <= 8 && N % 8 == 0 && ceil_div(N, 256) <= kCUs / 8 && (long long)ceil_div(M, 64) * ceil_div(N, 256) >= kCUs) {
    p.kind = 3;
    p.tiles = kCUs / (8 * ceil_div(N, 256)) * 8;     // chunk lists: at most one workgroup per CU
    return p;
  }
  // The largest tile that still gives every CU one: 4096^3 66 (256) against 71 (128); 8192 x 1024 x 4096 38 (128) against 57 (256), 55
  // (64); 1024^3 6 (64) against 10 (128).  Few tiles and a long K axis: larger tiles, which load less, and more pieces
  // (256 x 128 or 128 x 256 never won: 4096 x 1024 x 8192 61 against 48 of 128 x 128, 8192^3 513 .. 544 against 457 of 256 x 256)
  const long long t128 = (long long)ceil_div(M, 128) * ceil_div(N, 128);
  if (!exact && M >= 256 && N >= 256 && (long long)ceil_div(M, 256) * ceil_div(N, 256) >= kCUs) p.kind = 2;
  else p.kind = t128 >= kCUs || steps >= 64 ? 1 : 4;
  const int edge = p.kind == 2 ? 256 : p.kind == 1 ? 128 : 64;
  p.tiles = ceil_div(M, edge) * ceil_div(N, edge);
  // pieces of at least 8 steps, up to one workgroup of 64 x 64 or two of 128 x 128 per CU: 33 x 4096 x 4096 11 -> 9.4, 100 x 4096 x
  // 4096 11.5 -> 10.7; 256 x 4096 x 4096, a tile per CU, 12.2 -> 15.8, and cut at 128 x 128 8192 x 1024 x 4096 38 -> 61
  const int want = std::min((p.kind == 1 && t128 < kCUs ? 2 : 1) * kCUs / p.tiles, steps / 8);
  if (p.kind != 2 && want > 1) {
    p.per_split = ceil_div(ceil_div(steps, want), 4) * 4;
    p.splits = ceil_div(steps, p.per_split);
  }
  return p;
}

template <int FA, int FB, int KS = 1>
void launch_stationary(const MmArgs &a, int n_series, hipStream_t st) {
  if constexpr (KS < 8) {
    if (a.steps > KS) return launch_stationary<FA, FB, KS + 1>(a, n_series, st);
  }
  const dim3 grid(n_series * ceil_div(a.N, 256));
  if (a.N % 32 == 0) hipLaunchKernelGGL((mm_stationary_kernel<FA, FB, KS, true>), grid, dim3(512), 0, st, a, n_series);
  else hipLaunchKernelGGL((mm_stationary_kernel<FA, FB, KS, false>), grid, dim3(512), 0, st, a, n_series);
}

}  // namespace

extern "C" {

size_t snipper_fp8_quantize_workspace_bytes(int rows, int cols, int with_colsum) {
  if (!dim_ok(rows) || !dim_ok(cols) || !with_colsum) return 0;
  return (size_t)ceil_div(rows, 128) * cols * sizeof(float);
}

int snipper_fp8_quantize(void *stream, const void *x, int x_dtype, long long ldx, int rows, int cols, int tile_rows, int fmt,
                         const float *mean, const float *rstd, const void *gamma, const void *beta, int p_dtype, uint8_t *data,
                         uint8_t *scale, uint8_t *data_t, uint8_t *scale_t, void *colsum, int colsum_dtype, void *workspace,
                         size_t workspace_bytes) {
  if (!x || (!data && !data_t) || (data && !scale) || (data_t && !scale_t) || ((mean == nullptr) != (rstd == nullptr))) return SNIPPER_E_NULL;
  if (!dim_ok(rows) || !dim_ok(cols) || ldx < cols || !type_ok(x_dtype) || !type_ok(p_dtype) || !type_ok(colsum_dtype) || !fmt_ok(fmt))
    return SNIPPER_E_SHAPE;
  if (tile_rows != 1 && (tile_rows != 128 || mean)) return SNIPPER_E_SHAPE;
  if (!mean && (gamma || beta)) return SNIPPER_E_SHAPE;
  if (((uintptr_t)data | (uintptr_t)data_t) & 15 || ((uintptr_t)scale | (uintptr_t)scale_t) & 3) return SNIPPER_E_SHAPE;
  if (colsum && (!workspace || workspace_bytes < snipper_fp8_quantize_workspace_bytes(rows, cols, 1))) return SNIPPER_E_SHAPE;
  const QuantArgs a{x, ldx, rows, cols, mean, rstd, gamma, beta, p_dtype, data, scale, data_t, scale_t, colsum ? (float *)workspace : nullptr};
  hipStream_t st = (hipStream_t)stream;
  if (tile_rows == 1 && !data_t && !mean && !colsum) {
    const long long wgs = ((long long)rows * ceil_div(cols, 512) + 3) / 4;
    const dim3 grid((unsigned)std::min<long long>(wgs, 16 * kCUs));
    with_type(x_dtype, [&](auto t) {
      with_fmt(fmt, [&](auto f) { hipLaunchKernelGGL((quant_rows_kernel<decltype(t), decltype(f)::value>), grid, dim3(256), 0, st, a); });
    });
    return launch_status();
  }
  const int rb = ceil_div(rows, 128);
  const dim3 grid(ceil_div(cols, 128), std::min(rb, 32768), ceil_div(rb, 32768));
  with_type(x_dtype, [&](auto t) {
    with_fmt(fmt, [&](auto f) {
      using T = decltype(t);
      constexpr int F = decltype(f)::value;
      if (tile_rows == 128) hipLaunchKernelGGL((quant_tile_kernel<T, F, true, false>), grid, dim3(512), 0, st, a);
      else if (mean) hipLaunchKernelGGL((quant_tile_kernel<T, F, false, true>), grid, dim3(512), 0, st, a);
      else hipLaunchKernelGGL((quant_tile_kernel<T, F, false, false>), grid, dim3(512), 0, st, a);
    });
  });
  if (colsum) hipLaunchKernelGGL(colsum_parts_kernel, dim3(ceil_div(cols, 32)), dim3(1024), 0, st, (const float *)workspace, rb, cols, colsum, colsum_dtype);
  return launch_status();
}

size_t snipper_fp8_matmul_workspace_bytes(int M, int N, int K, int out_dtype) {
  if (!dim_ok(M) || !dim_ok(N) || !dim_ok(K) || !result_ok(M, N) || !type_ok(element_type(out_dtype))) return 0;
  const MmPlan p = mm_plan(M, N, K, full_sums(out_dtype));
  return p.splits > 1 ? (size_t)p.splits * M * N * sizeof(float) : 0;
}

int snipper_fp8_matmul(void *stream, const uint8_t *A, const uint8_t *a_scale, int a_fmt, const uint8_t *B, const uint8_t *b_scale,
                       int b_fmt, int M, int N, int K, const void *bias, int bias_dtype, int relu, void *out, int out_dtype,
                       void *workspace, size_t workspace_bytes) {
  if (!A || !a_scale || !B || !b_scale || !out) return SNIPPER_E_NULL;
  if (!dim_ok(M) || !dim_ok(N) || !dim_ok(K) || !result_ok(M, N) || !fmt_ok(a_fmt) || !fmt_ok(b_fmt) || !type_ok(element_type(out_dtype)) || !type_ok(bias_dtype))
    return SNIPPER_E_SHAPE;
  if (((uintptr_t)A | (uintptr_t)B | (uintptr_t)out) & 15 || ((uintptr_t)a_scale | (uintptr_t)b_scale) & 3) return SNIPPER_E_SHAPE;
  const bool exact = full_sums(out_dtype);
  const MmPlan p = mm_plan(M, N, K, exact);
  const size_t need = snipper_fp8_matmul_workspace_bytes(M, N, K, out_dtype);
  if (need && (!workspace || workspace_bytes < need)) return SNIPPER_E_SHAPE;
  const MmArgs a{A, a_scale, B, b_scale, M, N, ceil_div(K, 128), bias, bias_dtype, relu, out, element_type(out_dtype),
                 p.splits > 1 ? (float *)workspace : nullptr, p.splits, p.per_split};
  hipStream_t st = (hipStream_t)stream;
  with_fmt(a_fmt, [&](auto fa) {
    with_fmt(b_fmt, [&](auto fb) {
      constexpr int FA = decltype(fa)::value, FB = decltype(fb)::value;
      auto go = [&](auto ex) {
        constexpr bool E = decltype(ex)::value;
        if (p.kind == 0) {
          hipLaunchKernelGGL((mm_rows_kernel<FA, FB>), dim3(ceil_div(N, 16)), dim3(64 * p.waves), 0, st, a);
        } else if (p.kind == 4) {
          hipLaunchKernelGGL((mm_tile_kernel<FA, FB, E, 2, 2, 2, 2, false>), dim3(p.tiles * p.splits), dim3(256), 0, st, a);
        } else if (p.kind == 1) {
          hipLaunchKernelGGL((mm_tile_kernel<FA, FB, E, 2, 2, 4, 4, false>), dim3(p.tiles * p.splits), dim3(256), 0, st, a);
        } else if constexpr (E) {
        } else if (p.kind == 3) {
          launch_stationary<FA, FB>(a, p.tiles, st);
        } else {
          hipLaunchKernelGGL((mm_tile_kernel<FA, FB, false, 2, 4, 8, 4, true>), dim3(p.tiles * p.splits), dim3(512), 0, st, a);
        }
      };
      if (exact) go(std::true_type{});
      else go(std::false_type{});
    });
  });
  if (p.splits > 1) {
    const long long units = (long long)M * ((N + 3) / 4);
    hipLaunchKernelGGL(mm_join_kernel, dim3((unsigned)std::min<long long>((units + 255) / 256, 16 * kCUs)), dim3(256), 0, st, a);
  }
  return launch_status();
}

int snipper_layernorm_forward(void *stream, const void *x, int x_dtype, long long ldx, const void *gamma, const void *beta, int p_dtype,
                              int rows, int cols, float eps, void *y, float *mean, float *rstd, uint8_t *data, uint8_t *scale, int fmt) {
  if (!x || (!y && !mean && !data) || ((mean == nullptr) != (rstd == nullptr)) || ((data == nullptr) != (scale == nullptr))) return SNIPPER_E_NULL;
  if (rows <= 0 || cols <= 0 || cols > kLnMaxCols || ldx < cols || !type_ok(x_dtype) || !type_ok(p_dtype) || !fmt_ok(fmt) || !(eps >= 0.f))
    return SNIPPER_E_SHAPE;
  if ((uintptr_t)data & 15 || (uintptr_t)scale & 3) return SNIPPER_E_SHAPE;
  LnRowsArgs a{};
  a.x = x; a.ldx = ldx; a.gamma = gamma; a.beta = beta; a.p_dtype = p_dtype; a.R = rows; a.C = cols; a.eps = eps;
  a.y = y; a.mean = mean; a.rstd = rstd; a.data = data; a.scale = scale;
  hipStream_t st = (hipStream_t)stream;
  with_type(x_dtype, [&](auto t) {
    using T = decltype(t);
    with_ln_shape<T>(cols, [&](auto lpr, auto nit) {
      constexpr int L = decltype(lpr)::value, I = decltype(nit)::value;
      const dim3 grid(ln_fwd_blocks(rows, LnShape<T, L, I>::RPW, cols));
      if (!data) hipLaunchKernelGGL((ln_rows_fwd_kernel<T, L, I, -1>), grid, dim3(ln_threads(L)), 0, st, a);
      else if (fmt == 0) hipLaunchKernelGGL((ln_rows_fwd_kernel<T, L, I, 0>), grid, dim3(ln_threads(L)), 0, st, a);
      else hipLaunchKernelGGL((ln_rows_fwd_kernel<T, L, I, 1>), grid, dim3(ln_threads(L)), 0, st, a);
    });
  });
  return launch_status();
}

size_t snipper_layernorm_backward_workspace_bytes(int rows, int cols) {
  if (rows <= 0 || cols <= 0 || cols > kLnMaxCols) return 0;
  return (size_t)ln_bwd_blocks(rows, cols <= 1024 ? 4 : 1, cols) * 2 * cols * sizeof(float);        // (4: the fewest rows of a workgroup there)
}

int snipper_layernorm_backward(void *stream, const void *g, const void *x, int x_dtype, long long ldx, const float *mean, const float *rstd,
                               const void *gamma, int p_dtype, int rows, int cols, void *dx, void *dgamma, void *dbeta, void *workspace,
                               size_t workspace_bytes) {
  if (((dgamma == nullptr) != (dbeta == nullptr)) || (!dx && !dgamma)) return SNIPPER_E_NULL;
  if (rows < 0 || cols <= 0 || cols > kLnMaxCols || ldx < cols || !type_ok(x_dtype) || !type_ok(p_dtype)) return SNIPPER_E_SHAPE;
  if (rows > 0 && (!g || !x || !mean || !rstd)) return SNIPPER_E_NULL;
  if (rows > 0 && dgamma && (!workspace || workspace_bytes < snipper_layernorm_backward_workspace_bytes(rows, cols))) return SNIPPER_E_SHAPE;
  int blocks = 0;
  LnRowsArgs a{};
  a.x = x; a.ldx = ldx; a.gamma = gamma; a.p_dtype = p_dtype; a.R = rows; a.C = cols;
  a.mean = const_cast<float *>(mean); a.rstd = const_cast<float *>(rstd);
  a.g = g; a.dx = dx; a.part = dgamma ? (float *)workspace : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (rows > 0)
    with_type(x_dtype, [&](auto t) {
      using T = decltype(t);
      with_ln_shape<T>(cols, [&](auto lpr, auto nit) {
        constexpr int L = decltype(lpr)::value, I = decltype(nit)::value;
        blocks = ln_bwd_blocks(rows, LnShape<T, L, I>::RPW, cols);
        hipLaunchKernelGGL((ln_rows_bwd_kernel<T, L, I>), dim3(blocks), dim3(ln_threads(L)), 0, st, a);
      });
    });
  if (dgamma)
    hipLaunchKernelGGL(ln_rows_join_kernel, dim3(ceil_div(2 * cols, 32)), dim3(1024), 0, st, (const float *)workspace, blocks, cols, dgamma, dbeta, p_dtype);
  return launch_status();
}

}  // extern "C"
