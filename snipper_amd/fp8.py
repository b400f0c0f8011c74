"""8-bit products with a power-of-two scale for each 128 elements (include/snipper_fp8.h, csrc/gemm_fp8.cuh, quant_fp8.cuh).

What the bf16 products of ``dense.py`` are for Linears in 16 bits, these are in 8:

    quantize_rows / quantize_both / quantize_tiles   a matrix into blocks (``Fp8Blocks``)
    matmul_fp8(a, b, bias)                           a @ b.T + bias of two matrices in blocks
    linear_fp8(x, lin)                               ``lin(x)``, differentiable: all three products of a training step in 8 bits
    layer_norm_fp8(x, norm)                          ``norm(x)`` straight into blocks, for inference
    layer_norm_linear_fp8(x, norm, lin)              ``lin(norm(x))``, differentiable, the norm's result held in 8 bits only

At inference a weight is laid out once, ``w8, _ = quantize_tiles(lin.weight)``, and used as
``matmul_fp8(quantize_rows(x), w8, lin.bias)`` or ``matmul_fp8(layer_norm_fp8(x, norm), w8, lin.bias)``.

Blocks run along the axis that a product sums over.  The training step therefore rounds x and the gradient twice, along their rows
(y = x W^T, dx = g W) and along their columns (dW = g^T x), both from one read; a weight has one scale for each 128 x 128 tile, so its
transpose holds the same values.  Scales are powers of two that keep the largest element of a block in range: nothing saturates, and
an element is its input rounded once.  CUDA tensors only, as everywhere in this package.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._autograd import Function
from .fused import _ROW_DT, _layer_norm_backward, _layer_norm_forward, _norm_rows, _opt

_FMT = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}
_MAX_DIM = 1 << 23


class Fp8Blocks:
    """A matrix [rows, cols] in 8-bit blocks: ``data`` [rows, 128 ceil(cols / 128)] float8_e4m3fn / float8_e5m2, zeros behind the last
    column, ``scale`` [rows, 4 ceil(cols / 512)] float8_e8m0fnu, one for each 128 elements of a row, 1 behind the last block; both
    contiguous.  The quantizers make them; a program that keeps a weight in a file stores the two tensors and ``cols``."""

    __slots__ = ("data", "scale", "cols")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, cols: int):
        if data.dtype not in _FMT or scale.dtype is not torch.float8_e8m0fnu:
            raise TypeError(f"Fp8Blocks: data in float8_e4m3fn or float8_e5m2 and scale in float8_e8m0fnu, got {data.dtype} and {scale.dtype}")
        if (cols < 1 or data.dim() != 2 or data.shape[1] != -(-cols // 128) * 128 or
                scale.shape != (data.shape[0], -(-cols // 512) * 4)):
            raise ValueError(f"Fp8Blocks: data {tuple(data.shape)} and scale {tuple(scale.shape)} are not those of {cols} columns")
        if not data.is_contiguous() or not scale.is_contiguous() or data.device != scale.device:
            raise ValueError("Fp8Blocks: data and scale are contiguous and on one device")
        self.data, self.scale, self.cols = data, scale, cols

    @property
    def shape(self) -> Tuple[int, int]:
        return self.data.shape[0], self.cols

    def dequantize(self) -> torch.Tensor:
        """The matrix that the blocks stand for, float32 (elementary torch operations: for checks and exports)."""
        R, P = self.data.shape
        s = self.scale.float()[:, :P // 128]
        return (self.data.float().view(R, P // 128, 128) * s[:, :, None]).view(R, P)[:, :self.cols]


def _empty_blocks(rows: int, cols: int, dtype, device):
    return (torch.empty((rows, -(-cols // 128) * 128), dtype=dtype, device=device),
            torch.empty((rows, -(-cols // 512) * 4), dtype=torch.float8_e8m0fnu, device=device))


def _matrix(x: torch.Tensor, what: str):
    """x [..., cols] as a matrix with unit stride inside a row, and its row stride."""
    if not x.is_cuda:
        raise RuntimeError(f"{what}: Not implemented on the CPU")
    if x.dtype not in _ROW_DT:
        raise TypeError(f"{what}: float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() < 2:
        raise ValueError(f"{what}: a matrix or a batch of rows, got {tuple(x.shape)}")
    C = x.shape[-1]
    x2 = x if x.dim() == 2 else x.reshape(-1, C) if C else x
    if not 1 <= C <= _MAX_DIM or x2.shape[0] > _MAX_DIM:
        raise ValueError(f"{what}: up to 2^23 rows of 1 to 2^23 elements, got {tuple(x.shape)}")
    if x2.stride(1) != 1 or (x2.shape[0] > 1 and x2.stride(0) < C):
        x2 = x2.contiguous()
    return x2, (x2.stride(0) if x2.shape[0] > 1 else C)


def _format(dtype, what: str) -> int:
    if dtype not in _FMT:
        raise TypeError(f"{what}: float8_e4m3fn or float8_e5m2, got {dtype}")
    return _FMT[dtype]


def _no_graph(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} is not differentiable: use linear_fp8 / layer_norm_linear_fp8, or call it under torch.no_grad()")


def _quantize(x2, ld, dtype, rows=True, cols=False, tile=False, colsum=False, norm=None):
    """(blocks of x or None, blocks of x^T or None, column sums or None), as tensors.  ``norm``: (stats [2, R], gamma, beta, p_dtype)."""
    fmt = _FMT[dtype]
    R, C = x2.shape
    dev = x2.device
    a = _empty_blocks(R, C, dtype, dev) if rows else None
    b = _empty_blocks(C, R, dtype, dev) if cols else None
    s = torch.empty(C, dtype=torch.float32, device=dev) if colsum else None
    stats, gamma, beta, p_dtype = norm if norm is not None else (None, None, None, torch.float32)
    lib = _lib.load()
    nbytes = lib.snipper_fp8_quantize_workspace_bytes(R, C, 1) if colsum else 0
    ws = torch.empty(nbytes // 4, dtype=torch.float32, device=dev) if nbytes else None
    with _lib.device_guard(dev):
        rc = lib.snipper_fp8_quantize(
            _lib.raw_stream(dev), x2.data_ptr(), _ROW_DT[x2.dtype], ld, R, C, 128 if tile else 1, fmt,
            stats[0].data_ptr() if norm is not None else None, stats[1].data_ptr() if norm is not None else None, _opt(gamma), _opt(beta),
            _ROW_DT[p_dtype], a[0].data_ptr() if rows else None, a[1].data_ptr() if rows else None, b[0].data_ptr() if cols else None,
            b[1].data_ptr() if cols else None, _opt(s), _opt(ws), nbytes)
    _lib.check(rc, "snipper_fp8_quantize")
    return a, b, s


def quantize_rows(x: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn) -> Fp8Blocks:
    """x [..., cols] (float32 / bfloat16 / float16, leading axes as rows) into blocks of 128 elements of a row."""
    _format(dtype, "quantize_rows")
    _no_graph("quantize_rows", x)
    x2, ld = _matrix(x, "quantize_rows")
    if x2.shape[0] == 0:
        return Fp8Blocks(*_empty_blocks(0, x2.shape[1], dtype, x.device), x2.shape[1])
    return Fp8Blocks(*_quantize(x2, ld, dtype)[0], x2.shape[1])


def quantize_both(x: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn) -> Tuple[Fp8Blocks, Fp8Blocks]:
    """(blocks of x, blocks of x^T) from one read: the second has a scale for each 128 elements of a COLUMN of x."""
    _format(dtype, "quantize_both")
    _no_graph("quantize_both", x)
    x2, ld = _matrix(x, "quantize_both")
    if x2.shape[0] == 0:
        raise ValueError("quantize_both: a matrix without rows has no columns to cut into blocks")
    a, b, _ = _quantize(x2, ld, dtype, cols=True)
    return Fp8Blocks(*a, x2.shape[1]), Fp8Blocks(*b, x2.shape[0])


def quantize_tiles(w: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn) -> Tuple[Fp8Blocks, Fp8Blocks]:
    """(blocks of w, blocks of w^T) of a weight [out, in] with one scale for each 128 x 128 tile: the two hold the same values."""
    _format(dtype, "quantize_tiles")
    _no_graph("quantize_tiles", w)
    if w.dim() != 2 or w.shape[0] == 0:
        raise ValueError(f"quantize_tiles: a matrix with rows, got {tuple(w.shape)}")
    w2, ld = _matrix(w, "quantize_tiles")
    a, b, _ = _quantize(w2, ld, dtype, cols=True, tile=True)
    return Fp8Blocks(*a, w2.shape[1]), Fp8Blocks(*b, w2.shape[0])


def _matmul(a_data, a_scale, b_data, b_scale, K, bias, relu, out_dtype):
    M, N = a_data.shape[0], b_data.shape[0]
    dev = a_data.device
    out = torch.empty((M, N), dtype=out_dtype, device=dev)
    if M == 0 or N == 0:
        return out
    lib = _lib.load()
    od = _ROW_DT[out_dtype]
    nbytes = lib.snipper_fp8_matmul_workspace_bytes(M, N, K, od)
    ws = torch.empty(nbytes // 4, dtype=torch.float32, device=dev) if nbytes else None
    with _lib.device_guard(dev):
        rc = lib.snipper_fp8_matmul(
            _lib.raw_stream(dev), a_data.data_ptr(), a_scale.data_ptr(), _FMT[a_data.dtype], b_data.data_ptr(), b_scale.data_ptr(),
            _FMT[b_data.dtype], M, N, K, bias.data_ptr() if bias is not None else None, _ROW_DT[bias.dtype] if bias is not None else 0,
            relu, out.data_ptr(), od, ws.data_ptr() if nbytes else None, nbytes)
    _lib.check(rc, "snipper_fp8_matmul")
    return out


def _check_bias(bias, N, device, what):
    if bias.dtype not in _ROW_DT or bias.shape != (N,) or bias.device != device or (N > 1 and bias.stride(0) != 1):
        raise ValueError(f"{what}: bias [{N}] contiguous, of a floating type, on the operands' device")


def matmul_fp8(a: Fp8Blocks, b: Fp8Blocks, bias: Optional[torch.Tensor] = None, relu: bool = False,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """act(a @ b.T + bias): a [M, K], b [N, K] in blocks (either type each), bias [N] or None -> [M, N] of ``out_dtype``.

    A bfloat16 / float16 result comes from the 8-bit matrix instructions (relative error of their sums 1.5e-5, far inside the
    result's own rounding); a float32 result from the bfloat16 ones on exactly widened operands, at a quarter of the rate."""
    if a.cols != b.cols:
        raise ValueError(f"matmul_fp8: a {a.shape} and b {b.shape} have rows of different length")
    if not a.data.is_cuda:
        raise RuntimeError("matmul_fp8: Not implemented on the CPU")
    if a.data.device != b.data.device:
        raise ValueError("matmul_fp8: operands on one device")
    if out_dtype not in _ROW_DT:
        raise TypeError(f"matmul_fp8: out_dtype float32, bfloat16 or float16, got {out_dtype}")
    if max(a.shape[0], b.shape[0], a.cols) > _MAX_DIM:
        raise ValueError("matmul_fp8: sizes up to 2^23")
    if bias is not None:
        _no_graph("matmul_fp8", bias)
        _check_bias(bias, b.data.shape[0], a.data.device, "matmul_fp8")
    return _matmul(a.data, a.scale, b.data, b.scale, a.cols, bias, int(relu), out_dtype)


def _linear_params(x, weight, bias, what):
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] == 0:
        raise ValueError(f"{what}: x {tuple(x.shape)} and weight {tuple(weight.shape)}")
    if weight.device != x.device:
        raise ValueError(f"{what}: weight on x's device")
    if bias is not None:
        _check_bias(bias, weight.shape[0], x.device, what)


def _linear_backward(ctx, g2, xt, wt, K, x_dtype, want, grad_dtype):
    """(dx [M, K] or None, dW or None, db or None) from the gradient [M, N]; want = which."""
    wx, ww, wb = want
    gr, gt, db = _quantize(g2, g2.stride(0) if g2.shape[0] > 1 else g2.shape[1], grad_dtype, rows=wx, cols=ww or not wx, colsum=wb)
    dx = _matmul(*gr, *wt, g2.shape[1], None, 0, x_dtype) if wx else None
    dw = _matmul(*gt, *xt, g2.shape[0], None, 0, ctx.param_dtypes[0]) if ww else None
    return dx, dw, db.to(ctx.param_dtypes[1]) if wb else None


class LinearFp8(Function):
    """apply(x, weight, bias, grad_dtype): see ``linear_fp8``."""

    @staticmethod
    def forward(ctx, x, weight, bias, grad_dtype):
        x2, ld = _matrix(x, "linear_fp8")
        w2, ldw = _matrix(weight, "linear_fp8")
        M, K = x2.shape
        N = w2.shape[0]
        nx, nw, nb = ctx.needs_input_grad[:3]
        ctx.param_dtypes = (weight.dtype, bias.dtype if bias is not None else None)
        ctx.dims, ctx.grad_dtype, ctx.x_dtype = (M, N, K), grad_dtype, x.dtype
        if M == 0:
            ctx.save_for_backward()
            return x.new_empty((*x.shape[:-1], N))
        wr, wt, _ = _quantize(w2, ldw, torch.float8_e4m3fn, cols=nx, tile=True)
        xr, xt, _ = _quantize(x2, ld, torch.float8_e4m3fn, cols=nw)
        y = _matmul(*xr, *wr, K, bias, 0, x.dtype)
        ctx.save_for_backward(*(xt if nw else (None, None)), *(wt if nx else (None, None)))
        return y.view(*x.shape[:-1], N)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        M, N, K = ctx.dims
        nx, nw, nb = ctx.needs_input_grad[:3]
        if M == 0:
            return (g.new_empty((*g.shape[:-1], K), dtype=ctx.x_dtype) if nx else None,
                    g.new_zeros((N, K), dtype=ctx.param_dtypes[0]) if nw else None,
                    g.new_zeros(N, dtype=ctx.param_dtypes[1]) if nb else None, None)
        saved = ctx.saved_tensors
        g2, _ = _matrix(g.reshape(M, N), "linear_fp8")
        dx, dw, db = _linear_backward(ctx, g2, saved[:2], saved[2:], K, ctx.x_dtype, (nx, nw, nb), ctx.grad_dtype)
        return dx.view(*g.shape[:-1], K) if nx else None, dw, db, None


def linear_fp8(x: torch.Tensor, lin: torch.nn.Linear, grad_dtype: torch.dtype = torch.float8_e4m3fn) -> torch.Tensor:
    """``lin(x)`` with 8-bit products, differentiable: ``dense.big_linear`` in 8 bits.

    x [..., K] float32 / bfloat16 / float16 -> [..., N] of x's type; lin's parameters in any of the three, their gradients in theirs.
    y = x W^T + b, dx = g W and dW = g^T x are products of blocks along the axis that each sums over; g is rounded to ``grad_dtype``
    (e4m3, or e5m2 for more range inside a block); db is the sum of the unrounded g."""
    _format(grad_dtype, "linear_fp8")
    _linear_params(x, lin.weight, lin.bias, "linear_fp8")
    return LinearFp8.apply(x, lin.weight, lin.bias, grad_dtype)


def layer_norm_fp8(x: torch.Tensor, norm: torch.nn.LayerNorm, dtype: torch.dtype = torch.float8_e4m3fn) -> Fp8Blocks:
    """``norm(x)`` as blocks, rounded once from float32, in one launch: the left operand of ``matmul_fp8`` at inference."""
    fmt = _format(dtype, "layer_norm_fp8")
    _no_graph("layer_norm_fp8", x, norm.weight, norm.bias)
    x2, ld, gamma, beta, p_dtype = _norm_rows(x, norm, "layer_norm_fp8")
    blocks = _empty_blocks(*x2.shape, dtype, x.device)
    _layer_norm_forward(x2, ld, gamma, beta, p_dtype, norm.eps, None, None, blocks, fmt)
    return Fp8Blocks(*blocks, x2.shape[1])


class LayerNormLinearFp8(Function):
    """apply(x, gamma, beta, weight, bias, norm, grad_dtype): see ``layer_norm_linear_fp8``."""

    @staticmethod
    def forward(ctx, x, gamma, beta, weight, bias, norm, grad_dtype):
        what = "layer_norm_linear_fp8"
        x2, ld, gamma, beta, p_dtype = _norm_rows(x, norm, what)
        w2, ldw = _matrix(weight, what)
        M, K = x2.shape
        N = w2.shape[0]
        if M > _MAX_DIM:
            raise ValueError(f"{what}: up to 2^23 rows")
        nx, ng, nbt, nw, nb = ctx.needs_input_grad[:5]
        ctx.param_dtypes = (weight.dtype, bias.dtype if bias is not None else None)
        ctx.dims, ctx.grad_dtype, ctx.p_dtype, ctx.ld = (M, N, K), grad_dtype, p_dtype, ld
        if M == 0:
            ctx.x_dtype = x.dtype
            ctx.save_for_backward()
            return x.new_empty((*x.shape[:-1], N))
        before = nx or ng or nbt                       # something in front of the product wants a gradient
        wr, wt, _ = _quantize(w2, ldw, torch.float8_e4m3fn, cols=before, tile=True)
        stats = torch.empty((2, M), dtype=torch.float32, device=x.device) if before or nw else None
        if nw:                                         # both forms: statistics first, then one more read normalises and rounds
            _layer_norm_forward(x2, ld, gamma, beta, p_dtype, norm.eps, None, stats)
            xr, xt, _ = _quantize(x2, ld, torch.float8_e4m3fn, cols=True, norm=(stats, gamma, beta, p_dtype))
        else:
            xr, xt = _empty_blocks(M, K, torch.float8_e4m3fn, x.device), (None, None)
            _layer_norm_forward(x2, ld, gamma, beta, p_dtype, norm.eps, None, stats, xr)
        y = _matmul(*xr, *wr, K, bias, 0, x.dtype)
        ctx.save_for_backward(*xt, *(wt if before else (None, None)), x2 if before else None, stats, gamma)
        return y.view(*x.shape[:-1], N)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        M, N, K = ctx.dims
        nx, ng, nbt, nw, nb = ctx.needs_input_grad[:5]
        if M == 0:
            z = lambda want, shape, dtype: g.new_zeros(shape, dtype=dtype) if want else None
            return (z(nx, (*g.shape[:-1], K), ctx.x_dtype), z(ng, K, ctx.p_dtype), z(nbt, K, ctx.p_dtype),
                    z(nw, (N, K), ctx.param_dtypes[0]), z(nb, N, ctx.param_dtypes[1]), None, None)
        *blocks, x2, stats, gamma = ctx.saved_tensors
        before = nx or ng or nbt
        g2, _ = _matrix(g.reshape(M, N), "layer_norm_linear_fp8")
        x_dtype = x2.dtype if before else None
        dz, dw, db = _linear_backward(ctx, g2, blocks[:2], blocks[2:], K, x_dtype, (before, nw, nb), ctx.grad_dtype)
        dx, dp = _layer_norm_backward(dz, x2, ctx.ld, stats, gamma, ctx.p_dtype, nx, ng or nbt) if before else (None, None)
        return (dx.view(*g.shape[:-1], K) if nx else None, dp[0] if ng else None, dp[1] if nbt else None, dw, db, None, None)


def layer_norm_linear_fp8(x: torch.Tensor, norm: torch.nn.LayerNorm, lin: torch.nn.Linear,
                          grad_dtype: torch.dtype = torch.float8_e4m3fn) -> torch.Tensor:
    """``lin(norm(x))``, differentiable, as ``linear_fp8`` after ``fused.layer_norm`` without the norm's result in 16 or 32 bits: it is
    rounded from float32 straight into the blocks that the two products read.  The gradient between the two has x's type."""
    what = "layer_norm_linear_fp8"
    _format(grad_dtype, what)
    _linear_params(x, lin.weight, lin.bias, what)
    return LayerNormLinearFp8.apply(x, norm.weight, norm.bias, lin.weight, lin.bias, norm, grad_dtype)
