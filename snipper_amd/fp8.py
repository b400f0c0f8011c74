"""8-bit products with a power-of-two scale for each 128 elements (include/snipper_fp8.h, csrc/gemm_fp8.cuh, quant_fp8.cuh).

What the bf16 products of ``dense.py`` are for Linears in 16 bits, these are in 8:

    quantize_rows / quantize_both / quantize_tiles   a matrix into blocks (``Fp8Blocks``)
    matmul_fp8(a, b, bias)                           a @ b.T + bias of two matrices in blocks
    linear_fp8(x, lin)                               ``lin(x)``, differentiable: all three products of a training step in 8 bits
    layer_norm_fp8(x, norm)                          ``norm(x)`` straight into blocks, for inference
    layer_norm_linear_fp8(x, norm, lin)              ``lin(norm(x))``, differentiable, the norm's result held in 8 bits only

At inference, under ``torch.no_grad()``, a weight is laid out once, ``w8, _ = quantize_tiles(lin.weight)``, and used as
``matmul_fp8(quantize_rows(x), w8, lin.bias)`` or ``matmul_fp8(layer_norm_fp8(x, norm), w8, lin.bias)``.

Blocks run along the axis that a product sums over.  The training step therefore rounds x and the gradient twice, along their rows
(y = x W^T, dx = g W) and along their columns (dW = g^T x), both from one read; a weight has one scale for each 128 x 128 tile, so its
transpose holds the same values.  Scales are powers of two that keep the largest element of a block in range: nothing saturates, and
an element is its input rounded once.  CUDA tensors only, as everywhere in this package; autocast changes nothing here, a result has
x's type.

Every call can be captured into a graph.  A captured backward pass needs what PyTorch asks of any: leaves whose eager graphs are gone
(the engine would otherwise join the capture to the stream that those were made on).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._autograd import Function
from .fused import (_ROW_DT, _call, _differentiates, _layer_norm_backward, _layer_norm_forward, _norm_rows, _once_differentiable, _opt,
                    _row_stride)

_FMT = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}
_MAX_DIM = 1 << 23
_FULL_SUMS = 16                        # SNIPPER_FP8_FULL_SUMS


class Fp8Blocks:
    """A matrix [rows, cols] in 8-bit blocks: ``data`` [rows, 128 ceil(cols / 128)] float8_e4m3fn / float8_e5m2, zeros behind the last
    column, ``scale`` [rows, 4 ceil(cols / 512)] float8_e8m0fnu, one for each 128 elements of a row, 1 behind the last block; both
    contiguous.  The quantizers make them; a program that keeps a weight in a file stores the two tensors and ``cols``."""

    __slots__ = ("data", "scale", "cols")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, cols: int):
        if data.dtype not in _FMT or scale.dtype is not torch.float8_e8m0fnu:
            raise TypeError(f"Fp8Blocks: data in float8_e4m3fn or float8_e5m2 and scale in float8_e8m0fnu, got {data.dtype} and {scale.dtype}")
        shape = data.shape
        if cols < 1 or len(shape) != 2 or shape[1] != -(-cols // 128) * 128 or scale.shape != (shape[0], -(-cols // 512) * 4):
            raise ValueError(f"Fp8Blocks: data {tuple(shape)} and scale {tuple(scale.shape)} are not those of {cols} columns")
        if not (data.is_contiguous() and scale.is_contiguous()) or data.device != scale.device:
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


# Inside this file a matrix in blocks is (address of its data, of its scales): several lie in one buffer, each from a multiple of 256 on.
def _room(rows: int, cols: int) -> int:
    return (rows * (-(-cols // 128) * 128 + -(-cols // 512) * 4) + 255) & -256


def _at(address: int, rows: int, cols: int) -> Tuple[int, int]:
    return address, address + rows * (-(-cols // 128) * 128)


def _parts(b: Fp8Blocks) -> Tuple[int, int]:
    return b.data.data_ptr(), b.scale.data_ptr()


def _new_blocks(rows: int, cols: int, dtype, device) -> Fp8Blocks:
    return Fp8Blocks(torch.empty((rows, -(-cols // 128) * 128), dtype=dtype, device=device),
                     torch.empty((rows, -(-cols // 512) * 4), dtype=torch.float8_e8m0fnu, device=device), cols)


def _matrix(x: torch.Tensor, what: str):
    """x [..., cols] as a matrix with unit stride inside a row, and its row stride."""
    if not x.is_cuda:
        raise RuntimeError(f"{what}: Not implemented on the CPU")
    if x.dtype not in _ROW_DT:
        raise TypeError(f"{what}: float32, bfloat16 or float16, got {x.dtype}")
    shape = x.shape
    if len(shape) < 2:
        raise ValueError(f"{what}: a matrix or a batch of rows, got {tuple(shape)}")
    C = shape[-1]
    x2 = x if len(shape) == 2 else x.reshape(-1, C) if C else x
    R = x2.shape[0]
    if not 1 <= C <= _MAX_DIM or R > _MAX_DIM:
        raise ValueError(f"{what}: up to 2^23 rows of 1 to 2^23 elements, got {tuple(shape)}")
    return _row_stride(x2)


def _format(dtype, what: str) -> int:
    if dtype not in _FMT:
        raise TypeError(f"{what}: float8_e4m3fn or float8_e5m2, got {dtype}")
    return _FMT[dtype]


def _no_graph(what: str, *tensors) -> None:
    if _differentiates(*tensors):
        raise RuntimeError(f"{what} is not differentiable: use linear_fp8 / layer_norm_linear_fp8, or call it under torch.no_grad() "
                           "(and, in forward mode, on tensors without a tangent)")


_NONE = (None, None)


def _quantize(x2, ld, fmt, a=_NONE, b=_NONE, tile=1, norm=None, colsum=None, ws=None, ws_bytes=0):
    """x into a (blocks of x) and / or b (blocks of x^T); the sums over the rows into ``colsum`` if given.  ``norm``: (stats [2, R],
    gamma, beta, p_dtype)."""
    R, C = x2.shape
    mean = rstd = gamma = beta = None
    p_dtype = 0
    if norm is not None:
        mean, gamma, beta, p_dtype = norm[0].data_ptr(), _opt(norm[1]), _opt(norm[2]), _ROW_DT[norm[3]]
        rstd = mean + 4 * R
    _call(_lib.load().snipper_fp8_quantize, x2.get_device(), x2.data_ptr(), _ROW_DT[x2.dtype], ld, R, C, tile, fmt, mean, rstd, gamma, beta, p_dtype,
          a[0], a[1], b[0], b[1], _opt(colsum), _ROW_DT[colsum.dtype] if colsum is not None else 0, ws, ws_bytes)


def quantize_rows(x: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn) -> Fp8Blocks:
    """x [..., cols] (float32 / bfloat16 / float16, leading axes as rows) into blocks of 128 elements of a row."""
    fmt = _format(dtype, "quantize_rows")
    _no_graph("quantize_rows", x)
    x2, ld = _matrix(x, "quantize_rows")
    a = _new_blocks(*x2.shape, dtype, x.device)
    if x2.shape[0]:
        _quantize(x2, ld, fmt, _parts(a))
    return a


def quantize_both(x: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn) -> Tuple[Fp8Blocks, Fp8Blocks]:
    """(blocks of x, blocks of x^T) from one read: the second has a scale for each 128 elements of a COLUMN of x."""
    fmt = _format(dtype, "quantize_both")
    _no_graph("quantize_both", x)
    x2, ld = _matrix(x, "quantize_both")
    if x2.shape[0] == 0:
        raise ValueError("quantize_both: a matrix without rows has no columns to cut into blocks")
    a, b = _new_blocks(*x2.shape, dtype, x.device), _new_blocks(x2.shape[1], x2.shape[0], dtype, x.device)
    _quantize(x2, ld, fmt, _parts(a), _parts(b))
    return a, b


def quantize_tiles(w: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn) -> Tuple[Fp8Blocks, Fp8Blocks]:
    """(blocks of w, blocks of w^T) of a weight [out, in] with one scale for each 128 x 128 tile: the two hold the same values."""
    fmt = _format(dtype, "quantize_tiles")
    _no_graph("quantize_tiles", w)
    if w.dim() != 2 or w.shape[0] == 0:
        raise ValueError(f"quantize_tiles: a matrix with rows, got {tuple(w.shape)}")
    w2, ld = _matrix(w, "quantize_tiles")
    a, b = _new_blocks(*w2.shape, dtype, w.device), _new_blocks(w2.shape[1], w2.shape[0], dtype, w.device)
    _quantize(w2, ld, fmt, _parts(a), _parts(b), tile=128)
    return a, b


def _product(like, a, a_fmt, b, b_fmt, M, N, K, bias, relu, out_dtype, full):
    """act(a b^T + bias) [M, N] on the device of ``like``; full: _FULL_SUMS or 0."""
    out = like.new_empty((M, N), dtype=out_dtype)
    if M == 0 or N == 0:
        return out
    lib = _lib.load()
    od = _ROW_DT[out_dtype] | full
    nbytes = lib.snipper_fp8_matmul_workspace_bytes(M, N, K, od)
    ws = like.new_empty(nbytes // 4, dtype=torch.float32) if nbytes else None
    _call(lib.snipper_fp8_matmul, like.get_device(), a[0], a[1], a_fmt, b[0], b[1], b_fmt, M, N, K, _opt(bias),
          _ROW_DT[bias.dtype] if bias is not None else 0, relu, out.data_ptr(), od, _opt(ws), nbytes)
    return out


def _check_bias(bias, N, device, what):
    if bias.dtype not in _ROW_DT or bias.shape != (N,) or bias.device != device or (N > 1 and bias.stride(0) != 1):
        raise ValueError(f"{what}: bias [{N}] contiguous, of a floating type, on the operands' device")


def matmul_fp8(a: Fp8Blocks, b: Fp8Blocks, bias: Optional[torch.Tensor] = None, relu: bool = False,
               out_dtype: torch.dtype = torch.bfloat16, full_sums: bool = False) -> torch.Tensor:
    """act(a @ b.T + bias): a [M, K], b [N, K] in blocks (either type each), bias [N] or None -> [M, N] of ``out_dtype``.

    A bfloat16 / float16 result comes from the 8-bit matrix instructions, which cut the products of eight neighbours off at 2^-13 of the
    largest: before its own rounding an element is off by less than 8.5e-4 of the sum of its products' magnitudes (on random data by
    1.5e-5 of the result's norm).  With ``full_sums``, and always in a float32 result or one of up to 16 rows, the sums are float32 ones (1e-7), from
    the bfloat16 instructions on exactly widened operands at a quarter of the rate."""
    K, ad, bd = a.cols, a.data, b.data
    if K != b.cols:
        raise ValueError(f"matmul_fp8: a {a.shape} and b {b.shape} have rows of different length")
    if not ad.is_cuda:
        raise RuntimeError("matmul_fp8: Not implemented on the CPU")
    if ad.get_device() != bd.get_device():
        raise ValueError("matmul_fp8: operands on one device")
    if out_dtype not in _ROW_DT:
        raise TypeError(f"matmul_fp8: out_dtype float32, bfloat16 or float16, got {out_dtype}")
    M, N = ad.shape[0], bd.shape[0]
    if M > _MAX_DIM or N > _MAX_DIM or K > _MAX_DIM:
        raise ValueError("matmul_fp8: sizes up to 2^23")
    if bias is not None:
        _no_graph("matmul_fp8", bias)
        _check_bias(bias, N, ad.device, "matmul_fp8")
    return _product(ad, _parts(a), _FMT[ad.dtype], _parts(b), _FMT[bd.dtype], M, N, K, bias, int(relu), out_dtype,
                    _FULL_SUMS if full_sums else 0)


def _linear_params(x, weight, bias, what):
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] == 0:
        raise ValueError(f"{what}: x {tuple(x.shape)} and weight {tuple(weight.shape)}")
    if weight.device != x.device:
        raise ValueError(f"{what}: weight on x's device")
    if bias is not None:
        _check_bias(bias, weight.shape[0], x.device, what)


def _linear_forward(x2, ld, weight, bias, out_dtype, want_wt, want_xt, full, what, norm=None):
    """y [M, N] of x2 [M, K] (normalised first with ``norm``), and a buffer of what the backward pass reads: the columns' blocks of the
    input (for dW; in front) and of the weight (for dx)."""
    w2, ldw = _matrix(weight, what)
    M, K = x2.shape
    N = w2.shape[0]
    if M == 0:
        return x2.new_empty((0, N), dtype=out_dtype), None
    x_room = _room(M, K)
    xt_room = _room(K, M) if want_xt else 0
    rows = x2.new_empty(x_room + _room(N, K), dtype=torch.uint8)
    keep = x2.new_empty(xt_room + (_room(K, N) if want_wt else 0), dtype=torch.uint8) if want_xt or want_wt else None
    p = rows.data_ptr()
    xr, wr = _at(p, M, K), _at(p + x_room, N, K)
    _quantize(w2, ldw, 0, wr, _at(keep.data_ptr() + xt_room, K, N) if want_wt else _NONE, tile=128)
    xt = _at(keep.data_ptr(), K, M) if want_xt else _NONE
    if norm is None:
        _quantize(x2, ld, 0, xr, xt)
    else:
        stats, gamma, beta, p_dtype, eps = norm
        if want_xt:                                    # both forms: statistics first, then one more read normalises and rounds
            _layer_norm_forward(x2, ld, gamma, beta, p_dtype, eps, None, stats)
            _quantize(x2, ld, 0, xr, xt, norm=(stats, gamma, beta, p_dtype))
        else:
            _layer_norm_forward(x2, ld, gamma, beta, p_dtype, eps, None, stats, xr)
    return _product(x2, xr, 0, wr, 0, M, N, K, bias, 0, out_dtype, full), keep


def _linear_backward(g, dims, keep, dtypes, want, grad_fmt, full):
    """(dx [M, K] or None, dW or None, db or None) from the gradient [..., N]; dims (M, N, K); dtypes of the three; want = which, the
    first two as in the forward pass."""
    M, N, K = dims
    wx, ww, wb = want
    g2, ld = _matrix(g if g.dim() == 2 else g.reshape(M, N), "linear_fp8")
    ws_bytes = _lib.load().snipper_fp8_quantize_workspace_bytes(M, N, 1) if wb else 0
    g_room, t_room = _room(M, N) if wx else 0, _room(N, M) if ww or not wx else 0
    buf = g2.new_empty(g_room + t_room + ws_bytes, dtype=torch.uint8)
    p = buf.data_ptr()
    gr, gt = _at(p, M, N) if wx else _NONE, _at(p + g_room, N, M) if t_room else _NONE
    db = g2.new_empty(N, dtype=dtypes[2]) if wb else None
    _quantize(g2, ld, grad_fmt, gr, gt, colsum=db, ws=p + g_room + t_room if wb else None, ws_bytes=ws_bytes)
    keep = keep.contiguous() if keep is not None else None          # (saved-tensor hooks may have changed its stride)
    k = keep.data_ptr() if keep is not None else 0
    dx = _product(g2, gr, grad_fmt, _at(k + (_room(K, M) if ww else 0), K, N), 0, M, K, N, None, 0, dtypes[0], full) if wx else None
    dw = _product(g2, gt, grad_fmt, _at(k, K, M), 0, N, K, M, None, 0, dtypes[1], full) if ww else None
    return dx, dw, db


def _zero_grads(g, shapes, dtypes, want):
    return tuple(g.new_zeros(s, dtype=d) if w else None for s, d, w in zip(shapes, dtypes, want))


class LinearFp8(Function):
    """apply(x, weight, bias, grad_fmt, full): see ``linear_fp8``."""

    @staticmethod
    def forward(ctx, x, weight, bias, grad_fmt, full):
        x2, ld = _matrix(x, "linear_fp8")
        M, K = x2.shape
        N = weight.shape[0]
        ctx.meta = (M, N, K), (x.dtype, weight.dtype, bias.dtype if bias is not None else None), grad_fmt, full, x.shape
        if M == 0:
            ctx.save_for_backward()
            return x.new_empty((*x.shape[:-1], N))
        y, keep = _linear_forward(x2, ld, weight, bias, x.dtype, ctx.needs_input_grad[0], ctx.needs_input_grad[1], full, "linear_fp8")
        ctx.save_for_backward(keep)
        return y if x2 is x else y.view(*x.shape[:-1], N)

    @staticmethod
    @_once_differentiable
    def backward(ctx, g):
        dims, dtypes, grad_fmt, full, shape = ctx.meta
        want = ctx.needs_input_grad[:3]
        if dims[0] == 0:
            return *_zero_grads(g, (shape, dims[1:], dims[1]), dtypes, want), None, None
        keep, = ctx.saved_tensors
        dx, dw, db = _linear_backward(g, dims, keep, dtypes, want, grad_fmt, full)
        return dx.view(shape) if dx is not None and len(shape) != 2 else dx, dw, db, None, None


def linear_fp8(x: torch.Tensor, lin: torch.nn.Linear, grad_dtype: torch.dtype = torch.float8_e4m3fn, full_sums: bool = False) -> torch.Tensor:
    """``lin(x)`` with 8-bit products, differentiable: ``dense.big_linear`` in 8 bits.

    x [..., K] float32 / bfloat16 / float16 -> [..., N] of x's type; lin's parameters in any of the three, their gradients in theirs.
    y = x W^T + b, dx = g W and dW = g^T x are products of blocks along the axis that each sums over; g is rounded to ``grad_dtype``
    (e4m3, or e5m2 for more range inside a block); db is the sum of the unrounded g.  ``full_sums``: as for ``matmul_fp8``, of all three."""
    fmt, full = _format(grad_dtype, "linear_fp8"), _FULL_SUMS if full_sums else 0
    weight, bias = lin.weight, lin.bias
    _linear_params(x, weight, bias, "linear_fp8")
    if _differentiates(x, weight, bias):
        return LinearFp8.apply(x, weight, bias, fmt, full)
    x2, ld = _matrix(x, "linear_fp8")
    y, _ = _linear_forward(x2, ld, weight, bias, x.dtype, False, False, full, "linear_fp8")
    return y if x2 is x else y.view(*x.shape[:-1], weight.shape[0])


def layer_norm_fp8(x: torch.Tensor, norm: torch.nn.LayerNorm, dtype: torch.dtype = torch.float8_e4m3fn) -> Fp8Blocks:
    """``norm(x)`` as blocks, rounded once from float32, in one launch: the left operand of ``matmul_fp8`` at inference."""
    fmt = _format(dtype, "layer_norm_fp8")
    gamma, beta = norm.weight, norm.bias
    _no_graph("layer_norm_fp8", x, gamma, beta)
    x2, ld, p_dtype = _norm_rows(x, gamma, beta, norm.normalized_shape, "layer_norm_fp8")
    blocks = _new_blocks(*x2.shape, dtype, x.device)
    _layer_norm_forward(x2, ld, gamma, beta, p_dtype, norm.eps, None, None, (blocks.data.data_ptr(), blocks.scale.data_ptr()), fmt)
    return blocks


def _norm_linear_rows(x, gamma, beta, normalized_shape, what):
    """``_norm_rows`` within the sizes of the products."""
    x2, ld, p_dtype = _norm_rows(x, gamma, beta, normalized_shape, what)
    if x2.shape[0] > _MAX_DIM:
        raise ValueError(f"{what}: up to 2^23 rows")
    return x2, ld, p_dtype


class LayerNormLinearFp8(Function):
    """apply(x, gamma, beta, weight, bias, normalized_shape, eps, grad_fmt, full): see ``layer_norm_linear_fp8``."""

    @staticmethod
    def forward(ctx, x, gamma, beta, weight, bias, normalized_shape, eps, grad_fmt, full):
        what = "layer_norm_linear_fp8"
        x2, ld, p_dtype = _norm_linear_rows(x, gamma, beta, normalized_shape, what)
        M, K = x2.shape
        N = weight.shape[0]
        nx, ng, nbt, nw, nb = ctx.needs_input_grad[:5]
        ctx.meta = (M, N, K), (x.dtype, p_dtype, p_dtype, weight.dtype, bias.dtype if bias is not None else None), grad_fmt, full, x.shape
        if M == 0:
            ctx.save_for_backward()
            return x.new_empty((*x.shape[:-1], N))
        before = nx or ng or nbt                       # something in front of the product wants a gradient
        stats = x.new_empty((2, M), dtype=torch.float32) if before or nw else None
        y, keep = _linear_forward(x2, ld, weight, bias, x.dtype, before, nw, full, what, (stats, gamma, beta, p_dtype, eps))
        ctx.save_for_backward(keep, *((x2, stats, gamma) if before else (None, None, None)))
        return y if x2 is x else y.view(*x.shape[:-1], N)

    @staticmethod
    @_once_differentiable
    def backward(ctx, g):
        dims, dtypes, grad_fmt, full, shape = ctx.meta
        M, N, K = dims
        want = ctx.needs_input_grad[:5]
        if M == 0:
            return *_zero_grads(g, (shape, K, K, (N, K), N), dtypes, want), None, None, None, None
        nx, ng, nbt, nw, nb = want
        keep, x2, stats, gamma = ctx.saved_tensors
        before = nx or ng or nbt
        dz, dw, db = _linear_backward(g, dims, keep, (dtypes[0], dtypes[3], dtypes[4]), (before, nw, nb), grad_fmt, full)
        dx = dgamma = dbeta = None
        if before:
            dx, dgamma, dbeta = _layer_norm_backward(dz, x2, stats, gamma, dtypes[1], nx, ng or nbt)
        return (dx.view(shape) if nx and len(shape) != 2 else dx, dgamma if ng else None, dbeta if nbt else None, dw, db, None, None, None, None)


def layer_norm_linear_fp8(x: torch.Tensor, norm: torch.nn.LayerNorm, lin: torch.nn.Linear,
                          grad_dtype: torch.dtype = torch.float8_e4m3fn, full_sums: bool = False) -> torch.Tensor:
    """``lin(norm(x))``, differentiable, as ``linear_fp8`` after ``fused.layer_norm`` without the norm's result in 16 or 32 bits: it is
    rounded from float32 straight into the blocks that the two products read.  The gradient between the two has x's type."""
    what = "layer_norm_linear_fp8"
    fmt, full = _format(grad_dtype, what), _FULL_SUMS if full_sums else 0
    weight, bias = lin.weight, lin.bias
    _linear_params(x, weight, bias, what)
    gamma, beta = norm.weight, norm.bias
    if _differentiates(x, gamma, beta, weight, bias):
        return LayerNormLinearFp8.apply(x, gamma, beta, weight, bias, norm.normalized_shape, norm.eps, fmt, full)
    x2, ld, p_dtype = _norm_linear_rows(x, gamma, beta, norm.normalized_shape, what)
    y, _ = _linear_forward(x2, ld, weight, bias, x.dtype, False, False, full, what, (None, gamma, beta, p_dtype, norm.eps))
    return y if x2 is x else y.view(*x.shape[:-1], weight.shape[0])
