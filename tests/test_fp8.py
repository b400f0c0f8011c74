"""What the 8-bit operators and the layer norm of wide rows refuse, and the format's reference itself: all on the CPU."""
import ctypes

import pytest
import torch

from tests import fp8_reference as R
from snipper_amd import _lib, fp8, fused

E4M3, E5M2 = R.E4M3, R.E5M2


def _cpu_blocks(rows=4, cols=200, dtype=E4M3):
    return R.random_blocks(rows, cols, dtype, "cpu", torch.Generator().manual_seed(0))


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_reference_rounds_like_the_types(dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.cat([torch.randn(4096, generator=g) * 100, torch.randn(4096, generator=g) * 1e-3, torch.tensor([0.0, 448, -448, 17, 19, 2.0 ** -10])])
    x = x.clamp(-448, 448)
    assert torch.equal(R.round_to(x.double(), dtype), x.to(dtype).double())


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_reference_scales_are_the_smallest_that_hold(dtype):
    most = R.MOST[dtype]
    a = torch.tensor([most, most * 2 ** 10, most * 1.0001, most * 0.5, most * 0.5001, 1e-44, 3e38, 0.0], dtype=torch.float32).double()
    e = R.exponents(a, dtype)
    ok = a > 0
    assert (a <= most * R.pow2(e))[ok].all()
    assert ((a > most * R.pow2(e - 1)) | (e == -127))[ok].all()
    assert e.tolist()[:5] == [0, 10, 1, -1, 0] and e[-1] == 0


def test_blocks_check_their_parts():
    b = _cpu_blocks()
    assert b.shape == (4, 200) and b.dequantize().shape == (4, 200)
    assert torch.equal(b.dequantize().double(), R.held(b))
    for bad in (lambda: fp8.Fp8Blocks(b.data, b.scale, 300), lambda: fp8.Fp8Blocks(b.data[:, :128], b.scale, 200),
                lambda: fp8.Fp8Blocks(b.data, b.scale[:, :2], 200), lambda: fp8.Fp8Blocks(b.data[:2], b.scale, 200),
                lambda: fp8.Fp8Blocks(b.data, b.scale, 0), lambda: fp8.Fp8Blocks(b.data.t(), b.scale, 200)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        fp8.Fp8Blocks(b.data.float(), b.scale, 200)
    with pytest.raises(TypeError):
        fp8.Fp8Blocks(b.data, b.scale.float(), 200)


def test_cpu_tensors_are_refused():
    x, lin, norm = torch.randn(4, 200), torch.nn.Linear(200, 8), torch.nn.LayerNorm(200)
    with torch.no_grad():
        for call in (lambda: fp8.quantize_rows(x), lambda: fp8.quantize_both(x), lambda: fp8.quantize_tiles(lin.weight),
                     lambda: fp8.matmul_fp8(_cpu_blocks(), _cpu_blocks()), lambda: fp8.linear_fp8(x, lin),
                     lambda: fp8.layer_norm_fp8(x, norm), lambda: fp8.layer_norm_linear_fp8(x, norm, lin), lambda: fused.layer_norm(x, norm)):
            with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
                call()


def test_types_and_sizes_are_refused():
    x, lin, norm = torch.randn(4, 200), torch.nn.Linear(200, 8), torch.nn.LayerNorm(200)
    with pytest.raises(TypeError):
        fp8.quantize_rows(x, torch.float16)
    with pytest.raises(TypeError):
        fp8.linear_fp8(x, lin, grad_dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        fp8.linear_fp8(torch.randn(4, 100), lin)
    with pytest.raises(ValueError):
        fp8.matmul_fp8(_cpu_blocks(cols=200), _cpu_blocks(cols=201))


def test_inference_calls_do_not_drop_gradients_in_silence():
    x, norm = torch.randn(4, 200, requires_grad=True), torch.nn.LayerNorm(200)
    for call in (lambda: fp8.quantize_rows(x), lambda: fp8.quantize_both(x), lambda: fp8.quantize_tiles(x), lambda: fp8.layer_norm_fp8(x, norm)):
        with pytest.raises(RuntimeError, match="not differentiable"):
            call()


# ---- the C entries: arguments are checked before anything is launched --------------------------------------------------
P = ctypes.c_void_p(4096)
NULL, SHAPE = -1, -2


def test_c_quantize_refuses():
    f = _lib.load().snipper_fp8_quantize

    def call(x=P, dt=0, ld=200, rows=4, cols=200, tile=1, fmt=0, mean=None, rstd=None, gamma=None, beta=None, pdt=0, d=P, s=P, dt_=None,
             st_=None, cs=None, cdt=0, ws=None, nb=0):
        return f(None, x, dt, ld, rows, cols, tile, fmt, mean, rstd, gamma, beta, pdt, d, s, dt_, st_, cs, cdt, ws, nb)
    assert call(x=None) == NULL and call(d=None) == NULL and call(s=None) == NULL and call(dt_=P) == NULL and call(mean=P) == NULL
    for bad in (dict(rows=0), dict(cols=0), dict(rows=(1 << 23) + 1), dict(cols=(1 << 23) + 1, ld=1 << 24), dict(ld=199), dict(dt=2), dict(dt=7),
                dict(tile=64), dict(fmt=2), dict(pdt=2), dict(gamma=P), dict(d=ctypes.c_void_p(4104)), dict(s=ctypes.c_void_p(4098)),
                dict(cs=P), dict(cs=P, cdt=2, ws=P, nb=4 * 200), dict(cs=P, ws=P, nb=4 * 200 - 1), dict(tile=128, mean=P, rstd=P)):
        assert call(**bad) == SHAPE, bad
    assert _lib.load().snipper_fp8_quantize_workspace_bytes(129, 200, 1) == 2 * 200 * 4
    assert _lib.load().snipper_fp8_quantize_workspace_bytes(129, 200, 0) == 0


def test_c_matmul_refuses():
    lib = _lib.load()

    def call(a=P, sa=P, fa=0, b=P, sb=P, fb=0, M=4, N=8, K=200, bias=None, bdt=0, out=P, odt=1, ws=None, nb=0):
        return lib.snipper_fp8_matmul(None, a, sa, fa, b, sb, fb, M, N, K, bias, bdt, 0, out, odt, ws, nb)
    for n in ("a", "sa", "b", "sb", "out"):
        assert call(**{n: None}) == NULL, n
    for bad in (dict(M=0), dict(N=0), dict(K=0), dict(K=(1 << 23) + 1), dict(fa=2), dict(fb=-1), dict(odt=2), dict(bdt=2),
                dict(a=ctypes.c_void_p(4104)), dict(sb=ctypes.c_void_p(4098)), dict(out=ctypes.c_void_p(4104))):
        assert call(**bad) == SHAPE, bad
    assert call(M=1 << 23, N=1 << 17) == SHAPE                                # (2^40 elements of a result)
    need = lib.snipper_fp8_matmul_workspace_bytes(384, 1024, 79000, 0)         # (a weight gradient: the reduction is split)
    assert need > 0 and need % (384 * 1024 * 4) == 0
    assert call(M=384, N=1024, K=79000, odt=0) == SHAPE and call(M=384, N=1024, K=79000, odt=0, ws=P, nb=need - 1) == SHAPE
    assert lib.snipper_fp8_matmul_workspace_bytes(1, 4096, 4096, 1) == 0


def test_c_layer_norm_refuses():
    lib = _lib.load()

    def fwd(x=P, dt=0, ld=200, g=P, b=P, pdt=0, rows=4, cols=200, eps=1e-5, y=P, mean=None, rstd=None, d=None, s=None, fmt=0):
        return lib.snipper_layernorm_forward(None, x, dt, ld, g, b, pdt, rows, cols, eps, y, mean, rstd, d, s, fmt)

    def bwd(g=P, x=P, dt=0, ld=200, mean=P, rstd=P, gamma=P, pdt=0, rows=4, cols=200, dx=P, dg=None, db=None, ws=None, nb=0):
        return lib.snipper_layernorm_backward(None, g, x, dt, ld, mean, rstd, gamma, pdt, rows, cols, dx, dg, db, ws, nb)
    assert fwd(x=None) == NULL and fwd(y=None) == NULL and fwd(mean=P) == NULL and fwd(d=P) == NULL
    for bad in (dict(rows=0), dict(cols=0), dict(cols=16385, ld=16385), dict(ld=100), dict(dt=2), dict(pdt=4), dict(fmt=3), dict(eps=-1.0),
                dict(eps=float("nan")), dict(d=ctypes.c_void_p(4100), s=P)):
        assert fwd(**bad) == SHAPE, bad
    assert lib.snipper_layernorm_backward_workspace_bytes((1 << 31) - 1, 100) > 0       # (the largest number of rows)
    assert bwd(g=None) == NULL and bwd(mean=None) == NULL and bwd(dx=None) == NULL and bwd(dg=P) == NULL
    need = lib.snipper_layernorm_backward_workspace_bytes(4, 200)
    assert need == 2 * 200 * 4
    for bad in (dict(rows=-1), dict(cols=16385, ld=16385), dict(ld=100), dict(dt=2), dict(pdt=5), dict(dg=P, db=P), dict(dg=P, db=P, ws=P, nb=need - 1)):
        assert bwd(**bad) == SHAPE, bad
