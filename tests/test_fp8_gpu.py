"""The 8-bit operators (snipper_amd/fp8.py) against their definitions in 64 bits, at the sizes and values where they can go wrong."""
import pytest
import torch

from tests import fp8_reference as R
from snipper_amd import fp8, fused

pytestmark = pytest.mark.gpu
E4M3, E5M2 = R.E4M3, R.E5M2
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda:0"


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _x(rows, cols, dtype, seed=0, spread=2.0):
    g = _gen(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(spread * torch.randn(rows, 1, generator=g)) * torch.exp(torch.randn(cols, generator=g))
    if rows > 3:
        x[rows // 2] = 0
    return x.to(dtype).to(DEV)


def _same_blocks(blocks, v, e):
    """blocks hold exactly the elements v and exponents e, zeros and 2^0 behind the matrix."""
    got = blocks.data.double().cpu()
    v = v.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(v))
    assert torch.equal(got.nan_to_num(0, 1e9, -1e9), v.nan_to_num(0, 1e9, -1e9))
    s = blocks.scale.view(torch.uint8).int().cpu()
    nb = v.shape[1] // 128
    assert torch.equal(s[:, :nb], e.cpu().int() + 127)
    assert (s[:, nb:] == 127).all()


SIZES = [(1, 1), (1, 4096), (3, 127), (5, 128), (2, 129), (7, 511), (33, 513), (127, 130), (128, 384), (129, 1000), (300, 257)]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantizers_give_the_definition_bit_for_bit(rows, cols, dtype, kind):
    x = _x(rows, cols, DT[kind])
    _same_blocks(fp8.quantize_rows(x, dtype), *R.quantize(x.cpu(), dtype))
    a, b = fp8.quantize_both(x, dtype)
    _same_blocks(a, *R.quantize(x.cpu(), dtype))
    _same_blocks(b, *R.quantize(x.cpu().t(), dtype))
    a, b = fp8.quantize_tiles(x, dtype)
    _same_blocks(a, *R.quantize(x.cpu(), dtype, 128))
    _same_blocks(b, *R.quantize(x.cpu().t(), dtype, 128))
    assert torch.equal(a.dequantize(), b.dequantize().t())


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_quantizers_at_the_ends_of_the_range(dtype):
    most = R.MOST[dtype]
    rows = [[0.0, -0.0], [1e-45, 3e-45], [2.0 ** -126, 1e-39], [2.0 ** -119, 2.0 ** -130], [3.4e38, -1e38], [most, -most], [most * 1.0001, 1.0],
            [most * 2 ** 20, 1.0], [float("inf"), 3.0], [float("nan"), 5.0], [-float("inf"), float("nan")], [float("nan"), float("nan")],
            [1.0 + 2 ** -23, 17 / 16], [19 / 16, 21 / 16], [most, most / 2 ** 17]]
    x = torch.zeros(len(rows), 200)
    x[:, 3], x[:, 150] = torch.tensor(rows).t()
    x[:, 4] = x[:, 150]
    want = R.quantize(x, dtype)
    _same_blocks(fp8.quantize_rows(x.to(DEV), dtype), *want)
    _same_blocks(fp8.quantize_both(x.to(DEV), dtype)[0], *want)
    _same_blocks(fp8.quantize_both(x.t().contiguous().to(DEV), dtype)[1], *want)
    _same_blocks(fp8.quantize_tiles(x.to(DEV), dtype)[0], *R.quantize(x, dtype, 128))


@pytest.mark.parametrize("skip,at", [(1, 0), (3, 1), (8, 5)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_quantizers_take_rows_of_a_wider_buffer(kind, skip, at):
    buf = _x(70, 300 + skip + at, DT[kind])
    x = buf[:, at:at + 300]
    want = R.quantize(x.cpu(), E4M3)
    _same_blocks(fp8.quantize_rows(x), *want)
    a, b = fp8.quantize_both(x)
    _same_blocks(a, *want)
    _same_blocks(b, *R.quantize(x.cpu().t(), E4M3))
    _same_blocks(fp8.quantize_rows(x.t()), *R.quantize(x.cpu().t(), E4M3))                 # (a transposed view: copied)
    _same_blocks(fp8.quantize_rows(x.view(7, 10, 300) if x.is_contiguous() else x.unflatten(0, (7, 10))), *want)
    _same_blocks(fp8.quantize_rows(x[:1].expand(5, 300)), *R.quantize(x.cpu()[:1].expand(5, 300), E4M3))


def test_no_rows():
    b = fp8.quantize_rows(torch.empty(0, 200, device=DEV))
    assert b.shape == (0, 200)
    w, _ = fp8.quantize_tiles(_x(16, 200, torch.float32))
    assert fp8.matmul_fp8(b, w).shape == (0, 16)


# ---- products ----------------------------------------------------------------------------------------------------------
def _check_product(y, a, b, bias, relu, out_dtype):
    A, B = R.held(a), R.held(b)
    e = A @ B.t()
    if bias is not None:
        e = e + bias.double()
    each, norm = R.product_bounds(A, B, e, out_dtype, bias)
    if relu:
        e = e.clamp(min=0)
    assert y.dtype == out_dtype and y.shape == e.shape
    d = (y.double() - e).abs()
    assert (d <= each).all(), (d / each).max()
    assert d.norm() <= norm, (d.norm(), norm)


@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("fa,fb", [(E4M3, E4M3), (E5M2, E4M3), (E4M3, E5M2), (E5M2, E5M2)])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 17, 128), (3, 300, 1000), (16, 64, 2100), (17, 33, 640), (40, 130, 512), (64, 16, 130),
                                   (65, 1, 300), (130, 127, 129), (200, 257, 1025)])
def test_matmul(M, N, K, fa, fb, out):
    g = _gen(M * N + K)
    a, b = R.random_blocks(M, K, fa, DEV, g, 4), R.random_blocks(N, K, fb, DEV, g, 4)
    bias = torch.randn(N, generator=g).to(DEV) * 1000 if N % 2 else None
    if out == "f16":                       # (in its range)
        a.scale.view(torch.uint8)[:, :-(-K // 128)] -= 14
    _check_product(fp8.matmul_fp8(a, b, bias, relu=N % 3 == 0, out_dtype=DT[out]), a, b, bias, N % 3 == 0, DT[out])


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(257, 129, 9000), (128, 128, 4096), (65, 70, 16385), (300, 200, 79001)])
def test_matmul_split_over_long_rows(M, N, K, out):
    """Few tiles and a long reduction: the K axis is cut, and the pieces are added in a fixed order."""
    g = _gen(K)
    x, w = torch.randn(M, K, generator=g).to(DEV), torch.randn(N, K, generator=g).to(DEV)
    a, b = fp8.quantize_rows(x), fp8.quantize_rows(w, E5M2)
    A, B = R.held(a), R.held(b)
    e = A @ B.t()
    y = fp8.matmul_fp8(a, b, out_dtype=DT[out])
    # float32: K + (pieces) additions; 16 bits: half a step and what a block's products lose (2^-13 of the largest, |p| <= 9 rms here)
    S = A.abs() @ B.abs().t()
    half = torch.finfo(DT[out]).eps / 2
    lost = 0.0 if out == "f32" else 9 * 2.0 ** -13 * S
    assert ((y.double() - e).abs() <= half * e.abs() + lost + (K + 64) * 2.0 ** -24 * S).all()
    assert (y.double() - e).norm() <= (half + (1e-6 if out == "f32" else 2e-4)) * e.norm()
    assert torch.equal(y, fp8.matmul_fp8(a, b, out_dtype=DT[out]))


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(4100, 4097, 300), (2300, 8200, 128), (9001, 1900, 1030), (79000, 384, 1024)])
def test_matmul_of_many_tiles(M, N, K, out):
    g = torch.Generator(device=DEV).manual_seed(K)
    x, w = torch.randn(M, K, generator=g, device=DEV), torch.randn(N, K, generator=g, device=DEV)
    bias = torch.randn(N, generator=g, device=DEV)
    a, b = fp8.quantize_rows(x), fp8.quantize_tiles(w)[0]
    e = R.held(a) @ R.held(b).t() + bias.double()
    y = fp8.matmul_fp8(a, b, bias, out_dtype=DT[out]).double()
    half = torch.finfo(DT[out]).eps / 2
    # rms of a sum of K unit products is sqrt(K); every element within what 2^-13 of the block's largest product (< 25 here) can lose
    lost = K * 2.0 ** -24 * K if out == "f32" else K * 25 * 2.0 ** -13
    assert ((y - e).abs() <= half * e.abs() + lost).all()
    assert (y - e).norm() <= (half + (1e-6 if out == "f32" else 2e-4)) * e.norm()


def test_a_poisoned_row_poisons_its_own_results_only():
    """NaN and infinite elements, and a scale that stands for NaN, in rows of both sides; every kernel."""
    for M, N, K in ((5, 40, 300), (200, 300, 300), (4100, 4100, 140)):
        for out in (torch.bfloat16, torch.float32):
            x, w = torch.randn(M, K, generator=_gen(1)).to(DEV), torch.randn(N, K, generator=_gen(2)).to(DEV)
            clean = fp8.matmul_fp8(fp8.quantize_rows(x, E5M2), fp8.quantize_rows(w), out_dtype=out)
            x[1, 7], x[2, 130], w[3, 5] = float("nan"), float("inf"), float("nan")
            a, b = fp8.quantize_rows(x, E5M2), fp8.quantize_rows(w)
            a.scale.view(torch.uint8)[3, 1] = 255
            y = fp8.matmul_fp8(a, b, out_dtype=out)
            assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all() and torch.isnan(y[:, 3]).all()
            assert not torch.isfinite(y[2]).any()
            rows, cols = [i for i in range(M) if i not in (1, 2, 3)], [j for j in range(N) if j != 3]
            assert torch.equal(y[rows][:, cols], clean[rows][:, cols])
            r = fp8.matmul_fp8(a, b, relu=True, out_dtype=out)
            assert torch.isnan(r[1]).all() and torch.isnan(r[3]).all()


def test_matmul_beyond_32_bit_offsets():
    """The left operand's elements lie more than 2^31 bytes behind its first."""
    M, K, N = 70000, 32768, 24
    a = fp8.quantize_rows(torch.ones(1, K, device=DEV))
    data, scale = a.data.expand(M, K).contiguous(), a.scale.expand(M, -1).contiguous()
    tail = torch.randn(100, K, generator=_gen(3)).to(DEV)
    t = fp8.quantize_rows(tail)
    data[-100:], scale.view(torch.uint8)[-100:] = t.data, t.scale.view(torch.uint8)
    w = fp8.quantize_rows(torch.randn(N, K, generator=_gen(4)).to(DEV))
    for out in (torch.bfloat16, torch.float32):
        y = fp8.matmul_fp8(fp8.Fp8Blocks(data, scale, K), w, out_dtype=out)
        e = R.held(t) @ R.held(w).t()
        assert (y[-100:].double() - e).norm() <= (torch.finfo(out).eps / 2 + 2e-4) * e.norm()
        e = R.held(a) @ R.held(w).t()
        assert (y[:-100].double() - e).norm() <= (torch.finfo(out).eps / 2 + 2e-4) * e.norm() * (M - 100) ** 0.5


def test_the_longest_rows():
    """2^23 elements: few rows, pieces of tiles, and whole tiles whose rows end 2^31 bytes behind a tile's first."""
    K = 1 << 23
    for M, N in ((3, 5), (20, 40)):
        a, b = (fp8.quantize_rows(torch.randn(n, K, device=DEV, dtype=torch.bfloat16)) for n in (M, N))
        e = torch.zeros(M, N, dtype=torch.float64, device=DEV)
        for at in range(0, K, 1 << 20):
            A, B = (x.data[:, at:at + (1 << 20)].double() * x.scale.float().double()[:, at // 128:at // 128 + 8192].repeat_interleave(128, 1) for x in (a, b))
            e += A @ B.t()
        # up to 2^15 additions in turn, each off by 2^-24 of a partial sum at most: 2^-24 sqrt(2^15) = 1.1e-5 where they are independent,
        # taken ten times; the 8-bit instructions' own 1.5e-5 twenty times; a block of 128 left out would be 2^-8
        for out, most in ((torch.float32, 1.1e-4), (torch.bfloat16, 2.0 ** -9 + 3e-4)):
            assert (fp8.matmul_fp8(a, b, out_dtype=out).double() - e).norm() <= most * e.norm()
    M = 4096
    bytes_ = [torch.zeros(M, K, dtype=torch.uint8, device=DEV) for _ in range(2)]
    scale = torch.full((M, K // 128), 127, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
    one, two = 0x38, 0x40                                                          # (1 and 2 in e4m3)
    for row, at in ((0, 0), (255, K - 1), (4095, K - 1), (3841, K // 2)):
        bytes_[0][row, at], bytes_[1][row, at] = one, two
    y = fp8.matmul_fp8(*(fp8.Fp8Blocks(d.view(E4M3), scale, K) for d in bytes_))
    e = torch.zeros(M, M, device=DEV, dtype=torch.bfloat16)
    for r, c in ((0, 0), (255, 255), (4095, 4095), (255, 4095), (4095, 255), (3841, 3841)):
        e[r, c] = 2
    assert torch.equal(y, e)


def test_more_than_four_million_rows():
    """The quantizers' third grid axis, and results whose last rows lie more than 2^32 bytes behind the first."""
    rows, K, N = (1 << 22) + 300, 70, 520
    x = torch.randn(rows, K, device=DEV, dtype=torch.bfloat16)
    a, at = fp8.quantize_both(x)
    ta, tat = fp8.quantize_both(x[-300:])                                         # (2^22 is a multiple of 128: the same blocks)
    u8 = lambda t: t.view(torch.uint8)
    assert torch.equal(u8(a.data)[-300:], u8(ta.data)) and torch.equal(u8(a.scale)[-300:], u8(ta.scale))
    assert torch.equal(u8(at.data)[:, 1 << 22:], u8(tat.data)) and torch.equal(u8(at.scale)[:, 1 << 15:(1 << 15) + 3], u8(tat.scale)[:, :3])
    r = fp8.quantize_rows(x)
    assert torch.equal(u8(r.data), u8(a.data)) and torch.equal(u8(r.scale), u8(a.scale))
    assert torch.equal(at.dequantize()[:, :1000], fp8.quantize_both(x[:1024])[1].dequantize()[:, :1000])
    w = fp8.quantize_rows(torch.randn(N, K, generator=_gen(4)).to(DEV))
    bias = torch.randn(N, generator=_gen(5)).to(DEV)
    for out in (torch.bfloat16, torch.float32):
        y = fp8.matmul_fp8(a, w, bias, out_dtype=out)
        _check_product(y[-300:], ta, w, bias, False, out)
        _check_product(y[:300], fp8.quantize_rows(x[:300]), w, bias, False, out)


# ---- training ----------------------------------------------------------------------------------------------------------
def _linear(n, k, dtype, bias=True, seed=5):
    lin = torch.nn.Linear(k, n, bias=bias)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(n, k, generator=_gen(seed)) / k ** 0.5)
        if bias:
            lin.bias.copy_(torch.randn(n, generator=_gen(seed + 1)))
    return lin.to(DEV, dtype)


def _close(y, A, B, extra=None):
    """y against A @ B.T (+ extra), A and B rounded matrices in 64 bits."""
    e = A @ B.t()
    S = A.abs() @ B.abs().t()
    if extra is not None:
        e, S = e + extra.double(), S + extra.double().abs()
    half = torch.finfo(y.dtype).eps / 2
    lost = 0.0 if y.dtype == torch.float32 else 2.0 ** -13 * S * 12          # (largest product of a block under 12 times the mean one)
    tiny = torch.finfo(y.dtype).smallest_normal * half
    assert ((y.double() - e).abs() <= half * e.abs() + lost + (A.shape[1] + 64) * 2.0 ** -24 * S + tiny).all()
    assert (y.double() - e).norm() <= (half + (1e-6 if y.dtype == torch.float32 else 3e-4)) * e.norm() + tiny * y.numel() ** 0.5


@pytest.mark.parametrize("kind,param,gd", [("bf16", "f32", E4M3), ("f32", "f32", E5M2), ("f16", "f16", E4M3), ("bf16", "bf16", E5M2)])
@pytest.mark.parametrize("M,N,K", [(1, 40, 70), (150, 130, 200), (1000, 384, 129)])
def test_linear_fp8_against_its_formulas(M, N, K, kind, param, gd):
    x = _x(M, K, DT[kind], spread=0.5).requires_grad_()
    lin = _linear(N, K, DT[param])
    g = (torch.randn(M, N, generator=_gen(9)) * 0.1).to(DT[kind]).to(DEV)
    y = fp8.linear_fp8(x, lin, grad_dtype=gd)
    dx, dw, db = torch.autograd.grad(y, (x, lin.weight, lin.bias), g)
    assert (y.dtype, dx.dtype, dw.dtype, db.dtype) == (x.dtype, x.dtype, lin.weight.dtype, lin.bias.dtype)
    w8 = R.rounded(lin.weight.detach().cpu(), E4M3, 128).to(DEV)
    q = lambda t, d=E4M3: R.rounded(t.detach().cpu(), d).to(DEV)
    _close(y.detach(), q(x), w8, lin.bias.detach())
    _close(dx, q(g, gd), w8.t().contiguous())
    _close(dw, q(g.t(), gd), q(x.t()))
    S = g.double().abs().sum(0)
    assert ((db.double() - g.double().sum(0)).abs() <= torch.finfo(db.dtype).eps / 2 * g.double().sum(0).abs() + 64 * 2.0 ** -24 * S).all()


def test_linear_fp8_gradients_against_differences():
    """The rounded map is linear in the rounded x and W: its differences in 64 bits give what the backward pass has to return when g is
    a value that e4m3 holds exactly."""
    M, N, K = 64, 48, 72
    x, lin = _x(M, K, torch.float32, spread=0.3).requires_grad_(), _linear(N, K, torch.float32)
    g = torch.randint(-2, 3, (M, N), generator=_gen(4)).float().to(DEV)
    dx, dw, db = torch.autograd.grad(fp8.linear_fp8(x, lin), (x, lin.weight, lin.bias), g)
    x8, xt8 = R.rounded(x.detach().cpu(), E4M3), R.rounded(x.detach().cpu().t(), E4M3).t()
    w8, b, gd = R.rounded(lin.weight.detach().cpu(), E4M3, 128), lin.bias.detach().cpu().double(), g.cpu().double()
    loss = lambda xx, ww, bb: ((xx @ ww.t() + bb) * gd).sum()
    for seed in range(3):
        u, v, t = (torch.randn(s, generator=_gen(seed), dtype=torch.float64) for s in ((M, K), (N, K), (N,)))
        h = 1e-4
        for grad, want in ((dx, (loss(x8 + h * u, w8, b) - loss(x8 - h * u, w8, b)) / (2 * h)),
                           (dw, (loss(xt8, w8 + h * v, b) - loss(xt8, w8 - h * v, b)) / (2 * h)),
                           (db, (loss(x8, w8, b + h * t) - loss(x8, w8, b - h * t)) / (2 * h))):
            d = {dx.shape: u, dw.shape: v, db.shape: t}[grad.shape]
            got = (grad.cpu().double() * d).sum()
            # linear, so the difference is exact but for 64-bit rounding; the gradients are float32 sums of up to 72 products
            assert (got - want).abs() <= 128 * 2.0 ** -24 * (grad.cpu().double().abs() * d.abs()).sum() + 1e-6 * want.abs()


@pytest.mark.parametrize("want", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)])
def test_linear_fp8_gives_the_gradients_that_are_asked_for(want):
    x, lin = _x(140, 72, torch.bfloat16, spread=0.5), _linear(48, 72, torch.float32)
    g = torch.randn(140, 48, generator=_gen(2)).bfloat16().to(DEV)
    leaves = [x, lin.weight, lin.bias]
    for t in leaves:
        t.requires_grad_(True)
    full = torch.autograd.grad(fp8.linear_fp8(x, lin), leaves, g)
    for t, w in zip(leaves, want):
        t.requires_grad_(bool(w))
    got = torch.autograd.grad(fp8.linear_fp8(x, lin), [t for t, w in zip(leaves, want) if w], g)
    for a, b in zip(got, [f for f, w in zip(full, want) if w]):
        assert torch.equal(a, b)


def test_linear_fp8_leading_axes_broadcast_rows_and_no_rows():
    lin = _linear(48, 72, torch.float32)
    x = _x(6, 72, torch.float32, spread=0.5).view(2, 3, 72)
    y = fp8.linear_fp8(x, lin)
    assert y.shape == (2, 3, 48) and torch.equal(y.view(6, 48), fp8.linear_fp8(x.view(6, 72), lin))
    row = _x(1, 72, torch.float32).requires_grad_()
    fp8.linear_fp8(row.expand(5, 72), lin).sum().backward()
    one = row.detach().expand(5, 72).contiguous().requires_grad_()
    lin.zero_grad()
    fp8.linear_fp8(one, lin).sum().backward()
    assert torch.equal(row.grad, one.grad.sum(0, keepdim=True))
    empty = torch.empty(0, 72, device=DEV, requires_grad=True)
    lin.zero_grad()
    y = fp8.linear_fp8(empty, lin)
    y.sum().backward()
    assert y.shape == (0, 48) and empty.grad.shape == (0, 72) and not lin.weight.grad.any() and not lin.bias.grad.any()
    nb = _linear(48, 72, torch.float32, bias=False)
    fp8.linear_fp8(x, nb).sum().backward()
    assert nb.weight.grad.abs().sum() > 0


def _norm(c, dtype=torch.float32, seed=11):
    n = torch.nn.LayerNorm(c)
    with torch.no_grad():
        n.weight.copy_(1 + 0.3 * torch.randn(c, generator=_gen(seed)))
        n.bias.copy_(0.3 * torch.randn(c, generator=_gen(seed + 1)))
    return n.to(DEV, dtype)


def _norm64(x, norm):
    x = x.detach().double().cpu()
    d = x - x.mean(1, keepdim=True)
    h = d / torch.sqrt((d * d).mean(1, keepdim=True) + norm.eps)
    return h * norm.weight.detach().double().cpu() + norm.bias.detach().double().cpu()


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 100), (17, 128), (5, 129), (33, 256), (18, 300), (9, 512), (4, 600), (3, 1100), (2, 2049), (2, 4097), (3, 8192), (2, 8193), (2, 16384)])
def test_layer_norm_fp8(rows, cols, kind, dtype):
    x, norm = _x(rows, cols, DT[kind], spread=0.5), _norm(cols)
    with torch.no_grad():
        b = fp8.layer_norm_fp8(x, norm, dtype)
    y = _norm64(x, norm)
    v, e = R.quantize(y, dtype)
    assert not b.data.view(torch.uint8)[:, cols:].any()
    s = b.scale.view(torch.uint8).int().cpu()
    assert (s[:, v.shape[1] // 128:] == 127).all()
    # float32 statistics move a value by up to 64 * 2^-24 of its parts: an element next to a border may land on the other side of it,
    # one step further, and so may a scale whose maximum lies at a power of two
    eb = s[:, :v.shape[1] // 128] - 127
    assert ((eb - e).abs() <= 1).all() and (eb != e).float().mean() <= 0.02
    got = R.held(b).cpu()
    step = 2.0 ** (-3 if dtype == E4M3 else -2)
    small = R.pow2(torch.maximum(eb, e)).repeat_interleave(128, 1)[:, :cols] * (2.0 ** -9 if dtype == E4M3 else 2.0 ** -16)
    assert ((got - y).abs() <= step / 2 * y.abs() + small / 2 + 1e-4 * (1 + y.abs())).all()
    assert (got != R.values(v, e, cols)).double().mean() <= 0.01


@pytest.mark.parametrize("param", ["f32", "bf16"])
def test_layer_norm_linear_fp8_is_the_two_together(param):
    """The run that a feed-forward block makes: norm, 8-bit product, ReLU, 8-bit product, backward through all of it."""
    M, K, N = 300, 200, 260
    x = _x(M, K, torch.bfloat16, spread=0.5).requires_grad_()
    norm, up, down = _norm(K, DT[param]), _linear(N, K, DT[param]), _linear(K, N, DT[param], seed=8)
    g = torch.randn(M, K, generator=_gen(3)).bfloat16().to(DEV)
    leaves = [x, norm.weight, norm.bias, up.weight, up.bias, down.weight, down.bias]

    def plain(round_=True):
        """The same in 64 bits on the CPU, straight through the rounding."""
        L = [t.detach().cpu().double().requires_grad_() for t in leaves]
        ste = lambda t, tile=1: t + (R.rounded(t.detach(), E4M3, tile) - t.detach()) if round_ else t
        d = L[0] - L[0].mean(1, keepdim=True)
        z = d / torch.sqrt((d * d).mean(1, keepdim=True) + norm.eps) * L[1] + L[2]
        h = torch.relu(ste(z) @ ste(L[3], 128).t() + L[4])
        y = ste(h) @ ste(L[5], 128).t() + L[6]
        return (y.detach(),) + torch.autograd.grad(y, L, g.cpu().double())
    h = torch.relu(fp8.layer_norm_linear_fp8(x, norm, up))
    y = fp8.linear_fp8(h, down)
    got = (y.detach(),) + torch.autograd.grad(y, leaves, g)
    for a, b, c in zip(got, plain(), plain(False)):
        off = (a.cpu().double() - b).norm() / b.norm()
        # rounding to 8 bits is off by at most 2^-4, about 2^-4 / sqrt(3) on average, once for each operand of each of up to four
        # products on the way (the reference rounds x and W, not the gradients, and rounds dW's operands along other blocks)
        assert off <= 4 * 2 * 2.0 ** -4 / 3 ** 0.5 / 2, off
        assert (a.cpu().double() - c).norm() / c.norm() <= 4 * 2 * 2.0 ** -4 / 3 ** 0.5
    # the composition of the public calls on the same values gives the same product
    with torch.no_grad():
        two = fp8.matmul_fp8(fp8.layer_norm_fp8(x, norm), fp8.quantize_tiles(up.weight)[0], up.bias)
        one = fp8.layer_norm_linear_fp8(x, norm, up)
    assert torch.equal(one, two)


@pytest.mark.parametrize("want", ["x", "norm", "weight", "bias", "all"])
def test_layer_norm_linear_fp8_gives_the_gradients_that_are_asked_for(want):
    x, norm, lin = _x(200, 150, torch.float32, spread=0.5), _norm(150), _linear(60, 150, torch.float32)
    groups = {"x": [x], "norm": [norm.weight, norm.bias], "weight": [lin.weight], "bias": [lin.bias]}
    leaves = [x, norm.weight, norm.bias, lin.weight, lin.bias]
    g = torch.randn(200, 60, generator=_gen(3)).to(DEV)
    for t in leaves:
        t.requires_grad_(True)
    full = dict(zip(map(id, leaves), torch.autograd.grad(fp8.layer_norm_linear_fp8(x, norm, lin), leaves, g)))
    # dx, dgamma and dbeta are the layer norm's own adjoint of the product's dx
    z = fused.layer_norm(x, norm)
    dz = torch.autograd.grad(fp8.linear_fp8(z, lin), z, g)[0]
    for a, t in zip(torch.autograd.grad(fused.layer_norm(x, norm), leaves[:3], dz), leaves[:3]):
        assert torch.equal(a, full[id(t)])
    asked = leaves if want == "all" else groups[want]
    for t in leaves:
        t.requires_grad_(any(t is u for u in asked))
    for t, a in zip(asked, torch.autograd.grad(fp8.layer_norm_linear_fp8(x, norm, lin), asked, g)):
        assert torch.equal(a, full[id(t)])


# ---- streams and graphs ------------------------------------------------------------------------------------------------
def test_another_stream_and_two_at_once():
    a = fp8.quantize_rows(_x(300, 9000, torch.float32, spread=0.2))
    b = fp8.quantize_rows(_x(200, 9000, torch.float32, seed=2, spread=0.2))
    want = fp8.matmul_fp8(a, b, out_dtype=torch.float32)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(fp8.matmul_fp8(a, b, out_dtype=torch.float32))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


def test_two_captured_graphs_replayed_in_turn():
    """Training steps in two graphs, new values in their inputs before each replay, eager work between; the eager calls' results."""
    lin, norm = _linear(130, 200, torch.float32), _norm(200)
    x, g = [_x(150, 200, torch.bfloat16, seed=s, spread=0.3).requires_grad_() for s in (1, 2)], torch.randn(150, 130, generator=_gen(7)).bfloat16().to(DEV)
    leaves = [norm.weight, norm.bias, lin.weight, lin.bias]

    def step(x):
        y = fp8.layer_norm_linear_fp8(x, norm, lin)
        return (y.detach(),) + torch.autograd.grad(y, [x] + leaves, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in x:
            step(t)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t in x:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(t))
        graphs.append(graph)
    for k in range(4):
        for i in (0, 1):
            with torch.no_grad():
                x[i].copy_(_x(150, 200, torch.bfloat16, seed=10 * k + i, spread=0.3))
            graphs[i].replay()
            torch.cuda.synchronize()
            for a, b in zip(outs[i], step(x[i])):
                assert torch.equal(a, b)


def test_threads_at_once():
    """Two threads on streams of their own: the library keeps nothing between calls."""
    import threading
    lin, norm = _linear(130, 200, torch.float32), _norm(200)
    xs = [_x(257, 200, torch.bfloat16, seed=s, spread=0.3) for s in (1, 2)]
    g = torch.randn(257, 130, generator=_gen(7)).bfloat16().to(DEV)

    def step(x):
        x = x.detach().requires_grad_()
        y = fp8.layer_norm_linear_fp8(x, norm, lin)
        return (y.detach(),) + torch.autograd.grad(y, (x, norm.weight, norm.bias, lin.weight, lin.bias), g)
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def loop(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = step(xs[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)
    threads = [threading.Thread(target=loop, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_second_derivatives_are_refused():
    x, lin, norm = _x(20, 72, torch.float32, spread=0.3).requires_grad_(), _linear(48, 72, torch.float32), _norm(72)
    for f in (lambda: fp8.linear_fp8(x, lin), lambda: fp8.layer_norm_linear_fp8(x, norm, lin), lambda: fused.layer_norm(x, norm)):
        y = f()
        first = torch.autograd.grad(y.sum(), x)[0]
        graph = torch.autograd.grad(f().square().sum(), x, create_graph=True)[0]
        assert graph.shape == first.shape
        with pytest.raises(RuntimeError, match="differentiate twice"):
            graph.sum().backward()


def test_rows_of_blocks_and_one_matrix_on_both_sides():
    """A run of rows of blocks is blocks again; a product of a matrix with itself is symmetric."""
    x = _x(300, 700, torch.float32, spread=0.3)
    a = fp8.quantize_rows(x)
    part = fp8.Fp8Blocks(a.data[37:201], a.scale[37:201], 700)
    for out in (torch.bfloat16, torch.float32):
        y = fp8.matmul_fp8(a, a, out_dtype=out)
        assert torch.equal(y, y.t())
        _check_product(fp8.matmul_fp8(part, a, out_dtype=out), part, a, None, False, out)


def test_autocast_and_inference_mode_change_nothing():
    x, lin = _x(33, 72, torch.float32, spread=0.3), _linear(48, 72, torch.float32)
    with torch.no_grad():
        y = fp8.linear_fp8(x, lin)
        with torch.autocast("cuda", torch.bfloat16):
            z = fp8.linear_fp8(x, lin)
    assert y.dtype == z.dtype == torch.float32 and torch.equal(y, z)
    with torch.inference_mode():
        assert torch.equal(fp8.linear_fp8(x, lin), y)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one():
    x, lin = _x(33, 72, torch.float32, spread=0.3).to("cuda:1").requires_grad_(), _linear(48, 72, torch.float32).to("cuda:1")
    with torch.cuda.device(0):
        fp8.linear_fp8(x, lin).sum().backward()
    assert x.grad.device == x.device and torch.isfinite(x.grad).all()
