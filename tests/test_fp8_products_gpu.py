"""8-bit products where their sums can go wrong, kernel by kernel, against the formula in 64 bits: scales at the ends of their range, a few
large products beside many small ones, sums that cancel."""
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


def _group_largest(a, b):
    """sum over the groups of eight neighbours of a row of the largest |product| of a group: [M, N], 64 bits."""
    pad = -a.shape[1] % 8
    a, b = torch.nn.functional.pad(a.abs(), (0, pad)), torch.nn.functional.pad(b.abs(), (0, pad))
    g = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device=a.device)
    for k in range(0, a.shape[1], 8):
        most = a[:, None, k] * b[None, :, k]
        for j in range(k + 1, k + 8):
            most = torch.maximum(most, a[:, None, j] * b[None, :, j])
        g += most
    return g


def _bound(a, b, y, out_dtype, eight_bit, bias=None):
    """Element by element: half a step of the result; float32 additions, each off by at most 2^-23 of a partial sum (the matrix
    instructions cut off instead of rounding) that is at most S = sum |a b|: K / 8 groups, K / 128 blocks and 64 pieces for the 8-bit
    instructions, K for the others; and what the 8-bit instructions drop, for each of seven products of a group of eight at most 2^-13 of
    the largest."""
    K = a.shape[1]
    half = torch.finfo(out_dtype).eps / 2
    S = a.abs() @ b.abs().t() + (0 if bias is None else bias.double().abs())
    adds = K / 8 + K / 128 + 64 if eight_bit else K + 64
    lost = 7 * 2.0 ** -13 * _group_largest(a, b) if eight_bit else 0
    tiny = 2.0 ** -126 if out_dtype == torch.float32 else torch.finfo(out_dtype).smallest_normal * half
    return half * (y.abs() + adds * 2.0 ** -23 * S + lost) + adds * 2.0 ** -23 * S + lost + tiny


def _check(y, a, b, eight_bit, bias=None, relu=False):
    A, B = R.held(a), R.held(b)
    e = A @ B.t() + (0 if bias is None else bias.double())
    bound = _bound(A, B, e, y.dtype, eight_bit, bias)
    if relu:
        e = e.clamp(min=0)
    off = (y.double() - e).abs()
    assert y.shape == e.shape and (off <= bound).all(), (off / bound).max()


# sizes that reach each of the kernels: few rows, tiles of 64, tiles of 64 and of 128 with the K axis cut, tiles of 128
SHAPES = [(1, 5, 130), (5, 40, 300), (16, 70, 1100), (200, 300, 300), (130, 127, 1100), (128, 130, 4096), (130, 140, 9000), (2100, 2090, 300)]


def _far_blocks(M, N, K, fa, fb, seed):
    """Two matrices whose scales go from 2^-127 to 2^127, block by block in opposite directions, ordinary blocks among them, with zeros
    opposite large elements: the products themselves are of ordinary size."""
    g = _gen(seed)
    blocks = -(-K // 128)
    base = torch.tensor([(-127, 0, 127, -60, 97, 3, -96, 126, -3)[i % 9] for i in range(blocks)])
    out = []
    for rows, dtype, sign in ((M, fa, 1), (N, fb, -1)):
        b = R.random_blocks(rows, K, dtype, "cpu", g)
        d = b.data.float() * (torch.rand(rows, b.data.shape[1], generator=g) < 0.7)
        s = b.scale.view(torch.uint8)
        s[:, :blocks] = (127 + sign * base + torch.randint(-3, 4, (rows, blocks), generator=g)).clamp(0, 254).to(torch.uint8)
        out.append(fp8.Fp8Blocks(d.to(dtype).to(DEV), s.view(torch.float8_e8m0fnu).to(DEV), K))
    return out


@pytest.mark.parametrize("fa,fb", [(E4M3, E4M3), (E5M2, E4M3), (E5M2, E5M2)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_scales_from_end_to_end_of_their_range(M, N, K, out, fa, fb):
    a, b = _far_blocks(M, N, K, fa, fb, M + K)
    bias = torch.randn(N, generator=_gen(1)).to(DEV)
    for bi in (None, bias):
        y = fp8.matmul_fp8(a, b, bi, out_dtype=DT[out])
        _check(y, a, b, out != "f32" and M > 16, bi)          # (up to 16 rows: float32 sums for every type)
        assert torch.equal(y, fp8.matmul_fp8(a, b, bi, out_dtype=DT[out]))


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_one_far_block_changes_its_own_products_only(M, N, K):
    """Ordinary matrices, then one block of one row with another scale: every other row of the result keeps its value to float32
    rounding, whichever way its tile was summed up."""
    g = _gen(K)
    a, b = R.random_blocks(M, K, E4M3, DEV, g), R.random_blocks(N, K, E4M3, DEV, g)
    a.scale.view(torch.uint8)[M - 1, (K - 1) // 128] = 250
    b.data[:, (K - 1) // 128 * 128:] = 0
    _check(fp8.matmul_fp8(a, b, out_dtype=torch.float32), a, b, False)
    a.scale.view(torch.uint8)[M - 1, 0] = 255                                       # (stands for NaN)
    y = fp8.matmul_fp8(a, b, out_dtype=torch.float32)
    assert torch.isnan(y[M - 1]).all() and torch.isfinite(y[:M - 1]).all()


@pytest.mark.parametrize("M,N,K", [(5, 40, 300), (200, 300, 300)])
def test_float32_values_next_to_the_largest_stay_finite(M, N, K):
    """Magnitudes of 3.4e38 are held as 256 x 2^120; opposite zeros and small weights their products are ordinary."""
    x, w = torch.randn(M, K, generator=_gen(1)), torch.randn(N, K, generator=_gen(2)) * 1e-30
    x[:, 130] = 3.4e38
    x[M - 1, 131] = -3.4e38
    w[0, 130] = 0
    a, b = fp8.quantize_rows(x.to(DEV)), fp8.quantize_rows(w.to(DEV))
    y = fp8.matmul_fp8(a, b, out_dtype=torch.float32)
    assert torch.isfinite(y).all()
    _check(y, a, b, False)


@pytest.mark.parametrize("fa", [E4M3, E5M2])
@pytest.mark.parametrize("M,N,K", [(5, 40, 300), (200, 300, 300), (2100, 2090, 300)])
def test_infinities_and_nan_beside_far_scales(M, N, K, fa):
    a, b = _far_blocks(M, N, K, E4M3, E4M3, 3)
    clean = fp8.matmul_fp8(a, b, out_dtype=torch.float32)
    a = fp8.Fp8Blocks(a.data.float().to(fa), a.scale, K)
    d = a.data.float()
    d[1, 3], d[2, 140] = float("nan"), float("inf") if fa == E5M2 else float("nan")
    a = fp8.Fp8Blocks(d.to(fa), a.scale, K)
    y = fp8.matmul_fp8(a, b, out_dtype=torch.float32)
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()
    rest = [i for i in range(M) if i not in (1, 2)]
    assert torch.isfinite(y[rest]).all()
    if fa == E4M3:
        assert torch.equal(y[rest], clean[rest])



@pytest.mark.parametrize("out,full", [("f32", False), ("bf16", False), ("bf16", True)])
@pytest.mark.parametrize("M,N,K", [(5, 40, 300), (200, 300, 300), (2100, 2090, 300)])
def test_a_scale_that_stands_for_nan(M, N, K, out, full):
    """Whatever the elements under it, zeros too; the other rows keep their bits."""
    g = _gen(K)
    for kind in ("zeros", "positive", "random"):
        x, w = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g)
        if kind != "random":
            x, w = x.abs(), w.abs()
        if kind == "zeros":
            x[3] = 0
        a, b = fp8.quantize_rows(x.to(DEV)), fp8.quantize_rows(w.to(DEV))
        clean = fp8.matmul_fp8(a, b, out_dtype=DT[out], **({"full_sums": True} if full else {}))
        a.scale.view(torch.uint8)[3, 1] = 255
        y = fp8.matmul_fp8(a, b, out_dtype=DT[out], **({"full_sums": True} if full else {}))
        assert torch.isnan(y[3]).all()
        assert torch.equal(torch.cat([y[:3], y[4:]]), torch.cat([clean[:3], clean[4:]]))


# ... and those of 16-bit results: tiles of 128, of 256, and the kernel with B in registers
SHAPES16 = SHAPES + [(4097, 4100, 140), (2111, 2048, 300), (16400, 200, 1000)]


def _outliers(rows, K, seed, cancel):
    """In each group of eight one large element and seven whose products lie just under 2^-13 of the large one's; with ``cancel`` the
    large ones come in pairs of opposite signs."""
    g = _gen(seed)
    d = torch.full((rows, -(-K // 128) * 128), 1.75 * 2.0 ** -7) if cancel else torch.full((rows, -(-K // 128) * 128), 2.0 ** -7)
    d[:, ::8] = 1
    if cancel:
        d[:, 8::16] = -1
    else:
        d *= torch.randint(0, 2, d.shape, generator=g) * 2 - 1
    d[:, K:] = 0
    s = torch.full((rows, -(-K // 512) * 4), 127, dtype=torch.uint8)
    s[:, :-(-K // 128)] = torch.randint(124, 130, (rows, 1), generator=g, dtype=torch.uint8)
    return fp8.Fp8Blocks(d.to(E4M3).to(DEV), s.view(torch.float8_e8m0fnu).to(DEV), K)


@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("cancel", [True, False])
@pytest.mark.parametrize("M,N,K", SHAPES16)
def test_large_products_beside_small_ones(M, N, K, cancel, out):
    """Each element within what the 8-bit instructions may drop; with full_sums within float32 sums."""
    a, b = _outliers(M, K, 1, cancel), _outliers(N, K, 2, False)
    if cancel:
        b.data.copy_(b.data.float().abs().to(E4M3))
    y = fp8.matmul_fp8(a, b, out_dtype=DT[out])
    _check(y, a, b, M > 16)
    z = fp8.matmul_fp8(a, b, out_dtype=DT[out], full_sums=True)
    _check(z, a, b, False)
    if cancel and K % 16 == 0:                  # the small ones are all that is left: 7 / 8 of K products of 1.75 * 2^-14
        assert not y.any() and (z > 0).all()


@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", SHAPES16)
def test_random_products_element_by_element(M, N, K, out):
    g = _gen(M + K)
    a, b = R.random_blocks(M, K, E5M2, DEV, g, 3), R.random_blocks(N, K, E4M3, DEV, g, 3)
    if out == "f16":                            # (in its range)
        a.scale.view(torch.uint8)[:, :-(-K // 128)] -= 14
    bias = torch.randn(N, generator=g).to(DEV)
    for full in (False, True):
        _check(fp8.matmul_fp8(a, b, bias, relu=full, out_dtype=DT[out], full_sums=full), a, b, M > 16 and not full, bias, relu=full)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_with_full_sums(dtype):
    """y, dx and dW of outliers whose small neighbours the 8-bit instructions drop; the norm + Linear's are those of its parts."""
    M, N, K = 160, 48, 256
    big = _outliers(M, K, 1, True).data.float().to(dtype).requires_grad_()
    lin, norm = torch.nn.Linear(K, N, device=DEV, dtype=dtype), torch.nn.LayerNorm(K, device=DEV, dtype=dtype)
    with torch.no_grad():
        lin.weight.copy_(_outliers(N, K, 2, False).data.float().abs())
        lin.bias.zero_()
    gm = _outliers(M, N, 3, True).data.float()[:, :N].to(dtype)

    def step(call):
        y = call()
        return (y.detach(), *torch.autograd.grad(y, (big, lin.weight), gm))
    q = lambda t, tile=1: R.rounded(t.detach().cpu(), E4M3, tile).to(DEV)
    w8 = q(lin.weight, 128)
    for got, A, B in zip(step(lambda: fp8.linear_fp8(big, lin, full_sums=True)), (q(big), q(gm), q(gm.t())), (w8, w8.t(), q(big.t()))):
        e = A @ B.t()
        assert ((got.double() - e).abs() <= _bound(A, B, e, dtype, False)).all()
    y = fp8.linear_fp8(big, lin).detach()
    full = fp8.linear_fp8(big, lin, full_sums=True).detach()
    assert not y.any() and (full > 0).all()
    with torch.no_grad():
        assert torch.equal(full, fp8.linear_fp8(big, lin, full_sums=True))
    z = fused.layer_norm(big, norm)
    a = fp8.layer_norm_linear_fp8(big, norm, lin, full_sums=True)
    blocks, wt = fp8.quantize_rows(torch.nn.functional.layer_norm(big.detach().float(), (K,))), fp8.quantize_tiles(lin.weight.detach())[0]
    e = R.held(blocks) @ R.held(wt).t()
    # (the norm's own rounding may move an element to the next value of its type: 2^-3 of it)
    S = R.held(blocks).abs() @ R.held(wt).abs().t()
    assert ((a.double() - e).abs() <= torch.finfo(dtype).eps / 2 * e.abs() + 2.0 ** -3 * S).all()
    dz = torch.autograd.grad(fp8.linear_fp8(z, lin, full_sums=True), z, gm)[0]
    want = torch.autograd.grad(fused.layer_norm(big, norm), (big, norm.weight, norm.bias), dz)
    for p, w in zip(torch.autograd.grad(a, (big, norm.weight, norm.bias), gm), want):
        assert torch.equal(p, w)


# ---- the kernel with B in registers: K up to 1024 on many rows, N a multiple of 8 ------------------------------------------------------
def _check_many(y, a, b, bias, relu):
    """As ``_check`` with what a group drops taken relative to all of its products, for results of many elements."""
    A, B = R.held(a), R.held(b)
    e = A @ B.t() + (0 if bias is None else bias.double())
    S = A.abs() @ B.abs().t() + (0 if bias is None else bias.double().abs())
    half, K = torch.finfo(y.dtype).eps / 2, A.shape[1]
    lost = (7 * 2.0 ** -13 + (K / 8 + K / 128 + 64) * 2.0 ** -23) * S
    bound = half * (e.abs() + lost) + lost + torch.finfo(y.dtype).smallest_normal * half
    if relu:
        e = e.clamp(min=0)
    off = (y.double() - e).abs()
    assert (off <= bound).all(), (off / bound).max()
    # and, random as the elements are, near that in the norm: half a step (sqrt 3 below its largest on average), 1e-4 for what is dropped
    assert off.norm() <= (half / 3 ** 0.5 * 1.1 + 1e-4) * S.norm()


@pytest.mark.parametrize("short", [0, 60])
@pytest.mark.parametrize("steps", range(1, 9))
def test_many_rows_with_short_k(steps, short):
    """Each number of K steps (a ring of 4, 3 or 2 slots), each pair of types, more chunks of 64 rows than twice the ring, ragged rows and
    columns that end inside a wave's 32."""
    K, M, N = 128 * steps - short, 40007, 1000
    bias = torch.randn(N, generator=_gen(1)).to(DEV)
    for i, (fa, fb) in enumerate([(E4M3, E4M3), (E5M2, E4M3), (E4M3, E5M2), (E5M2, E5M2)]):
        g = torch.Generator(device=DEV).manual_seed(K + i)
        x = torch.randn(M, K, generator=g, device=DEV) * torch.exp(torch.randn(M, 1, generator=g, device=DEV))
        w = torch.randn(N, K, generator=g, device=DEV) / K ** 0.5
        a, b = fp8.quantize_rows(x, fa), fp8.quantize_rows(w, fb)
        for out, bi, relu in ((torch.bfloat16, bias, i % 2 == 0), (torch.float16, None if i % 2 else bias.to(torch.bfloat16), i % 2 == 1)):
            y = fp8.matmul_fp8(a, b, bi, relu=relu, out_dtype=out)
            _check_many(y, a, b, bi, relu)
            assert torch.equal(y, fp8.matmul_fp8(a, b, bi, relu=relu, out_dtype=out))
            tail = fp8.Fp8Blocks(a.data[-300:], a.scale[-300:], K)
            assert torch.equal(y[:, :8], fp8.matmul_fp8(a, fp8.Fp8Blocks(b.data[:8], b.scale[:8], K), None if bi is None else bi[:8], relu=relu, out_dtype=out))
            _check_many(fp8.matmul_fp8(tail, b, bi, relu=relu, out_dtype=out), tail, b, bi, relu)


@pytest.mark.parametrize("M,N,K", [(4100, 4104, 140), (16400, 264, 1000), (20000, 8, 70), (4164, 4104, 400)])
def test_poisoned_rows_with_b_in_registers(M, N, K):
    x, w = torch.randn(M, K, generator=_gen(1)).to(DEV), torch.randn(N, K, generator=_gen(2)).to(DEV)
    clean = fp8.matmul_fp8(fp8.quantize_rows(x, E5M2), fp8.quantize_rows(w))
    x[1, 7], x[2, K - 1], w[3, 5] = float("nan"), float("inf"), float("nan")
    x[M - 1, 0] = float("nan")
    a, b = fp8.quantize_rows(x, E5M2), fp8.quantize_rows(w)
    a.scale.view(torch.uint8)[3, 0] = 255
    b.scale.view(torch.uint8)[N - 2, 0] = 255
    y = fp8.matmul_fp8(a, b)
    assert all(torch.isnan(y[i]).all() for i in (1, 3, M - 1)) and all(torch.isnan(y[:, j]).all() for j in (3, N - 2))
    assert not torch.isfinite(y[2]).any()
    rows, cols = [i for i in range(M) if i not in (1, 2, 3, M - 1)], [j for j in range(N) if j not in (3, N - 2)]
    assert torch.equal(y[rows][:, cols], clean[rows][:, cols])
    r = fp8.matmul_fp8(a, b, relu=True)
    assert torch.isnan(r[1]).all() and torch.isnan(r[:, 3]).all()
    rest = y[rows][:, cols]
    assert torch.equal(r[rows][:, cols], rest.clamp(min=0))


@pytest.mark.parametrize("kind,grad", [("bf16", E5M2), ("f16", E4M3)])
def test_linear_of_many_rows(kind, grad):
    """y and dx from the kernel with B in registers, the gradient in either type, dW over many pieces of a long K axis."""
    M, N, K = 20011, 136, 264
    x = (torch.randn(M, K, generator=_gen(1)) * torch.exp(0.5 * torch.randn(M, 1, generator=_gen(2)))).to(DT[kind]).to(DEV).requires_grad_()
    lin = torch.nn.Linear(K, N, device=DEV)
    g = (torch.randn(M, N, generator=_gen(3)) * 0.1).to(DT[kind]).to(DEV)
    y = fp8.linear_fp8(x, lin, grad_dtype=grad)
    dx, dw, db = torch.autograd.grad(y, (x, lin.weight, lin.bias), g)
    xq, gq = fp8.quantize_both(x.detach()), fp8.quantize_both(g, grad)
    w, wt = fp8.quantize_tiles(lin.weight.detach())
    _check_many(y.detach(), xq[0], w, lin.bias.detach(), False)
    _check_many(dx, gq[0], wt, None, False)
    _check(dw, gq[1], xq[1], False)
    # the longest chain of additions of a sum over rows: 32 rows of a lane and wave, then 157 tiles in 32 slices
    assert ((db.double() - g.double().sum(0)).abs() <= 128 * 2.0 ** -24 * g.double().abs().sum(0)).all()


@pytest.mark.parametrize("M,N,K", [(700, 8192, 140), (700, 8200, 140), (2111, 2816, 1000), (8003, 520, 300), (8003, 544, 300)])
def test_wide_results_of_short_k(M, N, K):
    """On both sides of the number of columns up to which B stays in registers, and rows that are and are not whole pieces of 64 bytes."""
    g = torch.Generator(device=DEV).manual_seed(N)
    a, b = (fp8.quantize_rows(torch.randn(r, K, generator=g, device=DEV)) for r in (M, N))
    bias = torch.randn(N, generator=g, device=DEV)
    _check_many(fp8.matmul_fp8(a, b, bias), a, b, bias, False)
