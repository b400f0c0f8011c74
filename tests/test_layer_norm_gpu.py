"""``fused.layer_norm`` (rows of any width) against the formulas in 64 bits."""
import pytest
import torch

from snipper_amd import fused

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda:0"
U = 2.0 ** -24


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _norm(c, dtype, affine=True, bias=True):
    n = torch.nn.LayerNorm(c, elementwise_affine=affine, bias=bias)
    if affine:
        with torch.no_grad():
            n.weight.copy_(1 + 0.3 * torch.randn(c, generator=_gen(1)))
            if bias:
                n.bias.copy_(0.3 * torch.randn(c, generator=_gen(2)))
    return n.to(DEV, dtype)


def _formulas(x, g, norm):
    """y, dx, dgamma, dbeta in 64 bits, and for each the sum of magnitudes that float32 rounding is relative to."""
    x, g = x.detach().double(), g.double()
    w = norm.weight.detach().double() if norm.weight is not None else torch.ones(x.shape[1], device=DEV, dtype=torch.float64)
    b = norm.bias.detach().double() if norm.bias is not None else torch.zeros(x.shape[1], device=DEV, dtype=torch.float64)
    m = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + norm.eps)
    h = (x - m) * r
    t = g * w
    dx = r * (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True))
    # h's own magnitude: x and the mean are subtracted after rounding of the mean, relative to the mean magnitude of the row
    hm = (x.abs() + x.abs().mean(1, keepdim=True)) * r + h.abs()
    parts = (hm * w.abs() + b.abs(),
             r * (t.abs() + t.abs().mean(1, keepdim=True) + hm * (t.abs() * hm).mean(1, keepdim=True)),
             (g.abs() * hm).sum(0), g.abs().sum(0))
    return (h * w + b, dx, (g * h).sum(0), g.sum(0)), parts


def _check(got, want, parts, depth=64):
    """Half a step of the type, and `depth` float32 roundings (the longest chain of additions) of the parts."""
    for a, e, p in zip(got, want, parts):
        if a is None:
            continue
        half = torch.finfo(a.dtype).eps / 2
        tiny = torch.finfo(a.dtype).smallest_normal * half
        off = (a.double() - e).abs()
        bound = half * e.abs() + depth * U * p + tiny
        assert (off <= bound).all(), (off / bound).max()


def _run(x, g, norm):
    leaves = [t for t in (x, norm.weight, norm.bias) if t is not None]
    y = fused.layer_norm(x, norm)
    grads = list(torch.autograd.grad(y, leaves, g))
    return [y.detach(), grads[0]] + [grads[1] if norm.weight is not None else None, grads[2] if norm.bias is not None else None]


WIDTHS = [1, 2, 7, 127, 128, 129, 256, 257, 383, 384, 385, 511, 512, 513, 1024, 1027, 2048, 2050, 4096, 4099, 8192, 8200, 16383, 16384]


@pytest.mark.parametrize("kind,param", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("cols", WIDTHS)
def test_against_the_formulas(cols, kind, param):
    rows = 37
    x = (torch.randn(rows, cols, generator=_gen(cols)) * 2 + torch.randn(rows, 1, generator=_gen(3))).to(DT[kind]).to(DEV).requires_grad_()
    g = torch.randn(rows, cols, generator=_gen(4)).to(DT[kind]).to(DEV)
    norm = _norm(cols, DT[param])
    got = _run(x, g, norm)
    assert [t.dtype for t in got] == [DT[kind]] * 2 + [DT[param]] * 2
    _check(got, *_formulas(x, g, norm))


@pytest.mark.parametrize("rows", [1, 3, 16, 1000, 20011])
@pytest.mark.parametrize("cols", [60, 384, 1500, 5000])
def test_rows(rows, cols):
    if rows * cols > 3e7:
        rows = 4001
    x = torch.randn(rows, cols, generator=_gen(1)).to(DEV).requires_grad_()
    g = torch.randn(rows, cols, generator=_gen(2)).to(DEV)
    norm = _norm(cols, torch.float32)
    # the longest chain for dgamma: the rows of one lane, then the partial rows of a slice, then the slices
    _check(_run(x, g, norm), *_formulas(x, g, norm), depth=64 + rows // 256 + 32 + 40)


@pytest.mark.parametrize("skip,at", [(1, 0), (5, 1), (16, 8)])
def test_rows_of_a_wider_buffer(skip, at):
    for kind in DT:
        buf = torch.randn(50, 301 + skip + at, generator=_gen(1)).to(DT[kind]).to(DEV)
        x = buf[:, at:at + 301].requires_grad_()
        g = torch.randn(50, 301, generator=_gen(2)).to(DT[kind]).to(DEV)
        norm = _norm(301, torch.float32)
        a = _run(x, g, norm)
        b = _run(x.detach().contiguous().requires_grad_(), g, norm)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        t = buf.t().requires_grad_()                                # (columns as rows: copied)
        gt = torch.randn(t.shape, generator=_gen(2)).to(DT[kind]).to(DEV)
        nt = _norm(50, torch.float32)
        _check(_run(t, gt, nt), *_formulas(t, gt, nt))


def test_leading_axes_no_rows_and_broadcast():
    norm = _norm(96, torch.float32)
    x = torch.randn(2, 3, 4, 96, generator=_gen(1)).to(DEV).requires_grad_()
    y = fused.layer_norm(x, norm)
    assert y.shape == x.shape and torch.equal(y.view(24, 96), fused.layer_norm(x.view(24, 96), norm))
    v = torch.randn(96, generator=_gen(1)).to(DEV)
    assert torch.equal(fused.layer_norm(v, norm), fused.layer_norm(v[None], norm)[0])
    e = torch.empty(0, 96, device=DEV, requires_grad=True)
    dx, dw, db = torch.autograd.grad(fused.layer_norm(e, norm).sum(), (e, norm.weight, norm.bias))
    assert dx.shape == (0, 96) and not dw.any() and not db.any()
    row = torch.randn(1, 96, generator=_gen(5)).to(DEV).requires_grad_()
    g = torch.randn(7, 96, generator=_gen(6)).to(DEV)
    one = row.detach().expand(7, 96).contiguous().requires_grad_()
    a = torch.autograd.grad(fused.layer_norm(row.expand(7, 96), norm), row, g)[0]
    b = torch.autograd.grad(fused.layer_norm(one, norm), one, g)[0].sum(0, keepdim=True)
    assert torch.equal(a, b)


@pytest.mark.parametrize("affine,bias", [(False, False), (True, False)])
def test_without_parameters(affine, bias):
    norm = _norm(200, torch.float32, affine, bias)
    x = torch.randn(30, 200, generator=_gen(1)).to(DEV).requires_grad_()
    g = torch.randn(30, 200, generator=_gen(2)).to(DEV)
    _check(_run(x, g, norm), *_formulas(x, g, norm))


@pytest.mark.parametrize("want", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)])
def test_gradients_that_are_asked_for(want):
    x, norm = torch.randn(50, 300, generator=_gen(1)).to(DEV).requires_grad_(), _norm(300, torch.float32)
    g = torch.randn(50, 300, generator=_gen(2)).to(DEV)
    full = _run(x, g, norm)[1:]
    leaves = [x, norm.weight, norm.bias]
    for t, w in zip(leaves, want):
        t.requires_grad_(bool(w))
    got = torch.autograd.grad(fused.layer_norm(x, norm), [t for t, w in zip(leaves, want) if w], g)
    assert all(torch.equal(a, b) for a, b in zip(got, [f for f, w in zip(full, want) if w]))


@pytest.mark.parametrize("cols", [100, 384, 1100, 3001, 9000])
def test_rows_that_are_constant_far_off_or_poisoned(cols):
    x = torch.randn(12, cols, generator=_gen(1))
    x[0], x[1], x[2] = 0.0, 3.25, 1e4 + x[2]
    x[3, cols // 2], x[4, 0] = float("nan"), float("inf")
    x[5] *= 1e-20
    x = x.to(DEV).requires_grad_()
    g = torch.randn(12, cols, generator=_gen(2)).to(DEV)
    norm = _norm(cols, torch.float32)
    y, dx, dw, db = _run(x, g, norm)
    ok = [0, 1, 2, 5, 6, 7, 8, 9, 10, 11]
    sub = x.detach()[ok].requires_grad_()
    (ey, edx, _, edb), (py, pdx, _, pdb) = _formulas(sub, g[ok], norm)
    _check((y[ok], dx[ok]), (ey, edx), (py, pdx))
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).all() and torch.isnan(dx[3]).all() and torch.isnan(dx[4]).all()
    assert torch.isnan(dw).all()
    assert ((db.double() - g.double().sum(0)).abs() <= 64 * U * g.double().abs().sum(0)).all()


def test_against_differences():
    """dx, dgamma and dbeta along a direction against differences of the kernel's own forward pass."""
    cols = 211
    x, norm = torch.randn(40, cols, generator=_gen(1)).to(DEV).requires_grad_(), _norm(cols, torch.float32)
    g = torch.randn(40, cols, generator=_gen(2)).to(DEV)
    _, dx, dw, db = _run(x, g, norm)

    def loss(xx, w, b):
        n = _norm(cols, torch.float32)
        with torch.no_grad():
            n.weight.copy_(w), n.bias.copy_(b)
            return (fused.layer_norm(xx, n).double() * g.double()).sum()
    at = (x.detach(), norm.weight.detach(), norm.bias.detach())
    for i, grad in enumerate((dx, dw, db)):
        u = torch.randn(at[i].shape, generator=_gen(5 + i)).to(DEV)
        h = 1e-2
        move = lambda s: loss(*[t + s * h * u if j == i else t for j, t in enumerate(at)])
        want, got = (move(1) - move(-1)) / (2 * h), (grad.double() * u.double()).sum()
        scale = (grad.double().abs() * u.double().abs()).sum()
        # h^2 / 6 of a third derivative of the order of the first, and float32 roundings of 8440 terms over 2 h
        assert (want - got).abs() <= 2 * h * h * scale + 8440 ** 0.5 * 2 ** -22 / h * g.abs().max().double()


@pytest.mark.parametrize("cols", [300, 600])
def test_rows_beyond_32_bit_offsets(cols):
    """Two and a half (five) GB in bfloat16: the last rows' results are those of the same rows alone."""
    rows, last = (1 << 22) + 77, 77
    x = torch.randn(rows, cols, device=DEV, dtype=torch.bfloat16)
    g = torch.zeros(rows, cols, device=DEV, dtype=torch.bfloat16)
    g[-last:] = torch.randn(last, cols, device=DEV, dtype=torch.bfloat16)
    norm = torch.nn.LayerNorm(cols, device=DEV)

    def both(x, g):
        x = x.clone().requires_grad_()
        y = fused.layer_norm(x, norm)
        return (y.detach(), *torch.autograd.grad(y, (x, norm.weight, norm.bias), g))
    y, dx, dw, db = both(x, g)
    ys, dxs, dws, dbs = both(x[-last:], g[-last:])
    assert torch.equal(y[-last:], ys) and torch.equal(dx[-last:], dxs) and not dx[:-last].any()
    # the same 77 summands (and zeros) in another order: each of fewer than 77 additions is off by half a step of a sum
    h = torch.nn.functional.layer_norm(x[-last:].float(), (cols,))
    for a, b, S in ((dw, dws, (g[-last:].float() * h).abs().sum(0)), (db, dbs, g[-last:].float().abs().sum(0))):
        assert ((a - b).abs() <= 2 * 77 * 2.0 ** -24 * 1.01 * S).all()


def test_same_result_every_time_and_in_graphs():
    x, norm = torch.randn(3000, 384, generator=_gen(1)).to(DEV).requires_grad_(), _norm(384, torch.float32)
    g = torch.randn(3000, 384, generator=_gen(2)).to(DEV)
    first = _run(x, g, norm)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _run(x, g, norm)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(x, g, norm)
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(3000, 384, generator=_gen(20 + k)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, _run(x, g, norm)))


def test_refusals():
    x = torch.randn(4, 64, device=DEV)
    for bad, err in ((torch.nn.LayerNorm(63, device=DEV), ValueError), (torch.nn.LayerNorm((4, 64), device=DEV), ValueError),
                     (torch.nn.LayerNorm(64), TypeError), (torch.nn.LayerNorm(64, device=DEV, dtype=torch.float64), TypeError)):
        with pytest.raises(err):
            fused.layer_norm(x, bad)
    with pytest.raises(TypeError):
        fused.layer_norm(x.double(), torch.nn.LayerNorm(64, device=DEV))
    with pytest.raises(ValueError):
        fused.layer_norm(torch.randn(2, 16385, device=DEV), torch.nn.LayerNorm(16385, device=DEV))
