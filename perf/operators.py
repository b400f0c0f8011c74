"""The 8-bit operators and the layer norm of wide rows, as programs call them: inputs, one pass, and what a pass has to move.

Four operators, each in two forms.  ``own`` false: the plain form, elementary torch operations in 32 bits.  ``own`` true: the
calls of ``snipper_amd.fp8`` and ``snipper_amd.fused``.

    matmul       relu(A B^T + bias) of two matrices held in 8 bits with a power-of-two scale for each 128 elements of a row
    linear       a training step of nn.Linear in that format: y, dx, dW, db
    norm         a layer norm of rows of any width, forward and backward: y, dx, dgamma, dbeta
    norm_linear  a layer norm whose result goes straight into an 8-bit product: forward, or a whole training step

The 8-bit format.  A row is cut into blocks of 128 elements (weights of a Linear: tiles of 128 x 128).  A block's scale is 2^e with
the smallest e >= -127 for which the largest finite magnitude of the block over 2^e is not above the type's largest value (448 for
e4m3, 57344 for e5m2); a block of zeros has e = 0.  Elements are x / 2^e, rounded to the nearest value of the type, ties to even.
A matrix is kept as ``data`` [rows, pitch], pitch the columns rounded up to 128 (zeros behind the last column), and ``scale``
[rows, 4 * ceil(columns / 512)] in e8m0 (2^0 behind the last block).
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_MOST = {"e4m3": 448.0, "e5m2": 57344.0}
_EPS = 1e-5


def listed():
    return [
        # one row through a square projection held in 8 bits: the weight's bytes count
        dict(name="matmul one row 4096", op="matmul", m=1, n=4096, k=4096, a="e4m3", b="e4m3", out="bf16", bias=False, relu=False),
        # the object queries of two 4-frame snippets (2 x 4 x 60 rows) into the feed-forward block: latency counts
        dict(name="matmul queries 480x1024x384", op="matmul", m=480, n=1024, k=384, a="e4m3", b="e4m3", out="bf16", bias=True, relu=True),
        # the encoder's feed-forward block at 600 x 800: 8 frames of 9875 positions
        dict(name="matmul tokens 79000x1024x384", op="matmul", m=79000, n=1024, k=384, a="e4m3", b="e4m3", out="bf16", bias=True, relu=True),
        # a product that the matrix pipe bounds
        dict(name="matmul square 8192", op="matmul", m=8192, n=8192, k=8192, a="e4m3", b="e4m3", out="bf16", bias=False, relu=False),
        # no size a multiple of anything, gradients in e5m2, a result that is summed up further in 32 bits
        dict(name="matmul ragged 1999x777x1001", op="matmul", m=1999, n=777, k=1001, a="e5m2", b="e4m3", out="f32", bias=True, relu=False),
        # training: the encoder's linear1 with float32 master weights
        dict(name="linear tokens 79000x1024x384", op="linear", m=79000, n=1024, k=384, x="bf16", param="f32", grad="e4m3"),
        # training: odd rows, odd widths, float32 activations, gradients in e5m2
        dict(name="linear ragged 4999x333x650", op="linear", m=4999, n=333, k=650, x="f32", param="f32", grad="e5m2"),
        # training: the encoder's residual stream, float32
        dict(name="norm tokens 79000x384", op="norm", rows=79000, cols=384, x="f32", param="f32", skip=0),
        # training: wide rows
        dict(name="norm wide 16384x8192", op="norm", rows=16384, cols=8192, x="bf16", param="f32", skip=0),
        # a few rows of an odd width, taken out of a wider buffer
        dict(name="norm odd 61x1027", op="norm", rows=61, cols=1027, x="f16", param="f16", skip=5),
        # one token at inference: norm, then a projection whose weight was laid out once
        dict(name="norm_linear one row 4096", op="norm_linear", m=1, n=4096, k=4096, x="bf16", train=False),
        # training: norm and the first Linear of a feed-forward block, weights in bf16
        dict(name="norm_linear 8192x4096x1024", op="norm_linear", m=8192, n=4096, k=1024, x="bf16", train=True),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["matmul", "linear", "norm", "norm_linear"])
    if op == "norm":
        cols = _log(rng, 1, 16384)
        c = dict(op=op, rows=_log(rng, 1, max(1, min(131072, (1 << 27) // cols))), cols=cols, x=rng.choice(["f32", "bf16", "f16"]))
        return dict(c, param=rng.choice(["f32", c["x"]]), skip=rng.choice([0, 0, 3, 16]))
    if op == "matmul":
        n, k = _log(rng, 1, 8192), _log(rng, 1, 8192)
        return dict(op=op, m=_log(rng, 1, min(79000, (1 << 38) // (n * k))), n=n, k=k, a=rng.choice(["e4m3", "e5m2"]),
                    b=rng.choice(["e4m3", "e4m3", "e5m2"]), out=rng.choice(["bf16", "f16", "f32"]), bias=rng.random() < 0.5, relu=rng.random() < 0.5)
    n, k = _log(rng, 16, 4096), _log(rng, 16, 4096)
    m = _log(rng, 1, min(79000, (1 << 34) // (n * k)))
    if op == "linear":
        x = rng.choice(["f32", "bf16", "f16"])
        return dict(op=op, m=m, n=n, k=k, x=x, param=rng.choice(["f32", x]), grad=rng.choice(["e4m3", "e5m2"]))
    return dict(op=op, m=m, n=n, k=k, x=rng.choice(["bf16", "f16"]), train=rng.random() < 0.5)


# ---- the format, in 32 bits ------------------------------------------------------------------------------------------
def _exponents(most, kind):
    """e of the smallest 2^e >= most / largest, with the largest value of the type 0.875 * 2^9 or 0.875 * 2^16."""
    m, x = torch.frexp(most)
    e = torch.where(m <= 0.875, x - (9 if kind == "e4m3" else 16), x - (8 if kind == "e4m3" else 15))
    return torch.where(most == 0, torch.zeros_like(e), e.clamp(min=-127))


def _pow2(e):
    """2^e for whole -127 <= e <= 127, put together from its bits: exact on every device."""
    e = e.to(torch.int32)
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _pad(x, rows, cols):
    r, c = -x.shape[0] % rows, -x.shape[1] % cols
    return torch.nn.functional.pad(x, (0, c, 0, r)) if r or c else x


def _quantize(x, kind, rows=1):
    """Blocks of `rows` x 128: (data [R, pitch] 8-bit, exponents [R, blocks] int32) with R the rows rounded up to `rows`."""
    x = _pad(x.float(), rows, 128)
    R, P = x.shape
    b = x.view(R // rows, rows, P // 128, 128)
    most = torch.where(torch.isfinite(b), b.abs(), torch.zeros_like(b)).amax(dim=(1, 3))
    e = _exponents(most, kind)
    d = (b * _pow2(-e)[:, None, :, None]).to(_DT[kind]).view(R, P)
    return d, e.repeat_interleave(rows, 0)


def _values(d, e, cols):
    """The matrix that (data, exponents) stand for, float32."""
    R, P = d.shape
    return (d.float().view(R, P // 128, 128) * _pow2(e)[:, :, None]).reshape(R, P)[:, :cols]


def _rounded(x, kind, rows=1):
    """x, rounded to the format."""
    d, e = _quantize(x, kind, rows)
    return _values(d, e, x.shape[1])[:x.shape[0]]


def _held(x, kind, rows=1):
    """(data, scale) as programs keep them."""
    R, blocks = x.shape[0], -(-x.shape[1] // 128)
    d, e = _quantize(x, kind, rows)
    s = torch.full((R, -(-blocks // 4) * 4), 127, dtype=torch.uint8, device=x.device)
    s[:, :blocks] = (e[:R] + 127).to(torch.uint8)
    return d[:R].contiguous(), s.view(torch.float8_e8m0fnu)


def _taken(d, s, cols):
    """The matrix that (data, scale) stand for, float32."""
    e = s.view(torch.uint8)[:, :d.shape[1] // 128].int() - 127
    return _values(d, e, cols)


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _activations(g, m, k, dtype):
    """Tokens: a few channels much larger than the others, rows of different size, every 16th row behind a padding mask."""
    x = torch.randn(m, k, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(m, 1, generator=g, device="cuda"))
    x = x * torch.exp(torch.randn(k, generator=g, device="cuda"))
    if m >= 16:
        x[torch.randint(0, m, (m // 16,), generator=g, device="cuda")] = 0
    return x.to(dtype)


def _module(kind, dtype, *sizes, weight, bias):
    mod = kind(*sizes, device="meta")
    mod.weight = torch.nn.Parameter(weight.to(dtype))
    mod.bias = torch.nn.Parameter(bias.to(dtype))
    return mod


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    op, s = case["op"], dict(case=case)
    if op == "norm":
        R, C, dt, pt = case["rows"], case["cols"], _DT[case["x"]], _DT[case["param"]]
        x = (randn(R, C + case["skip"]) * torch.exp(0.5 * randn(R, 1)) + randn(R, 1)).to(dt)
        s["x"] = x[:, :C].requires_grad_()
        s["g"] = (randn(R, C) * 1e-2).to(dt)
        s["norm"] = _module(torch.nn.LayerNorm, pt, C, weight=1 + 0.2 * randn(C), bias=0.2 * randn(C))
        return s
    m, n, k = case["m"], case["n"], case["k"]
    w, b = randn(n, k) / math.sqrt(k), 0.1 * randn(n)
    if op == "matmul":
        s["a"] = _held(_activations(g, m, k, torch.float32), case["a"])
        s["b"] = _held(w, case["b"], rows=128)
        s["bias"] = b if case["bias"] else None
        return s
    dt = _DT[case["x"]]
    pt = _DT[case["param"]] if op == "linear" else dt
    s["x"] = _activations(g, m, k, dt)
    s["lin"] = _module(torch.nn.Linear, pt, k, n, weight=w, bias=b)
    if op == "norm_linear":
        s["norm"] = _module(torch.nn.LayerNorm, pt, k, weight=1 + 0.2 * randn(k), bias=0.2 * randn(k))
        if not case["train"]:
            s["w"] = _held(s["lin"].weight.detach(), "e4m3", rows=128)
            return s
    s["x"].requires_grad_()
    s["g"] = (randn(m, n) * torch.exp(randn(m, 1)) * 1e-4).to(dt) if dt != torch.float16 else (randn(m, n) * 1e-2).to(dt)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


def _run_own(s):
    from snipper_amd import fp8, fused
    c = s["case"]
    op = c["op"]
    if op == "matmul":
        a, b = fp8.Fp8Blocks(*s["a"], c["k"]), fp8.Fp8Blocks(*s["b"], c["k"])
        return fp8.matmul_fp8(a, b, s["bias"], relu=c["relu"], out_dtype=_DT[c["out"]])
    if op == "norm":
        norm = s["norm"]
        y = fused.layer_norm(s["x"], norm)
        return (y.detach(),) + torch.autograd.grad(y, (s["x"], norm.weight, norm.bias), s["g"])
    lin = s["lin"]
    if op == "linear":
        y = fp8.linear_fp8(s["x"], lin, grad_dtype=_DT[c["grad"]])
        return (y.detach(),) + torch.autograd.grad(y, (s["x"], lin.weight, lin.bias), s["g"])
    norm = s["norm"]
    if not c["train"]:
        with torch.no_grad():
            return fp8.matmul_fp8(fp8.layer_norm_fp8(s["x"], norm), fp8.Fp8Blocks(*s["w"], c["k"]), lin.bias, out_dtype=s["x"].dtype)
    y = fp8.layer_norm_linear_fp8(s["x"], norm, lin)
    return (y.detach(),) + torch.autograd.grad(y, (s["x"], norm.weight, norm.bias, lin.weight, lin.bias), s["g"])


def _norm_plain(x, w, b):
    """y, the normalised rows and 1 / deviation, in 32 bits."""
    x = x.float()
    d = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((d * d).mean(1, keepdim=True) + _EPS)
    h = d * r
    return h * w.float() + b.float(), h, r


def _norm_back_plain(g, h, r, w):
    """dx, dgamma, dbeta, in 32 bits."""
    g = g.float()
    t = g * w.float()
    return (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True)) * r, (g * h).sum(0), g.sum(0)


def _linear_plain(x, lin, out):
    """y and what the backward pass takes: the rounded weight."""
    w8 = _rounded(lin.weight, "e4m3", rows=128)
    return (_rounded(x, "e4m3") @ w8.t() + lin.bias.float()).to(out), w8


def _linear_back_plain(g, x, w8, kind):
    """dx, dW, db of y = x W^T + b, in 32 bits; x and g are rounded along the axis that each product sums over."""
    g = g.float()
    dw = _rounded(g.t(), kind) @ _rounded(x.t(), "e4m3").t()
    return _rounded(g, kind) @ w8, dw, g.sum(0)


def _run_plain(s):
    c = s["case"]
    op = c["op"]
    if op == "matmul":
        y = _taken(*s["a"], c["k"]) @ _taken(*s["b"], c["k"]).t()
        if s["bias"] is not None:
            y = y + s["bias"]
        return (torch.relu(y) if c["relu"] else y).to(_DT[c["out"]])
    x = s["x"].detach()
    dt = x.dtype
    if op == "norm":
        w, b = s["norm"].weight, s["norm"].bias
        y, h, r = _norm_plain(x, w, b)
        dx, dw, db = _norm_back_plain(s["g"], h, r, w)
        return y.to(dt), dx.to(dt), dw.to(w.dtype), db.to(w.dtype)
    lin = s["lin"]
    pt = lin.weight.dtype
    if op == "linear":
        y, w8 = _linear_plain(x, lin, dt)
        dx, dw, db = _linear_back_plain(s["g"], x, w8, c["grad"])
        return y, dx.to(dt), dw.to(pt), db.to(pt)
    w, b = s["norm"].weight, s["norm"].bias
    z, h, r = _norm_plain(x, w, b)
    if not c["train"]:
        return (_rounded(z, "e4m3") @ _taken(*s["w"], c["k"]).t() + lin.bias.float()).to(dt)
    y, w8 = _linear_plain(z, lin, dt)
    dz, dw, db = _linear_back_plain(s["g"], z, w8, "e4m3")
    dx, dgamma, dbeta = _norm_back_plain(dz.to(dt), h, r, w)     # (the gradient between the two layers has the activations' type)
    return y, dx.to(dt), dgamma.to(pt), dbeta.to(pt), dw.to(pt), db.to(pt)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
_SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "e5m2": 1}


def work(case):
    op = case["op"]
    if op == "norm":
        n, e, p = case["rows"] * case["cols"], _SIZE[case["x"]], _SIZE[case["param"]]
        return {"bytes": 4 * n * e + 4 * case["cols"] * p, "flops": 16 * n}       # x, g, y, dx; gamma, beta and their gradients
    m, n, k = case["m"], case["n"], case["k"]
    blocks = -(-k // 128)
    if op == "matmul":
        return {"bytes": (m + n) * (k + blocks) + m * n * _SIZE[case["out"]] + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    e = _SIZE[case["x"]]
    p = _SIZE[case["param"]] if op == "linear" else e
    if op == "norm_linear" and not case["train"]:
        return {"bytes": (m * k + m * n) * e + n * (k + blocks) + (2 * k + n) * p, "flops": 2 * m * n * k + 8 * m * k}
    nbytes = 2 * (m * k + m * n) * e + 2 * (n * k + n) * p                        # x, dx, y, g; W, b and their gradients
    return {"bytes": nbytes + (4 * k * p if op == "norm_linear" else 0), "flops": 6 * m * n * k + (16 * m * k if op == "norm_linear" else 0)}


# ---- the definition, in 64 bits --------------------------------------------------------------------------------------
def _exact_pow2(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_blocks(x, kind, rows=1):
    """x rounded to the format, from its definition alone: the scale by logarithm, each element by its own step."""
    x = x.detach().double()
    R, C = x.shape
    x = _pad(x, rows, 128)
    b = x.view(x.shape[0] // rows, rows, -1, 128)
    most = b.abs().nan_to_num(0, 0, 0).amax(dim=(1, 3), keepdim=True)
    q = most / _MOST[kind]
    e = torch.floor(torch.log2(torch.where(q > 0, q, torch.ones_like(q))))
    e = torch.where(_exact_pow2(e) < q, e + 1, e)                  # the smallest power of two that is not below q
    e = torch.where(_exact_pow2(e - 1) >= q, e - 1, e)
    e = torch.where(most > 0, e.clamp(min=-127), torch.zeros_like(e))
    v = b * _exact_pow2(-e)
    bits, low = (3, -6) if kind == "e4m3" else (2, -14)
    m = torch.where(v.abs() > 0, v.abs(), torch.ones_like(v))
    f = torch.floor(torch.log2(m))
    f = torch.where(_exact_pow2(f) > m, f - 1, f)
    step = _exact_pow2(f.clamp(min=low) - bits)
    return (torch.round(v / step) * step * _exact_pow2(e)).view(x.shape)[:R, :C]


def _exact_held(d, s, cols):
    f = s.view(torch.uint8).double() - 127
    return d.double()[:, :cols] * _exact_pow2(f).repeat_interleave(128, 1)[:, :cols]


def _exact_norm(x, w, b):
    x = x.double()
    mean = x.sum(1, keepdim=True) / x.shape[1]
    var = ((x - mean) ** 2).sum(1, keepdim=True) / x.shape[1]
    h = (x - mean) / torch.sqrt(var + _EPS)
    return h * w.double() + b.double(), h, 1 / torch.sqrt(var + _EPS)


def _exact_norm_back(g, h, r, w):
    g = g.double()
    t, c = g * w.double(), h.shape[1]
    return r * (t - t.sum(1, keepdim=True) / c - h * (t * h).sum(1, keepdim=True) / c), (g * h).sum(0), g.sum(0)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        op = case["op"]
        if op == "matmul":
            y = _exact_held(*s["a"], case["k"]) @ _exact_held(*s["b"], case["k"]).t()
            y = y + s["bias"].double() if s["bias"] is not None else y
            return y.clamp(min=0) if case["relu"] else y
        x = s["x"].detach()
        if op == "norm":
            y, h, r = _exact_norm(x, s["norm"].weight, s["norm"].bias)
            return (y,) + _exact_norm_back(s["g"], h, r, s["norm"].weight)
        lin, kind = s["lin"], case.get("grad", "e4m3")
        z, w8 = x, None
        if op == "norm_linear":
            z, h, r = _exact_norm(x, s["norm"].weight, s["norm"].bias)
            w8 = None if case["train"] else _exact_held(*s["w"], case["k"])
        w8 = _exact_blocks(lin.weight, "e4m3", rows=128) if w8 is None else w8
        y = _exact_blocks(z, "e4m3") @ w8.t() + lin.bias.double()
        if op == "norm_linear" and not case["train"]:
            return y
        g = s["g"].double()
        dz = _exact_blocks(g, kind) @ w8
        dw = _exact_blocks(g.t(), kind) @ _exact_blocks(z.double().t(), "e4m3").t()
        if op == "linear":
            return y, dz, dw, g.sum(0)
        return (y,) + _exact_norm_back(dz, h, r, s["norm"].weight) + (dw, g.sum(0))
