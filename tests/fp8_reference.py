"""The 8-bit block format and the operators over it in 64 bits, from their definitions (include/snipper_fp8.h)."""
import torch

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
MOST = {E4M3: 448.0, E5M2: 57344.0}


def pow2(e):
    return torch.ldexp(torch.ones((), dtype=torch.float64), e.to("cpu", torch.float64)).to(e.device)


def exponents(most, dtype):
    """Smallest e >= -127 with most / 2^e <= largest value of the type; 0 for a block of zeros."""
    q = most.double() / MOST[dtype]
    m, x = torch.frexp(q)                              # q = m 2^x, 0.5 <= m < 1: the smallest power of two not below q
    e = torch.where(m == 0.5, x - 1, x)
    return torch.where(most > 0, e.clamp(min=-127), torch.zeros_like(e))


def round_to(v, dtype):
    """Nearest value of the type, ties to even, in 64 bits; infinities: NaN in e4m3."""
    bits, low = (3, -6) if dtype == E4M3 else (2, -14)
    fin = torch.isfinite(v)
    m, x = torch.frexp(torch.where(fin, v, torch.zeros_like(v)).abs())
    step = pow2((x - 1).clamp(min=low) - bits)
    r = torch.round(torch.where(fin, v, torch.zeros_like(v)) / step) * step
    odd = v if dtype == E5M2 else torch.full_like(v, float("nan"))
    return torch.where(fin, r, odd)


def quantize(x, dtype, tile=1):
    """(elements [R, P] in units of their scale, exponents [R, P / 128]) of blocks of tile x 128, both 64-bit / whole."""
    x = x.detach().double()
    R, C = x.shape
    x = torch.nn.functional.pad(x, (0, -C % 128, 0, -R % tile))
    b = x.view(x.shape[0] // tile, tile, x.shape[1] // 128, 128)
    fin = torch.where(torch.isfinite(b), b.abs(), torch.zeros_like(b))
    e = exponents(fin.amax(dim=(1, 3)), dtype)
    v = round_to(b * pow2(-e)[:, None, :, None], dtype)
    return v.reshape(x.shape)[:R], e.repeat_interleave(tile, 0)[:R]


def values(v, e, cols):
    return (v.view(v.shape[0], -1, 128) * pow2(e)[:, :, None]).reshape(v.shape)[:, :cols]


def rounded(x, dtype, tile=1):
    return values(*quantize(x, dtype, tile), x.shape[1])


def held(blocks):
    """The matrix that an Fp8Blocks stands for, 64 bits."""
    v = blocks.data.double()
    e = blocks.scale.view(torch.uint8)[:, :v.shape[1] // 128].int() - 127
    return values(v, e, blocks.cols)


def random_blocks(R, C, dtype, device, gen, spread=6):
    """Blocks with random exponents, made without the quantizers."""
    from snipper_amd.fp8 import Fp8Blocks
    P, Q = -(-C // 128) * 128, -(-C // 512) * 4
    d = (torch.randn(R, P, generator=gen) * (100 if dtype == E4M3 else 2000)).clamp(-448, 448)
    d[:, C:] = 0
    s = torch.full((R, Q), 127, dtype=torch.uint8)
    s[:, :P // 128] = torch.randint(127 - spread, 127 + spread, (R, P // 128), generator=gen, dtype=torch.uint8)
    return Fp8Blocks(d.to(dtype).to(device), s.view(torch.float8_e8m0fnu).to(device), C)


def product_bounds(a, b, y, out_dtype, bias=None):
    """(y's bound element by element, bound of the norm of the error) for a product of matrices a [M, K], b [N, K] (64 bits).

    Rounding of the result: half a step.  Sums: a float32 result adds K products and K / 32 partial sums in float32, each addition off
    by at most 2^-24 of a partial sum that is at most S = sum |a b|; a 16-bit result loses of each product at most 2^-13 of the
    largest one of its block of 128 (or the product itself), plus the float32 additions."""
    half = torch.finfo(out_dtype).eps / 2
    K = a.shape[1]
    S = a.abs() @ b.abs().t()
    lost = torch.zeros_like(S)
    lost2 = torch.zeros_like(S)
    if out_dtype != torch.float32:
        for k in range(0, K, 128):
            p = (a[:, None, k:k + 128] * b[None, :, k:k + 128]).abs()
            c = torch.minimum(p, p.amax(2, keepdim=True) * 2.0 ** -13)
            lost += c.sum(2)
            lost2 += (c * c).sum(2)
    if bias is not None:
        S = S + bias.double().abs()
    tiny = torch.finfo(out_dtype).smallest_normal * half          # half a step of the type's smallest values
    each = half * y.abs() + lost + (K + 2) * 2.0 ** -24 * S + tiny
    # errors of single products and of single roundings do not add up in step: their squares do
    norm = ((half * y.abs()) ** 2 + lost2 + ((K + 2) ** 0.5 * 2.0 ** -24 * S) ** 2 + tiny ** 2).sum().sqrt()
    return each, norm
