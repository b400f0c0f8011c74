"""What the 8-bit operators' and the wide layer norm's wrappers hand to the native entries, on the CPU: the calls are recorded, not made."""
import ctypes

import pytest
import torch

from snipper_amd import _lib, fp8, fused


class OnCard(torch.Tensor):
    """A CPU tensor that says that it is on the card, and whose results do."""
    is_cuda = True


def _card(t):
    return t.as_subclass(OnCard)


@pytest.fixture
def calls(monkeypatch):
    """(entry's name, arguments without the stream) of each native call, in turn."""
    made = []

    def record(fn, index, *args):
        made.append((fn.__name__, args))
    _lib.load()
    for module in (fused, fp8):
        monkeypatch.setattr(module, "_call", record)
    return made


def _dense(t):
    return t.detach().clone(memory_format=torch.contiguous_format)


HOOKS = {"none": (lambda t: t, lambda t: t),
         "dense": (_dense, lambda t: t),                                     # what torch.autograd.graph.save_on_cpu gives back
         "columns": (lambda t: t, lambda t: _dense(t.t()).t() if t.dim() == 2 else torch.stack([t, t], 1)[:, 0]),
         "wider": (lambda t: t, lambda t: torch.cat([t, t], -1)[..., :t.shape[-1]] if t.dim() == 2 else t)}


def _layer_norm_backward_call(made):
    (_, args), = [c for c in made if c[0] == "snipper_layernorm_backward"]
    return dict(zip(("g", "x", "dtype", "ldx", "mean", "rstd", "gamma", "p_dtype", "rows", "cols"), args))


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("op", ["layer_norm", "layer_norm_linear_fp8"])
def test_backward_steps_by_the_stride_of_the_rows_that_it_gets(op, hook, calls):
    """Saved-tensor hooks may give x back in another layout: each row that the native call reads lies inside the tensor handed to it."""
    rows, cols, held = 6, 40, []
    pack, unpack = HOOKS[hook]

    def keep(t):
        t = unpack(t)
        held.append(t)
        return t
    x = _card(torch.randn(rows, cols + 9)[:, :cols]).requires_grad_()
    norm, lin = torch.nn.LayerNorm(cols), torch.nn.Linear(cols, 8)
    for m in (norm, lin):
        for n, p in list(m.named_parameters()):
            setattr(m, n, torch.nn.Parameter(_card(p.detach()), requires_grad=True))
    with torch.autograd.graph.saved_tensors_hooks(pack, keep):
        y = fused.layer_norm(x, norm) if op == "layer_norm" else fp8.layer_norm_linear_fp8(x, norm, lin)
        forward = len(calls)
        torch.autograd.grad(y, x, torch.ones_like(y))
    c = _layer_norm_backward_call(calls)
    assert (c["rows"], c["cols"]) == (rows, cols) and c["ldx"] >= cols
    given = [t for t in held if t.data_ptr() == c["x"]]
    # a copy made for the call is contiguous; anything else is one of the tensors that the hooks gave back
    if given:
        t, = given
        assert t.stride() == (c["ldx"], 1)
    else:
        assert c["ldx"] == cols
    last = c["x"] + 4 * ((rows - 1) * c["ldx"] + cols)
    # the statistics and what the products read are vectors for the native calls
    for t in held:
        if t.data_ptr() in (c["mean"], c["gamma"]):
            assert t.is_contiguous()
    assert c["rstd"] == c["mean"] + 4 * rows
    starts = {t.data_ptr(): t for t in held if not t.is_contiguous()}
    assert not any(a in starts for name, args in calls[forward:] if name == "snipper_fp8_matmul" for a in args)
    for t in given:
        assert last <= t.untyped_storage().data_ptr() + t.untyped_storage().nbytes()


def _differentiable_calls():
    x, norm, lin = _card(torch.randn(4, 40)), torch.nn.LayerNorm(40), torch.nn.Linear(40, 8)
    for m in (norm, lin):
        for n, p in list(m.named_parameters()):
            setattr(m, n, torch.nn.Parameter(_card(p.detach()), requires_grad=False))
    return x, norm, lin


CALLS = {"layer_norm": lambda x, norm, lin: fused.layer_norm(x, norm), "linear_fp8": lambda x, norm, lin: fp8.linear_fp8(x, lin),
         "layer_norm_linear_fp8": lambda x, norm, lin: fp8.layer_norm_linear_fp8(x, norm, lin),
         "quantize_rows": lambda x, norm, lin: fp8.quantize_rows(x), "quantize_both": lambda x, norm, lin: fp8.quantize_both(x),
         "quantize_tiles": lambda x, norm, lin: fp8.quantize_tiles(x), "layer_norm_fp8": lambda x, norm, lin: fp8.layer_norm_fp8(x, norm)}


@pytest.mark.parametrize("grad_mode", [torch.enable_grad, torch.no_grad])
@pytest.mark.parametrize("op", CALLS)
def test_forward_mode_derivatives_are_refused_not_dropped(op, grad_mode, calls):
    """A dual tensor has requires_grad false, and no_grad does not turn forward mode off."""
    from torch.autograd import forward_ad
    x, norm, lin = _differentiable_calls()
    with grad_mode(), forward_ad.dual_level():
        CALLS[op](x, norm, lin)                                              # (no tangent: as always)
        made = len(calls)
        assert made
        with pytest.raises((RuntimeError, NotImplementedError)):
            CALLS[op](forward_ad.make_dual(x, torch.ones_like(x)), norm, lin)
        if op in ("layer_norm", "layer_norm_fp8", "layer_norm_linear_fp8"):
            norm.weight.requires_grad_(False)
            dual = torch.nn.LayerNorm(40)
            del dual.weight
            dual.weight = forward_ad.make_dual(norm.weight.detach(), torch.ones_like(norm.weight))
            dual.bias = norm.bias
            with pytest.raises((RuntimeError, NotImplementedError)):
                CALLS[op](x, dual, lin)


def test_matmul_refuses_a_bias_with_a_tangent(calls):
    from torch.autograd import forward_ad
    a = fp8.Fp8Blocks(_card(torch.zeros(4, 128, dtype=torch.float8_e4m3fn)), _card(torch.ones(4, 4, dtype=torch.float32).to(torch.float8_e8m0fnu)), 40)
    bias = _card(torch.zeros(4))
    with forward_ad.dual_level():
        fp8.matmul_fp8(a, a, bias)
        with pytest.raises((RuntimeError, NotImplementedError)):
            fp8.matmul_fp8(a, a, forward_ad.make_dual(bias, torch.ones_like(bias)))


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_nothing_is_written_for_a_backward_pass_that_cannot_come(mode, calls):
    """Trainable modules under no_grad: x's and W's rows only, and the norm in one launch, straight into blocks."""
    x, norm, lin = _differentiable_calls()
    for p in (*norm.parameters(), *lin.parameters()):
        p.requires_grad_(True)
    with mode():
        y = fp8.linear_fp8(x, lin)
        z = fp8.layer_norm_linear_fp8(x, norm, lin)
    assert y.shape == z.shape == (4, 8) and not y.requires_grad and not z.requires_grad
    names = [n for n, _ in calls]
    assert names == ["snipper_fp8_quantize"] * 2 + ["snipper_fp8_matmul", "snipper_fp8_quantize", "snipper_layernorm_forward", "snipper_fp8_matmul"]
    for n, args in calls:
        if n == "snipper_fp8_quantize":
            data, scale, data_t, scale_t = args[12:16]
            assert data and scale and data_t is None and scale_t is None
        elif n == "snipper_layernorm_forward":
            y, mean, rstd, data, scale = args[9:14]
            assert data and scale and y is None and mean is None and rstd is None


@pytest.mark.parametrize("which", ["x", "norm", "weight", "bias"])
def test_what_a_backward_pass_reads_is_written_when_it_can_come(which, calls):
    x, norm, lin = _differentiable_calls()
    {"x": x, "norm": norm.weight, "weight": lin.weight, "bias": lin.bias}[which].requires_grad_(True)
    y = fp8.layer_norm_linear_fp8(x, norm, lin)
    assert y.requires_grad
    y.backward(torch.ones_like(y))
    made = [n for n, _ in calls].count("snipper_fp8_matmul")
    assert made == (1 if which == "bias" else 2)


def test_full_sums_reach_every_product(calls):
    x, norm, lin = _differentiable_calls()
    x, lin = x.bfloat16().as_subclass(OnCard).requires_grad_(), lin.requires_grad_()
    for full in (False, True):
        del calls[:]
        for y in (fp8.linear_fp8(x, lin, full_sums=full), fp8.layer_norm_linear_fp8(x, norm, lin, full_sums=full)):
            y.backward(torch.ones_like(y))
        types = [args[13] for n, args in calls if n == "snipper_fp8_matmul"]
        assert types == [1 + 16 * full] * 2 + [1 + 16 * full, 16 * full] * 2       # y, y; dx in bfloat16, dW in float32
    a = fp8.Fp8Blocks(_card(torch.zeros(4, 128, dtype=torch.float8_e4m3fn)), _card(torch.ones(4, 4).to(torch.float8_e8m0fnu)), 40)
    del calls[:]
    fp8.matmul_fp8(a, a, out_dtype=torch.float16, full_sums=True)
    assert calls[0][1][13] == 3 + 16


def test_c_matmul_takes_the_flag_of_full_sums():
    lib = _lib.load()
    p = ctypes.c_void_p(4096)
    need = lib.snipper_fp8_matmul_workspace_bytes
    for M, N, K in ((384, 1024, 79000), (1, 4096, 4096), (300, 200, 9000)):
        assert need(M, N, K, 1 | 16) == need(M, N, K, 3 | 16) == need(M, N, K, 0) == need(M, N, K, 16)
    assert need(384, 1024, 79000, 2 | 16) == 0 and need(384, 1024, 79000, 32) == 0

    def call(odt, nb=0):
        return lib.snipper_fp8_matmul(None, p, p, 0, p, p, 0, 384, 1024, 79000, None, 0, 0, p, odt, p if nb else None, nb)
    assert call(2 | 16) == call(32) == call(64 | 1) == -2
    assert call(1 | 16) == call(1 | 16, need(384, 1024, 79000, 0) - 1) == -2


def _first_values(monkeypatch):
    """The first float32 of the matrix that each native call reads, as the call finds it in memory."""
    seen = []

    def record(fn, index, *args):
        at = {"snipper_fp8_quantize": 0, "snipper_layernorm_forward": 0, "snipper_layernorm_backward": 0}.get(fn.__name__)
        if at is not None and args[at]:
            seen.append(ctypes.c_float.from_address(args[at]).value)
    _lib.load()
    for module in (fused, fp8):
        monkeypatch.setattr(module, "_call", record)
    return seen


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 1), (5, 7)])
@pytest.mark.parametrize("op", CALLS)
def test_a_lazily_negated_tensor_is_read_with_its_own_signs(op, rows, cols, monkeypatch):
    """conj().imag is a view whose memory holds the opposite signs, with or without another stride."""
    seen = _first_values(monkeypatch)
    norm, lin = torch.nn.LayerNorm(cols), torch.nn.Linear(cols, 8)
    for m in (norm, lin):
        for n, p in list(m.named_parameters()):
            setattr(m, n, torch.nn.Parameter(_card(p.detach().abs() + 1), requires_grad=False))
    for x in (torch._neg_view(torch.rand(rows, cols) + 1), (torch.rand(rows, cols, dtype=torch.complex64) + 1 + 1j).conj().imag):
        del seen[:]
        assert x.is_neg() and (x < 0).all()
        CALLS[op](_card(x), norm, lin)
        assert min(seen) == x[0, 0].item()                                  # (the weight's are above 1)


@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("op", ["layer_norm", "linear_fp8"])
def test_a_lazily_negated_gradient_is_read_with_its_own_signs(op, rows, monkeypatch):
    seen = _first_values(monkeypatch)
    x, norm, lin = _card(torch.randn(rows, 1)).requires_grad_(), torch.nn.LayerNorm(1), torch.nn.Linear(1, 1)
    for m in (norm, lin):
        for n, p in list(m.named_parameters()):
            setattr(m, n, torch.nn.Parameter(_card(p.detach()), requires_grad=False))
    y = CALLS[op](x, norm, lin)
    del seen[:]
    torch.autograd.grad(y, x, _card(torch._neg_view(torch.rand(rows, 1) + 1)))
    assert seen and seen[0] < 0
