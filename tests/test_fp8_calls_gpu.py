"""Calls of the 8-bit operators and the wide layer norm as programs make them: saved-tensor hooks, inference, threads."""
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from snipper_amd import fp8, fused

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _x(rows, cols, dtype=torch.float32, seed=0):
    g = _gen(seed)
    return (torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(rows, 1, generator=g))).to(dtype).to(DEV)


def _modules(k, n, dtype=torch.float32):
    norm, lin = torch.nn.LayerNorm(k), torch.nn.Linear(k, n)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.3 * torch.randn(k, generator=_gen(11)))
        norm.bias.copy_(0.3 * torch.randn(k, generator=_gen(12)))
        lin.weight.copy_(torch.randn(n, k, generator=_gen(5)) / k ** 0.5)
        lin.bias.copy_(torch.randn(n, generator=_gen(6)))
    return norm.to(DEV, dtype), lin.to(DEV, dtype)


CALLS = {"layer_norm": lambda x, norm, lin: fused.layer_norm(x, norm), "linear_fp8": lambda x, norm, lin: fp8.linear_fp8(x, lin),
         "layer_norm_linear_fp8": lambda x, norm, lin: fp8.layer_norm_linear_fp8(x, norm, lin)}


def _step(op, x, norm, lin, g, hooks=None):
    leaves = [x] + ([*norm.parameters()] if op != "linear_fp8" else []) + ([*lin.parameters()] if op != "layer_norm" else [])
    if hooks is None:
        y = CALLS[op](x, norm, lin)
    else:
        with hooks:
            y = CALLS[op](x, norm, lin)
    return (y.detach(), *torch.autograd.grad(y, leaves, g[:, :y.shape[1]].to(y.dtype)))


@pytest.mark.parametrize("op", CALLS)
@pytest.mark.parametrize("rows,cols,skip", [(1, 40, 5), (50, 301, 6), (130, 1030, 3)])
def test_saved_tensors_that_come_back_in_another_layout(op, rows, cols, skip):
    """save_on_cpu gives a dense tensor back for a row slice; the other hooks change the strides of everything saved."""
    norm, lin = _modules(cols, 77)
    g = torch.randn(rows, max(cols, 77), generator=_gen(3)).to(DEV)
    x = _x(rows, cols + skip)[:, 2:cols + 2].requires_grad_()
    want = _step(op, x, norm, lin, g)
    apart = torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else torch.stack([t, t], 1)[:, 0])
    for hooks in (torch.autograd.graph.save_on_cpu(), apart):
        for a, b in zip(_step(op, x, norm, lin, g, hooks), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("op", CALLS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 130), (40, 384), (129, 1000), (70, 2100), (33, 100), (9, 1500), (5, 5000), (3, 9000)])
def test_inference_gives_the_training_step_s_result(op, dtype, rows, cols):
    norm, lin = _modules(cols, 60)
    x = _x(rows, cols, dtype)
    want = CALLS[op](x.clone().requires_grad_(), norm, lin)
    assert want.requires_grad
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            y = CALLS[op](x, norm, lin)
            assert torch.equal(CALLS[op](x.view(1, rows, 1, cols), norm, lin), y.view(1, rows, 1, -1))
            assert CALLS[op](x[:0], norm, lin).shape == (0, y.shape[1])
        assert not y.requires_grad and torch.equal(y, want)


@pytest.mark.parametrize("op", CALLS)
def test_threads_at_once_each_to_its_end(op):
    """Two threads on streams of their own; what a thread raises is raised here."""
    norm, lin = _modules(200, 130)
    xs = [_x(257, 200, torch.bfloat16, seed) for seed in (1, 2)]
    g = torch.randn(257, 200, generator=_gen(7)).to(DEV)
    want = [_step(op, x.requires_grad_(), norm, lin, g) for x in xs]
    torch.cuda.synchronize()

    def loop(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = _step(op, xs[i].detach().requires_grad_(), norm, lin, g)
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
        return 10
    with ThreadPoolExecutor(2) as pool:
        assert [f.result() for f in [pool.submit(loop, i) for i in (0, 1)]] == [10, 10]
