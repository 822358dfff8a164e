"""The microscaled operators where torch looks on or steps in: dispatch modes, traces, vmap.  A recorded program computes
with the inputs that it is given later."""

import warnings

import pytest
import torch

from tests.conftest import announce
from tests.test_gpu_mx import _acts, _gen

pytestmark = pytest.mark.gpu


def _calls(gpu):
    """name -> (a function of one tensor, an input, another input)"""
    from dimq_amd import mx
    c, s = mx.quantize_mxfp4(torch.randn(24, 64, generator=_gen(1)).to(gpu))
    x8, xs = mx.compress_activation(torch.randn(10, 64, generator=_gen(2)).to(gpu))
    b = torch.randn(24, generator=_gen(3)).to(gpu)
    x = [_acts(10, 64, torch.bfloat16, i).to(gpu) for i in (4, 5)]
    g = [_acts(10, 24, torch.bfloat16, i).to(gpu) for i in (6, 7)]
    c2 = mx.quantize_mxfp4(torch.randn(24, 64, generator=_gen(8)).to(gpu))[0]
    y8 = mx.compress_activation(torch.randn(10, 64, generator=_gen(9)).to(gpu))[0]
    return {
        "quantize_mxfp4": (mx.quantize_mxfp4, *x),
        "compress_activation": (mx.compress_activation, *x),
        "quantize_and_compress": (mx.quantize_and_compress, *x),
        "dequantize_mxfp4": (lambda t: mx.dequantize_mxfp4(t, s, 64), c, c2),
        "decompress_activation": (lambda t: mx.decompress_activation(t, xs, 64), x8, y8),
        "mxfp4_linear": (lambda t: mx.mxfp4_linear(t, c, s, b, activation="gelu"), *x),
        "mxfp4_linear_grad_input": (lambda t: mx.mxfp4_linear_grad_input(t, c, s, 64), *g),
        "linear_grad_weight": (lambda t: mx.linear_grad_weight(t, x8, xs, 64), *g),
    }


NAMES = ["quantize_mxfp4", "compress_activation", "quantize_and_compress", "dequantize_mxfp4", "decompress_activation",
         "mxfp4_linear", "mxfp4_linear_grad_input", "linear_grad_weight"]


def _same(a, b):
    a, b = (t if isinstance(t, (tuple, list)) else (t,) for t in (a, b))
    return len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("name", NAMES)
def test_dispatch_mode_sees_the_operator(gpu, name):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Record(TorchDispatchMode):
        seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    announce(f"mode {name}")
    f, x, _ = _calls(gpu)[name]
    want = f(x)
    with Record() as mode:
        got = f(x)
    assert _same(got, want) and f"dimq.{name}.default" in mode.seen


@pytest.mark.parametrize("name", NAMES)
def test_traced_to_a_graph(gpu, name):
    from torch.fx.experimental.proxy_tensor import make_fx
    announce(f"make_fx {name}")
    f, x, other = _calls(gpu)[name]
    assert not _same(f(x), f(other))
    assert _same(make_fx(f)(x)(other), f(other))


def test_traced_module(gpu):
    import torch.nn as nn

    from dimq_amd import DIMQMXFP4Linear
    announce("traced module")
    mod = DIMQMXFP4Linear.from_linear(nn.Linear(64, 24).to(gpu))
    x, other = (_acts(10, 64, torch.bfloat16, i).to(gpu) for i in (4, 5))
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(mod, (x,))
    assert torch.equal(traced(other), mod(other)) and not torch.equal(mod(x), mod(other))


def test_vmap(gpu):
    from dimq_amd import mx
    announce("vmap")
    c, s = mx.quantize_mxfp4(torch.randn(24, 64, generator=_gen(1)).to(gpu))
    x = _acts(40, 64, torch.bfloat16, 4).view(4, 10, 64).to(gpu)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        y = torch.vmap(lambda t: mx.mxfp4_linear(t, c, s))(x)
    assert torch.equal(y, torch.stack([mx.mxfp4_linear(t, c, s) for t in x]))


def test_training_functions_refuse_a_trace(gpu):
    """They are no operators that a trace could record."""
    from dimq_amd import mx
    w = torch.randn(24, 64, device=gpu)
    x = torch.randn(10, 64, device=gpu)
    for f in (lambda t: mx.linear(t, w), mx.gelu):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (x,), check_trace=False)


def test_proxies_refused_by_training_functions(gpu):
    from torch.fx.experimental.proxy_tensor import make_fx

    from dimq_amd import mx
    w = torch.randn(24, 64, device=gpu)
    c, s = mx.quantize_mxfp4(w)
    x = torch.randn(10, 64, device=gpu)

    def through_a_frozen_layer(t):
        t = t.detach().requires_grad_()
        return torch.autograd.grad(mx.mxfp4_linear(t, c, s).sum(), t)[0]

    for f in (lambda t: mx.linear(t, w), mx.gelu, through_a_frozen_layer):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(f)(x)


def test_modes_autocast_and_inference_with_gradients(gpu):
    """The same values and gradients, and the operator seen, where the input needs a gradient."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from dimq_amd import mx
    seen = []

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    c, s = mx.quantize_mxfp4(torch.randn(24, 64, generator=_gen(1)).to(gpu))
    x = _acts(10, 64, torch.bfloat16, 4).to(gpu).requires_grad_()
    g = _acts(10, 24, torch.bfloat16, 5).to(gpu)
    y = mx.mxfp4_linear(x, c, s)
    gx, = torch.autograd.grad(y, x, g)
    for call in (mx.mxfp4_linear, lambda x, c, s: torch.ops.dimq.mxfp4_linear(x, c, s, None)):
        seen.clear()
        with Record():
            z = call(x, c, s)
            gz, = torch.autograd.grad(z, x, g)
        assert torch.equal(z, y) and torch.equal(gz, gx) and "dimq.mxfp4_linear.default" in seen
        with torch.autocast("cuda", dtype=torch.bfloat16):
            z = call(x, c, s)
        assert torch.equal(z, y) and torch.equal(torch.autograd.grad(z, x, g)[0], gx)
        with torch.inference_mode():
            z = call(x, c, s)
        assert torch.equal(z, y) and not z.requires_grad
