"""Gradients through a frozen layer on packed 4-bit weights: to its input, bias and residual, by the entry point, the torch op
and the module; an adapter in front of such a layer learns; what has no gradient says so.

Tolerances as in test_gpu_mx.py."""

import pytest
import torch
import torch.nn as nn

from oracle import mx as omx
from tests.conftest import announce
from tests.test_gpu_mx import _acts, _check, _gen

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _packed(N, K, gpu, seed=2):
    from dimq_amd import mx
    w = torch.randn(N, K, generator=_gen(seed)) / K ** 0.5
    return omx.q4(w), *mx.quantize_mxfp4(w.to(gpu))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 32, 16), (5, 100, 37), (300, 520, 130), (0, 64, 24)])
def test_to_the_input(gpu, dt, M, K, N):
    from dimq_amd import mx
    announce(f"frozen {dt} {M}x{K} -> {N}")
    wq, c, s = _packed(N, K, gpu)
    x, g = _acts(M, K, dt, 3).to(gpu).requires_grad_(), _acts(M, N, dt, 4)
    gd = g.double()
    for call in (mx.mxfp4_linear, lambda x, c, s: torch.ops.dimq.mxfp4_linear(x, c, s, None)):
        y = call(x, c, s)
        assert y.requires_grad and torch.equal(y, mx.mxfp4_linear(x.detach(), c, s))
        gx, = torch.autograd.grad(y, x, g.to(gpu))
        assert gx.dtype == dt and gx.shape == x.shape
        if M:
            _check(gx, gd @ wq, gd.abs() @ wq.abs(), 3 * N)
        with torch.no_grad():
            assert not call(x, c, s).requires_grad
        assert not call(x.detach(), c, s).requires_grad


@pytest.mark.parametrize("need", [(1, 1, 1), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)])
@pytest.mark.parametrize("bias,res", [(True, True), (True, False), (False, True)])
def test_to_every_input(gpu, need, bias, res):
    from dimq_amd import mx
    M, K, N = 24, 96, 50
    announce(f"frozen {need} bias {bias} residual {res}")
    wq, c, s = _packed(N, K, gpu)
    x = _acts(M, K, torch.bfloat16, 3).view(4, 6, K).to(gpu)
    b, r = torch.randn(1, N, generator=_gen(5), dtype=torch.float64), torch.randn(4, 6, N, generator=_gen(6)).half()
    leaves = [t for t, there in ((x, True), (b.to(gpu), bias), (r.to(gpu), res)) if there]
    asked = [n for n, there in zip(need, (True, bias, res)) if there]
    for t, n in zip(leaves, asked):
        t.requires_grad_(bool(n))
    if not any(asked):
        return
    args = iter(leaves[1:])
    y = mx.mxfp4_linear(leaves[0], c, s, next(args) if bias else None, residual=next(args) if res else None,
                        out_dtype=torch.float32)
    g = torch.randn(M, N, generator=_gen(7))
    y.backward(g.view(4, 6, N).to(gpu))
    gd = g.double()
    refs = [v for v, there in (((gd @ wq, gd.abs() @ wq.abs()), True), ((gd.sum(0), gd.abs().sum(0)), bias),
                               ((gd, gd.abs()), res)) if there]
    for t, n, (ref, S) in zip(leaves, asked, refs):
        assert (t.grad is not None) == bool(n)
        if n:
            assert t.grad.shape == t.shape and t.grad.dtype == t.dtype
            got = t.grad.float() if t.dtype == torch.float64 else t.grad  # the bias's is a sum in fp32
            _check(got.reshape(ref.shape), ref, S, 3 * N)


def test_to_one_after_the_other(gpu):
    """autograd.grad for one input of several that could have one."""
    from dimq_amd import mx
    wq, c, s = _packed(40, 64, gpu)
    x, b = torch.randn(9, 64, device=gpu, requires_grad=True), torch.randn(40, device=gpu, requires_grad=True)
    r = torch.randn(9, 40, device=gpu, requires_grad=True)
    g = torch.randn(9, 40, device=gpu)
    y = mx.mxfp4_linear(x, c, s, b, residual=r)
    full = torch.autograd.grad(y, (x, b, r), g, retain_graph=True)
    for t, want in zip((x, b, r), full):
        assert torch.equal(torch.autograd.grad(y, t, g, retain_graph=True)[0], want)
    assert torch.equal(full[2], g)


def test_differences(gpu):
    """On values of the format the layer is linear: the gradient times a step is what the output moves by."""
    from dimq_amd import mx
    wq, c, s = _packed(24, 64, gpu)
    wq = wq.to(gpu)
    x = omx.q4(torch.randn(8, 64, generator=_gen(1))).float().to(gpu).requires_grad_()
    g = torch.randn(8, 24, generator=_gen(5)).to(gpu)
    y = mx.mxfp4_linear(x, c, s)
    gx, = torch.autograd.grad(y, x, g)
    S = ((x.detach().double().abs() @ wq.abs().t()) * g.double().abs()).sum()  # the same for both outputs
    for i, j in ((0, 0), (5, 17), (7, 63)):
        moved = x.detach().clone()
        moved[i, j] = -moved[i, j]  # another value of the same block
        diff = ((mx.mxfp4_linear(moved, c, s).double() - y.detach().double()) * g.double()).sum()
        step = (moved - x.detach()).double()[i, j]
        part = (g[i].double().abs() * wq[:, j].abs()).sum() * step.abs()
        # two outputs of 64 terms and a gradient of 24 x 3, each within (terms + 8) 2^-23 of their magnitudes
        assert abs(diff - gx[i, j].double() * step) <= 2.0 ** -23 * (2 * 72 * S + 80 * part)


def test_adapter_in_front_of_a_frozen_layer(gpu):
    from dimq_amd import DIMQMXFP4Linear
    announce("adapter")
    torch.manual_seed(0)
    frozen = DIMQMXFP4Linear.from_linear(nn.Linear(64, 32).to(gpu))
    adapter = nn.Linear(64, 64).to(gpu)
    x, target = torch.randn(256, 64, device=gpu), torch.randn(256, 32, device=gpu)
    optimiser = torch.optim.Adam(adapter.parameters(), lr=1e-2)
    losses = []
    for _ in range(30):
        loss = (frozen(x + adapter(x)) - target).square().mean()
        optimiser.zero_grad()
        loss.backward()
        assert adapter.weight.grad.abs().sum() > 0
        optimiser.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.9 * losses[0], losses


def test_what_has_no_gradient_raises(gpu):
    from dimq_amd import mx
    _, c, s = _packed(40, 64, gpu)
    x = torch.randn(9, 64, device=gpu, requires_grad=True)
    for act in ("relu", "gelu"):
        y = mx.mxfp4_linear(x, c, s, activation=act)
        assert torch.equal(y.detach(), mx.mxfp4_linear(x.detach(), c, s, activation=act))
        with pytest.raises(RuntimeError, match="no gradient through its fused activation"):
            y.sum().backward()
    with pytest.raises(RuntimeError, match="gradients of its gradients"):
        torch.autograd.grad(mx.mxfp4_linear(x, c, s).sum(), x, create_graph=True)
    y = mx.mxfp4_linear(x, c, s)
    c += 0  # written to in between
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_nothing_kept_but_the_weights(gpu):
    from dimq_amd import mx
    _, c, s = _packed(48, 2048, gpu)
    x = torch.randn(1024, 2048, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    y = mx.mxfp4_linear(x, c, s)
    torch.cuda.synchronize()
    assert torch.cuda.memory_stats()["requested_bytes.all.current"] - before == y.numel() * 2


def test_captured_in_a_graph(gpu):
    from dimq_amd import mx
    _, c, s = _packed(96, 160, gpu)
    x, g = torch.zeros(300, 160, device=gpu, dtype=torch.bfloat16), torch.zeros(300, 96, device=gpu, dtype=torch.bfloat16)

    def step():
        t = x.detach().requires_grad_()
        y = mx.mxfp4_linear(t, c, s)
        return y.detach(), *torch.autograd.grad(y, t, g)

    announce("captured frozen layer")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        x.copy_(torch.randn(300, 160, generator=_gen(10 + i)))
        g.copy_(torch.randn(300, 96, generator=_gen(20 + i)))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
