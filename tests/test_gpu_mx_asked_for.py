"""A backward pass of mx.linear computes the gradients that it is asked for, and takes memory for no others."""

import ctypes

import pytest
import torch

from tests.conftest import announce
from tests.test_gpu_mx import _acts, _gen

pytestmark = pytest.mark.gpu

M, K, N = 96, 2048, 1536


def _grown(f):
    """(f(), bytes asked of the allocator at most during it beyond those held before)"""
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    r = f()
    torch.cuda.synchronize()
    return r, torch.cuda.memory_stats()["requested_bytes.all.peak"] - before


@pytest.mark.parametrize("asked", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1), (1, 1, 0), (1, 1, 1)])
def test_memory_and_values(gpu, asked):
    from dimq_amd import _C, mx
    announce(f"asked for {asked}")
    x = _acts(M, K, torch.bfloat16, 1).to(gpu).requires_grad_()
    w = (torch.randn(N, K, generator=_gen(2)) / 45).to(gpu).requires_grad_()
    b = torch.randn(N, generator=_gen(3)).to(gpu).requires_grad_()
    g = (torch.randn(M, N, generator=_gen(4)) * 0.01).to(gpu, torch.bfloat16)
    leaves = (x, w, b)
    want = torch.autograd.grad(mx.linear(*leaves), leaves, g)
    y = mx.linear(*leaves)
    some = [t for t, a in zip(leaves, asked) if a]
    got, bytes_ = _grown(lambda: torch.autograd.grad(y, some, g))
    for t, r in zip(got, [r for r, a in zip(want, asked) if a]):
        assert t.dtype == r.dtype and torch.equal(t, r)
    need = _C.lib.dimq_mx_linear_backward_workspace_bytes(ctypes.c_void_p(g.data_ptr()), _C.BF16, M, N, N, K,
                                                          sum(a << i for i, a in enumerate(asked)))
    # the outputs and the workspace of that choice, each rounded up by the allocator to at most 512 bytes
    assert bytes_ <= need + sum(t.numel() * t.element_size() for t in got) + 4 * 512


def test_one_step_through_some_leaves(gpu):
    """backward(inputs=...) fills those leaves and leaves the others alone."""
    from dimq_amd import mx
    announce("backward(inputs=)")
    x = torch.randn(40, 64, generator=_gen(5)).to(gpu).requires_grad_()
    layer = mx.MXFP4TrainLinear(64, 24).to(gpu)
    layer(x).sum().backward(inputs=[layer.bias])
    assert x.grad is None and layer.weight.grad is None
    assert torch.equal(layer.bias.grad, torch.full((24,), 40.0, device=gpu))
