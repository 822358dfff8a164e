"""GELU of the largest finite numbers, by itself and in the epilogue of each route of the 4-bit layer.

There h Phi(h) is h for positive h and 0 for negative: tolerances as in test_gpu_mx.py."""

import pytest
import torch

from oracle import mx as omx
from tests.conftest import announce
from tests.test_gpu_mx import _check

pytestmark = pytest.mark.gpu


def _large(dt):
    top = torch.finfo(dt).max
    v = [top, top / 2, top * 0.51, top * 0.6, top * 0.75, 1e4, 300.0, 2.0]
    return torch.tensor(v + [-a for a in v], dtype=torch.float64).to(dt)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
def test_gelu(gpu, dt):
    from dimq_amd import mx
    announce(f"large gelu {dt}")
    h = _large(dt)
    for shape in ((1, 16), (16, 1)):
        x = h.view(shape).to(gpu).requires_grad_()
        y = mx.gelu(x)
        ref = omx.gelu(h.view(shape))
        _check(y, ref, torch.zeros(()), 0, 3e-6 * ref.abs() + 1e-37)
        with torch.no_grad():
            assert torch.equal(mx.gelu(x), y)
        assert torch.equal(torch.ops.dimq.gelu_forward(x.detach())[0], y.detach())
        gh, = torch.autograd.grad(y, x, torch.ones_like(x))
        slope = omx.gelu_slope(omx.q8(h.view(shape)))
        _check(gh, slope, torch.zeros(()), 0, 3e-6 * slope.abs() + 1e-37)


# few rows in one launch; the tiled product; its split reduction
@pytest.mark.parametrize("M,K", [(3, 64), (700, 64), (130, 8224)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_epilogue(gpu, M, K, out):
    """One value of the 4-bit format a row against ones: the sum is that value."""
    from dimq_amd import mx
    announce(f"large epilogue {M}x{K} {out}")
    v = torch.tensor([1.5 * 2.0 ** 127, 2.0 ** 127, 1.5 * 2.0 ** 126, 3.0, -1.5 * 2.0 ** 127, -2.0 ** 127, 0.0])
    x = torch.zeros(M, K)
    x[:, K - 7] = v[torch.arange(M) % 7]
    c, s = mx.quantize_mxfp4(torch.ones(40, K, device=gpu))
    y = mx.mxfp4_linear(x.to(gpu), c, s, activation="gelu", out_dtype=out)
    ref = omx.gelu(x.double().sum(1, keepdim=True)).expand(M, 40)
    _check(y, ref, torch.zeros(()), 0, 3e-6 * ref.abs() + 1e-37)
