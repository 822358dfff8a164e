"""Gradients in fp32 so small that bf16 parts cannot hold all of their 24 bits: the least step of a part is 2^-133, so a
gradient of 2^-110 and more is split exactly and a smaller one to the nearest multiple of 2^-133, off by at most 2^-134.
The tolerances are test_gpu_mx.py's and that for each term, 2^-134 times the other factor."""

import pytest
import torch

from oracle import mx as omx
from tests.conftest import announce
from tests.test_gpu_mx import _check, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("exponent", [-100, -109, -112, -118, -125, -130, -136, -148])
@pytest.mark.parametrize("M,K,N", [(40, 72, 1), (1, 33, 40), (70, 160, 130), (600, 264, 520)])
def test_gradients(gpu, M, K, N, exponent):
    """All factors positive, so that errors towards zero would add up."""
    from dimq_amd import mx
    announce(f"tiny gradients 2^{exponent} {M}x{K} -> {N}")
    g = ((1 + torch.rand(M, N, generator=_gen(M + N), dtype=torch.float64)) * 2.0 ** exponent).float()
    x = (1 + torch.rand(M, K, generator=_gen(1))) * 2.0 ** 30
    w = (1 + torch.rand(N, K, generator=_gen(2))) * 2.0 ** 30
    gd, wq, xq = g.double(), omx.q4(w), omx.q8(x)
    step = 2.0 ** -134 if exponent < -110 else 0.0
    gx, gw = gd @ wq, gd.t() @ xq
    c, s = mx.quantize_mxfp4(w.to(gpu))
    _check(mx.mxfp4_linear_grad_input(g.to(gpu), c, s, K), gx, gx, 3 * N, step * wq.sum(0))
    got, gb = mx.linear_grad_weight(g.to(gpu), *mx.compress_activation(x.to(gpu)), K)
    _check(got, gw, gw, 3 * M, step * xq.sum(0))
    _check(gb, gd.sum(0), gd.sum(0), M)
