"""What the microscaled layers keep for a backward pass, in bytes asked of the allocator: the 8-bit form of an input (33 bytes
a block of 32) and the 4-bit one of a weight (17), each only where a gradient needs it, and nothing where none can follow.
And the 4-bit codes and scales by themselves against those of the call for both forms."""

import pytest
import torch

from tests.conftest import announce
from tests.test_gpu_mx import _acts, _gen, _same_codes, _special

pytestmark = pytest.mark.gpu


def _bytes(which):
    torch.cuda.synchronize()
    return torch.cuda.memory_stats()[f"requested_bytes.all.{which}"]


def _kept(f):
    """(f(), bytes more than before while its result lives, at most during the call)"""
    before = _bytes("current")
    torch.cuda.reset_peak_memory_stats()
    r = f()
    return r, _bytes("current") - before, _bytes("peak") - before


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(700, 1024), (301, 1001), (3, 40)])
def test_gelu(gpu, dt, rows, cols):
    from dimq_amd import mx
    announce(f"kept by gelu {dt} {rows}x{cols}")
    h = torch.randn(rows, cols, generator=_gen(1)).to(gpu, dt).requires_grad_()
    size, codes = rows * cols * h.element_size(), rows * -(-cols // 32) * 33
    y, now, peak = _kept(lambda: mx.gelu(h))
    assert now == peak == size + codes
    with torch.no_grad():
        z, now, peak = _kept(lambda: mx.gelu(h))
    assert now == peak == size
    z, now, peak = _kept(lambda: mx.gelu(h.detach()))
    assert now == peak == size


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(600, 1024, 96), (301, 1001, 130), (4, 64, 32)])
def test_linear(gpu, dt, M, K, N):
    from dimq_amd import _C, mx
    announce(f"kept by linear {dt} {M}x{K} -> {N}")
    x, w = _acts(M, K, dt, 1).to(gpu), torch.randn(N, K, generator=_gen(2)).to(gpu)
    nb = -(-K // 32)
    y, wq, xq = M * N * x.element_size(), N * nb * 17, M * nb * 33
    work = _C.lib.dimq_mxfp4_linear_workspace_bytes(M, K, N)
    for to_x, to_w in ((1, 1), (1, 0), (0, 1), (0, 0)):
        a, b = x.detach().requires_grad_(bool(to_x)), w.detach().requires_grad_(bool(to_w))
        r, now, peak = _kept(lambda: mx.linear(a, b))
        assert now == y + to_x * wq + to_w * xq
        assert peak == y + wq + to_w * xq + work
        del r
        with torch.no_grad():
            r, now, peak = _kept(lambda: mx.linear(a, b))
        assert now == y and peak == y + wq + work
        del r


def test_released_after_the_backward_pass(gpu):
    from dimq_amd import mx
    x, w = _acts(600, 512, torch.bfloat16, 1).to(gpu).requires_grad_(), torch.randn(256, 512, device=gpu, requires_grad=True)
    mx.gelu(mx.linear(x, w)).sum().backward()  # the gradients' memory
    before = _bytes("current")
    mx.gelu(mx.linear(x, w)).sum().backward()
    assert _bytes("current") == before


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 33), (65, 1000), (40, 4096)])
def test_four_bits_alone(gpu, dt, rows, cols):
    from dimq_amd import mx
    announce(f"quantize_mxfp4 {dt} {rows}x{cols}")
    x = _special(rows, cols, dt, rows + 7 * cols)
    c4, s4, c8, s8 = mx.quantize_and_compress(x.to(gpu))
    c, s = mx.quantize_mxfp4(x.to(gpu))
    assert torch.equal(c, c4) and torch.equal(s, s4)
    _same_codes(x, c, s, c8, s8)
