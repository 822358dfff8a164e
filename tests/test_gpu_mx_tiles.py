"""The tiled products of the microscaled layers at sizes that take each of their tiles, with whole and split reductions, odd
ends in every dimension, and one gradient plane or several; the single launch for few rows against the tiled route.

Tolerances as in test_gpu_mx.py: operands are exact, so a product is off by its fp32 sums, (r + 8) 2^-23 sum |a b| over
r terms, and its output's rounding."""

import pytest
import torch

from oracle import mx as omx
from tests.conftest import announce
from tests.test_gpu_mx import _acts, _check, _gen, _special

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _w(N, K, seed):
    return torch.randn(N, K, generator=_gen(seed)) / K ** 0.5


def _mm(a, b):
    """float64 a @ b on the GPU."""
    return (a.cuda().contiguous() @ b.cuda().contiguous()).cpu()


# 256 x 256 and 256 x 192 tiles; 128 x 128; 64 x 64, the last two with slices of a long reduction
@pytest.mark.parametrize("M,K,N,dt", [(3000, 140, 4100, F16), (12608, 72, 1032, F32), (6000, 96, 1288, BF16),
                                      (4100, 1100, 2050, F32), (4097, 2080, 2049, F16),
                                      (1500, 300, 2050, BF16), (3000, 1056, 1025, F32), (1030, 2560, 2050, F16),
                                      (257, 4128, 770, BF16), (100, 8200, 130, BF16), (40, 16416, 65, F32)])
def test_linear(gpu, M, K, N, dt):
    from dimq_amd import mx
    announce(f"tiled linear {dt} {M}x{K} -> {N}")
    x, w = _acts(M, K, dt, M + K), _w(N, K, N)
    b, r = torch.randn(N, generator=_gen(1)), torch.randn(M, N, generator=_gen(2)).to(dt)
    c, s = mx.quantize_mxfp4(w.to(gpu))
    xq, wq = omx.q4(x), omx.q4(w)
    ref = _mm(xq, wq.t()) + b.double() + r.double()
    S = _mm(xq.abs(), wq.abs().t()) + b.double().abs() + r.double().abs()
    y = mx.mxfp4_linear(x.to(gpu), c, s, b.to(gpu), residual=r.to(gpu))
    _check(y, ref, S, K)
    assert torch.equal(y, mx.mxfp4_linear(x.to(gpu), c, s, b.to(gpu), residual=r.to(gpu)))
    relu = mx.mxfp4_linear(x.to(gpu), c, s, b.to(gpu), residual=r.to(gpu), activation="relu")
    assert torch.equal(relu, y.clamp_min(0))


GRADS = [(6000, 2080, 2050, BF16), (1500, 2080, 2056, F32), (4100, 1000, 2050, F16), (4100, 2080, 40, BF16),
         (2049, 1056, 2056, BF16), (1030, 1000, 1025, F32), (6000, 544, 40, F16), (4096, 1056, 1032, BF16),
         (17, 96, 2056, BF16), (3000, 96, 40, F16), (64, 40, 5000, F32), (8200, 72, 136, BF16),
         (515, 4128, 4096, BF16), (130, 4128, 2056, F32), (2049, 1000, 4104, F16), (4100, 1000, 4104, BF16)]


@pytest.mark.parametrize("M,K,N,dt", GRADS)
def test_gradients(gpu, M, K, N, dt):
    from dimq_amd import mx
    announce(f"tiled gradients {dt} {M}x{K} -> {N}")
    x, w, g = _acts(M, K, dt, M), _w(N, K, N), _acts(M, N, dt, 11, 1.0) * 2.0 ** -6
    c, s = mx.quantize_mxfp4(w.to(gpu))
    x8, xs = mx.compress_activation(x.to(gpu))
    wq, xq, gd = omx.q4(w), omx.q8(x), g.double()
    parts = {F32: 3, F16: 2, BF16: 1}[dt]  # a term is the sum of as many products
    _check(mx.mxfp4_linear_grad_input(g.to(gpu), c, s, K), _mm(gd, wq), _mm(gd.abs(), wq.abs()), parts * N)
    gw, gb = mx.linear_grad_weight(g.to(gpu), x8, xs, K)
    _check(gw, _mm(gd.t(), xq), _mm(gd.abs().t(), xq.abs()), parts * M)
    _check(gb, gd.sum(0), gd.abs().sum(0), M)
    again = mx.linear_grad_weight(g.to(gpu), x8, xs, K)
    assert torch.equal(again[0], gw) and torch.equal(again[1], gb)


def test_rows_that_are_not_finite(gpu):
    """In tiles of every size, at the ends of the operands too: only the rows and columns concerned become NaN."""
    from dimq_amd import mx
    for M, K, N in ((4097, 300, 2049), (1500, 300, 2050), (200, 300, 130)):
        announce(f"not finite {M}x{K} -> {N}")
        x, w = _acts(M, K, BF16, 5), _w(N, K, 6)
        x[M - 1, K - 1], x[3, 0] = float("nan"), float("inf")
        w[N - 1, K - 1] = float("inf")
        c, s = mx.quantize_mxfp4(w.to(gpu))
        y = mx.mxfp4_linear(x.to(gpu), c, s)
        bad = torch.isnan(y).cpu()
        assert bad[M - 1].all() and bad[3].all() and bad[:, N - 1].all()
        assert bad.sum() == 2 * N + M - 2
        g = _acts(M, N, BF16, 7)
        g[M - 1, 0] = float("inf")
        x8, xs = mx.compress_activation(x.to(gpu))
        gw, gb = mx.linear_grad_weight(g.to(gpu), x8, xs, K)
        assert torch.isinf(gb[0]) and torch.isfinite(gb[1:]).all()
        nan = torch.isnan(gw).cpu()
        assert nan[:, :32].all() and nan[:, K // 32 * 32:].all() and not nan[1:, 32:K // 32 * 32].any()


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("M,K,N", [(1, 64, 33), (5, 1000, 70), (16, 4128, 48), (13, 200, 16), (61, 776, 100), (250, 100, 50)])
def test_few_rows_as_many(gpu, dt, M, K, N):
    """The single launch quantizes x by itself: the same rows within a larger batch give the same values, whatever they
    hold (subnormal numbers, ties, whole blocks of zeros, blocks that are not finite), up to the order of the fp32 sums."""
    from dimq_amd import mx
    announce(f"few rows {dt} {M}x{K} -> {N}")
    x, w = _special(M, K, dt, M + K + N), _w(N, K, 3)
    c, s = mx.quantize_mxfp4(w.to(gpu))
    few = mx.mxfp4_linear(x.to(gpu), c, s, out_dtype=F32)
    xq, wq = omx.q4(x), omx.q4(w)
    ref, S = xq @ wq.t(), torch.nan_to_num(xq).abs() @ wq.abs().t()
    ok = S.max(dim=1).values < 1e37  # no sum overflows fp32
    _check(few[ok.to(gpu)], ref[ok], S[ok], K)
    many = mx.mxfp4_linear(x.repeat(300, 1).to(gpu), c, s, out_dtype=F32)[:M]
    _check(many[ok.to(gpu)], ref[ok], S[ok], K)


def test_each_block_alone(gpu):
    """One block of x against a one in the weights: the products are the codes' values, bit for bit, by either route."""
    from dimq_amd import mx
    w = torch.zeros(32, 32)
    w.fill_diagonal_(1.0)
    c, s = mx.quantize_mxfp4(w.to(gpu))
    for dt in (F32, F16, BF16):
        x = _special(2000, 32, dt, 17)
        want = omx.q4(x).float()
        for got in (mx.mxfp4_linear(x.to(gpu), c, s, out_dtype=F32),
                    torch.cat([mx.mxfp4_linear(r.to(gpu), c, s, out_dtype=F32) for r in x.split(16)])):
            got = got.cpu()
            # a product's smallest step: subnormal results may be flushed
            tiny = want.abs() < 2.0 ** -126
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            same = (got == want) | torch.isnan(want) | (tiny & (got == 0))
            assert same.all(), (dt, want[~same][:5], got[~same][:5])
