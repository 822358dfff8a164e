"""Microscaled 4-bit linear layers and 8-bit checkpoints against the float64 oracle (oracle/mx.py).

Codes and scales are compared bit for bit.  A product's operands are exact, so its error is that of the fp32 sums and of
the output's rounding: with S = sum |a b| over the r terms, at most (r + 8) 2^-23 S (each addition within one fp32 step of a
partial sum, the epilogue's few included) plus eps / 2 of the value.  GELU and its slope are within 3e-6 of the value (the
distribution function's 5e-7, an exponential of an argument up to 100 known to 2^-24, their products) plus 1e-37."""

import pytest
import torch

from oracle import mx as omx
from tests.conftest import announce

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _acts(rows, cols, dt, seed, spread=0.6):
    g = _gen(seed)
    return (torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(cols, generator=g) * spread)).to(dt)


def _check(got, ref, S, terms, extra=0.0):
    """got within its tolerance of the float64 ref; NaN and infinities where ref has them."""
    dt, got = got.dtype, got.detach().cpu().double()
    ref = ref.to(dt).double() if dt == torch.float16 and not torch.isfinite(ref.to(dt)).all() else ref
    assert got.shape == ref.shape
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    fin = torch.isfinite(ref)
    assert torch.equal(got[~fin & ~torch.isnan(ref)], ref[~fin & ~torch.isnan(ref)])
    tol = (terms + 8) * 2.0 ** -23 * S + torch.finfo(dt).eps / 2 * ref.abs() * 1.01 + torch.finfo(dt).smallest_normal * \
        torch.finfo(dt).eps + extra
    err = (got - ref).abs()
    worst = (err - tol)[fin].max() if fin.any() else torch.tensor(-1.0)
    assert worst <= 0, f"{(err / tol)[fin].max()} times the tolerance"


# ---- formats ----------------------------------------------------------------------------------------------------

SPECIAL = [0.0, -0.0, 1.0, -6.0, 2.0 ** -149, 2.0 ** -130, 3e38, -2.5, 1.75, 5.0, 0.25]


def _special(rows, cols, dt, seed):
    """Random magnitudes over the type's whole range, whole blocks of zeros and of tiny values, ties, and in some blocks
    a NaN or an infinity."""
    g = _gen(seed)
    lo, hi = (-24, 15) if dt == torch.float16 else (-149, 127)
    nb = -(-cols // 32)
    e = torch.randint(lo, hi + 1, (rows, nb, 1), generator=g).double()
    v = torch.randint(-64, 65, (rows, nb, 32), generator=g).double() / 64 * torch.exp2(e)
    pick = torch.rand(rows, nb, 1, generator=g)
    v = torch.where(pick < 0.1, 0.0, v)
    one = torch.zeros(rows, nb, 32, dtype=torch.bool)
    one[..., 7] = True
    v = torch.where((pick > 0.85) & one, torch.inf, v)
    v = torch.where((pick > 0.92) & one, torch.nan, v)
    return v.flatten(1)[:, :cols].to(dt)


def _same_codes(x, c4, s4, c8, s8):
    rows, cols = x.shape
    for bits, codes, scales, unpack in ((4, c4, s4, omx.unpack4), (8, c8, s8, omx.unpack8)):
        level, scale = omx.quantize(x, bits)
        assert torch.equal(scales.cpu(), scale)
        got, want = unpack(codes, scales, scale.shape[1] * 32), omx.values(level, scale, bits, scale.shape[1] * 32)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 64), (9, 100), (65, 1000), (40, 4096), (300, 8)])
def test_codes_and_values(gpu, dt, rows, cols):
    from dimq_amd import mx
    announce(f"quantize {dt} {rows}x{cols}")
    x = _special(rows, cols, dt, rows * 10007 + cols)
    c4, s4, c8, s8 = mx.quantize_and_compress(x.to(gpu))
    _same_codes(x, c4, s4, c8, s8)
    assert torch.equal(torch.stack([*mx.quantize_mxfp4(x.to(gpu))][:1]), torch.stack([c4]))
    a, b = mx.compress_activation(x.to(gpu))
    assert torch.equal(a, c8) and torch.equal(b, s8)
    for out in DTYPES:
        for got, ref in ((mx.dequantize_mxfp4(c4, s4, cols, out), omx.q4(x)),
                         (mx.decompress_activation(c8, s8, cols, out), omx.q8(x))):
            ref = ref.float().to(out)
            assert got.dtype == out and torch.equal(torch.isnan(got.cpu()), torch.isnan(ref))
            assert torch.equal(torch.nan_to_num(got.cpu()), torch.nan_to_num(ref))


def test_padding_is_zero(gpu):
    from dimq_amd import mx
    c4, s4, c8, s8 = mx.quantize_and_compress(torch.full((3, 33), 5.0, device=gpu))
    assert c4.shape == (3, 32) and s4.shape == (3, 2) and c8.shape == (3, 64) and s8.shape == (3, 2)
    assert (c4[:, 17:] == 0).all() and (c8[:, 33:] == 0).all() and (c4[:, 16] < 16).all()


@pytest.mark.parametrize("shape", [(0, 64), (4, 0), (2, 0, 32), (5,), (2, 3, 4, 40)])
def test_shapes(gpu, shape):
    from dimq_amd import mx
    announce(f"shape {shape}")
    x = _special(1, max(1, int(torch.tensor(shape).prod())), torch.float32, 3).flatten()[:int(torch.tensor(shape).prod())]
    x = x.view(shape).to(gpu)
    nb = -(-shape[-1] // 32)
    c4, s4, c8, s8 = mx.quantize_and_compress(x)
    assert c4.shape == (*shape[:-1], 16 * nb) and s8.shape == (*shape[:-1], nb) and c8.shape == (*shape[:-1], 32 * nb)
    y = mx.dequantize_mxfp4(c4, s4, shape[-1])
    assert y.shape == x.shape
    if x.numel():
        ref = omx.q4(x.cpu().reshape(-1, shape[-1])).view(shape).float()
        assert torch.equal(torch.nan_to_num(y.cpu()), torch.nan_to_num(ref))


def test_views_and_strides(gpu):
    from dimq_amd import mx
    big = _acts(70, 400, torch.bfloat16, 5).to(gpu)
    for x in (big[:, :256], big[3:, 8:264], big[:, 1:257], big[::2, :96], big.t(), big[:1].expand(9, 400),
              big[:, 5:6].expand(70, 64), big.view(7, 10, 400)[:, ::2, :320], big[:, ::3]):
        announce(f"view {tuple(x.shape)} {x.stride()}")
        flat = x.reshape(-1, x.shape[-1])
        c4, s4, c8, s8 = mx.quantize_and_compress(x)
        _same_codes(flat.cpu(), c4.reshape(flat.shape[0], -1), s4.reshape(flat.shape[0], -1),
                    c8.reshape(flat.shape[0], -1), s8.reshape(flat.shape[0], -1))
        y, p, q = torch.ops.dimq.gelu_forward(x)
        assert torch.equal(p, c8) and torch.equal(q, s8)
        _check(y.reshape(flat.shape), omx.gelu(flat), 3e-6 / 2 ** -23 * omx.gelu(flat).abs(), -7)


def test_more_than_two_to_the_31_elements(gpu):
    from dimq_amd import mx
    announce("2^31 elements")
    rows, cols = 66000, 32800
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=gpu)
    tail = _acts(3, cols, torch.bfloat16, 9).to(gpu)
    x[-3:] = tail
    c4, s4, c8, s8 = mx.quantize_and_compress(x)
    for got, want in zip((c4, s4, c8, s8), mx.quantize_and_compress(tail)):
        assert torch.equal(got[-3:], want) and int(got[:-3].max()) == 0
    y = mx.decompress_activation(c8, s8, cols, torch.bfloat16)
    assert torch.equal(y[-3:], mx.decompress_activation(c8[-3:], s8[-3:], cols, torch.bfloat16))


# ---- linear layer -----------------------------------------------------------------------------------------------

def _linear_case(M, K, N, dt, seed):
    x, w = _acts(M, K, dt, seed), torch.randn(N, K, generator=_gen(seed + 1)) / K ** 0.5
    return x, w, omx.q4(x), omx.q4(w)


SIZES = [(1, 32, 16), (1, 4096, 512), (2, 31, 3), (3, 1, 1), (5, 100, 64), (8, 544, 40), (15, 128, 17), (16, 1024, 256),
         (17, 768, 768), (33, 129, 130), (64, 512, 255), (65, 256, 300), (100, 1000, 77), (129, 640, 512), (197, 768, 768),
         (256, 256, 256), (257, 384, 1025), (511, 96, 640), (700, 1056, 514), (1030, 160, 2048)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear(gpu, dt, M, K, N):
    from dimq_amd import mx
    announce(f"linear {dt} {M}x{K} -> {N}")
    x, w, xq, wq = _linear_case(M, K, N, dt, M + K + N)
    b = torch.randn(N, generator=_gen(7))
    c, s = mx.quantize_mxfp4(w.to(gpu))
    ref, S = xq @ wq.t() + b.double(), xq.abs() @ wq.abs().t() + b.double().abs()
    _check(mx.mxfp4_linear(x.to(gpu), c, s, b.to(gpu)), ref, S, K)


@pytest.mark.parametrize("M", [1, 4, 16, 48, 200, 640])
@pytest.mark.parametrize("act", [None, "relu", "gelu"])
@pytest.mark.parametrize("out", DTYPES)
def test_epilogues(gpu, M, act, out):
    from dimq_amd import mx
    K, N = 320, 300
    announce(f"epilogue M={M} {act} {out}")
    x, w, xq, wq = _linear_case(M, K, N, torch.bfloat16, M)
    b, r = torch.randn(N, generator=_gen(7)).to(torch.float16), torch.randn(M, N, generator=_gen(8)).to(torch.bfloat16)
    c, s = mx.quantize_mxfp4(w.to(gpu))
    for bias, res in ((None, None), (b, r), (None, r.float()), (b.double(), None)):
        y = mx.mxfp4_linear(x.to(gpu), c, s, None if bias is None else bias.to(gpu), activation=act, out_dtype=out,
                            residual=None if res is None else res.to(gpu))
        assert y.dtype == out
        ref, S = xq @ wq.t(), xq.abs() @ wq.abs().t()
        for t in (bias, res):
            if t is not None:
                ref, S = ref + t.double(), S + t.double().abs()
        extra = 0.0
        if act == "relu":
            ref = ref.clamp_min(0)
        if act == "gelu":  # the slope stays below 1.13
            ref, S = omx.gelu(ref), S * 1.13
            extra = 3e-6 * ref.abs() + 1e-37
        _check(y, ref, S, K, extra)


def test_linear_inputs_that_are_not_finite(gpu):
    """They make their own rows NaN (their weights' columns), and no others."""
    from dimq_amd import mx
    for M in (3, 16, 40, 300):
        announce(f"not finite M={M}")
        x, w, _, _ = _linear_case(M, 160, 70, torch.float32, M)
        x[1, 100] = float("inf")
        x[M - 1, 159] = float("nan")
        w[69, 0] = float("nan")
        xq, wq = omx.q4(x), omx.q4(w)
        c, s = mx.quantize_mxfp4(w.to(gpu))
        _check(mx.mxfp4_linear(x.to(gpu), c, s), xq @ wq.t(), torch.nan_to_num(xq).abs() @ torch.nan_to_num(wq).abs().t(), 160)


def test_linear_extreme_scales(gpu):
    from dimq_amd import mx
    for M in (2, 130):
        announce(f"scales M={M}")
        x, w = _acts(M, 192, torch.float32, 3) * 2.0 ** 100, torch.randn(96, 192, generator=_gen(4)) * 2.0 ** -126
        x[:, 32:64] *= 2.0 ** -140
        xq, wq = omx.q4(x), omx.q4(w)
        c, s = mx.quantize_mxfp4(w.to(gpu))
        _check(mx.mxfp4_linear(x.to(gpu), c, s), xq @ wq.t(), xq.abs() @ wq.abs().t(), 192)


def test_linear_views(gpu):
    """Rows of a wider tensor, codes at an odd address, a 3-D input, a transposed one, none at all."""
    from dimq_amd import mx
    K, N = 128, 96
    big = _acts(60, 300, torch.float16, 1).to(gpu)
    w = torch.randn(N, K, generator=_gen(2))
    c, s = mx.quantize_mxfp4(w.to(gpu))
    room = torch.empty(c.numel() + 3, dtype=torch.uint8, device=gpu)
    off = room[3:].view(c.shape).copy_(c)
    wq = omx.q4(w)
    for x in (big[:, 4:132], big[:2, 9:137], big.view(5, 12, 300)[:, :, :128], big[:, :256:2], big[:0, :128]):
        announce(f"linear view {tuple(x.shape)} {x.stride()}")
        y = mx.mxfp4_linear(x, off, s)
        assert y.shape == (*x.shape[:-1], N)
        xq = omx.q4(x.reshape(-1, K).cpu())
        _check(y.reshape(-1, N), xq @ wq.t(), xq.abs() @ wq.abs().t(), K) if x.numel() else None


# ---- gradients --------------------------------------------------------------------------------------------------

GRADS = [(1, 32, 16), (2, 31, 3), (3, 1, 1), (7, 100, 65), (16, 1024, 256), (33, 129, 130), (65, 256, 300), (130, 1000, 77),
         (200, 512, 640), (257, 384, 1025), (515, 96, 770), (1500, 264, 288), (4000, 72, 40)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,K,N", GRADS)
def test_gradients(gpu, dt, M, K, N):
    from dimq_amd import mx
    announce(f"gradients {dt} {M}x{K} -> {N}")
    x, w, _, wq = _linear_case(M, K, N, dt, M * 3 + K + N)
    g = _acts(M, N, dt, 11, 1.0) * 2.0 ** -6
    gd = g.double()
    c, s = mx.quantize_mxfp4(w.to(gpu))
    _check(mx.mxfp4_linear_grad_input(g.to(gpu), c, s, K), gd @ wq, gd.abs() @ wq.abs(), 3 * N)
    _check(mx.mxfp4_linear_grad_input(g.to(gpu), c, s, K, torch.float32), gd @ wq, gd.abs() @ wq.abs(), 3 * N)
    x8, xs = mx.compress_activation(x.to(gpu))
    xq = omx.q8(x)
    for out in (torch.float32, torch.bfloat16):
        gw, gb = mx.linear_grad_weight(g.to(gpu), x8, xs, K, out_dtype=out)
        assert gw.dtype == out and gb.dtype == out
        _check(gw, gd.t() @ xq, gd.abs().t() @ xq.abs(), 3 * M)
        _check(gb, gd.sum(0), gd.abs().sum(0), M)
    gw2, none = mx.linear_grad_weight(g.to(gpu), x8, xs, K, bias=False)
    assert none is None and torch.equal(gw2, mx.linear_grad_weight(g.to(gpu), x8, xs, K)[0])


def test_gradients_that_are_not_finite(gpu):
    from dimq_amd import mx
    for dt in DTYPES:
        announce(f"gradients not finite {dt}")
        M, K, N = 100, 96, 68
        x, w, _, _ = _linear_case(M, K, N, dt, 2)
        g = _acts(M, N, dt, 12)
        g[5, 67], g[99, 3] = float("inf"), float("nan")
        x[7, 40] = float("nan")
        w[8, 95] = float("inf")
        wq, xq, gd = omx.q4(w), omx.q8(x), g.double()
        c, s = mx.quantize_mxfp4(w.to(gpu))
        big = torch.nan_to_num
        ref = gd @ wq
        got = mx.mxfp4_linear_grad_input(g.to(gpu), c, s, K, torch.float32)
        _check(got, ref, big(gd, 0, 0, 0).abs() @ big(wq).abs(), 3 * N)
        x8, xs = mx.compress_activation(x.to(gpu))
        gw, gb = mx.linear_grad_weight(g.to(gpu), x8, xs, K)
        _check(gw, gd.t() @ xq, big(gd, 0, 0, 0).abs().t() @ big(xq).abs(), 3 * M)
        _check(gb, gd.sum(0), big(gd, 0, 0, 0).abs().sum(0), M)


def test_gradients_of_no_rows(gpu):
    from dimq_amd import mx
    x8, xs = mx.compress_activation(torch.zeros(0, 40, device=gpu))
    gw, gb = mx.linear_grad_weight(torch.zeros(0, 24, device=gpu), x8, xs, 40)
    assert gw.shape == (24, 40) and not gw.any() and gb.shape == (24,) and not gb.any()


def test_gradient_views(gpu):
    from dimq_amd import mx
    big = _acts(64, 400, torch.bfloat16, 3).to(gpu)
    K, N = 96, 128
    w = torch.randn(N, K, generator=_gen(2))
    c, s = mx.quantize_mxfp4(w.to(gpu))
    wq = omx.q4(w)
    for g in (big[:, 3:131], big[::2, :128], big[:, :256:2], big[:1, :128].expand(64, 128), big[:, :1].expand(64, 128)):
        announce(f"gradient view {g.stride()}")
        x = _acts(g.shape[0], K, torch.bfloat16, 4)
        xq, gd = omx.q8(x), g.cpu().double()
        _check(mx.mxfp4_linear_grad_input(g, c, s, K), gd @ wq, gd.abs() @ wq.abs(), 3 * N)
        gw, gb = mx.linear_grad_weight(g, *mx.compress_activation(x.to(gpu)), K)
        _check(gw, gd.t() @ xq, gd.abs().t() @ xq.abs(), 3 * g.shape[0])
        _check(gb, gd.sum(0), gd.abs().sum(0), g.shape[0])


@pytest.mark.parametrize("bias,need", [(True, (1, 1, 1)), (False, (1, 1)), (True, (1, 0, 0)), (True, (0, 1, 0)),
                                       (True, (0, 0, 1)), (False, (0, 1)), (True, (1, 0, 1))])
def test_autograd(gpu, bias, need):
    """mx.linear over a 3-D input: each asked-for gradient, and only those."""
    from dimq_amd import mx
    x, w, xq, wq = _linear_case(60, 72, 50, torch.bfloat16, 21)
    b, g = torch.randn(50, generator=_gen(1)), _acts(60, 50, torch.bfloat16, 22)
    leaves = [x.view(5, 12, 72).to(gpu), w.to(gpu)] + ([b.to(gpu)] if bias else [])
    for t, n in zip(leaves, need):
        t.requires_grad_(bool(n))
    y = mx.linear(*leaves)
    ref = xq @ wq.t() + (b.double() if bias else 0)
    _check(y.reshape(60, 50), ref, xq.abs() @ wq.abs().t() + b.double().abs(), 72)
    y.backward(g.view(5, 12, 50).to(gpu))
    gd, x8 = g.double(), omx.q8(x)
    refs = (gd @ wq, gd.t() @ x8, gd.sum(0))
    sums = (gd.abs() @ wq.abs(), gd.abs().t() @ x8.abs(), gd.abs().sum(0))
    for t, n, r, S in zip(leaves, need, refs, sums):
        assert (t.grad is not None) == bool(n)
        if n:
            assert t.grad.dtype == t.dtype
            _check(t.grad.reshape(r.shape), r, S, 180)


def test_gradients_are_the_differences(gpu):
    """Where x and w are values of the format the layer is linear in each: moving one of them by a representable step
    moves g . y by the gradient times the step."""
    from dimq_amd import mx
    M, K, N = 24, 64, 40
    x, w, xq, wq = _linear_case(M, K, N, torch.float32, 31)
    x, w = xq.float().to(gpu).requires_grad_(), wq.float().to(gpu).requires_grad_()
    g = torch.randn(M, N, generator=_gen(5)).to(gpu)
    gx, gw = torch.autograd.grad(mx.linear(x, w), (x, w), g)
    base = mx.linear(x, w).double()
    for t, grad in ((x, gx), (w, gw)):
        for i, j in ((0, 0), (5, 17), (23, 63)):
            moved = t.detach().clone()
            moved[i, j] = -moved[i, j] if moved[i, j] != 0 else moved[i, 32 * (j // 32):32 * (j // 32) + 32].abs().max()
            y = mx.linear(moved, w) if t is x else mx.linear(x, moved)
            diff = ((y.double() - base) * g.double()).sum()
            step = (moved - t).double()[i, j]
            assert abs(diff - grad[i, j].double() * step) <= 1e-4 * (abs(diff) + (base.abs() * g.abs()).sum() * 1e-3)


def test_no_gradient_of_gradients(gpu):
    from dimq_amd import mx
    x = torch.randn(4, 32, device=gpu, requires_grad=True)
    w = torch.randn(8, 32, device=gpu, requires_grad=True)
    for y in (mx.linear(x, w), mx.gelu(x)):
        with pytest.raises(RuntimeError, match="not supported"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


# ---- GELU -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 33), (64, 96), (197, 777), (50, 2048)])
def test_gelu(gpu, dt, rows, cols):
    from dimq_amd import mx
    announce(f"gelu {dt} {rows}x{cols}")
    h = (torch.randn(rows, cols, generator=_gen(rows)) * 3).to(dt)
    if cols > 8:
        h[0, :6] = torch.tensor([0.0, -13.0, 40.0, -1e-3, 1e-20, -6.0]).to(dt)
    g = torch.randn(rows, cols, generator=_gen(2)).to(dt)
    hd = h.to(gpu).requires_grad_()
    y = mx.gelu(hd)
    ref = omx.gelu(h)
    _check(y, ref, torch.zeros(()), 0, 3e-6 * ref.abs() + 1e-37)
    gh, = torch.autograd.grad(y, hd, g.to(gpu))
    hq = omx.q8(h)
    slope = omx.gelu_slope(hq)
    # near the slope's zero its two terms cancel: 3e-6 of the larger
    part = (omx.gelu(hq) / torch.where(hq == 0, 1.0, hq)).abs() + (hq * torch.exp(-hq * hq / 2)).abs()
    _check(gh, g.double() * slope, torch.zeros(()), 0, 3e-6 * g.double().abs() * part + 1e-37)


def test_gelu_not_finite(gpu):
    from dimq_amd import mx
    h = torch.zeros(2, 64, device=gpu)
    h[0, 3], h[1, 40], h[1, 41] = float("inf"), float("nan"), 1.0
    h.requires_grad_()
    y = mx.gelu(h)
    assert torch.isinf(y[0, 3]) and torch.isnan(y[1, 40]) and torch.isnan(y).sum() == 1
    gh, = torch.autograd.grad(y, h, torch.ones_like(h))
    bad = torch.isnan(gh)
    assert bad[0, :32].all() and bad[1, 32:].all() and bad.sum() == 64


# ---- streams, graphs, order -------------------------------------------------------------------------------------

def _step(x, w, b, g):
    from dimq_amd import mx
    x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
    y = mx.gelu(mx.linear(x, w, b))
    return (y.detach(), *torch.autograd.grad(y, (x, w, b), g))


def test_same_bits_every_time_and_on_another_stream(gpu):
    g0 = _gen(3)
    x, w = torch.randn(1000, 320, generator=g0).to(gpu, torch.bfloat16), torch.randn(416, 320, generator=g0).to(gpu)
    b, g = torch.randn(416, generator=g0).to(gpu), torch.randn(1000, 416, generator=g0).to(gpu, torch.bfloat16)
    want = _step(x, w, b, g)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _step(x, w, b, g)
    side.synchronize()
    for a, c, d in zip(want, got, _step(x, w, b, g)):
        assert torch.equal(a, c) and torch.equal(a, d)


@pytest.mark.parametrize("M", [1, 16, 500])
def test_captured_in_a_graph(gpu, M):
    from dimq_amd import mx
    announce(f"graph M={M}")
    g0 = _gen(4)
    w = torch.randn(384, 640, generator=g0).to(gpu)
    c, s = mx.quantize_mxfp4(w)
    c8, s8 = mx.compress_activation(torch.randn(M, 640, generator=g0).to(gpu))
    x, g = torch.zeros(M, 640, device=gpu, dtype=torch.bfloat16), torch.zeros(M, 384, device=gpu, dtype=torch.bfloat16)

    def work():
        return (mx.mxfp4_linear(x, c, s), mx.mxfp4_linear_grad_input(g, c, s, 640),
                *mx.linear_grad_weight(g, c8, s8, 640))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(3):
        x.copy_(torch.randn(M, 640, generator=_gen(i)))
        g.copy_(torch.randn(M, 384, generator=_gen(i + 9)))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, work()):
            assert torch.equal(a, b)


# ---- refusals on the device -------------------------------------------------------------------------------------

def test_refusals(gpu):
    from dimq_amd import mx
    x, w = torch.randn(4, 64, device=gpu), torch.randn(8, 64, device=gpu)
    c, s = mx.quantize_mxfp4(w)
    c8, s8 = mx.compress_activation(x)
    g = torch.randn(4, 8, device=gpu)
    for call, text in (
            (lambda: mx.quantize_mxfp4(x.double()), "must be fp32, fp16 or bf16, not torch.float64"),
            (lambda: mx.quantize_mxfp4(x.int()), "not torch.int32"),
            (lambda: mx.quantize_mxfp4(x[0, 0]), "at least one dimension"),
            (lambda: mx.mxfp4_linear(x[:, :32], c, s), "rows of 32 have codes"),
            (lambda: mx.mxfp4_linear(x, c, s[:4]), "rows of 64 have codes"),
            (lambda: mx.mxfp4_linear(x, c.to(torch.int8), s), "codes must be uint8"),
            (lambda: mx.mxfp4_linear(x, c, s.int()), "scales must be uint8"),
            (lambda: mx.mxfp4_linear(x, c.cpu(), s), "must be on cuda"),
            (lambda: mx.mxfp4_linear(x, c, s, torch.zeros(7, device=gpu)), "bias numel must equal out_features"),
            (lambda: mx.mxfp4_linear(x, c, s, torch.zeros(8)), "bias must be CUDA"),
            (lambda: mx.mxfp4_linear(x, c, s, residual=x), "must equal the output shape"),
            (lambda: mx.mxfp4_linear(x, c, s, out_dtype=torch.float64), "output dtype"),
            (lambda: mx.dequantize_mxfp4(c, s, 65), "rows of 65 have codes"),
            (lambda: mx.dequantize_mxfp4(c, s, 64, torch.int32), "output dtype"),
            (lambda: mx.decompress_activation(c, s, 64), "codes must be int8"),
            (lambda: mx.mxfp4_linear_grad_input(x, c, s, 64), "must equal the weights' rows 8"),
            (lambda: mx.linear_grad_weight(g[:3], c8, s8, 64), "the gradient has 3 rows, the checkpoint 4"),
            (lambda: mx.linear_grad_weight(g.double(), c8, s8, 64), "not torch.float64"),
            (lambda: mx.linear(x, w[:, :32]), "must equal the weight's"),
            (lambda: mx.linear(x, w.double()), "not torch.float64"),
            (lambda: mx.linear(x, w, torch.zeros(8, device=gpu, dtype=torch.int32)), "bias must be"),
            (lambda: mx.gelu(x.double()), "not torch.float64")):
        with pytest.raises(RuntimeError, match=text):
            call()
