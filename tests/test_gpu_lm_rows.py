"""RMS norm, token log probabilities and distillation from top logits against the float64 oracle (oracle/lm.py).

Tolerances, e = 2^-24 (an fp32 rounding):

* a sum over a row is formed by 64 threads or more, each adding at most n = 64 + cols / 256 terms in turn, and then over the
  threads: relative to the sum of magnitudes, (n + 16) e;
* y = h s w: half that from the mean of squares, then 8 roundings; gradients of the norm: (2 n + 64) e of the magnitudes
  they are made of; each output type's own rounding, eps / 2, on top;
* exp(d) is known to (1.5 |d| + 4) e relative, so with D = sum p |d| over a row (d = x - max) log s is within
  (n + 16 + 1.5 D + 4) e + |log s| e, a log probability within that plus 2 e (|d| + |log s|), and the entropy within that
  plus D's own (n + 20) e + 1.5 e sum p d^2."""

import pytest
import torch

from oracle import lm
from tests.conftest import announce

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _terms(cols):
    return 64 + cols / 256


def _tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def _close(got, ref, tol, name=""):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), name
    same = (got == ref) | torch.isnan(ref)
    err = torch.where(same, 0.0, (got - ref).abs() - tol)
    assert (err <= 0).all(), f"{name}: {err.max()} above the tolerance"


def _half(ref, dt):
    return torch.finfo(dt).eps / 2 * ref.abs() * 1.0001 + _tiny(dt)


# ---- RMS norm -----------------------------------------------------------------------------------------------------

WIDTHS = [1, 7, 8, 63, 512, 513, 520, 1000, 1024, 1032, 2048, 2047, 4096, 4104, 8192, 8200, 8191, 32768, 40000, 33001]


def _rows(rows, cols, dt, seed):
    g = _gen(seed)
    return (torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(cols, generator=g) * 0.6)).to(dt)


def _check_norm(x, w, eps, r, y, h):
    ref, want_h = lm.rms_norm(x, w, eps, r)
    if r is not None:
        assert torch.equal(h.cpu(), want_h)
    _close(y, ref, (_terms(x.shape[-1]) + 32) * E * ref.abs() + _half(ref, y.dtype), "y")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_rms_norm(gpu, cols, dt):
    from dimq_amd import ops
    announce(f"rms_norm {cols} {dt}")
    for rows, residual, wdt, odt in ((5, True, dt, None), (1, False, torch.float32, torch.float32),
                                     (3, True, None, torch.bfloat16)):
        x, r = _rows(rows, cols, dt, 1).to(gpu), _rows(rows, cols, dt, 2).to(gpu) if residual else None
        w = None if wdt is None else (1 + 0.3 * torch.randn(cols, generator=_gen(3))).to(wdt).to(gpu)
        got = ops.rms_norm(x, w, 1e-5, residual=r, out_dtype=odt)
        y, h = got if residual else (got, None)
        assert y.dtype == (odt or dt)
        _check_norm(x, w, 1e-5, r, y, h)


@pytest.mark.parametrize("rows,cols", [(2500, 64), (9000, 8), (2300, 1500), (70000, 16)])
def test_rms_norm_more_rows_than_work_groups(gpu, rows, cols):
    from dimq_amd import ops
    announce(f"rms_norm rows {rows} {cols}")
    x, r = _rows(rows, cols, torch.bfloat16, 1).to(gpu), _rows(rows, cols, torch.bfloat16, 2).to(gpu)
    y, h = ops.rms_norm(x, None, 1e-6, residual=r)
    _check_norm(x, None, 1e-6, r, y, h)


@pytest.mark.parametrize("dt", DTYPES)
def test_rms_norm_strides_and_places(gpu, dt):
    """Rows of a larger tensor, odd starts, transposed and 3-D inputs: the output is contiguous, the neighbours stay."""
    from dimq_amd import ops
    announce(f"rms_norm strides {dt}")
    big = _rows(40, 300, dt, 1).to(gpu)
    for x in (big[3:9, 8:264], big[3:9, 5:200], big[::2, 1:], big.t(), big[:, :256].view(4, 10, 256), big[4], big[7:7]):
        y = ops.rms_norm(x, None, 1e-6)
        assert y.shape == x.shape and y.is_contiguous()
        ref, _ = lm.rms_norm(x, None, 1e-6)
        _close(y, ref, (_terms(300) + 32) * E * ref.abs() + _half(ref, dt))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("cols", [1, 40, 1000, 1001, 4096, 4100, 16384, 33000])
def test_rms_norm_e4m3(gpu, cols, dt):
    from dimq_amd import ops
    announce(f"rms_norm_e4m3 {cols} {dt}")
    x, r = _rows(6, cols, dt, 1), _rows(6, cols, dt, 2)
    x[2], r[2] = 0, 0
    x[3, 0] = torch.inf
    x[4, cols // 2] = torch.nan
    x, r = x.to(gpu), r.to(gpu)
    w = (1 + 0.3 * torch.randn(cols, generator=_gen(3))).to(gpu)
    q, s, h = ops.rms_norm_e4m3(x, w, 1e-6, residual=r)
    assert q.dtype == torch.float8_e4m3fn and s.shape == (6,)
    ref, want_h = lm.rms_norm(x, w, 1e-6, r)
    assert torch.equal(torch.nan_to_num(h.cpu(), 7.0), torch.nan_to_num(want_h, 7.0))
    s, q = s.cpu().double(), q.cpu().float().double()
    assert torch.isnan(s).tolist() == [False, False, False, True, True, False]
    assert s[2] == 0 and (q[2] == 0).all()
    d = (_terms(cols) + 32) * E
    for i in (0, 1, 5):
        top = ref[i].abs().max() / 448
        assert abs(s[i] - top) <= 2 * d * top
        v = ref[i] / top
        assert ((q[i] - v).abs() <= lm.e4m3_step(v) / 2 + 4 * d * v.abs()).all()


def test_rms_norm_e4m3_of_tiny_and_huge_rows(gpu):
    """|y| down to fp32's least normal numbers and up to its largest: scales stay normal, codes stay below 448."""
    from dimq_amd import ops
    announce("rms_norm_e4m3 range")
    x = torch.ones(3, 64, device=gpu)
    x[:, ::2] = -0.5
    for factor in (2.0 ** -120, 2.0 ** -126, 2.0 ** 120):
        w = torch.full((64,), factor, device=gpu)
        q, s = ops.rms_norm_e4m3(x, w, 0.0)
        ref, _ = lm.rms_norm(x, w, 0.0)
        scale = (ref.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
        assert ((s.cpu().double() - scale).abs() <= 100 * E * scale).all()
        v = ref / scale[:, None]
        assert ((q.cpu().float().double() - v).abs() <= lm.e4m3_step(v) / 2 + 400 * E * v.abs()).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (9, 7), (37, 512), (5, 1000), (2100, 40), (3, 4096), (1100, 1040), (6, 8200), (4, 33000)])
def test_rms_norm_gradients(gpu, rows, cols, dt):
    from dimq_amd import ops
    announce(f"rms_norm grad {rows} {cols} {dt}")
    x, r = _rows(rows, cols, dt, 1).to(gpu).requires_grad_(), _rows(rows, cols, dt, 2).to(gpu).requires_grad_()
    w = (1 + 0.3 * torch.randn(cols, generator=_gen(3))).to(gpu).requires_grad_()
    gy, gh = _rows(rows, cols, dt, 4).to(gpu), _rows(rows, cols, dt, 5).to(gpu)
    n = _terms(cols)

    def check(h, g_y, g_h, got_x, got_w):
        ref, ref_w, terms = lm.rms_norm_grads(h, w, 1e-5, g_y, g_h)
        _close(got_x, ref, (2 * n + 64) * E * terms + _half(ref, dt), "gx")
        if got_w is not None:
            mag = lm.rms_norm_grads(h.abs(), w, 1e-5, g_y.abs(), None)[1]
            _close(got_w, ref_w, (rows + n + 32) * E * mag + _half(ref_w, w.dtype), "gw")

    y, h = ops.rms_norm(x, w, 1e-5, residual=r)
    gx, gr, gw = torch.autograd.grad((y, h), (x, r, w), (gy, gh), retain_graph=True)
    assert torch.equal(gx, gr)
    check(h, gy, gh, gx, gw)
    gx2, = torch.autograd.grad(y, x, gy, retain_graph=True)
    check(h, gy, None, gx2, None)
    gr3, = torch.autograd.grad(h, r, gh, retain_graph=True)
    assert torch.equal(gr3, gh)
    # fp32 outputs of the layer, without a residual
    y = ops.rms_norm(x, w, 1e-5, out_dtype=torch.float32)
    g32 = gy.float() * 1.5
    gx, gw = torch.autograd.grad(y, (x, w), g32)
    check(x, g32, None, gx, gw)
    # a weight alone, and a broadcast gradient
    y = ops.rms_norm(x.detach(), w, 1e-5)
    gw, = torch.autograd.grad(y.sum(), w)
    mag = lm.rms_norm_grads(x.abs(), w, 1e-5, torch.ones_like(gy), None)[1]
    _close(gw, lm.rms_norm_grads(x, w, 1e-5, torch.ones_like(gy), None)[1], (rows + n + 32) * E * mag + 1e-30, "gw of ones")


def test_rms_norm_gradient_by_differences(gpu):
    from dimq_amd import ops
    announce("rms_norm differences")
    x = _rows(2, 24, torch.float32, 1).to(gpu).requires_grad_()
    r = _rows(2, 24, torch.float32, 2).to(gpu)
    w = (1 + 0.3 * torch.randn(24, generator=_gen(3))).to(gpu)
    c, d = _rows(2, 24, torch.float32, 4).to(gpu), _rows(2, 24, torch.float32, 5).to(gpu)
    y, h = ops.rms_norm(x, w, 1e-5, residual=r)
    g, = torch.autograd.grad((y, h), x, (c, d))

    def f(v):
        y, _ = lm.rms_norm(v, w, 1e-5)
        return (y * lm.f64(c)).sum() + (lm.f64(v) * lm.f64(d)).sum()

    base = lm.f64(x) + lm.f64(r)
    for i in range(0, 48, 5):
        step = torch.zeros(48, dtype=torch.float64)
        step[i] = 1e-6
        diff = (f(base + step.view(2, 24)) - f(base - step.view(2, 24))) / 2e-6
        # differences: 1e-16 * 100 / 1e-6, and the fp32 gradient
        assert abs(diff - g.cpu().double().view(-1)[i]) <= 1e-6 + 200 * E * (1 + abs(diff))


def test_rms_norm_gradients_of_some_inputs(gpu):
    """Any of the three absent or without a gradient of its own; the same tensor twice; accumulation into .grad."""
    from dimq_amd import ops
    announce("rms_norm some inputs")
    leaf = lambda seed, on: _rows(4, 48, torch.float32, seed).to(gpu).requires_grad_(on)  # noqa: E731
    gy, gh = _rows(4, 48, torch.float32, 8).to(gpu), _rows(4, 48, torch.float32, 9).to(gpu)
    for has_w in (None, False, True):
        for on_x, on_r in ((True, True), (True, False), (False, True), (False, False)):
            w = None if has_w is None else (1 + 0.1 * torch.randn(48, generator=_gen(1))).to(gpu).requires_grad_(has_w)
            x, r = leaf(2, on_x), leaf(3, on_r)
            y, h = ops.rms_norm(x, w, 1e-5, residual=r)
            if not (on_x or on_r or has_w):
                assert not y.requires_grad
                continue
            torch.autograd.backward((y, h), (gy, gh)) if h.requires_grad else y.backward(gy)
            ref, ref_w, terms = lm.rms_norm_grads(h, w, 1e-5, gy, gh)
            for t, on in ((x, on_x), (r, on_r)):
                assert (t.grad is not None) == on
                if on:
                    _close(t.grad, ref, 300 * E * terms + _half(ref, torch.float32))
            if on_x and on_r:
                assert x.grad.data_ptr() != r.grad.data_ptr()
            if has_w:
                _close(w.grad, ref_w, 400 * E * lm.rms_norm_grads(h.abs(), w, 1e-5, gy.abs(), None)[1] + 1e-30)
    x = leaf(2, True)
    y, h = ops.rms_norm(x, None, 1e-5, residual=x)
    torch.autograd.backward((y, h), (gy, gh))
    ref, _, terms = lm.rms_norm_grads(h, None, 1e-5, gy, gh)
    _close(x.grad, 2 * ref, 700 * E * terms + _half(2 * ref, torch.float32))


def test_rms_norm_of_a_row_added_to_itself(gpu):
    """The residual may be the input itself: its gradient is both's."""
    from dimq_amd import ops
    announce("norm of x + x")
    x = torch.randn(9, 520, generator=_gen(5)).to(gpu).requires_grad_()
    two = x.detach().clone().requires_grad_()
    gy, gh = (torch.randn(9, 520, generator=_gen(s)).to(gpu) for s in (6, 7))
    got, = torch.autograd.grad(ops.rms_norm(x, residual=x), x, (gy, gh))
    ref, = torch.autograd.grad(ops.rms_norm(two, residual=x.detach()), two, (gy, gh))
    assert torch.equal(got, 2 * ref)
    # the sum alone, and the norm alone
    got, = torch.autograd.grad(ops.rms_norm(x, residual=x)[1], x, gh)
    assert torch.equal(got, 2 * gh)
    a, b = torch.autograd.grad(ops.rms_norm(x, residual=two)[1], (x, two), gh)
    assert torch.equal(a, gh) and torch.equal(b, gh)


def test_rms_norm_no_rows(gpu):
    from dimq_amd import ops
    x, w = torch.zeros(0, 16, device=gpu, requires_grad=True), torch.ones(16, device=gpu, requires_grad=True)
    y = ops.rms_norm(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert gx.shape == (0, 16) and (gw == 0).all()


def test_rms_norm_module(gpu):
    from dimq_amd.modules import DIMQRMSNorm
    announce("DIMQRMSNorm")
    torch.manual_seed(0)
    ref = torch.nn.RMSNorm(96, eps=1e-5)
    ref.weight.data.uniform_(0.5, 1.5)
    m = DIMQRMSNorm.from_rms_norm(ref).to(gpu)
    x, r = _rows(4, 96, torch.float32, 1).to(gpu), _rows(4, 96, torch.float32, 2).to(gpu)
    _check_norm(x, m.weight, 1e-5, None, m(x), None)
    y, h = m(x, residual=r)
    _check_norm(x, m.weight, 1e-5, r, y, h)
    q, s, h8 = m.e4m3(x, residual=r)
    assert q.dtype == torch.float8_e4m3fn and torch.equal(h8, h)
    m.eps = None  # torch's default: the type's epsilon
    _check_norm(x, m.weight, torch.finfo(torch.float32).eps, None, m(x), None)


# ---- log probabilities --------------------------------------------------------------------------------------------

def _logits(rows, vocab, dt, seed):
    g = _gen(seed)
    x = torch.randn(rows, vocab, generator=g) * 2.5
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 8), generator=g), torch.rand(rows, 8, generator=g) * 12)
    return x.to(dt)


def _score_tols(x):
    """(of log s + ..., of the entropy, d, log s)"""
    bad = lm.no_distribution(x)
    v = torch.where(bad[:, None], 0.0, lm.f64(x))
    d = v - v.amax(-1, keepdim=True)
    p, ls = torch.softmax(v, -1), torch.logsumexp(d, -1)
    dd = torch.where(p > 0, d, 0.0)
    D, n = (p * dd.abs()).sum(-1), _terms(x.shape[1])
    of_ls = (n + 20 + 1.5 * D + ls) * E
    return of_ls, of_ls + ((n + 24) * D + 1.5 * (p * dd * dd).sum(-1) + ls) * E, dd, ls


def _check_scores(x, tokens, top, got):
    lp, H, tlp, tid = (t.cpu() for t in got)
    want = lm.scores(x, tokens, top)
    of_ls, of_h, d, ls = _score_tols(x)
    wide = lambda v: torch.where(torch.isfinite(v), v.abs(), 0.0)  # noqa: E731
    # |d| <= |log p| + log s
    _close(lp, want[0], of_ls + 2 * E * (wide(want[0]) + 2 * ls), "logprobs")
    _close(H, want[1], of_h, "entropy")
    assert torch.equal(tid, want[3])
    _close(tlp, want[2], (of_ls + 4 * E * ls)[:, None] + 2 * E * wide(want[2]), "top")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 5, 5), (2, 130, 128), (7, 1000, 20), (4, 2048, 1), (1, 50021, 64),
                                            (3, 128000, 128), (1030, 333, 8), (1100, 4099, 5), (5, 32768, 0), (2, 8193, 40)])
def test_token_logprobs(gpu, rows, vocab, top, dt):
    from dimq_amd import ops
    announce(f"token_logprobs {rows} {vocab} {top} {dt}")
    x = _logits(rows, vocab, dt, rows + vocab).to(gpu)
    t = torch.randint(0, vocab, (rows,), generator=_gen(5)).to(gpu)
    t[rows // 2:] = x[rows // 2:].float().argmax(1)
    _check_scores(x, t, top, ops.token_logprobs(x, t, top))
    t[0] = -100
    _check_scores(x, t.int(), top, ops.token_logprobs(x, t.int(), top))


@pytest.mark.parametrize("rows", [9, 1100])
@pytest.mark.parametrize("dt", DTYPES)
def test_token_logprobs_of_masked_rows(gpu, dt, rows):
    """-infinity, the type's lowest number, NaN and infinities in a row's logits; one row cut over several work-groups and
    rows of one work-group."""
    from dimq_amd import ops
    announce(f"token_logprobs masks {dt} {rows}")
    vocab, top = 9000, 12
    x = _logits(rows, vocab, dt, 3)
    low = torch.finfo(dt).min
    x[0] = -torch.inf
    x[1, 5:] = -torch.inf       # fewer than `top` tokens left
    x[2] = low
    x[3, 100:] = low
    x[4, 8500] = torch.nan
    x[5, 17] = torch.inf
    x[6, ::2] = -torch.inf
    x[7, :] = -torch.inf
    x[7, 8999] = low
    x[8] = 0.25                 # all alike: every logit ties
    t = torch.tensor([3, 7, 0, 150, 1, 17, 2, 8999, 8000] + [4] * (rows - 9))
    got = ops.token_logprobs(x.to(gpu), t.to(gpu), top)
    _check_scores(x, t, top, got)
    assert got[0][1].item() == -torch.inf and got[3][0].tolist() == [-1] * top
    assert got[3][2].tolist() == list(range(top)) and got[3][8].tolist() == list(range(top))


@pytest.mark.parametrize("rows", [2, 1030])
def test_token_logprobs_ties(gpu, rows):
    """Many equal logits around the last alternative, on both sides of the candidates' capacity."""
    from dimq_amd import ops
    announce(f"token_logprobs ties {rows}")
    g = _gen(7)
    for levels in (2, 5, 40, 3000):
        x = (torch.randint(0, levels, (rows, 6001), generator=g).float() / 8).to(gpu)
        t = torch.zeros(rows, dtype=torch.long, device=gpu)
        _check_scores(x, t, 33, ops.token_logprobs(x, t, 33))
    x = torch.zeros(rows, 6001, device=gpu)
    x[:, ::2] = -0.0  # equal to 0
    assert (ops.token_logprobs(x, t, 50)[3].cpu() == torch.arange(50)).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_token_logprobs_strides_and_places(gpu, dt):
    from dimq_amd import ops
    announce(f"token_logprobs strides {dt}")
    big = _logits(24, 1300, dt, 9).to(gpu)
    for x in (big[2:9, 3:1203], big[::3, 1:], big[:, 8:1288], big.t().contiguous().t(), big[5:5]):
        t = torch.arange(x.shape[0], device=gpu)
        _check_scores(x, t, 9, ops.token_logprobs(x, t, 9))
    x = big[:, :1200].reshape(4, 6, 1200)
    t = torch.arange(24, device=gpu).view(4, 6)
    got = ops.token_logprobs(x, t, 3)
    assert got[0].shape == (4, 6) and got[2].shape == (4, 6, 3)
    _check_scores(x.reshape(24, 1200), t.view(-1), 3, [v.flatten(0, 1) for v in got])
    one = ops.token_logprobs(big[0], torch.tensor(7, device=gpu), 2)
    assert one[0].shape == () and one[3].shape == (2,)


def _check_score_grad(x, t, a, b, gx):
    keep = ~((a.cpu() == 0) | (t.cpu() < 0)) | ~(b.cpu() == 0)
    ref = torch.where(keep[:, None], lm.score_grads(x, t, a, b), 0.0)
    of_ls, of_h, d, ls = _score_tols(x)
    p = torch.softmax(lm.f64(x), -1)
    A, B = lm.f64(a).abs() * (t.cpu() >= 0), lm.f64(b).abs()
    lp = torch.where(p > 0, d - ls[:, None], 0.0).abs()
    H = torch.where(p > 0, p * lp, 0.0).sum(-1)
    rel = of_ls[:, None] + (4 * (d.abs() + ls[:, None]) + 8) * E   # of p
    tol = p * (A[:, None] + B[:, None] * (lp + H[:, None])) * (rel + 8 * E) + p * B[:, None] * (rel + of_h[:, None])
    tol = torch.where(torch.isfinite(tol), tol, 0.0) + A[:, None] * 2 * E + 1e-37
    _close(gx, ref, tol + _half(ref, x.dtype), "gx")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 6), (5, 1000), (2, 50021), (1040, 515), (1, 131072)])
def test_token_logprobs_gradients(gpu, rows, vocab, dt):
    from dimq_amd import ops
    announce(f"token_logprobs grad {rows} {vocab} {dt}")
    x = _logits(rows, vocab, dt, 11).to(gpu).requires_grad_()
    t = torch.randint(0, vocab, (rows,), generator=_gen(5)).to(gpu)
    if rows > 2:
        t[1] = -1
    a, b = torch.randn(rows, generator=_gen(6)).to(gpu), torch.randn(rows, generator=_gen(7)).to(gpu)
    lp, H, _, _ = ops.token_logprobs(x, t, min(3, vocab))
    gx, = torch.autograd.grad((lp, H), x, (a, b), retain_graph=True)
    _check_score_grad(x, t, a, b, gx)
    gx, = torch.autograd.grad(lp, x, a, retain_graph=True)
    _check_score_grad(x, t, a, torch.zeros_like(b), gx)
    gx, = torch.autograd.grad(H.sum(), x)  # a broadcast gradient
    _check_score_grad(x, t, torch.zeros_like(a), torch.ones_like(b), gx)


def test_token_logprobs_gradient_of_rows_without_one(gpu):
    """A row that is all masked and whose token is none gets zeros, not NaNs; a masked token's p is 0."""
    from dimq_amd import ops
    announce("token_logprobs grad masks")
    x = _logits(4, 700, torch.float32, 1)
    x[0] = -torch.inf
    x[1, 3] = torch.nan
    x[2, 100:] = -torch.inf
    x = x.to(gpu).requires_grad_()
    t = torch.tensor([-1, -1, 5, 6], device=gpu)
    lp, H, _, _ = ops.token_logprobs(x, t)
    a = torch.ones(4, device=gpu)
    gx, = torch.autograd.grad(lp, x, a, retain_graph=True)
    assert (gx[:2] == 0).all()
    _check_score_grad(x[2:], t[2:], a[2:], torch.zeros(2), gx[2:])
    gx, = torch.autograd.grad(H, x, torch.tensor([0.0, 0.0, 1.0, 0.5], device=gpu))
    assert (gx[:2] == 0).all()
    _check_score_grad(x[2:], t[2:], torch.zeros(2), torch.tensor([1.0, 0.5]), gx[2:])


def test_token_logprobs_gradient_of_strided_logits(gpu):
    from dimq_amd import ops
    announce("token_logprobs grad strides")
    big = _logits(6, 1301, torch.bfloat16, 2).to(gpu).requires_grad_()
    t = torch.arange(6, device=gpu)
    a = torch.ones(6, device=gpu)
    gx, = torch.autograd.grad(ops.token_logprobs(big[:, 3:1203], t)[0], big, a)
    assert (gx[:, :3] == 0).all() and (gx[:, 1203:] == 0).all()
    _check_score_grad(big[:, 3:1203], t, a, torch.zeros(6), gx[:, 3:1203])


# ---- distillation -------------------------------------------------------------------------------------------------

def _teacher(x, k, seed):
    g = _gen(seed)
    t = x.float() + torch.randn(x.shape, generator=g)
    return torch.topk(t, k, dim=-1)


def _check_distill(x, values, ids, tau, reduction, loss, gx, g):
    """gx: the gradient for the upstream g (a number, or one a row for "none")."""
    row, some, grad = lm.distill(x, values, ids, tau)
    n = max(1, int(some.sum()))
    z = lm.f64(x) / tau
    z = torch.where(torch.isfinite(z).all(-1, keepdim=True) | True, z, z)
    d = z - z.amax(-1, keepdim=True)
    p, ls = torch.softmax(z, -1), torch.logsumexp(d, -1)
    dd = torch.where(p > 0, d, 0.0)
    of_ls = (_terms(x.shape[1]) + 20 + 2.5 * (p * dd.abs()).sum(-1) + ls) * E
    keep = (ids.cpu() >= 0) & (lm.f64(values) != -torch.inf)
    v = torch.where(keep, lm.f64(values) / tau, -torch.inf)
    v = torch.where(some[:, None], v, 0.0)
    dt_ = torch.where(keep, v - v.amax(-1, keepdim=True), 0.0)
    lt = torch.log_softmax(v, -1)
    pt = torch.where(keep, torch.exp(lt), 0.0)
    dq = dd.gather(1, ids.cpu().long().clamp(min=0)).abs()
    # the teacher's p to (4 |d| + 2 |log s| + 40) e relative, its log p and the student's log q absolutely
    rel_t = (4 * dt_.abs() + 2 * ids.shape[1] + 40) * E
    lq = dq + ls[:, None]
    each = tau ** 2 * (pt * (rel_t * (torch.where(pt > 0, lt, 0.0).abs() + lq + 1) + of_ls[:, None] + 4 * E * lq + 8 * E)).sum(-1)
    each = torch.where(some, each, 0.0)
    if reduction == "none":
        _close(loss, row, each + 1e-37, "loss")
        scale = lm.f64(g)[:, None]
    else:
        by = n if reduction == "mean" else 1
        _close(loss, row.sum() / by, (each.sum() + row.abs().sum() * (row.numel() / 1024 + 16) * E) / by + 1e-37, "loss")
        scale = torch.full((row.numel(), 1), float(g) / by, dtype=torch.float64)
    ref = grad * scale
    tol = p * (of_ls[:, None] + (4 * (dd.abs() + ls[:, None]) + 12) * E)
    tol.scatter_add_(1, ids.cpu().long().clamp(min=0), pt * (rel_t + (2 * ids.shape[1] + 8) * E))
    tol = torch.where(some[:, None], tol, 0.0) * tau * scale.abs()
    _close(gx, ref, tol + _half(ref, x.dtype) + 1e-37, "gx")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,vocab,k,tau,reduction", [
    (1, 1, 1, 1.0, "mean"), (5, 40, 40, 0.5, "sum"), (7, 1000, 20, 2.0, "none"), (2, 50021, 64, 1.0, "mean"),
    (1050, 515, 5, 4.0, "mean"), (3, 128000, 300, 2.0, "sum"), (1, 4104, 1, 1.0, "none")])
def test_distillation(gpu, rows, vocab, k, tau, reduction, dt):
    from dimq_amd import qat
    announce(f"distillation {rows} {vocab} {k} {dt}")
    x = _logits(rows, vocab, dt, 13)
    values, ids = _teacher(x, k, 4)
    if rows > 2:
        ids[1] = -1            # a row without entries
        ids[2, k // 2:] = -1   # one with fewer
    x = x.to(gpu).requires_grad_()
    for vdt, idt in ((torch.float32, torch.int64), (torch.bfloat16, torch.int32)):
        v, i = values.to(vdt).to(gpu), ids.to(idt).to(gpu)
        loss = qat.top_logits_distillation_loss(x, v, i, tau, reduction)
        g = torch.randn(rows, generator=_gen(8)).to(gpu) if reduction == "none" else torch.tensor(1.7, device=gpu)
        gx, = torch.autograd.grad(loss, x, g)
        _check_distill(x, v, i, tau, reduction, loss, gx, g if reduction == "none" else 1.7)


@pytest.mark.parametrize("rows,vocab", [(2, 5000), (1, 40000)])
def test_distillation_of_most_entries(gpu, rows, vocab):
    """As many teacher entries as there may be, tokens among them more than once."""
    from dimq_amd import qat
    announce(f"distillation of 4096 entries, {rows} {vocab}")
    x = _logits(rows, vocab, torch.float32, 19).to(gpu).requires_grad_()
    values = torch.randn(rows, 4096, generator=_gen(3)).to(gpu)
    ids = torch.randint(0, vocab, (rows, 4096), generator=_gen(4)).to(gpu)
    loss = qat.top_logits_distillation_loss(x, values, ids, 2.0, "none")
    g = torch.randn(rows, generator=_gen(8)).to(gpu)
    gx, = torch.autograd.grad(loss, x, g)
    _check_distill(x, values, ids, 2.0, "none", loss, gx, g)


def test_distillation_special_rows(gpu):
    from dimq_amd import qat
    announce("distillation special")
    x = _logits(8, 600, torch.float32, 1)
    values, ids = _teacher(x, 6, 2)
    values[0, 3:] = -torch.inf      # left out
    values[1] = -torch.inf          # nothing left
    ids[2, 4] = ids[2, 1]           # the same token twice: both count
    ids[2, 5] = ids[2, 1]
    x[3] = torch.nan
    ids[3] = -1                     # a row without entries, whatever its logits
    x[4, ids[4, 5] + 0] = -torch.inf
    ids[4, 5] = -1
    x[5, :500] = torch.finfo(torch.float32).min
    ids[5] = torch.arange(500, 506)
    xg = x.to(gpu).requires_grad_()
    loss = qat.top_logits_distillation_loss(xg, values.to(gpu), ids.to(gpu), 1.5, "none")
    gx, = torch.autograd.grad(loss, xg, torch.ones(8, device=gpu))
    assert loss[3].item() == 0 and (gx[3] == 0).all() and loss[1].item() == 0 and (gx[1] == 0).all()
    rows = [0, 1, 2, 4, 5, 6, 7]
    _check_distill(x[rows], values[rows], ids[rows], 1.5, "none", loss[rows], gx[rows], torch.ones(7))
    # a student that rules a kept token out: infinite loss, finite gradient
    x2 = x[6:].clone()
    x2[0, ids[6, 0]] = -torch.inf
    xg = x2.to(gpu).requires_grad_()
    loss = qat.top_logits_distillation_loss(xg, values[6:].to(gpu), ids[6:].to(gpu), 1.0, "none")
    gx, = torch.autograd.grad(loss.sum(), xg)
    assert loss[0].item() == torch.inf and torch.isfinite(gx).all()
    # a token beyond the vocabulary, a NaN logit, a NaN value: NaN loss and gradient, of that row alone
    for spoil in ("id", "x", "value"):
        v, i, xx = values[6:].clone(), ids[6:].clone(), x[6:].clone()
        if spoil == "id":
            i[0, 2] = 600
        elif spoil == "x":
            xx[0, 7] = torch.nan
        else:
            v[0, 1] = torch.nan
        xg = xx.to(gpu).requires_grad_()
        loss = qat.top_logits_distillation_loss(xg, v.to(gpu), i.to(gpu), 1.0, "none")
        gx, = torch.autograd.grad(loss, xg, torch.ones(2, device=gpu))
        assert torch.isnan(loss).tolist() == [True, False] and torch.isnan(gx[0]).all() and torch.isfinite(gx[1]).all()


def test_distillation_without_any_entry(gpu):
    from dimq_amd import qat
    announce("distillation empty")
    x = _logits(3, 50, torch.float16, 1).to(gpu).requires_grad_()
    for k in (0, 2):
        v, i = torch.zeros(3, k, device=gpu), torch.full((3, k), -1, device=gpu)
        loss = qat.top_logits_distillation_loss(x, v, i)
        gx, = torch.autograd.grad(loss, x)
        assert loss.item() == 0 and (gx == 0).all()
    x = torch.zeros(0, 50, device=gpu, requires_grad=True)
    loss = qat.top_logits_distillation_loss(x, torch.zeros(0, 2, device=gpu), torch.zeros(0, 2, device=gpu, dtype=torch.long))
    assert loss.item() == 0 and torch.autograd.grad(loss, x)[0].shape == (0, 50)


def test_distillation_gradient_by_differences(gpu):
    from dimq_amd import qat
    announce("distillation differences")
    x = _logits(2, 30, torch.float32, 3)
    values, ids = _teacher(x, 5, 4)
    xg = x.to(gpu).requires_grad_()
    loss = qat.top_logits_distillation_loss(xg, values.to(gpu), ids.to(gpu), 2.0, "sum")
    g, = torch.autograd.grad(loss, xg)
    for i in range(0, 60, 7):
        step = torch.zeros(60, dtype=torch.float64)
        step[i] = 1e-6
        up, down = (lm.distill(x.double() + s * step.view(2, 30), values, ids, 2.0)[0].sum() for s in (1, -1))
        assert abs((up - down) / 2e-6 - g.cpu().double().view(-1)[i]) <= 1e-7 + 300 * E * 4


def test_teacher_rows_feed_the_distillation(gpu):
    """token_logprobs' alternatives as the teacher's entries: log probabilities give the loss that logits give."""
    from dimq_amd import ops, qat
    announce("teacher to distillation")
    teacher, student = _logits(6, 3001, torch.bfloat16, 1), _logits(6, 3001, torch.bfloat16, 2)
    teacher[2] = -torch.inf  # a row without a distribution: tokens -1, nothing to learn from it
    xg = student.to(gpu).requires_grad_()
    _, _, v, i = ops.token_logprobs(teacher.to(gpu), torch.full((6,), -1, device=gpu), 16)
    loss = qat.top_logits_distillation_loss(xg, v, i, 2.0)
    gx, = torch.autograd.grad(loss, xg)
    assert (gx[2] == 0).all()
    _check_distill(student, torch.nan_to_num(v), i, 2.0, "mean", loss, gx, 1.0)


# ---- streams, graphs, autograd ------------------------------------------------------------------------------------

def _all_ops(gpu, seed):
    """Inputs and a pass through everything, forward and backward."""
    from dimq_amd import ops, qat
    x, r = _rows(20, 520, torch.bfloat16, seed).to(gpu).requires_grad_(), _rows(20, 520, torch.bfloat16, seed + 1).to(gpu)
    w = torch.ones(520, device=gpu, requires_grad=True)
    z = _logits(20, 9001, torch.bfloat16, seed + 2).to(gpu).requires_grad_()
    v, i = (t.to(gpu) for t in _teacher(z.detach().cpu(), 9, seed))
    t = torch.arange(20, device=gpu)
    gy, one = _rows(20, 520, torch.bfloat16, seed + 3).to(gpu), torch.ones(20, device=gpu)

    def run():
        y, h = ops.rms_norm(x, w, residual=r)
        q, s, h8 = ops.rms_norm_e4m3(x.detach(), w.detach(), residual=r)
        lp, H, tlp, tid = ops.token_logprobs(z, t, 5)
        loss = qat.top_logits_distillation_loss(z, v, i, 2.0)
        gx, gw = torch.autograd.grad((y, h), (x, w), (gy, gy))
        g1, = torch.autograd.grad((lp, H), z, (one, one))
        g2, = torch.autograd.grad(loss, z)
        return [y, h, q.float(), s, h8, lp, H, tlp, tid, loss, gx, gw, g1, g2]

    return (x, r, z), run


def test_on_another_stream(gpu):
    announce("other stream")
    _, run = _all_ops(gpu, 1)
    want = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_and_replayed(gpu):
    announce("graph")
    (x, r, z), run = _all_ops(gpu, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in (5, 6, 7):
        with torch.no_grad():
            for to, like in zip((x, r, z), _all_ops(gpu, seed)[0]):
                to.copy_(like)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = run()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_calls_give_the_same_bits(gpu):
    _, run = _all_ops(gpu, 3)
    assert all(torch.equal(a, b) for a, b in zip([t.clone() for t in run()], run()))


def test_autograd_refusals(gpu):
    from dimq_amd import ops, qat
    x = _rows(4, 64, torch.float32, 1).to(gpu).requires_grad_()
    t = torch.zeros(4, dtype=torch.long, device=gpu)
    v = torch.zeros(4, 2, device=gpu)
    i = torch.zeros(4, 2, dtype=torch.long, device=gpu)
    for out in (ops.rms_norm(x).sum(), ops.token_logprobs(x, t)[0].sum(), qat.top_logits_distillation_loss(x, v, i)):
        with pytest.raises(RuntimeError, match="gradients of its gradients"):
            torch.autograd.grad(out, x, create_graph=True)
    q, s = ops.rms_norm_e4m3(x)
    with pytest.raises(RuntimeError, match="not implemented"):
        s.sum().backward()
    lp, H, tlp, tid = ops.token_logprobs(x, t, 3)
    assert not tlp.requires_grad and not tid.requires_grad
    y, h = ops.rms_norm(x, residual=x.detach().clone())
    with torch.no_grad():
        h.add_(1.0)  # what the gradient reads is changed
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_below_no_grad_and_under_autocast(gpu):
    from dimq_amd import ops
    x = _rows(4, 64, torch.bfloat16, 1).to(gpu).requires_grad_()
    with torch.no_grad():
        assert not ops.rms_norm(x).requires_grad
    with torch.autocast("cuda"):
        assert torch.equal(ops.rms_norm(x), ops.rms_norm(x))
    assert torch.equal(ops.rms_norm(x), torch.ops.dimq.rms_norm(x, None, 1e-6)[0])
