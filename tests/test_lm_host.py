"""Language-model operators without a GPU: the float64 oracle against differences and hand-worked values, the packing of
grouped weights, and what the entry points refuse before anything is launched."""

import ctypes

import pytest
import torch

from oracle import lm


# ---- the oracle ---------------------------------------------------------------------------------------------------

def test_e4m3_values():
    v = torch.tensor([448.0, 449.0, 1.0, 1.0625, 1.1875, 0.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, -17.0], dtype=torch.float64)
    want = [448.0, 448.0, 1.0, 1.0, 1.25, 0.0, 2.0 ** -9, 0.0, 2.0 ** -8, -16.0]
    assert lm.e4m3(v).tolist() == want
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[torch.isfinite(every)]
    assert torch.equal(lm.e4m3(every), every)


def test_norm_gradients_are_the_differences():
    g = torch.Generator().manual_seed(1)
    h, w, gy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((3, 7), (7,), (3, 7)))
    grad, gw, _ = lm.rms_norm_grads(h, w, 1e-3, gy, None)
    f = lambda a, b: (lm.rms_norm(a, b, 1e-3)[0] * gy).sum()  # noqa: E731
    for i in range(21):
        e = torch.zeros(21, dtype=torch.float64)
        e[i] = 1e-6
        e = e.view(3, 7)
        assert abs((f(h + e, w) - f(h - e, w)) / 2e-6 - grad.view(-1)[i]) < 1e-8
    for i in range(7):
        e = torch.zeros(7, dtype=torch.float64)
        e[i] = 1e-6
        assert abs((f(h, w + e) - f(h, w - e)) / 2e-6 - gw[i]) < 1e-8


def test_scores_by_hand():
    x = torch.log(torch.tensor([[0.5, 0.25, 0.25], [1.0, 1.0, 2.0]]))
    lp, H, tlp, tid = lm.scores(x, torch.tensor([1, -1]), 2)
    assert torch.allclose(lp, torch.tensor([0.25, 1.0]).log().double(), atol=1e-7) and lp[1] == 0
    assert torch.allclose(H, torch.tensor([1.5, 1.5]).double() * 0.6931471805599453, atol=1e-7)
    assert tid.tolist() == [[0, 1], [2, 0]]


def test_distillation_by_hand():
    x = torch.tensor([[0.0, 0.0, 0.0, 0.0]])
    loss, some, grad = lm.distill(x, torch.tensor([[1.0, 1.0, 9.0]]), torch.tensor([[2, 0, -1]]), 1.0)
    assert abs(loss.item() - torch.log(torch.tensor(2.0)).item()) < 1e-7  # log(1/2) - log(1/4)
    assert some.tolist() == [True]
    assert torch.allclose(grad, torch.tensor([[-0.25, 0.25, -0.25, 0.25]]).double())


# ---- packing ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (3, 40, 32), (5, 256, 128), (2, 200, 64), (4, 96, 96), (2, 70, 256)])
@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_quantize_grouped(n, k, group, symmetric, dt):
    from dimq_amd import ops
    g = torch.Generator().manual_seed(n + k)
    w = torch.randn(n, k, generator=g) + 0.3
    w[0] = w[0].abs()       # a row above 0: its grid starts there
    if n > 1:
        w[1] = 0
    codes, scales, zeros = ops.quantize_grouped(w, group, symmetric=symmetric, scale_dtype=dt)
    groups, blocks = -(-k // group), -(-k // 32)
    assert codes.shape == (n, 16 * blocks) and codes.dtype == torch.uint8 and scales.shape == (n, groups)
    assert scales.dtype == dt and (zeros is None) == symmetric
    step = scales.double().repeat_interleave(group, 1)[:, :k]
    # half a step, and the scale's own rounding over 15 steps
    tol = step * (0.5 + 16 * torch.finfo(dt).eps) + 1e-30
    err = (lm.grouped_weight(codes, scales, zeros, group, k) - w.double()).abs()
    assert (err <= tol).all()
    if n > 1:
        assert (lm.grouped_weight(codes, scales, zeros, group, k)[1] == 0).all()


def test_quantize_grouped_refuses():
    from dimq_amd import ops
    w = torch.randn(4, 64)
    for bad, match in ((lambda: ops.quantize_grouped(w[0]), "expects a weight"), (lambda: ops.quantize_grouped(w, 48), "multiple of 32"),
                       (lambda: ops.quantize_grouped(w, 0), "multiple of 32"), (lambda: ops.quantize_grouped(w[:0]), "expects a weight"),
                       (lambda: ops.quantize_grouped(w / 0), "finite"),
                       (lambda: ops.quantize_grouped(w, 32, scale_dtype=torch.float64), "scales must be"),
                       (lambda: ops.quantize_grouped(w, 32, scale_dtype=torch.int8), "scales must be")):
        with pytest.raises(RuntimeError, match=match):
            bad()


# ---- refusals -----------------------------------------------------------------------------------------------------

def test_ops_refuse_cpu_tensors():
    from dimq_amd import ops, qat
    x, t = torch.ones(2, 32), torch.zeros(2, dtype=torch.long)
    c, s = torch.zeros(4, 16, dtype=torch.uint8), torch.ones(4, 1)
    for call in (lambda: ops.rms_norm(x), lambda: ops.rms_norm(x, residual=x), lambda: ops.rms_norm_e4m3(x),
                 lambda: ops.token_logprobs(x, t), lambda: ops.dimq_linear_grouped(x, c, s, None, 32),
                 lambda: qat.top_logits_distillation_loss(x, x[:, :2], t[:, None].expand(2, 2)),
                 lambda: ops.rms_norm(x.requires_grad_())):
        with pytest.raises(NotImplementedError):
            call()


def test_modules_refuse_cpu_tensors():
    from dimq_amd import DIMQGroupedLinear, DIMQRMSNorm
    m = DIMQGroupedLinear.from_linear(torch.nn.Linear(32, 4), 32)
    for call in (lambda: m(torch.ones(1, 32)), lambda: DIMQRMSNorm(32)(torch.ones(1, 32)), lambda: DIMQRMSNorm(32).e4m3(torch.ones(1, 32))):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        DIMQRMSNorm.from_rms_norm(torch.nn.RMSNorm((2, 32)))


def test_names_are_checked():
    from dimq_amd import ops, qat
    x, t = torch.ones(2, 32), torch.zeros(2, dtype=torch.long)
    with pytest.raises(ValueError, match="reduction"):
        qat.top_logits_distillation_loss(x, x, t, 1.0, "avg")
    c, s = torch.zeros(4, 16, dtype=torch.uint8), torch.ones(4, 1)
    with pytest.raises(KeyError):
        ops.dimq_linear_grouped(x, c, s, None, 32, activation="tanh")
    with pytest.raises(KeyError):
        ops.dimq_linear_grouped(x, c, s, None, 32, variant="small")


_BUF = ctypes.create_string_buffer(1 << 16)
P = (ctypes.addressof(_BUF) + 255) // 256 * 256
F32, F16, E4M3 = 0, 1, 5


def _refused(rc, match):
    from dimq_amd import _C
    assert rc == 1, "accepted"
    assert match in _C.lib.dimq_last_error().decode(), _C.lib.dimq_last_error()


def test_c_abi_norm_refusals():
    """Arguments alone: every one of these returns before a launch."""
    from dimq_amd import _C
    f = _C.lib.dimq_rms_norm
    ok = dict(x=P, xd=F32, rows=2, dim=8, ldx=8, r=None, ldr=8, w=None, wd=0, eps=1e-6, y=P, yd=F32, scales=None, h=None)

    def call(**k):
        a = {**ok, **k}
        return f(*a.values(), None)

    _refused(call(xd=3), "input must be")
    _refused(call(dim=0), "dimensions")
    _refused(call(rows=-1), "dimensions")
    _refused(call(ldx=7), "row stride")
    _refused(call(w=P, wd=4), "weight must be")
    _refused(call(eps=-1.0), "eps")
    _refused(call(eps=float("nan")), "eps")
    _refused(call(x=None), "null")
    _refused(call(x=P + 2), "misaligned")
    _refused(call(dim=1 << 30, ldx=1 << 30), "2^30")
    _refused(call(y=None), "null")
    _refused(call(yd=E4M3), "with scales")
    _refused(call(scales=P), "with scales")
    _refused(call(r=P), "go together")
    _refused(call(r=P, h=P, ldr=3), "residual row stride")
    assert call(rows=0) == 0
    b = _C.lib.dimq_rms_norm_backward
    _refused(b(P, F32, 2, 8, 8, None, 0, 1e-6, P, 3, 8, None, 0, P, None, 0, None, 0, None), "gradient must be")
    _refused(b(P, F32, 2, 8, 8, None, 0, 1e-6, P, F32, 4, None, 0, P, None, 0, None, 0, None), "row stride")
    _refused(b(P, F32, 2, 8, 8, None, 0, 1e-6, P, F32, 8, None, 0, None, P, F32, P, 8, None), "workspace")
    _refused(b(P, F32, 2, 8, 8, None, 0, 1e-6, None, F32, 8, None, 0, P, None, 0, None, 0, None), "null")


def test_c_abi_score_refusals():
    from dimq_amd import _C
    f = _C.lib.dimq_token_logprobs
    ok = dict(x=P, dt=F32, rows=2, vocab=100, ldx=100, tokens=P, t64=1, top=4, lp=P, H=P, norm=None, tlp=P, tid=P, ws=P, wsb=1 << 20)

    def call(**k):
        a = {**ok, **k}
        return f(*a.values(), None)

    _refused(call(dt=3), "logits must be")
    _refused(call(vocab=0), "at least one logit")
    _refused(call(ldx=99), "row stride")
    _refused(call(top=129), "top must be")
    _refused(call(top=-1), "top must be")
    _refused(call(vocab=3, ldx=3), "top must be")
    _refused(call(tokens=None), "null")
    _refused(call(tid=None), "null")
    _refused(call(vocab=1 << 31, ldx=1 << 31), "2^31")
    assert call(rows=0) == 0
    q = _C.lib.dimq_logits_workspace_bytes
    assert q(0, 100, 4) == 0 and q(1, 128000, 20) > 0
    _refused(call(rows=1, vocab=128000, ldx=128000, wsb=8), "workspace")
    _refused(call(rows=1, vocab=128000, ldx=128000, ws=P + 4), "workspace")
    d = _C.lib.dimq_distill_loss
    ok = dict(x=P, dt=F32, rows=2, vocab=100, ldx=100, v=P, vd=F32, ids=P, i64=1, k=4, t=1.0, red=1, rl=P, loss=P, by=P, norm=P, p=P,
              ws=P, wsb=1 << 20)

    def call(**k):
        a = {**ok, **k}
        return d(*a.values(), None)

    _refused(call(vd=3), "teacher values")
    _refused(call(t=0.0), "temperature")
    _refused(call(t=float("nan")), "temperature")
    _refused(call(t=-1.0), "temperature")
    _refused(call(t=0.0009), "temperature")
    _refused(call(t=1001.0), "temperature")
    _refused(call(t=float("inf")), "temperature")
    _refused(call(red=3), "reduction")
    _refused(call(k=-1), "entries")
    _refused(call(k=4097), "entries")
    _refused(call(x=P + 2), "misaligned")
    b = _C.lib.dimq_distill_loss_backward
    _refused(b(P, F32, 2, 100, 100, P, 1, 4097, P, P, 1.0, P, 0, None, P, None), "entries")
    _refused(call(ids=None), "null")
    _refused(call(norm=None), "null")
    _refused(call(rows=1, vocab=128000, ldx=128000, wsb=8), "workspace")


def test_c_abi_grouped_refusals():
    from dimq_amd import _C
    f = _C.lib.dimq_linear_grouped
    ok = dict(x=P, xd=F32, M=2, K=64, ldx=64, xs=None, codes=P, scales=P, sd=F16, zeros=None, group=32, bias=None, bd=0, N=4, y=P,
              yd=F32, res=None, rd=0, act=0, variant=0, ws=None, wsb=0)

    def call(**k):
        a = {**ok, **k}
        return f(*a.values(), None)

    _refused(call(xd=3), "input must be")
    _refused(call(xd=E4M3), "have scales")
    _refused(call(xs=P), "have scales")
    _refused(call(sd=4), "scales must be")
    _refused(call(yd=E4M3), "output must be")
    _refused(call(K=0), "positive")
    _refused(call(N=0), "positive")
    _refused(call(group=48), "multiple of 32")
    _refused(call(group=-32), "multiple of 32")
    _refused(call(ldx=63), "row stride")
    _refused(call(act=3), "activation")
    _refused(call(variant=3), "variant")
    _refused(call(bias=P, bd=5), "bias must be")
    _refused(call(res=P, rd=4), "residual must be")
    _refused(call(codes=None), "null")
    _refused(call(codes=P + 8), "aligned")
    _refused(call(x=P + 2), "misaligned")
    _refused(call(scales=P + 1), "misaligned")
    _refused(call(N=(1 << 31) - 1, variant=1, ws=P, wsb=1 << 60), "one launch")
    _refused(call(M=1 << 30, variant=2, ws=P, wsb=1 << 60), "one launch")
    _refused(call(K=1 << 31, ldx=1 << 31), "2^31")
    assert call(M=0) == 0
    q = _C.lib.dimq_linear_grouped_workspace_bytes
    assert q(P, F32, 2, 64, 64, 32, 4, 0) == 0 and q(P, F32, 2, 64, 64, 32, 4, 1) == 0 and q(P, F32, 2, 64, 64, 32, 4, 2) > 0
    assert q(P, F16, 2048, 4096, 4096, 32, 4096, 0) > 0 and q(P, 3, 2048, 4096, 4096, 32, 4096, 0) == 0
    _refused(call(variant=2), "workspace")
    need = q(P, F32, 2, 64, 64, 32, 4, 2)
    _refused(call(variant=2, ws=P, wsb=need - 1), "workspace")
    _refused(call(variant=2, ws=P + 8, wsb=need), "workspace")
    # copies are made of rows that cannot be read in place
    assert q(P, F16, 4096, 4096, 4096, 32, 4096, 2) < q(P + 2, F16, 4096, 4096, 4096, 32, 4096, 2)
    assert q(P, F16, 4096, 4096, 4096, 32, 4096, 2) < q(P, F16, 4096, 4096, 4097, 32, 4096, 2)
