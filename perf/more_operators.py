"""Layers, scoring and distillation of quantized language models: what they compute, and on which sizes.

Kinds of cases:

* ``linear``   4-bit weights with a scale (and a zero point, or 8) per group of a row's elements:
  y[m, n] = sum_g s[n, g] sum_{k in g} (q[n, k] - z[n, g]) x[m, k] + b[n]; x in fp32, fp16, bf16, or in e4m3 codes with one
  scale per row, which multiplies the sum.  Codes: two a byte, the earlier element in the low half, rows padded to whole
  blocks of 32;
* ``norm``     h = x + r, rounded to their type; y = h / sqrt(mean(h^2) + eps) w, as e4m3 codes of y / scale with
  scale = max|y| / 448 per row, or (``train``) as y itself with the gradients to x, r and w;
* ``score``    of rows of logits x: log p of a given token (0 where the token is negative), the entropy -sum p log p, and the
  largest log p's with their tokens (ties: the lower token first), p = softmax(x); or (``train``) the first two with the
  gradient to x;
* ``distill``  the mean over the rows that keep a teacher entry of tau^2 sum_j p_j (log p_j - log q[id_j]),
  p = softmax(values / tau) over a row's kept entries (id >= 0), q = softmax(student / tau); with the gradient to the student.
"""

import math

import torch

own = False

_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2, "e4m3": 1}
_EPS = 1e-6


def listed():
    return [
        # one token through a square layer: latency and the weights' bytes
        dict(name="linear_1x4096_4096", kind="linear", rows=1, k=4096, n=4096, dtype="bf16", group=128, zeros=True),
        # sixteen sequences' next tokens from the norm's 8-bit rows through three such layers in one
        dict(name="linear_16x4096_12288_e4m3", kind="linear", rows=16, k=4096, n=12288, dtype="e4m3", group=128, zeros=True),
        # odd sizes, a short last group, single precision, no zero points
        dict(name="linear_37x1000_1030", kind="linear", rows=37, k=1000, n=1030, dtype="fp32", group=64, zeros=False),
        # a prompt of 2,048 tokens
        dict(name="linear_2048x4096_4096", kind="linear", rows=2048, k=4096, n=4096, dtype="bf16", group=128, zeros=True),
        # the norm in front of a decode step's layers, and of a prompt batch's
        dict(name="norm_1x4096", kind="norm", rows=1, d=4096, dtype="bf16", train=False),
        dict(name="norm_16384x4096", kind="norm", rows=16384, d=4096, dtype="bf16", train=False),
        # training: an odd width
        dict(name="norm_train_8191x1000", kind="norm", rows=8191, d=1000, dtype="fp16", train=True),
        # the next token's log probability with 20 alternatives, as a server returns them
        dict(name="score_1x128000", kind="score", rows=1, v=128000, dtype="bf16", top=20, train=False),
        # a teacher's pass over 4,096 tokens: 32 alternatives to keep
        dict(name="score_4096x32768", kind="score", rows=4096, v=32768, dtype="fp16", top=32, train=False),
        # token log probabilities with an entropy bonus, trained; odd sizes
        dict(name="score_train_1021x50021", kind="score", rows=1021, v=50021, dtype="bf16", top=0, train=True),
        # a distillation step: a long batch over a large vocabulary, and a small odd one in single precision
        dict(name="distill_2048x128000", kind="distill", rows=2048, v=128000, dtype="bf16", top=64, tau=2.0),
        dict(name="distill_99x32003", kind="distill", rows=99, v=32003, dtype="fp32", top=20, tau=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "norm", "score", "distill"])
    if kind == "linear":
        case = dict(kind=kind, rows=_log(rng, 1, 2048), k=_log(rng, 64, 4096), n=_log(rng, 16, 4096),
                    dtype=rng.choice(["bf16", "fp16", "fp32", "e4m3"]), group=rng.choice([32, 64, 128, 256]),
                    zeros=rng.random() < 0.7)
        if rng.random() < 0.6:  # the sizes of most layers
            case["k"], case["n"] = max(64, case["k"] // 64 * 64), max(16, case["n"] // 16 * 16)
        return case
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if kind == "norm":
        case = dict(kind=kind, rows=_log(rng, 1, 16384), d=_log(rng, 32, 8192), dtype=dtype, train=rng.random() < 0.4)
        if rng.random() < 0.6:
            case["d"] = case["d"] // 32 * 32
        return case
    v = _log(rng, 1000, 131072)
    if rng.random() < 0.5:
        v = max(1024, v // 64 * 64)
    case = dict(kind=kind, rows=_log(rng, 1, max(1, min(4096, 2 ** 26 // v))), v=v, dtype=dtype, top=_log(rng, 1, 64))
    if kind == "distill":
        return dict(case, tau=rng.choice([1.0, 2.0, 0.5]))
    case["train"] = rng.random() < 0.4
    if case["train"]:
        case["top"] = 0
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, rows, dt = case["kind"], case["rows"], _DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": case}
    if kind in ("linear", "norm"):
        k = case["k"] if kind == "linear" else case["d"]
        # activations: a common spread and, as trained networks show, some features that are much larger
        x = normal(rows, k) * torch.exp(normal(k) * 0.6)
    if kind == "linear":
        n, size = case["n"], case["group"]
        groups, blocks = -(-k // size), -(-k // 32)
        w = normal(n, k) / math.sqrt(k)
        wg = torch.nn.functional.pad(w, (0, groups * size - k)).view(n, groups, size)
        low, high = wg.amin(2).clamp(max=0), wg.amax(2).clamp(min=0)
        if case["zeros"]:
            s["scales"] = ((high - low) / 15).clamp(min=1e-6).half()
            s["zeros"] = torch.round(-low / s["scales"].float()).clamp(0, 15).to(torch.uint8)
        else:
            s["scales"], s["zeros"] = (torch.maximum(-low, high) / 7.5).clamp(min=1e-6).half(), None
        zero = 8.0 if s["zeros"] is None else s["zeros"].float()[..., None]
        q = torch.round(wg / s["scales"].float()[..., None] + zero).clamp(0, 15).to(torch.uint8).view(n, -1)[:, :k]
        q = torch.nn.functional.pad(q, (0, blocks * 32 - k)).view(n, blocks * 16, 2)
        s["codes"] = q[..., 0] + q[..., 1] * 16
        s["b"] = normal(n) * 0.1
        if case["dtype"] == "e4m3":
            s["xs"] = x.abs().amax(1) / 448
            x = x / s["xs"][:, None]
        s["x"] = x.to(dt)
    elif kind == "norm":
        s["x"], s["r"] = x.to(dt), (normal(rows, k) * 4).to(dt)
        s["w"] = 1 + 0.2 * normal(k)
        if case["train"]:
            s["gy"], s["gh"] = (normal(rows, k) * 1e-2).to(dt), (normal(rows, k) * 1e-2).to(dt)
        else:
            s["w"] = s["w"].to(dt)
    else:
        v, top = case["v"], case["top"]
        # logits: a broad bulk, and some tokens of each row that stand out
        x = normal(rows, v).mul_(2.5)
        x.scatter_add_(1, torch.randint(0, v, (rows, 16), generator=g, device="cuda"), normal(rows, 16).abs() * 5 + 3)
        if kind == "score":
            s["x"] = x.to(dt)
            token = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, s["x"].float().argmax(1),
                                torch.randint(0, v, (rows,), generator=g, device="cuda"))
            token[rows // 2 + 1:][::13] = -100  # padding
            s["token"] = token
            if case["train"]:
                s["ga"], s["gb"] = normal(rows) / rows, normal(rows) * 0.01 / rows
        else:
            s["values"], s["ids"] = torch.topk(x, top, dim=1)
            # rows behind a sequence's end keep nothing, and some keep fewer entries
            s["ids"][rows // 3 + 1:][::11] = -1
            s["ids"][::7, top - top // 4:] = -1
            s["x"] = x.add_(normal(rows, v).mul_(0.7)).to(dt)
    return s


# ---- plain forms, 32 bits -----------------------------------------------------------------------------------------

def _linear(s):
    case, x = s["case"], s["x"].float()
    k, size, n = case["k"], case["group"], case["n"]
    q = torch.stack([s["codes"] & 15, s["codes"] >> 4], dim=-1).view(n, -1)[:, :k].float()
    wide = lambda t: t.float().repeat_interleave(size, dim=1)[:, :k]  # noqa: E731
    w = (q - (8.0 if s["zeros"] is None else wide(s["zeros"]))) * wide(s["scales"])
    y = x @ w.t()
    if case["dtype"] == "e4m3":
        y = y * s["xs"][:, None]
    return (y + s["b"]).to(torch.bfloat16 if case["dtype"] == "e4m3" else s["x"].dtype)


def _norm(s):
    dt = s["x"].dtype
    h = (s["x"].float() + s["r"].float()).to(dt)
    hf, w = h.float(), s["w"].float()
    inv = 1 / torch.sqrt(hf.square().mean(1, keepdim=True) + _EPS)
    y = hf * inv * w
    if not s["case"]["train"]:
        scale = y.abs().amax(1, keepdim=True) / 448
        return (y / scale).to(torch.float8_e4m3fn), scale[:, 0], h
    gw = s["gy"].float() * w
    xhat = hf * inv
    gh = inv * (gw - xhat * (gw * xhat).mean(1, keepdim=True)) + s["gh"].float()
    gh = gh.to(dt)
    return y.to(dt), h, gh, gh, (s["gy"].float() * xhat).sum(0)


def _logsumexp(x):
    top = x.amax(1, keepdim=True)
    return top + torch.log(torch.exp(x - top).sum(1, keepdim=True))


def _score(s):
    case, x, token = s["case"], s["x"].float(), s["token"]
    lse = _logsumexp(x)
    logp = x - lse
    p = torch.exp(logp)
    h = -(p * logp).sum(1)
    given = token >= 0
    lp = torch.where(given, logp.gather(1, token.clamp(min=0)[:, None])[:, 0], 0.0)
    if case["train"]:
        a = torch.where(given, s["ga"], 0.0)
        grad = -p * (a[:, None] + s["gb"][:, None] * (logp + h[:, None]))
        grad.scatter_add_(1, token.clamp(min=0)[:, None], a[:, None])
        return lp, h, grad.to(s["x"].dtype)
    # keys that order like the logits, the lower token first among equals: no two alike
    bits = x.view(torch.int32).to(torch.int64)
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * 2 ** 31 - torch.arange(case["v"], device=x.device)
    ids = torch.topk(key, case["top"], dim=1).indices
    return lp, h, logp.gather(1, ids), ids


def _distill(s):
    case, x, ids = s["case"], s["x"].float(), s["ids"]
    tau = case["tau"]
    kept = ids >= 0
    some = kept.any(1)
    at = ids.clamp(min=0)
    logq = x / tau - _logsumexp(x / tau)
    values = torch.where(kept, s["values"] / tau, -math.inf)
    values = torch.where(some[:, None], values, 0.0)  # rows without entries: any finite values, p is cleared below
    logp = values - _logsumexp(values)
    p = torch.where(kept, torch.exp(logp), 0.0)
    each = torch.where(kept, p * (logp - logq.gather(1, at)), 0.0).sum(1) * tau * tau
    count = some.sum().clamp(min=1)
    grad = torch.where(some[:, None], torch.exp(logq), 0.0)
    grad.scatter_add_(1, at, -p)
    return each.sum() / count, (grad * (tau / count)).to(s["x"].dtype)


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from dimq_amd import ops, qat

        if kind == "linear":
            return ops.dimq_linear_grouped(s["x"], s["codes"], s["scales"], s["zeros"], case["group"], s["b"],
                                           x_scales=s.get("xs"))
        if kind == "norm" and not case["train"]:
            return ops.rms_norm_e4m3(s["x"], s["w"], _EPS, residual=s["r"])
        if kind == "norm":
            x, r, w = (s[name].detach().requires_grad_() for name in ("x", "r", "w"))
            y, h = ops.rms_norm(x, w, _EPS, residual=r)
            return (y.detach(), h.detach(), *torch.autograd.grad((y, h), (x, r, w), (s["gy"], s["gh"])))
        if kind == "score" and not case["train"]:
            return ops.token_logprobs(s["x"], s["token"], case["top"])
        x = s["x"].detach().requires_grad_()
        if kind == "score":
            lp, h, _, _ = ops.token_logprobs(x, s["token"])
            return (lp.detach(), h.detach(), *torch.autograd.grad((lp, h), x, (s["ga"], s["gb"])))
        loss = qat.top_logits_distillation_loss(x, s["values"], s["ids"], case["tau"])
        return loss.detach(), torch.autograd.grad(loss, x)[0]
    return {"linear": _linear, "norm": _norm, "score": _score, "distill": _distill}[kind](s)


# ---- 64 bits ------------------------------------------------------------------------------------------------------

def _to_e4m3(v):
    """v in 64 bits to the nearest value of 4 exponent and 3 mantissa bits, ties to even."""
    step = torch.exp2((torch.frexp(v).exponent.double() - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    kind, x = case["kind"], s["x"].double()
    if kind == "linear":
        n, k, size = case["n"], case["k"], case["group"]
        w = torch.empty(n, s["codes"].shape[1] * 2, dtype=torch.float64, device=x.device)
        w[:, 0::2], w[:, 1::2] = s["codes"] % 16, s["codes"] // 16
        group = torch.arange(k, device=x.device) // size
        w = w[:, :k] - (8 if s["zeros"] is None else s["zeros"][:, group].double())
        y = x @ (w * s["scales"].double()[:, group]).t()
        return (y if "xs" not in s else y * s["xs"].double()[:, None]) + s["b"].double()
    if kind == "norm":
        h = x + s["r"].double()
        z, w = h.to(s["x"].dtype).double(), s["w"].double()
        rms = torch.sqrt(torch.einsum("ij,ij->i", z, z) / case["d"] + _EPS)[:, None]
        unit = z / rms
        y = unit * w
        if not case["train"]:
            scale = y.abs().max(dim=1).values / 448
            return _to_e4m3(y / scale[:, None]), scale, h
        gu = s["gy"].double() * w
        gh = (gu - unit * (gu * unit).sum(1, keepdim=True) / case["d"]) / rms + s["gh"].double()
        return y, h, gh, gh, (s["gy"].double() * unit).sum(0)
    if kind == "score":
        lse = torch.logsumexp(x, 1)
        p = torch.softmax(x, 1)
        h = lse - (p * x).sum(1)
        rows = torch.arange(case["rows"], device=x.device)
        given = s["token"] >= 0
        lp = (x[rows, s["token"].clamp(min=0)] - lse) * given
        if not case["train"]:
            values, ids = torch.sort(x, dim=1, descending=True, stable=True)
            return lp, h, values[:, :case["top"]] - lse[:, None], ids[:, :case["top"]].contiguous()
        a, b = s["ga"].double() * given, s["gb"].double()
        grad = -p * (a + b * (h - lse))[:, None] - p * x * b[:, None]
        grad[rows, s["token"].clamp(min=0)] += a
        return lp, h, grad
    tau, kept = case["tau"], s["ids"] >= 0
    logq = torch.log_softmax(x / tau, 1)
    logp = torch.log_softmax((s["values"].double() / tau).masked_fill(~kept, -1e300), 1)
    p = torch.exp(logp) * kept
    some = kept.any(1)
    at = s["ids"].clamp(min=0)
    loss = tau ** 2 * (p * (logp - logq.gather(1, at))).sum() / max(1, int(some.sum()))
    grad = torch.exp_(logq) * some[:, None]
    grad.scatter_add_(1, at, -p)
    return loss, grad * (tau / max(1, int(some.sum())))


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    m, e = case["rows"], _SIZE[case["dtype"]]
    if case["kind"] == "linear":
        n, k = case["n"], case["k"]
        groups = -(-k // case["group"])
        out = 2 if case["dtype"] == "e4m3" else e
        return {"bytes": m * k * e + (4 * m if out > e else 0) + n * k // 2 + n * groups * (3 if case["zeros"] else 2) + 4 * n
                + m * n * out, "flops": 2 * m * n * k}
    if case["kind"] == "norm":
        d = case["d"]
        if case["train"]:  # x, r, gy, gh read; y, h and the two gradients (the same one) written; the weight and its gradient
            return {"bytes": m * d * 7 * e + 8 * d, "flops": 16 * m * d}
        return {"bytes": m * d * (3 * e + 1) + 4 * m + d * e, "flops": 8 * m * d}
    v, top = case["v"], case["top"]
    if case["kind"] == "score":
        if case["train"]:  # logits read, their gradient written
            return {"bytes": 2 * m * v * e + 24 * m, "flops": 12 * m * v}
        return {"bytes": m * v * e + m * (16 + 12 * top), "flops": 6 * m * v}
    return {"bytes": 2 * m * v * e + 12 * m * top, "flops": 10 * m * v}
