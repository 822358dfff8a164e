"""Operators of language models in float64 on the CPU, from their definitions: RMS norm (with e4m3 rows), log probabilities
with entropy and top alternatives, distillation from top logits, 4-bit weights with group scales; with the gradients."""

from __future__ import annotations

import torch
from torch import Tensor


def f64(t: Tensor) -> Tensor:
    return t.detach().cpu().double()


def rms_norm(x: Tensor, w: Tensor | None, eps: float, r: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """(y, h): h rounded to x's type, y not rounded."""
    h = x.detach().cpu() if r is None else (f64(x) + f64(r)).to(x.dtype)
    v = h.double()
    y = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
    return (y if w is None else y * f64(w)), h


def rms_norm_grads(h: Tensor, w: Tensor | None, eps: float, gy: Tensor, gh: Tensor | None) -> tuple[Tensor, Tensor, Tensor]:
    """(grad h, grad w, the sum of the first one's terms' magnitudes)."""
    v, g = f64(h), f64(gy)
    gw = g if w is None else g * f64(w)
    s = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
    n = v * s
    grad = s * (gw - n * (gw * n).mean(-1, keepdim=True))
    terms = s * (gw.abs() + n.abs() * (gw * n).abs().mean(-1, keepdim=True))
    if gh is not None:
        grad, terms = grad + f64(gh), terms + f64(gh).abs()
    return grad, (g * n).flatten(0, -2).sum(0), terms


def e4m3(v: Tensor) -> Tensor:
    """The nearest value with 4 exponent and 3 mantissa bits, ties to even, of |v| <= 448."""
    step = e4m3_step(v)
    return torch.round(v / step) * step


def e4m3_step(v: Tensor) -> Tensor:
    return torch.exp2((torch.frexp(v).exponent.double() - 1).clamp(min=-6) - 3)


def no_distribution(x: Tensor) -> Tensor:
    """Rows with a NaN or +infinity, or nothing above -infinity."""
    x = f64(x)
    return torch.isnan(x).any(-1) | (x == torch.inf).any(-1) | (x == -torch.inf).all(-1)


def scores(x: Tensor, tokens: Tensor, top: int) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(logprobs, entropy, top log p, top tokens) of rows [n, vocab]."""
    bad = no_distribution(x)
    x = torch.where(bad[:, None], 0.0, f64(x))
    d = x - x.amax(-1, keepdim=True)  # a maximum of -1e38 would swallow the rest even here
    lp = d - torch.logsumexp(d, -1, keepdim=True)
    p = torch.exp(lp)
    H = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    t = tokens.cpu().long()
    at = torch.where(bad | (t >= x.shape[1]), torch.nan, lp.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0])
    values, ids = torch.sort(lp, dim=-1, descending=True, stable=True)
    nan = torch.tensor(torch.nan, dtype=torch.float64)
    return (torch.where(t < 0, 0.0, at), torch.where(bad, nan, H), torch.where(bad[:, None], nan, values[:, :top]),
            torch.where(bad[:, None], -1, ids[:, :top]))


def score_grads(x: Tensor, tokens: Tensor, a: Tensor, b: Tensor) -> Tensor:
    v = f64(x).requires_grad_()
    lp = torch.log_softmax(v, -1)
    p = torch.exp(lp)
    H = -torch.where(p > 0, p * torch.where(p > 0, lp, 0.0), 0.0).sum(-1)
    t = tokens.cpu().long()
    at = torch.where(t < 0, 0.0, lp.gather(1, t.clamp(min=0)[:, None])[:, 0])
    return torch.autograd.grad((f64(a) * at + f64(b) * H).sum(), v)[0]


def distill(x: Tensor, values: Tensor, ids: Tensor, tau: float) -> tuple[Tensor, Tensor, Tensor]:
    """(row losses, rows with entries, the gradient of the sum of the row losses) of rows [n, vocab]."""
    values, ids = f64(values), ids.cpu().long()
    keep = (ids >= 0) & (values != -torch.inf)
    some = keep.any(-1)
    v = torch.where(some[:, None], f64(x), 0.0).requires_grad_()
    lt = torch.log_softmax(torch.where(keep, values, torch.where(some[:, None], -torch.inf, 0.0)) / tau, -1)
    p = torch.where(keep, torch.exp(lt), 0.0)
    lq = torch.log_softmax(v / tau, -1).gather(1, ids.clamp(min=0))
    loss = tau ** 2 * torch.where(p > 0, p * (torch.where(p > 0, lt, 0.0) - lq), 0.0).sum(-1)
    grad = torch.autograd.grad(loss.sum(), v)[0]
    return loss.detach(), some, grad


# ---- 4-bit weights with group scales ----------------------------------------------------------------------------

def grouped_weight(codes: Tensor, scales: Tensor, zeros: Tensor | None, group: int, k: int) -> Tensor:
    """[n, k] values of packed codes (two a byte, the earlier element in the low half)."""
    c = codes.cpu().long()
    q = torch.stack([c % 16, c // 16], -1).flatten(1)[:, :k].double()
    at = torch.arange(k) // group
    z = 8.0 if zeros is None else f64(zeros)[:, at]
    return (q - z) * f64(scales)[:, at]
