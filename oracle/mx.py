"""Microscaled formats in float64 on the CPU, from their definition: blocks of 32 along the last dimension share a power
of two; 4-bit floats {0, .5, 1, 1.5, 2, 3, 4, 6} or 8-bit integers in units of 1/64, to nearest, ties to the even code."""

from __future__ import annotations

import math

import torch
from torch import Tensor

FP4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
INT8 = [i / 64 for i in range(128)]


def quantize(x: Tensor, bits: int) -> tuple[Tensor, Tensor]:
    """(level numbers with the sign, [rows, blocks, 32], and scale bytes [rows, blocks]) of x [rows, cols]; a block with a NaN
    or an infinity has level 0 throughout and scale 255.  The sign of a zero is not kept."""
    levels, emax = (FP4, 2) if bits == 4 else (INT8, 0)
    x = x.detach().cpu().double()
    rows, cols = x.shape
    nb = -(-cols // 32)
    v = torch.zeros(rows, nb * 32, dtype=torch.float64)
    v[:, :cols] = x
    v = v.view(rows, nb, 32)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    top = torch.where(bad, 1.0, top)
    e = torch.where(top > 0, torch.frexp(top).exponent.double() - 1 - emax, -127.0).clamp_min(-127)
    a = torch.where(bad[..., None], 0.0, v.abs()) / torch.exp2(e)[..., None]
    lev = torch.tensor(levels, dtype=torch.float64)
    mid = (lev[:-1] + lev[1:]) / 2
    up = torch.searchsorted(mid, a, right=True)    # a tie counted to the level above
    down = torch.searchsorted(mid, a, right=False)  # and below
    i = torch.where(up % 2 == 0, up, down)
    scale = torch.where(bad, 255.0, e + 127).to(torch.uint8)
    return torch.where(v < 0, -i, i), scale


def values(level: Tensor, scale: Tensor, bits: int, cols: int) -> Tensor:
    lev = torch.tensor(FP4 if bits == 4 else INT8, dtype=torch.float64)
    v = lev[level.abs()] * torch.sign(level) * torch.exp2(scale.double() - 127)[..., None]
    v = torch.where((scale == 255)[..., None], torch.nan, v)
    return v.flatten(-2)[..., :cols]


def q4(x: Tensor) -> Tensor:
    return values(*quantize(x, 4), 4, x.shape[1])


def q8(x: Tensor) -> Tensor:
    return values(*quantize(x, 8), 8, x.shape[1])


def unpack4(codes: Tensor, scales: Tensor, cols: int) -> Tensor:
    """Values of packed 4-bit codes [rows, 16 blocks] as the layout says."""
    c = codes.cpu().long()
    c = torch.stack([c % 16, c // 16], -1).view(c.shape[0], -1, 32)
    return values(torch.where(c >= 8, -(c - 8), c), scales.cpu(), 4, cols)


def unpack8(codes: Tensor, scales: Tensor, cols: int) -> Tensor:
    return values(codes.cpu().long().view(codes.shape[0], -1, 32), scales.cpu(), 8, cols)


def gelu(h: Tensor) -> Tensor:
    h = h.detach().cpu().double()
    return h * torch.special.erfc(-h / math.sqrt(2)) / 2


def gelu_slope(h: Tensor) -> Tensor:
    h = h.detach().cpu().double()
    return torch.special.erfc(-h / math.sqrt(2)) / 2 + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi)
