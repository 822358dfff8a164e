"""Microscaled formats: what the 4-bit products and the 8-bit activation checkpoints compute, and on which sizes.

Formats, along the last dimension in blocks of 32 (a last block may be short), one power of two per block:

* 4 bits: scale 2^(floor(log2(max|v|)) - 2), elements sign, 2 exponent bits, 1 mantissa bit
  ({0, .5, 1, 1.5, 2, 3, 4, 6} and their negatives), to nearest, ties to the even code, saturating at 6;
* 8 bits: scale 2^floor(log2(max|v|)), elements integers of -127..127 in units of 1/64 of the scale, to nearest even,
  saturating.

Both scales are at least 2^-127; a block that holds a NaN or an infinity stands for NaN throughout.

Kinds of cases (Q4, Q8: the value a tensor's codes stand for):

* ``quantize``  x -> Q4(x), Q8(x), from one read of x;
* ``linear``    serving: y = act(Q4(x) W^T + b) on weights kept as 4-bit codes;
* ``train``     a linear layer's training step with straight-through gradients: y = Q4(x) Q4(W)^T + b, and for the
  upstream g: gx = g Q4(W), gw = g^T Q8(x) (all that is kept of x is its 8-bit form), gb = sum of g over the rows;
* ``gelu``      y = gelu(h), h kept in 8 bits, and gh = g gelu'(Q8(h)).
"""

import math

import torch

own = False

_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # one token, and sixteen sequences' next tokens, through a square layer: latency and the weights' bytes
        dict(name="linear_1x4096_4096", kind="linear", rows=1, k=4096, n=4096, dtype="bf16", act="none"),
        dict(name="linear_16x4096_4096", kind="linear", rows=16, k=4096, n=4096, dtype="bf16", act="none"),
        # odd sizes throughout, single precision
        dict(name="linear_1003x1000_1030", kind="linear", rows=1003, k=1000, n=1030, dtype="fp32", act="gelu"),
        # ViT-B/16's qkv layer on 64 images of 197 tokens
        dict(name="linear_12608x768_2304", kind="linear", rows=12608, k=768, n=2304, dtype="bf16", act="none"),
        # a long prompt batch through a wide layer
        dict(name="linear_16384x8192_8192", kind="linear", rows=16384, k=8192, n=8192, dtype="bf16", act="none"),
        # the same qkv layer trained; an odd layer trained in half precision; a wide one
        dict(name="train_12608x768_2304", kind="train", rows=12608, k=768, n=2304, dtype="bf16"),
        dict(name="train_515x1000_770", kind="train", rows=515, k=1000, n=770, dtype="fp16"),
        dict(name="train_8192x4096_4096", kind="train", rows=8192, k=4096, n=4096, dtype="bf16"),
        # the activation between an MLP's layers: 64 images' tokens, and a small odd one
        dict(name="gelu_12608x2048", kind="gelu", rows=12608, k=2048, dtype="bf16"),
        dict(name="gelu_197x777", kind="gelu", rows=197, k=777, dtype="fp32"),
        # a layer's master weights, and a batch of activations of odd width
        dict(name="quantize_4096x4096", kind="quantize", rows=4096, k=4096, dtype="fp32"),
        dict(name="quantize_3001x1001", kind="quantize", rows=3001, k=1001, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "train", "gelu", "quantize"])
    case = dict(kind=kind, rows=_log(rng, 1, 16384), k=_log(rng, 40, 8192), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    if rng.random() < 0.5:  # the sizes of most layers
        case["k"] = max(64, case["k"] // 64 * 64)
    if kind in ("linear", "train"):
        case["n"] = _log(rng, 40, 8192)
        if rng.random() < 0.5:
            case["n"] = max(64, case["n"] // 64 * 64)
    if kind == "linear":
        case["act"] = rng.choice(["none", "relu", "gelu"])
    if kind == "train":  # three products and as many types of gradients: not above the largest listed one
        case["rows"] = max(2, case["rows"] // 2)
        case["n"] = min(case["n"], 4096)
        case["k"] = min(case["k"], 4096)
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, k, dt = case["rows"], case["k"], _DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    # activations: a common spread and, as trained networks show, some features that are much larger
    wide = torch.exp(normal(k) * 0.6)
    s = {"case": case, "x": (normal(rows, k) * wide).to(dt)}
    if case["kind"] == "quantize":
        return s
    if case["kind"] == "gelu":
        s["x"] = (normal(rows, k) * 1.5).to(dt)
        s["g"] = (normal(rows, k) * 1e-2).to(dt)
        return s
    n = case["n"]
    w = normal(n, k) / math.sqrt(k)
    s["b"] = normal(n) * 0.1
    if case["kind"] == "train":
        s["w"] = w  # the optimiser's weights, in single precision
        s["g"] = (normal(rows, n) * 1e-2).to(dt)
        return s
    # serving: the program keeps the packed weights, as the format lays them out: two codes a byte, the earlier element
    # in the low half, rows padded to whole blocks, one scale byte (its exponent + 127) a block
    s["codes"], s["scales"] = _pack4(w)
    return s


# ---- plain forms, 32 bits -----------------------------------------------------------------------------------------

def _blocks(x):
    """x [rows, k] as fp32 [rows, blocks, 32], zeros past k."""
    k = x.shape[-1]
    pad = -k % 32
    return torch.nn.functional.pad(x.float(), (0, pad)).view(x.shape[0], (k + pad) // 32, 32)


def _exponent(v):
    """Biased exponent (that of 2^-127: 0) of each block's largest magnitude, and whether the block is all finite."""
    bits = v.abs().amax(-1, keepdim=True).view(torch.int32)
    return bits >> 23, bits < 0x7F800000


def _fp4_steps(v, scale):
    """|v| / scale rounded to the eight magnitudes, and the scale's reciprocal applied exactly (powers of two)."""
    a = (v.abs() / scale).clamp(max=6.0)
    # the step between neighbours is 1/2 below 2, 1 below 4, 2 from there; torch.round takes ties to even, which is
    # the even code in each of the three ranges
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.round(a / step) * step


def _pow2(e):
    """2^(e - 127), e in 0..254, from its bits."""
    return torch.where(e == 0, 0x400000, e << 23).to(torch.int32).view(torch.float32)


def _q4(x):
    v = _blocks(x)
    e, finite = _exponent(v)
    scale = _pow2((e - 2).clamp(min=0))
    q = torch.where(finite, torch.copysign(_fp4_steps(v, scale), v) * scale, torch.nan)
    return q.view(x.shape[0], -1)[:, :x.shape[1]]


def _q8(x):
    v = _blocks(x)
    e, finite = _exponent(v)
    scale = _pow2(e)
    q = torch.where(finite, torch.round(v / scale * 64).clamp(-127, 127) / 64 * scale, torch.nan)
    return q.view(x.shape[0], -1)[:, :x.shape[1]]


def _pack4(w):
    v = _blocks(w)
    e, _ = _exponent(v)
    e = (e - 2).clamp(min=0)
    a = _fp4_steps(v, _pow2(e))
    level = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (level + (v < 0).to(torch.uint8) * 8).view(w.shape[0], -1, 2)
    return code[..., 0] + code[..., 1] * 16, e.view(w.shape[0], -1).to(torch.uint8)


def _unpack4(codes, scales, k):
    c = torch.stack([codes & 15, codes >> 4], dim=-1).view(codes.shape[0], -1, 32).int()
    level = (c & 7).float()
    a = torch.where(level < 4, level / 2, torch.where(level < 6, level - 2, level * 2 - 8))
    v = torch.where(c >= 8, -a, a) * _pow2(scales.int())[..., None]
    return v.view(codes.shape[0], -1)[:, :k]


def _act(y, act):
    if act == "relu":
        return torch.where(y < 0, 0.0, y)
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y


def run(s):
    case, x = s["case"], s["x"]
    kind, dt = case["kind"], x.dtype
    if own:
        from dimq_amd import mx

        if kind == "quantize":
            c4, s4, c8, s8 = mx.quantize_and_compress(x)
            return (mx.dequantize_mxfp4(c4, s4, case["k"], torch.float32),
                    mx.decompress_activation(c8, s8, case["k"], torch.float32))
        if kind == "linear":
            return mx.mxfp4_linear(x, s["codes"], s["scales"], s["b"], activation=case["act"])
        x = x.detach().requires_grad_()
        if kind == "gelu":
            y = mx.gelu(x)
            return y.detach(), torch.autograd.grad(y, x, s["g"])[0]
        w, b = s["w"].detach().requires_grad_(), s["b"].detach().requires_grad_()
        y = mx.linear(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), s["g"]))

    if kind == "quantize":
        return _q4(x), _q8(x)
    if kind == "linear":
        y = _q4(x) @ _unpack4(s["codes"], s["scales"], case["k"]).t() + s["b"]
        return _act(y, case["act"]).to(dt)
    g = s["g"].float()
    if kind == "gelu":
        h, hq = x.float(), _q8(x)
        slope = 0.5 * (1 + torch.erf(hq * math.sqrt(0.5))) + hq * torch.exp(-0.5 * hq * hq) / math.sqrt(2 * math.pi)
        return _act(h, "gelu").to(dt), (g * slope).to(dt)
    wq = _q4(s["w"])
    y = _q4(x) @ wq.t() + s["b"]
    return y.to(dt), (g @ wq).to(dt), g.t() @ _q8(x), g.sum(0)


# ---- 64 bits ------------------------------------------------------------------------------------------------------

def _nearest(x, levels, ties_up, emax):
    """Every element of x to the nearest of `levels` (ascending magnitudes, times 2^(floor(log2 max) - emax) of its
    block); a tie between levels i and i + 1 goes up where i is in ties_up."""
    x = x.double()
    out = torch.empty_like(x)
    mid = [(a + b) / 2 for a, b in zip(levels, levels[1:])]
    mid = [math.nextafter(m, 0) if i in ties_up else m for i, m in enumerate(mid)]
    mid = torch.tensor(mid, dtype=torch.float64, device=x.device)
    lev = torch.tensor(levels, dtype=torch.float64, device=x.device)
    whole = x.shape[1] // 32 * 32
    for at, part in ((0, x[:, :whole].unflatten(1, (whole // 32, 32))), (whole, x[:, whole:].unsqueeze(1))):
        if part.numel() == 0:
            continue
        top = part.abs().amax(2, keepdim=True)
        e = torch.where(top > 0, torch.frexp(top).exponent.double() - 1 - emax, -127.0).clamp(min=-127)
        scale = torch.exp2(e)
        q = lev[torch.bucketize((part.abs() / scale).contiguous(), mid)] * scale * torch.sign(part)
        q = torch.where(torch.isfinite(top), q, torch.nan)
        out[:, at:at + q.shape[1] * q.shape[2]] = q.flatten(1)
    return out


def _exact4(x):
    return _nearest(x, [0, 0.5, 1, 1.5, 2, 3, 4, 6], (1, 3, 5), 2)


def _exact8(x):
    return _nearest(x, [i / 64 for i in range(128)], range(1, 127, 2), 0)


def exact(case, seed):
    s = prepare(case, seed)
    x, kind = s["x"], case["kind"]
    if kind == "quantize":
        return _exact4(x), _exact8(x)
    if kind == "gelu":
        h, hq = x.double(), _exact8(x)
        root = math.sqrt(2)
        return (h * torch.special.erfc(-h / root) / 2,
                s["g"].double() * (torch.special.erfc(-hq / root) / 2 + hq * torch.exp(-hq.square() / 2) / math.sqrt(2 * math.pi)))
    if kind == "linear":
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64,
                             device=x.device)
        codes = s["codes"].long()
        w = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device=x.device)
        w[:, 0::2], w[:, 1::2] = table[codes % 16], table[codes // 16]
        w *= torch.exp2(s["scales"].double() - 127).repeat_interleave(32, dim=1)
        y = torch.addmm(s["b"].double(), _exact4(x), w[:, :case["k"]].t())
        if case["act"] == "relu":
            y = torch.clamp(y, min=0)
        if case["act"] == "gelu":
            y = y * torch.special.erfc(-y / math.sqrt(2)) / 2
        return y
    w, g = _exact4(s["w"]), s["g"].double()
    return torch.addmm(s["b"].double(), _exact4(x), w.t()), g @ w, g.t() @ _exact8(x), g.sum(0)


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    m, k, e = case["rows"], case["k"], _SIZE[case["dtype"]]
    if case["kind"] == "quantize":
        return {"bytes": m * k * (e + 8), "flops": 6 * m * k}
    if case["kind"] == "gelu":  # h read, y written, g read, gh written
        return {"bytes": m * k * 4 * e, "flops": 60 * m * k}
    n = case["n"]
    if case["kind"] == "linear":
        return {"bytes": m * k * e + n * k * 17 // 32 + 4 * n + m * n * e, "flops": 2 * m * n * k}
    # x, w, b, g read; y, gx, gw, gb written
    return {"bytes": 2 * m * k * e + 2 * 4 * n * k + 8 * n + 2 * m * n * e, "flops": 6 * m * n * k}
