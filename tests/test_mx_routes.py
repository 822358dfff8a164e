"""Every kernel that the plan of the microscaled products can choose, over more stages of the reduction than its ring in
the LDS holds twice, with odd ends in all three sizes and a last stage that is not whole.

Each route is a kernel (its number in dimq_mx_linear_route) with a whole or a split reduction, for the forward product (0),
the gradient to the input (1) and to the weight (2); the gradients also with one plane of bf16 parts and with several.

Operands are values of the formats with common scales, so that products and sums are whole numbers of a step below 2^24 of
it: exact in fp32 in any order, and every output has to be equal.  Gradients with random bits are compared within
(r + 8) 2^-23 sum |a b| over r terms (test_gpu_mx.py)."""

import itertools

import pytest
import torch

from tests.conftest import announce
from tests.test_gpu_mx import _check, _gen

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
KERNELS = {1: "256x256", 2: "256x192", 3: "128x128", 4: "128x128 of four slots", 5: "64x64"}
SLOTS = {1: 2, 2: 2, 3: 2, 4: 4, 5: 3}
PARTS = {F32: 3, F16: 2, BF16: 1}

# product, kernel, split, dtype, M, K, N
CASES = [
    (0, 1, False, BF16, 3275, 1047, 3705), (0, 2, False, BF16, 2475, 1053, 3253), (0, 3, False, BF16, 1731, 1041, 1837),
    (0, 4, False, F32, 1281, 6467, 1619), (0, 5, False, F16, 279, 1553, 41),
    (0, 1, True, BF16, 2319, 14453, 1747), (0, 2, True, F16, 1733, 10015, 2307), (0, 3, True, F32, 1247, 11943, 793),
    (0, 4, True, BF16, 911, 12059, 1305), (0, 5, True, F16, 533, 5221, 451),
    (1, 1, False, BF16, 6545, 1837, 289), (1, 1, False, F32, 9273, 1205, 109), (1, 1, True, BF16, 2879, 1471, 7083),
    (1, 1, True, F32, 1105, 3929, 2319), (1, 2, False, BF16, 1187, 6649, 289), (1, 2, False, F32, 13135, 551, 71),
    (1, 2, True, BF16, 1927, 2131, 3403), (1, 2, True, F32, 2039, 2069, 1487), (1, 3, False, BF16, 1825, 1701, 305),
    (1, 3, False, F32, 1101, 2699, 65), (1, 3, True, BF16, 1007, 1049, 3347), (1, 3, True, F32, 739, 657, 2291),
    (1, 4, False, BF16, 1555, 1415, 1685), (1, 4, False, F32, 1805, 1117, 465), (1, 4, True, BF16, 825, 1323, 3277),
    (1, 4, True, F16, 769, 1223, 1659), (1, 5, False, BF16, 19, 41, 405), (1, 5, False, F32, 21, 39, 135),
    (1, 5, True, BF16, 19, 35, 8713), (1, 5, True, F32, 21, 33, 2613),
    (2, 1, False, BF16, 259, 3595, 3569), (2, 1, False, F16, 133, 4851, 2315), (2, 1, True, BF16, 4771, 463, 8987),
    (2, 1, True, F32, 2751, 1205, 3519), (2, 2, False, BF16, 277, 4619, 1699), (2, 2, False, F32, 101, 3687, 2185),
    (2, 2, True, BF16, 4055, 2077, 2129), (2, 2, True, F32, 1153, 2271, 1797), (2, 3, False, BF16, 323, 1737, 1783),
    (2, 3, False, F32, 73, 779, 3845), (2, 3, True, BF16, 4357, 1335, 859), (2, 3, True, F32, 1325, 1131, 905),
    (2, 4, False, BF16, 1577, 1793, 1221), (2, 4, False, F32, 495, 2721, 729), (2, 4, True, BF16, 3549, 1455, 805),
    (2, 4, True, F32, 3157, 593, 513), (2, 5, False, BF16, 507, 37, 17), (2, 5, False, F32, 139, 33, 17),
    (2, 5, True, BF16, 8173, 35, 19), (2, 5, True, F32, 2613, 37, 23),
]


def _route(product, dt, M, K, N):
    """(kernel, slices) or None for the single launch of few rows"""
    from dimq_amd import _C
    r = _C.lib.dimq_mx_linear_route(product, {F32: _C.F32, F16: _C.F16, BF16: _C.BF16}[dt], M, K, N)
    assert r >= 0
    return (r % 8, r // 8) if r else None


@pytest.mark.parametrize("case", CASES, ids=str)
def test_case_takes_its_route(case):
    product, kernel, split, dt, M, K, N = case
    got, slices = _route(product, dt, M, K, N)
    assert (got, slices > 1) == (kernel, split), f"{KERNELS[got]} in {slices} slices"
    if product == 0:
        blocks = -(-K // 32)
        stages, whole = -(-blocks // 8), blocks % 8 == 0 or K % 32 == 0
    else:
        length = N if product == 1 else M
        stages, whole = -(-length // 64) * PARTS[dt], length % 64 == 0
    assert stages // slices > 2 * SLOTS[kernel] and not whole
    assert M % 2 and K % 2 and N % 2


def test_no_other_route_is_chosen():
    """Over sizes from one tile to a large layer, each route that the plan takes is one that the cases run."""
    run = {(p, k, s, p > 0 and dt != BF16) for p, k, s, dt, *_ in CASES}
    ms = [1, 17, 65, 100, 197, 300, 515, 777, 1003, 1576, 2048, 2650, 4096, 6000, 8192, 12608, 16384, 20000]
    ks = [32, 72, 200, 512, 768, 1000, 1500, 2304, 4096, 6504, 8192, 11008, 16384]
    ns = [16, 40, 100, 256, 384, 768, 1138, 2048, 2304, 3895, 4096, 6000, 8192, 11008]
    taken = set()
    for product, dt, M, K, N in itertools.product((0, 1, 2), (F32, F16, BF16), ms, ks, ns):
        r = _route(product, dt, M, K, N)
        if r:
            taken.add((product, r[0], r[1] > 1, product > 0 and dt != BF16))
    assert taken <= run, taken - run
    assert len(taken) > 30  # and the sizes are not all of one kind


def test_sizes_without_a_route():
    from dimq_amd import _C
    R = _C.lib.dimq_mx_linear_route
    for a in ((0, _C.F32, 0, 32, 32), (0, _C.F32, 8, 0, 32), (1, _C.F32, 8, 32, 0), (3, _C.F32, 8, 32, 32),
              (-1, _C.F32, 8, 32, 32), (0, _C.F64, 8, 32, 32), (2, _C.U8, 8, 32, 32)):
        assert R(*a) == -1
    assert R(0, _C.BF16, 1, 4096, 4096) == 0


def _blocks(rows, cols, levels, top, units, seed, gpu):
    """Values of a block format: whole numbers of -levels..levels, the first of each block +-top so that the block's scale
    is the one meant, times 1 or 2 by the block, times `units`."""
    g = _gen(seed)
    nb = -(-cols // 32)
    v = levels[torch.randint(0, len(levels), (rows, nb, 32), generator=g)]
    v[..., 0] = top
    v *= 1 - 2 * torch.randint(0, 2, v.shape, generator=g, dtype=torch.int8)
    v = v.to(gpu).float() * torch.randint(1, 3, (rows, nb, 1), generator=g).to(gpu) * units
    return v.flatten(1)[:, :cols]


def _blocks4(rows, cols, seed, gpu):  # doubled levels of the 4-bit format
    return _blocks(rows, cols, torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], dtype=torch.int8), 12, 0.5, seed, gpu)


def _blocks8(rows, cols, seed, gpu):
    return _blocks(rows, cols, torch.arange(0, 128, dtype=torch.int8), 64, 1 / 64, seed, gpu)


def _mm(a, b):
    return a.double().contiguous() @ b.double().contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_products(gpu, case):
    from dimq_amd import mx
    product, kernel, split, dt, M, K, N = case
    announce(f"product {product} on {KERNELS[kernel]}{' split' if split else ''} {dt} {M}x{K} -> {N}")
    if product == 0:
        x, w = _blocks4(M, K, 1, gpu), _blocks4(N, K, 2, gpu)
        c, s = mx.quantize_mxfp4(w)
        y = mx.mxfp4_linear(x.to(dt), c, s, out_dtype=F32)
        assert torch.equal(y.double(), _mm(x, w.t()))  # below 14453 x 144 in steps of 1/4
        return
    other = _blocks4(N, K, 2, gpu) if product == 1 else _blocks8(M, K, 3, gpu)
    if product == 1:
        c, s = mx.quantize_mxfp4(other)

        def call(g):
            return mx.mxfp4_linear_grad_input(g, c, s, K, F32)
    else:
        c, s = mx.compress_activation(other)

        def call(g):
            return mx.linear_grad_weight(g, c, s, K, bias=False)[0]
    whole = torch.randint(-4, 5, (M, N), generator=_gen(4)).to(gpu, dt)
    # below 8713 x 4 x 12 in steps of 1/2, or 8173 x 4 x 254 in steps of 1
    ref = _mm(whole, other) if product == 1 else _mm(whole.t(), other)
    assert torch.equal(call(whole).double(), ref)
    bits = (torch.randn(M, N, generator=_gen(5)) * 0.01).to(gpu, dt)
    ref, S = ((_mm(bits, other), _mm(bits.abs(), other.abs())) if product == 1 else
              (_mm(bits.t(), other), _mm(bits.abs().t(), other.abs())))
    _check(call(bits), ref.cpu(), S.cpu(), PARTS[dt] * (N if product == 1 else M))
