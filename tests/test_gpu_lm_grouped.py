"""4-bit weights with group scales against the float64 oracle (oracle/lm.py).

With x and q - z small integers and power-of-two scales every partial sum is a multiple of 1/4 below 2^22, so fp32 sums are
exact in any order and the fp32 output is compared bit for bit.  With real values the error is at most one fp32 rounding for
each of the K + 32 additions of a sum, relative to T = |c| sum |s| (q + z) |x|, what is added up on the way (the zero
point's part is taken off each group's sum), plus the epilogue's 8, plus the output's own rounding."""

import pytest
import torch

from oracle import lm
from tests.conftest import announce

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
XTYPES = [torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _pack(q):
    n, k = q.shape
    q = torch.nn.functional.pad(q, (0, -k % 32)).view(n, -1, 2)
    return q[..., 0] + q[..., 1] * 16


def _layer(n, k, group, seed, zeros=True, exact=True, sdt=torch.float16):
    """(codes, scales, zeros); the codes behind a row's last element are not 0 (they must not matter)."""
    g = _gen(seed)
    groups = -(-k // group)
    q = torch.randint(0, 16, (n, -(-k // 32) * 32), generator=g).to(torch.uint8)
    s = 2.0 ** torch.randint(-2, 2, (n, groups), generator=g) if exact else torch.rand(n, groups, generator=g) * 0.02 + 1e-3
    z = torch.randint(0, 16, (n, groups), generator=g).to(torch.uint8) if zeros else None
    return _pack(q), s.to(sdt), z


def _ints(m, k, dt, seed):
    return torch.randint(-8, 9, (m, k), generator=_gen(seed)).float().to(dt)


def _c(x, m):
    return 2.0 ** torch.randint(-1, 2, (m,), generator=_gen(9)) if x.dtype == torch.float8_e4m3fn else None


def _run(gpu, x, layer, group, xs=None, **more):
    from dimq_amd import ops
    to = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    return ops.dimq_linear_grouped(to(x), to(layer[0]), to(layer[1]), to(layer[2]), group, x_scales=to(xs),
                                   **{k: to(v) if torch.is_tensor(v) else v for k, v in more.items()})


def _ref(x, layer, group, xs=None):
    y = x.float().double() @ lm.grouped_weight(*layer, group, x.shape[-1]).t()
    return y if xs is None else y * xs.double()[..., None]


SHAPES = [(1, 32, 1), (1, 33, 15), (3, 1000, 130), (16, 128, 16), (2, 4096, 48), (17, 96, 33), (31, 250, 16), (33, 1024, 100),
          (64, 160, 17), (65, 128, 128), (70, 1000, 130), (128, 64, 257), (130, 4100, 40), (300, 512, 384), (1, 20000, 5),
          (90, 31, 3)]


BOTH = pytest.mark.parametrize("variant", ["small_m", "mfma"])


@BOTH
@pytest.mark.parametrize("dt", XTYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_exact_sums(gpu, m, k, n, dt, variant):
    announce(f"grouped {m} {k} {n} {dt} {variant}")
    x = _ints(m, k, dt, m + k)
    xs = _c(x, m)
    for group, zeros in ((32, True), (64, True), (96, False), (128, True), (192, True), (256, False), (32768, True),
                         (2 ** 40, False), (2 ** 39 + 32, True)):
        layer = _layer(n, k, group, n + group % 1000, zeros, sdt=XTYPES[(group // 32) % 3])
        y = _run(gpu, x, layer, group, xs, out_dtype=torch.float32, variant=variant)
        assert torch.equal(y.cpu().double(), _ref(x, layer, group, xs)), (group, zeros)


@BOTH
@pytest.mark.parametrize("dt", XTYPES)
@pytest.mark.parametrize("m,k,n,group", [(1, 4096, 64, 128), (5, 64, 40, 32), (40, 1000, 70, 64), (100, 2048, 130, 128),
                                         (513, 640, 200, 128), (2, 96, 5, 96)])
def test_real_values(gpu, m, k, n, group, dt, variant):
    announce(f"grouped real {m} {k} {n} {dt} {variant}")
    g = _gen(m + k)
    x = torch.randn(m, k, generator=g) * torch.exp(torch.randn(k, generator=g) * 0.6)
    x = x.to(dt) if dt != torch.float8_e4m3fn else (x * 20).clamp(-448, 448).to(dt)
    xs = torch.rand(m, generator=g) if dt == torch.float8_e4m3fn else None
    bias, res = torch.randn(n, generator=g) * 0.1, torch.randn(m, n, generator=g)
    for zeros, act, sdt in ((True, None, torch.float16), (False, "relu", torch.float32), (True, "gelu", torch.bfloat16)):
        layer = _layer(n, k, group, 3, zeros, exact=False, sdt=sdt)
        r = res.bfloat16() if act == "relu" else None
        y = _run(gpu, x, layer, group, xs, bias=bias, residual=r, activation=act, variant=variant)
        assert y.dtype == (torch.bfloat16 if dt == torch.float8_e4m3fn else dt)
        ref = _ref(x, layer, group, xs) + bias.double() + (0 if r is None else r.double())
        plus = (layer[0], layer[1], torch.zeros_like(layer[1], dtype=torch.uint8))
        z = (torch.full_like(plus[2], 8) if layer[2] is None else layer[2]).double()
        T = (x.float().double().abs() @ (lm.grouped_weight(*plus, group, k) +
                                         (z * layer[1].double()).repeat_interleave(group, 1)[:, :k]).t())
        T = (T if xs is None else T * xs.double()[:, None]) + bias.abs().double() + (0 if r is None else r.double().abs())
        tol = (k + 40) * E * T
        if act == "relu":
            ref = ref.clamp(min=0)
        elif act == "gelu":
            tol = 1.13 * tol + 3e-7 * ref.abs()  # the slope's largest value; erf's error 1.5e-7, doubled for its arithmetic
            ref = 0.5 * ref * torch.special.erfc(-ref / 2 ** 0.5)
        tol = tol + torch.finfo(y.dtype).eps / 2 * ref.abs() * 1.0001 + torch.finfo(y.dtype).smallest_normal
        over = ((y.cpu().double() - ref).abs() / tol).max().item()
        assert over <= 1, f"{over} times the tolerance"


@BOTH
def test_fp32_inputs_are_not_rounded(gpu, variant):
    """24-bit numbers: the third of their parts counts.  One element a row, so the sum is one product."""
    announce("grouped fp32 bits")
    for m in (2, 80):
        x = torch.zeros(m, 256)
        at = torch.randint(0, 256, (m,), generator=_gen(1))
        v = torch.randint(2 ** 23, 2 ** 24, (m,), generator=_gen(2)).float() * 2.0 ** torch.randint(-60, 40, (m,), generator=_gen(3))
        x[torch.arange(m), at] = torch.where(torch.arange(m) % 2 == 0, v, -v)
        q = torch.ones(20, 256, dtype=torch.uint8)
        layer = (_pack(q), torch.ones(20, 2), torch.zeros(20, 2, dtype=torch.uint8))
        y = _run(gpu, x, layer, 128, variant=variant).cpu()
        assert torch.equal(y, x.sum(1, keepdim=True).expand(m, 20))


@BOTH
@pytest.mark.parametrize("m", [4, 100])
@pytest.mark.parametrize("dt", XTYPES)
def test_rows_that_are_not_finite_stay_alone(gpu, dt, m, variant):
    announce(f"grouped not finite {dt} {m}")
    k = 300
    x = _ints(m, k, torch.float32, 1)
    x[1, 5] = torch.nan
    if dt != torch.float8_e4m3fn:
        x[2, 299] = torch.inf
    x = x.to(dt)
    xs = _c(x, m)
    if xs is not None:
        xs[2] = torch.nan
    layer = _layer(50, k, 64, 2)
    y = _run(gpu, x, layer, 64, xs, out_dtype=torch.float32, variant=variant).cpu()
    assert not torch.isfinite(y[1:3]).any()
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(y[keep].double(), _ref(x[keep], layer, 64, None if xs is None else xs[keep]))


@BOTH
@pytest.mark.parametrize("dt", XTYPES)
@pytest.mark.parametrize("rows", [6, 150])
def test_strides_and_places(gpu, dt, rows, variant):
    """Rows of a larger tensor, odd starts, transposed and 3-D inputs; codes that do not start at 16 bytes."""
    from dimq_amd import ops
    announce(f"grouped strides {dt} {rows}")
    big = _ints(2 * rows, 700, dt, 1).to(gpu)
    flat = big.view(torch.uint8) if dt == torch.float8_e4m3fn else big
    codes, s, z = (t.to(gpu) for t in _layer(40, 256, 64, 2))
    odd = torch.empty(codes.numel() + 5, dtype=torch.uint8, device=gpu)
    odd[5:] = codes.flatten()
    for x in (big[::2, :256], big[:rows, 3:259], big[rows:, 8:264], flat[:256, :256].t().view(dt) if rows > 100 else big[:, 64:320],
              big[:rows, :512].view(rows, 2, 256) if dt == torch.float8_e4m3fn else big[:rows, :512].reshape(rows, 2, 256),
              big[4, 10:266], big[3:3, :256]):
        lead = x.shape[:-1]
        xs = torch.full(lead, 0.5, device=gpu) if dt == torch.float8_e4m3fn else None
        y = ops.dimq_linear_grouped(x, odd[5:].view(40, 128), s, z, 64, x_scales=xs, out_dtype=torch.float32, variant=variant)
        assert y.shape == (*lead, 40) and y.is_contiguous()
        assert torch.equal(y.cpu().double(), _ref(x.cpu(), (codes, s, z), 64, None if xs is None else xs.cpu()))


@BOTH
def test_more_columns_than_tiles_and_split_sums(gpu, variant):
    """Few tiles with a long reduction (cut along k), tiles beyond a multiple of the XCDs, and every number of row and column
    blocks that the single launch gives a work-group."""
    announce(f"grouped splits {variant}")
    for m, k, n in ((65, 16384, 64), (129, 8192, 300), (260, 256, 1300), (1000, 128, 1000), (3, 128, 2100), (20, 128, 2050),
                    (40, 256, 2049), (20, 128, 10300), (16, 128, 10245), (50, 128, 10250)):
        x = _ints(m, k, torch.bfloat16, 1)
        layer = _layer(n, k, 128, 2)
        y = _run(gpu, x, layer, 128, out_dtype=torch.float32, variant=variant)
        assert torch.equal(y.cpu().double(), _ref(x, layer, 128))
    for dt in (torch.float32, torch.float8_e4m3fn):
        for m, group in ((5, 32), (20, 32), (40, 32), (20, 64), (40, 64), (40, 128)):
            x = _ints(m, 128, dt, 1)
            layer = _layer(2050, 128, group, 2)
            y = _run(gpu, x, layer, group, _c(x, m), out_dtype=torch.float32, variant=variant)
            assert torch.equal(y.cpu().double(), _ref(x, layer, group, _c(x, m)))


# (rows, columns) that between them take every plan of the few-row kernel: 16, 32 or 64 rows by 16 to 64 columns a work-group
PLANS = [(5, 1001), (5, 8100), (16, 12280), (3, 16379), (33, 4099), (47, 8190), (30, 12271), (20, 16300), (60, 4090), (63, 8189),
         (50, 12280), (64, 16381), (130, 2050)]


@pytest.mark.parametrize("dt", XTYPES)
@pytest.mark.parametrize("m,n", PLANS)
def test_plans_of_few_rows(gpu, m, n, dt):
    announce(f"grouped plans {m} {n} {dt}")
    k = 1300
    x = _ints(m, k, dt, m)
    xs = _c(x, m)
    some = torch.cat([torch.randint(0, n, (60,), generator=_gen(4)), torch.arange(n - 20, n)])
    bias, res = torch.randint(-9, 9, (n,), generator=_gen(5)).float(), torch.randint(-9, 9, (m, n), generator=_gen(6)).float()
    for group in (32, 64, 128):
        g = _gen(group)
        codes = torch.randint(0, 256, (n, -(-k // 32) * 16), generator=g, dtype=torch.uint8)
        scales = 2.0 ** torch.randint(-2, 2, (n, -(-k // group)), generator=g)
        zeros = torch.randint(0, 16, scales.shape, generator=g, dtype=torch.uint8)
        y = _run(gpu, x, (codes, scales, zeros), group, xs, bias=bias, residual=res, out_dtype=torch.float32, variant="small_m")
        ref = _ref(x, (codes[some], scales[some], zeros[some]), group, xs) + bias[some] + res[:, some]
        assert torch.equal(y.cpu()[:, some].double(), ref), group


@pytest.mark.parametrize("group,most32,most16", [(128, 2.1e9, 4e9), (64, 2.1e9, 4e9), (96, 3.5e9, 8e9)])
@pytest.mark.parametrize("dt", XTYPES)
def test_products_that_auto_gives_to_each_kernel(gpu, dt, group, most32, most16):
    """On both sides of the sizes at which the kernels change."""
    from dimq_amd import _C
    announce(f"grouped routes {dt} {group}")
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 5}[dt]
    m = int((most32 if dt == torch.float32 else most16) / (1024 * 4096))
    for rows in (m, m + 1):
        x, layer = _ints(rows, 1024, dt, 1), _layer(4096, 1024, group, 2)
        xs = _c(x, rows)
        at = x.to(gpu)
        tiles = _C.lib.dimq_linear_grouped_workspace_bytes(at.data_ptr(), code, rows, 1024, 1024, group, 4096, 0) > 0
        assert tiles == (rows > m)
        y = _run(gpu, x, layer, group, xs, out_dtype=torch.float32)
        some = torch.randint(0, rows, (20,), generator=_gen(5))
        assert torch.equal(y.cpu()[some].double(), _ref(x[some], layer, group, None if xs is None else xs[some]))


def test_large_products_choose_tiles(gpu):
    announce("grouped large")
    x, layer = _ints(700, 1024, torch.bfloat16, 1), _layer(4096, 1024, 128, 2)
    y = _run(gpu, x, layer, 128, out_dtype=torch.float32)
    assert torch.equal(y, _run(gpu, x, layer, 128, out_dtype=torch.float32, variant="mfma"))
    rows = torch.randint(0, 700, (20,), generator=_gen(5))
    assert torch.equal(y.cpu()[rows].double(), _ref(x[rows], layer, 128))


def test_layer_of_a_linear(gpu):
    from dimq_amd import DIMQGroupedLinear
    announce("DIMQGroupedLinear")
    torch.manual_seed(0)
    lin = torch.nn.Linear(1000, 70)
    for symmetric in (False, True):
        mod = DIMQGroupedLinear.from_linear(lin, 64, symmetric=symmetric).to(gpu)
        w = lm.grouped_weight(mod.codes, mod.scales, mod.zeros, 64, 1000)
        # half a step, and the scale's own rounding (2^-11 of up to 15 steps)
        step = mod.scales.cpu().double().repeat_interleave(64, 1)[:, :1000]
        assert ((w - lin.weight.detach().double()).abs() <= step * (0.5 + 16 * 2.0 ** -11)).all()
        x = _ints(5, 1000, torch.float32, 1)
        y = mod(x.to(gpu))
        ref = x.double() @ w.t() + lin.bias.detach().double()
        T = x.double().abs() @ (step * 31).t() + 1
        assert ((y.cpu().double() - ref).abs() <= 1040 * E * T).all()
        state = mod.state_dict()
        again = DIMQGroupedLinear.from_linear(torch.nn.Linear(1000, 70), 64, symmetric=symmetric).to(gpu)
        again.load_state_dict(state)
        assert torch.equal(again(x.to(gpu)), y)


def test_norm_rows_feed_the_layer(gpu):
    """A decoder block's half as it would be served: norm with the residual to 8 bits, the grouped layer, its output added to
    the stream by the next norm; then the logits' alternatives."""
    from dimq_amd import DIMQGroupedLinear, ops
    from dimq_amd.modules import DIMQRMSNorm
    announce("served chain")
    torch.manual_seed(0)
    d, vocab = 256, 500
    norm1, norm2 = DIMQRMSNorm(d, eps=1e-6).to(gpu).bfloat16(), DIMQRMSNorm(d, eps=1e-6).to(gpu).bfloat16()
    lin, head = torch.nn.Linear(d, d), torch.nn.Linear(d, vocab, bias=False)
    layer, out = DIMQGroupedLinear.from_linear(lin).to(gpu), DIMQGroupedLinear.from_linear(head, out_dtype=torch.float32).to(gpu)
    for rows in (1, 7, 90):
        x, r = (torch.randn(rows, d, generator=_gen(i)).bfloat16().to(gpu) for i in (1, 2))
        with torch.no_grad():
            q, s, h = norm1.e4m3(x, residual=r)
            y = layer((q, s))
            q2, s2, h2 = norm2.e4m3(y, residual=h)
            logits = out((q2, s2))
            lp, H, tlp, tid = ops.token_logprobs(logits, torch.full((rows,), 3, device=gpu), 4)
        # each step from the values it was given
        w1, w2 = (lm.grouped_weight(m.codes, m.scales, m.zeros, 128, d) for m in (layer, out))
        ref = (q.float().double().cpu() * s.double().cpu()[:, None]) @ w1.t() + lin.bias.detach().double()
        assert ((y.double().cpu() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-3).all()
        assert torch.equal(h2, (y.float() + h.float()).bfloat16())
        ref = (q2.float().double().cpu() * s2.double().cpu()[:, None]) @ w2.t()
        assert ((logits.double().cpu() - ref).abs() <= 1e-4).all()
        want = lm.scores(logits, torch.full((rows,), 3), 4)
        assert torch.equal(tid.cpu(), want[3]) and ((lp.cpu().double() - want[0]).abs() < 1e-5).all()


def test_streams_and_graphs(gpu):
    announce("grouped graph")
    from dimq_amd import ops
    for m, dt, variant in ((3, torch.bfloat16, "small_m"), (100, torch.bfloat16, "mfma"), (70, torch.float32, "mfma"),
                           (200, torch.float8_e4m3fn, "mfma")):
        x = _ints(m, 1000, dt, 1).to(gpu)
        xs = torch.ones(m, device=gpu) if dt == torch.float8_e4m3fn else None
        codes, s, z = (t.to(gpu) for t in _layer(96, 1000, 128, 2))
        call = lambda: ops.dimq_linear_grouped(x, codes, s, z, 128, x_scales=xs, out_dtype=torch.float32, variant=variant)  # noqa: E731,B023
        want = call()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert torch.equal(call(), want)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call()
        for seed in (3, 4, 5):
            x.copy_(_ints(m, 1000, dt, seed).to(gpu))
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            assert torch.equal(got, call())


def test_gradients_are_refused(gpu):
    from dimq_amd import ops
    x = torch.randn(3, 64, device=gpu, requires_grad=True)
    codes, s, z = (t.to(gpu) for t in _layer(8, 64, 32, 2))
    y = ops.dimq_linear_grouped(x, codes, s, z, 32)
    with pytest.raises(RuntimeError, match="not implemented"):
        y.sum().backward()
    with torch.no_grad():
        assert not ops.dimq_linear_grouped(x, codes, s, z, 32).requires_grad
