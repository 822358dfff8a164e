"""The microscaled layers as a program uses them: the serving module, the example that trains and serves a block, the
gradients of a whole step captured into a graph, the backward entry point's outputs one by one, and its refusals."""

import ctypes

import pytest
import torch

from oracle import mx as omx
from tests.conftest import announce
from tests.test_gpu_mx import _acts, _check, _gen, _step

BF16 = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5, 300])
def test_serving_module(gpu, rows):
    import torch.nn as nn

    from dimq_amd import DIMQMXFP4Linear
    announce(f"module {rows}")
    torch.manual_seed(rows)
    lin = nn.Linear(200, 72)
    x, r = _acts(rows, 200, BF16, rows), torch.randn(rows, 72, generator=_gen(3)).to(BF16)
    mod = DIMQMXFP4Linear.from_linear(lin.to(gpu))
    assert (mod.in_features, mod.out_features) == (200, 72) and set(mod.state_dict()) == {"codes", "scales", "bias"}
    xq, wq = omx.q4(x), omx.q4(lin.weight.detach().cpu())
    b = lin.bias.detach().cpu().double()
    ref, S = xq @ wq.t() + b + r.double(), xq.abs() @ wq.abs().t() + b.abs() + r.double().abs()
    _check(mod(x.to(gpu), residual=r.to(gpu)), ref, S, 200)
    _check(mod(x.view(1, rows, 200).to(gpu), activation="relu").view(rows, 72), (ref - r.double()).clamp_min(0), S, 200)
    out = DIMQMXFP4Linear.from_linear(lin, out_dtype=torch.float32)(x.to(gpu))
    assert out.dtype == torch.float32
    _check(out, ref - r.double(), S, 200)


@pytest.mark.gpu
def test_example_trains_and_serves(gpu):
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parents[1] / "examples" / "mxfp4_mlp.py"
    spec = importlib.util.spec_from_file_location("mxfp4_mlp", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    announce("example")
    losses, trained, served, single = example.run(rows=512, width=256, steps=12)
    assert losses[-1] < 0.8 * losses[0], losses
    # the same products; serving rounds once (residual in fp32) where the training block rounds the layer's output and the
    # sum, and its hidden activations can fall on the other side of a 4-bit border: half a step of a few of 512 of them
    scale = trained.float().abs().max()
    assert (trained.float() - served.float()).abs().max() <= 0.05 * scale
    assert (single.float() - served[:8].float()).abs().max() <= 0.05 * scale


@pytest.mark.gpu
def test_linear_of_no_rows_trains(gpu):
    from dimq_amd import mx
    x = torch.zeros(0, 64, device=gpu, requires_grad=True)
    w, b = torch.randn(24, 64, device=gpu, requires_grad=True), torch.randn(24, device=gpu, requires_grad=True)
    y = mx.linear(x, w, b)
    assert y.shape == (0, 24)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    assert gx.shape == (0, 64) and gw.shape == (24, 64) and not gw.any() and not gb.any()


@pytest.mark.gpu
def test_without_gradients(gpu):
    """The same values where no backward pass can follow, and nothing kept for one."""
    from dimq_amd import mx
    x, h = _acts(200, 96, BF16, 1).to(gpu), torch.randn(70, 129, generator=_gen(2)).to(gpu).requires_grad_()
    w = torch.randn(48, 96, generator=_gen(3)).to(gpu).requires_grad_()
    announce("no gradients")
    y, z = mx.linear(x, w), mx.gelu(h)
    with torch.no_grad():
        y2, z2 = mx.linear(x, w), mx.gelu(h)
    assert torch.equal(y, y2) and torch.equal(z, z2)
    assert y.requires_grad and z.requires_grad and not y2.requires_grad and not z2.requires_grad
    assert torch.equal(mx.gelu(h.detach()), z2) and torch.equal(mx.linear(x, w.detach()), y2)


@pytest.mark.gpu
def test_step_captured_in_a_graph(gpu):
    """A layer's forward and backward pass in one graph; every replay against the eager step."""
    x, w = torch.zeros(300, 160, device=gpu, dtype=BF16), torch.randn(224, 160, generator=_gen(1)).to(gpu)
    b, g = torch.randn(224, generator=_gen(2)).to(gpu), torch.zeros(300, 224, device=gpu, dtype=BF16)
    announce("captured step")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _step(x, w, b, g)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(x, w, b, g)
    for i in range(3):
        x.copy_(torch.randn(300, 160, generator=_gen(10 + i)))
        g.copy_(torch.randn(300, 224, generator=_gen(20 + i)))
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, _step(x, w, b, g)):
            assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, BF16])
def test_backward_outputs_one_by_one(gpu, dt):
    """dimq_mx_linear_backward with every choice of outputs gives the bits of the call for all three."""
    from dimq_amd import _C, mx
    M, K, N = 333, 200, 137
    announce(f"backward {dt}")
    x, w = _acts(M, K, dt, 1).to(gpu), torch.randn(N, K, generator=_gen(2)).to(gpu)
    g = (_acts(M, N, dt, 3) * 2.0 ** -4).to(gpu)
    c, s = mx.quantize_mxfp4(w)
    c8, s8 = mx.compress_activation(x)
    code = {torch.float32: _C.F32, torch.float16: _C.F16, BF16: _C.BF16}[dt]
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def p(t):
        return None if t is None else ctypes.c_void_p(t.data_ptr())

    def call(which):
        out = [torch.full(shape, 7.0, device=gpu, dtype=d) if which >> i & 1 else None
               for i, (shape, d) in enumerate((((M, K), dt), ((N, K), torch.float32), ((N,), torch.float32)))]
        need = _C.lib.dimq_mx_linear_backward_workspace_bytes(p(g), code, M, N, N, K, which)
        ws = torch.empty(max(need, 256), dtype=torch.uint8, device=gpu)
        rc = _C.lib.dimq_mx_linear_backward(p(g), code, M, N, N, p(c), p(s), p(c8), p(s8), K, p(out[0]), code, p(out[1]),
                                            _C.F32, p(out[2]), _C.F32, p(ws), need, stream)
        assert rc == 0, _C.lib.dimq_last_error()
        return out

    full = call(7)
    assert torch.equal(full[0], mx.mxfp4_linear_grad_input(g, c, s, K))
    gw, gb = mx.linear_grad_weight(g, c8, s8, K)
    assert torch.equal(full[1], gw) and torch.equal(full[2], gb)
    for which in range(7):
        for a, b in zip(call(which), full):
            assert a is None or torch.equal(a, b)


def test_backward_refuses():
    from dimq_amd import _C
    L = _C.lib

    def ptr(a=4096):  # a non-null pointer that no refused call reads
        return ctypes.c_void_p(a)

    def refused(text, **change):
        a = dict(g=ptr(), gdt=_C.F32, M=2, N=8, ldg=8, c=ptr(), s=ptr(), c8=ptr(), s8=ptr(), K=32, gx=ptr(), xdt=_C.F32, gw=ptr(),
                 wdt=_C.F32, gb=ptr(), bdt=_C.F32, ws=None, n=0, stream=None)
        a.update(change)
        assert L.dimq_mx_linear_backward(*a.values()) == 1
        assert text in L.dimq_last_error().decode()

    refused("dtype must be fp32, fp16 or bf16", gdt=_C.F64)
    refused("row stride 7 is below", ldg=7)
    refused("must be positive", K=0)
    refused("must be positive", N=0, ldg=0)
    refused("null pointer", g=None)
    refused("null pointer", c=None)
    refused("null pointer", s8=None)
    refused("16-byte aligned", c=ptr(4104))
    refused("output dtype", xdt=_C.U8)
    refused("output dtype", wdt=_C.F64)
    refused("bias gradient must be", bdt=_C.U8)
    need = L.dimq_mx_linear_backward_workspace_bytes(ptr(), _C.F32, 2, 8, 8, 32, 7)
    assert need > 0
    refused("workspace is too small", ws=ptr(), n=need - 1)
    refused("256-byte aligned", ws=ptr(4100), n=need)
    # a part that is not asked for is not looked at, and nothing to do is no error
    assert L.dimq_mx_linear_backward(ptr(), _C.F32, 0, 8, 8, None, None, None, None, 32, ptr(), _C.F32, None, 0, None, 0, None, 0,
                                     None) == 0
    assert L.dimq_mx_linear_backward_workspace_bytes(ptr(), _C.F32, 0, 8, 8, 32, 1) == 0


def test_serving_module_has_no_cpu_path():
    from dimq_amd import DIMQMXFP4Linear
    mod = DIMQMXFP4Linear(torch.zeros(8, 16, dtype=torch.uint8), torch.zeros(8, 1, dtype=torch.uint8), 32)
    with pytest.raises(RuntimeError, match="runs on the GPU"):
        mod(torch.ones(2, 32))
