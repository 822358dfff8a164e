"""Microscaled formats without a GPU: the float64 oracle against values worked out by hand and against differences, and
what the entry points refuse before anything is launched."""

import ctypes

import pytest
import torch

from oracle import mx as omx


def test_four_bit_levels_ties_and_saturation():
    # one block whose largest magnitude 6 gives scale 1: ties to the even code, above 6 saturates
    v = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, 0.2, 0.3, 7.9, -7.0, 0.0, 2.6]
    want = [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 0.0, -1.0, 0.0, 0.5, 6.0, -6.0, 0.0, 3.0]
    assert omx.q4(torch.tensor([v])).tolist() == [want]


def test_eight_bit_levels_and_scales():
    v = torch.tensor([[1.0, 1.9999, 0.5 / 64, 1.5 / 64, -2.5 / 64, 1 / 3]])
    assert omx.q8(v).tolist() == [[1.0, 127 / 64, 0.0, 2 / 64, -2 / 64, 21 / 64]]


@pytest.mark.parametrize("top,byte4,byte8", [(1.0, 125, 127), (1.999, 125, 127), (2.0 ** 127, 252, 254), (2.0 ** -126, 0, 1),
                                             (2.0 ** -125, 0, 2), (2.0 ** -124, 1, 3), (2.0 ** -149, 0, 0), (0.0, 0, 0),
                                             (float("inf"), 255, 255), (float("nan"), 255, 255)])
def test_scale_bytes(top, byte4, byte8):
    x = torch.zeros(1, 40)
    x[0, 33] = top
    for bits, want in ((4, byte4), (8, byte8)):
        assert omx.quantize(x, bits)[1].tolist() == [[0, want]]


def test_a_value_that_is_not_finite_takes_its_block_only():
    x = torch.ones(2, 70)
    x[1, 40] = float("-inf")
    for q in (omx.q4, omx.q8):
        bad = torch.isnan(q(x))
        assert bad[1, 32:64].all() and bad.sum() == 32


def test_slope_is_the_differences_of_gelu():
    h = torch.linspace(-9, 9, 401, dtype=torch.float64)
    d = (omx.gelu(h + 1e-5) - omx.gelu(h - 1e-5)) / 2e-5
    assert (omx.gelu_slope(h) - d).abs().max() < 1e-9


# ---- refusals ---------------------------------------------------------------------------------------------------

def test_ops_refuse_cpu_tensors():
    from dimq_amd import mx
    x, w = torch.ones(2, 32), torch.ones(4, 32)
    c, s = torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8)
    c8 = torch.zeros(2, 32, dtype=torch.int8)
    for call in (lambda: mx.quantize_mxfp4(x), lambda: mx.compress_activation(x), lambda: mx.quantize_and_compress(x),
                 lambda: mx.mxfp4_linear(x, c, s), lambda: mx.dequantize_mxfp4(c, s, 32),
                 lambda: mx.decompress_activation(c8, s[:2], 32), lambda: mx.mxfp4_linear_grad_input(x, c, s, 32),
                 lambda: mx.linear_grad_weight(x, c8, s[:2], 32)):
        with pytest.raises(NotImplementedError):
            call()
    for call in (lambda: mx.linear(x, w), lambda: mx.gelu(x)):
        with pytest.raises(RuntimeError, match="expects a CUDA input"):
            call()


def test_unknown_activation():
    from dimq_amd import mx
    with pytest.raises(ValueError, match="unknown activation"):
        mx.mxfp4_linear(torch.ones(1, 32), torch.zeros(1, 16, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.uint8),
                        activation="tanh")


def _p(a=4096):  # a non-null pointer that no refused call reads
    return ctypes.c_void_p(a)


def test_entry_points_refuse():
    from dimq_amd import _C
    L = _C.lib

    def refused(rc, text):
        assert rc == 1 and text in L.dimq_last_error().decode()

    q = L.dimq_mx_quantize
    refused(q(_p(), _C.F64, 2, 32, 32, _p(), _p(), 1, None, None, None), "dtype must be fp32, fp16 or bf16")
    refused(q(_p(), _C.F32, -1, 32, 32, _p(), _p(), 1, None, None, None), "must not be negative")
    refused(q(_p(), _C.F32, 2, 32, 31, _p(), _p(), 1, None, None, None), "row stride 31 is below")
    refused(q(None, _C.F32, 2, 32, 32, _p(), _p(), 1, None, None, None), "null pointer")
    refused(q(_p(), _C.F32, 2, 32, 32, None, None, 1, None, None, None), "no output")
    refused(q(_p(), _C.F32, 2, 32, 32, _p(4100), _p(), 1, None, None, None), "16-byte aligned")
    refused(q(_p(), _C.F32, 2, 33, 33, _p(), _p(), 1, None, None, None), "1 blocks do not hold a row of 33")
    refused(q(_p(), _C.F32, 2, 33, 33, None, None, 0, _p(), None, None), "null pointer")
    d = L.dimq_mx_dequantize
    refused(d(_p(), _p(), 3, 2, 32, _p(), _C.F32, None), "bits must be 4 or 8")
    refused(d(_p(), _p(), 4, 2, 32, _p(), _C.U8, None), "dtype must be")
    refused(d(_p(4104), _p(), 8, 2, 32, _p(), _C.F32, None), "16-byte aligned")
    f = L.dimq_mxfp4_linear
    tail = (None, None, None, 0, None)
    refused(f(_p(), _C.F32, 1, 0, 0, _p(), _p(), None, 0, 8, _p(), _C.F32, None, 0, 0, *tail), "must be positive")
    refused(f(_p(), _C.F32, 1, 32, 32, _p(), _p(), None, 0, 8, _p(), _C.F32, None, 0, 7, *tail), "unknown activation 7")
    refused(f(_p(), _C.F32, 1, 32, 32, _p(), _p(), None, 0, 8, _p(), _C.F64, None, 0, 0, *tail), "output dtype")
    refused(f(_p(), _C.F32, 1, 32, 32, _p(), _p(), _p(), _C.U8, 8, _p(), _C.F32, None, 0, 0, *tail), "bias must be")
    refused(f(_p(), _C.F32, 1, 32, 32, _p(), _p(), None, 0, 8, _p(), _C.F32, _p(), _C.U8, 0, *tail), "residual must be")
    refused(f(_p(), _C.F64, 1, 32, 32, _p(), _p(), None, 0, 8, _p(), _C.F32, None, 0, 0, *tail), "dtype must be")
    need = L.dimq_mxfp4_linear_workspace_bytes(300, 64, 8)
    assert need > 0
    refused(f(_p(), _C.F32, 300, 64, 64, _p(), _p(), None, 0, 8, _p(), _C.F32, None, 0, 0, None, None, _p(), need - 1, None),
            "workspace is too small")
    gi = L.dimq_mxfp4_linear_grad_input
    refused(gi(_p(), _C.F64, 2, 8, 8, _p(), _p(), 32, _p(), _C.F32, None, 0, None), "dtype must be")
    refused(gi(_p(), _C.F32, 2, 8, 7, _p(), _p(), 32, _p(), _C.F32, None, 0, None), "row stride 7 is below")
    refused(gi(_p(), _C.F32, 2, 8, 8, _p(), _p(), 32, None, _C.F32, None, 0, None), "null pointer")
    gw = L.dimq_mx_linear_grad_weight
    refused(gw(_p(), _C.F32, 2, 8, 8, _p(), _p(), 0, _p(), _C.F32, None, 0, None, 0, None), "must be positive")
    refused(gw(_p(), _C.F32, 2, 8, 8, _p(), _p(), 32, _p(), _C.F32, _p(), _C.U8, None, 0, None), "bias gradient must be")
    refused(gw(_p(), _C.F32, 2, 8, 8, _p(), _p(), 32, None, _C.F32, None, 0, None, 0, None), "null pointer")
    gf, gb = L.dimq_mx_gelu_forward, L.dimq_mx_gelu_backward
    refused(gf(_p(), _C.F64, 2, 8, 8, _p(), _p(), _p(), None), "dtype must be")
    refused(gf(_p(), _C.F32, 2, 8, 8, None, _p(), _p(), None), "null pointer")
    refused(gb(_p(), _C.F32, 2, 8, 8, None, _p(), _p(), None), "null pointer")
    # nothing to do is no error
    assert q(None, _C.F32, 0, 32, 32, None, None, 1, None, None, None) == 0
    assert f(None, _C.F32, 0, 32, 32, None, None, None, 0, 8, None, _C.F32, None, 0, 0, *tail) == 0


def test_gelu_refuses_half_a_kept_form():
    from dimq_amd import _C
    gf = _C.lib.dimq_mx_gelu_forward
    for codes, scales in ((_p(), None), (None, _p())):
        assert gf(_p(), _C.F32, 2, 8, 8, _p(), codes, scales, None) == 1
        assert "null pointer" in _C.lib.dimq_last_error().decode()
