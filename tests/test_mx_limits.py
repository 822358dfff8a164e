"""Sizes beyond the microscaled layers' 32-bit steps are refused before anything is launched."""

import ctypes

import pytest


@pytest.mark.parametrize("M,N", [((1 << 28) - 255, 64), ((1 << 28) - 1, 64), (1 << 28, 64), (300, (1 << 28) - 255),
                                 (300, (1 << 28) - 1)])
def test_scale_steps_of_two_gigabytes(M, N):
    """A stage's scales are 8 bytes a row, rows padded to whole tiles: 2^31 bytes from 2^28 - 255 rows on."""
    from dimq_amd import _C
    L, K, p = _C.lib, 520, ctypes.c_void_p(4096)  # a non-null pointer that no refused call reads
    room = L.dimq_mxfp4_linear_workspace_bytes(M, K, N)
    for rc in (L.dimq_mxfp4_linear(p, _C.F32, M, K, K, p, p, None, 0, N, p, _C.F32, None, 0, 0, None, None, p, room, None),
               L.dimq_mx_linear_forward(p, _C.F32, M, K, K, p, _C.F32, K, None, 0, N, p, _C.F32, p, p, None, None, p, room,
                                        None)):
        assert rc == 1 and "too large" in L.dimq_last_error().decode()
