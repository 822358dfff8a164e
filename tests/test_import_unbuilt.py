"""The package without its compiled libraries: it imports, says so, and its operators raise; built later, it runs."""

import shutil
import subprocess
import sys
from pathlib import Path

PACKAGE = Path(__file__).resolve().parents[1] / "dimq_amd"

PROGRAM = """
import shutil, sys
import torch
import dimq_amd
from dimq_amd import mx, ops
assert not dimq_amd.is_available()
x, c, s = torch.ones(2, 32), torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8)
mod = dimq_amd.DIMQMXFP4Linear(c, s, 32)
for call in (lambda: mx.quantize_mxfp4(x), lambda: mx.mxfp4_linear(x, c, s), lambda: mx.linear(x, x), lambda: mx.gelu(x),
             lambda: mx.MXFP4TrainLinear(32, 4)(x)):
    try:
        call()
    except RuntimeError as e:
        assert "library is not available" in str(e), e
    else:
        raise AssertionError("no error")
indices = torch.tensor([[1, 2, 3, 4]], dtype=torch.uint8)
assert dimq_amd.unpack_indices(dimq_amd.pack_indices(indices, 4), 4, 4).tolist() == [1, 2, 3, 4]
# the libraries appear
for name in ("libdimq_hip.so", "_native.so"):
    shutil.copy(sys.argv[1] + "/" + name, "dimq_amd/" + name)
ops._extension_available.cache_clear()
try:
    mx.gelu(x)
except RuntimeError as e:
    assert "expects a CUDA input" in str(e), e
else:
    raise AssertionError("no error")
assert dimq_amd.is_available()
"""


def test_import_without_the_libraries(tmp_path):
    to = tmp_path / "dimq_amd"
    to.mkdir()
    for f in PACKAGE.glob("*.py"):
        shutil.copy(f, to / f.name)
    r = subprocess.run([sys.executable, "-c", PROGRAM, str(PACKAGE)], cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
