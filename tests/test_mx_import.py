"""The package imports, and its containers work, with a PyTorch that was built without CUDA."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

PROGRAM = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)  # a build without CUDA has none of them
import flashloop_b200 as fl
t = fl.MXTensor.from_row_scales(torch.zeros(3, 100, dtype=torch.uint8), torch.zeros(3, 4, dtype=torch.uint8), (3, 100), "mxfp8")
assert t.view(1, 3, 100).shape == (1, 3, 100)
try:
    fl.mx_quantize(torch.zeros(2, 64))
except RuntimeError as error:
    assert "no CPU fallback" in str(error)
else:
    raise AssertionError("not refused")
"""


def test_import_without_a_cuda_build():
    done = subprocess.run([sys.executable, "-c", PROGRAM], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]
