"""The package beside other builds of torch: one without CUDA, and one that the C++ binding was not or
cannot be compiled against."""
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

_NO_CUDA = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
import c3_b200
from c3_b200 import linear, norm, quant
try:
    quant.quantize_rows(torch.zeros(2, 16))
except c3_b200.C3CUError as e:
    assert "CUDA" in str(e)
    print("imported")
"""


def test_a_torch_without_cuda():
    r = subprocess.run([sys.executable, "-c", _NO_CUDA], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert "imported" in r.stdout, r.stderr[-2000:]
