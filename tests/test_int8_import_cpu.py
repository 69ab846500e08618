"""The package beside other builds of torch: one without CUDA, and one that the C++ binding was not or
cannot be compiled against."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from c3_b200 import _lib, build

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


def _broken(*a, **k):
    raise RuntimeError("compile failed: no headers")


def test_the_library_builds_without_the_binding(monkeypatch):
    monkeypatch.setattr(build, "build_fast_calls", _broken)
    with pytest.warns(RuntimeWarning, match="no headers"):
        assert build.build() == build.LIB
    monkeypatch.setattr(build, "build_fast_calls", lambda: (_ for _ in ()).throw(FileNotFoundError("g++")))
    with pytest.warns(RuntimeWarning, match="g[+][+]"):
        assert build.try_build_fast_calls() is None


@pytest.mark.parametrize("content", [None, b"not a library"])
def test_calls_go_through_ctypes_without_the_binding(monkeypatch, tmp_path, content):
    path = tmp_path / "_fast_calls.other.so"
    if content is not None:
        path.write_bytes(content)
    monkeypatch.setattr(build, "fast_calls_path", lambda: path)
    monkeypatch.setattr(build, "build_fast_calls", _broken)
    monkeypatch.setattr(_lib, "_fast", None)
    with pytest.warns(RuntimeWarning, match="ctypes"):
        module = _lib.fast()
    assert module.quantize_rows(torch.zeros(1, 16)) is None and module.forward_int8(1, 2, 3) is None
    assert _lib.fast() is module  # and says so once


def test_another_torch_is_another_file(monkeypatch):
    here = build.fast_calls_path()
    assert _lib.fast() is not None
    monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    assert build.fast_calls_path() != here and "9_9_9" in build.fast_calls_path().name


def test_another_header_is_another_file(monkeypatch, tmp_path):
    here = build.fast_calls_path()
    src, header = build._fast_calls_sources()
    other = tmp_path / "c3cu.h"
    other.write_text(header.read_text().replace("int64_t ldq", "int32_t ldq"))
    monkeypatch.setattr(build, "_fast_calls_sources", lambda: (src, other))
    assert build.fast_calls_path() != here
