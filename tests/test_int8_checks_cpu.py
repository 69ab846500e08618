"""The 8-bit path without a GPU: operand checks that come before any C call, the work split of the
weight gradient, and the C ABI's refusals. The library is a stub that fails the test if an entry
point is reached, except where its own host code is what is tested."""
from __future__ import annotations

import itertools
import subprocess

import pytest
import torch

from c3_b200 import _lib, linear, norm, quant
from c3_b200._lib import C3CUError
from c3_b200.build import CSRC, OUT_DIR

bf16, f32, i8, i32 = torch.bfloat16, torch.float32, torch.int8, torch.int32


class _NoCalls:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached although an operand check should have refused")


@pytest.fixture
def no_library(monkeypatch):
    monkeypatch.setattr(_lib, "load", lambda *a, **k: _NoCalls())


@pytest.fixture
def any_device(monkeypatch, no_library):
    monkeypatch.setattr(linear, "_device_ok", lambda t: True)


def z(*shape, dtype=bf16):
    return torch.zeros(shape, dtype=dtype)


def refused(fn, *args, match: str = "", **kwargs):
    with pytest.raises(C3CUError) as e:
        fn(*args, **kwargs)
    assert e.value.code == -1
    assert match in str(e.value), str(e.value)


M, N, K = 24, 40, 32


def test_quantize_rows_operands(any_device):
    refused(quant.quantize_rows, [1.0], match="torch.Tensor")
    refused(quant.quantize_rows, z(M, K, dtype=torch.float16), match="bfloat16")
    refused(quant.quantize_rows, z(M), match="2-D")
    refused(quant.quantize_rows, z(M, 0), match="at least one")
    refused(quant.quantize_rows, z(K, M).t(), match="column stride")
    refused(quant.quantize_rows, z(1, K).expand(M, K), match="row stride")
    refused(quant.quantize_rows, z(M, K), q=z(M, K + 1, dtype=i8), match="expected shape")
    refused(quant.quantize_rows, z(M, K), q=z(M, K, dtype=torch.uint8), match="int8")
    refused(quant.quantize_rows, z(M, K), scale=z(M - 1, dtype=f32), match="expected shape")
    refused(quant.quantize_rows, z(M, K), scale=z(M), match="float32")


def test_rms_norm_operands(any_device):
    x, w = z(M, K), z(K, dtype=f32)
    refused(norm.rms_norm_int8, x, z(K + 1, dtype=f32), match="expected shape")
    refused(norm.rms_norm_int8, x, z(K), match="float32")
    refused(norm.rms_norm_int8, x, w, -1e-6, match="eps")
    refused(norm.rms_norm_int8, x, w, float("nan"), match="eps")
    refused(norm.rms_norm_int8, x, w, float("inf"), match="eps")
    refused(norm.rms_norm_int8, x, w, residual=z(M, K, dtype=f32), match="bfloat16")
    refused(norm.rms_norm_int8, x, w, residual=z(M + 1, K), match="expected shape")
    refused(norm.rms_norm_int8, x, w, h=z(M, K), match="without a residual")
    refused(norm.rms_norm_int8, x, w, residual=x, h=z(M, K, dtype=f32), match="bfloat16")
    refused(norm.rms_norm_int8, x, w, rstd=z(M + 1, dtype=f32), match="expected shape")
    refused(norm.rms_norm_int8, z(M, 0), z(0, dtype=f32), match="at least one")


def test_outputs_that_overlap_inputs_in_part(any_device):
    """The same rows, or other columns of the same buffer, are fine; any other overlap is refused."""
    buf = z(M + 1, 2 * K)
    x, w, r = z(M, K), z(K, dtype=f32), z(M, dtype=f32)
    stream = buf[:M, :K]
    for h in (buf[1:, :K], buf[:M, 8:8 + K], buf.view(-1)[:M * K].view(M, K)):
        refused(norm.rms_norm_int8, x, w, residual=stream, h=h, match="overlaps")
        refused(norm.rms_norm_backward, x, stream, w, r, dx=h, match="overlaps")
        refused(norm.rms_norm_backward, stream, x, w, r, dx=h, match="overlaps")
        refused(norm.rms_norm_backward, x, x, w, r, dh=stream, dx=h, match="overlaps")
    for h in (stream, buf[:M, K:]):  # passes the overlap check: only the device (CPU) stops it
        with pytest.raises((AssertionError, AttributeError, C3CUError, RuntimeError)) as e:
            norm.rms_norm_int8(x, w, residual=stream, h=h)
        assert "overlaps" not in str(e.value)


def test_rms_norm_backward_operands(any_device):
    h, w, r = z(M, K), z(K, dtype=f32), z(M, dtype=f32)
    refused(norm.rms_norm_backward, z(M, K, dtype=f32), h, w, r, match="bfloat16")
    refused(norm.rms_norm_backward, z(M, K + 1), h, w, r, match="expected shape")
    refused(norm.rms_norm_backward, h, h, w, z(M + 1, dtype=f32), match="expected shape")
    refused(norm.rms_norm_backward, h, h, z(K), r, match="float32")
    refused(norm.rms_norm_backward, h, h, w, r, dh=z(M, K, dtype=f32), match="bfloat16")
    refused(norm.rms_norm_backward, h, h, w, r, dweight=z(K), match="float32")


def test_forward_int8_operands(any_device):
    xq, xs, wq, ws = z(M, K, dtype=i8), z(M, dtype=f32), z(N, K, dtype=i8), z(N, dtype=f32)
    words = (N + 31) // 32
    refused(linear.forward_int8, z(M, K), xs, wq, ws, match="int8")
    refused(linear.forward_int8, xq, xs, z(N, K + 16, dtype=i8), ws, match="expected shape")
    refused(linear.forward_int8, xq, z(M + 1, dtype=f32), wq, ws, match="expected shape")
    refused(linear.forward_int8, xq, xs, wq, z(N), match="float32")
    refused(linear.forward_int8, xq, xs, wq, ws, z(N - 1, dtype=f32), match="expected shape")
    refused(linear.forward_int8, xq, xs, wq, ws, out_dtype=torch.float16, match="float32 or bfloat16")
    refused(linear.forward_int8, xq, xs, wq, ws, Y=z(M, N, dtype=torch.float16), match="float32 or bfloat16")
    refused(linear.forward_int8, xq, xs, wq, ws, Y=z(M, N + 8), match="expected shape")
    refused(linear.forward_int8, xq, xs, wq, ws, mask=z(M, words + 1, dtype=i32), match="expected shape")
    refused(linear.forward_int8, xq, xs, wq, ws, relu=False, mask=z(M, words, dtype=i32), match="ReLU")
    refused(linear.forward_int8, xq, xs, wq, ws, save_mask=False, mask=z(M, words, dtype=i32), match="ReLU")
    long = linear.INT8_MAX_K + 1
    refused(linear.forward_int8, z(1, long, dtype=i8), xs[:1], z(1, long, dtype=i8), ws[:1], match="outside")
    refused(linear.forward_int8, z(M, 0, dtype=i8), xs, z(N, 0, dtype=i8), ws, match="outside")


def test_grad_weight_int8_operands(any_device):
    dz, xq, xs = z(M, N), z(M, K, dtype=i8), z(M, dtype=f32)
    refused(linear.grad_weight_int8, z(M, N, dtype=f32), xq, xs, match="bfloat16")
    refused(linear.grad_weight_int8, dz, z(M + 1, K, dtype=i8), xs, match="expected shape")
    refused(linear.grad_weight_int8, dz, xq, z(M - 1, dtype=f32), match="expected shape")
    refused(linear.grad_weight_int8, dz, xq, xs, dW=z(N, K, dtype=f32), match="bfloat16")
    refused(linear.grad_weight_int8, dz, xq, xs, dW=z(K, N), match="expected shape")


def test_cpu_tensors_are_refused(no_library):
    x, w, r = z(M, K), z(K, dtype=f32), z(M, dtype=f32)
    xq, wq, ws = z(M, K, dtype=i8), z(N, K, dtype=i8), z(N, dtype=f32)
    refused(quant.quantize_rows, x, match="CUDA")
    refused(norm.rms_norm_int8, x, w, match="CUDA")
    refused(norm.rms_norm_backward, x, x, w, r, match="CUDA")
    refused(linear.forward_int8, xq, r, wq, ws, match="CUDA")
    refused(linear.grad_weight_int8, z(M, N), xq, r, match="CUDA")


def test_entry_points_without_a_device():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present; the no-device path is not reachable")
    L = _lib.load()
    assert L.c3cu_quantize_rows(None, 8, 1, None, 8, None, 1, 8, None) == -5
    assert L.c3cu_rms_norm_int8(None, 8, None, 0, 1, None, 1e-6, None, 0, None, 8, None, None, 1, 8, None) == -5
    assert L.c3cu_rms_norm_bwd(None, 8, None, 8, None, 0, 1, None, None, None, 8, None, 1, 8, None, 0, None) == -5
    assert L.c3cu_linear_int8_fwd(None, 16, None, None, 16, None, None, None, 8, 1, 0, None, 0, 1, 8, 16, None) == -5
    assert L.c3cu_gemm_dw_int8(None, 8, None, 16, None, None, 16, 1, 8, 16, None, 0, None) == -5
    # sizes beyond the limits are refused first
    big = 2 ** 31
    assert L.c3cu_linear_int8_fwd(None, 16, None, None, 16, None, None, None, 8, 1, 0, None, 0, big, 8, 16, None) == -1
    assert L.c3cu_gemm_dw_int8(None, 8, None, 16, None, None, 16, 1, 8, big, None, 0, None) == -1


def test_workspace_queries():
    L = _lib.load()
    assert L.c3cu_rms_norm_bwd_workspace(0, 64) == 0 and L.c3cu_rms_norm_bwd_workspace(1, 64) == 0
    assert L.c3cu_rms_norm_bwd_workspace(1000, 4096) % (4096 * 4) == 0
    assert L.c3cu_rms_norm_bwd_workspace(1000, 20000) >= 1000 * 4
    assert L.c3cu_gemm_dw_int8_workspace(0, 64, 64) == 0
    assert L.c3cu_gemm_dw_int8_workspace(128, 256, 784) == 0  # widened in the kernel, in one piece


_COVER = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "ckpt_schedule.h"
using namespace c3cu::ckpt;
int main() {
  long checked = 0;
  for (int clusters : {1, 2, 3, 37, 73, 74})
    for (int tiles = 1; tiles <= 3 * clusters + 2; ++tiles)
      for (int blocks : {1, 2, 3, 7, 16, 33, 64, 100, 255, 256, 1000, 4097}) {
        const Plan p = make_plan(tiles, clusters, blocks);
        const int items = item_count(p);
        if (p.rest > 0 && (p.pieces < 2 || p.whole + p.rest != tiles || p.whole % clusters != 0 || p.rest * p.pieces > clusters)) return 1;
        if (p.rest == 0 && p.whole != tiles) return 2;
        std::vector<std::vector<char>> seen(tiles, std::vector<char>(blocks, 0));
        std::vector<char> slots(p.rest * p.pieces, 0);
        for (int c = 0; c < (items < clusters ? items : clusters); ++c) {
          int mine = 0;
          for (int i = c; i < items; i += clusters, ++mine) {
            const Item it = item_at(p, i, blocks);
            if (it.tile < 0 || it.tile >= tiles || it.kb0 >= it.kb1 || it.kb1 > blocks) return 3;
            for (int k = it.kb0; k < it.kb1; ++k)
              if (seen[it.tile][k]++) return 4;
            if ((it.slot >= 0) != (it.tile >= p.whole)) return 5;
            if (it.slot >= 0 && (it.slot >= (int)slots.size() || slots[it.slot]++ || it.slot / p.pieces != it.tile - p.whole)) return 6;
          }
          if (mine == 0) return 7;
        }
        for (auto& t : seen)
          for (char k : t)
            if (k != 1) return 8;
        for (char s : slots)
          if (s != 1) return 9;
        ++checked;
      }
  std::printf("%ld\n", checked);
  return 0;
}
"""


def test_weight_gradient_work_split_covers_each_block_once(tmp_path):
    """Every K block of every tile is computed exactly once, pieces map to their own slots in order,
    and every cluster that is launched has work."""
    src = tmp_path / "cover.cpp"
    src.write_text(_COVER)
    exe = tmp_path / "cover"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, f"check {r.returncode} failed"
    assert int(r.stdout) > 5000


def _converter_layout():
    """The converter warps' addresses (gemm_ckpt.cuh), restated: {(row, 16-byte piece of 128 columns)}
    -> byte offset, for one 64 x 128 tile."""
    out = {}
    for warp, lane in itertools.product(range(4), range(32)):
        u, r0 = lane & 7, warp * 16 + (lane >> 3)
        swap = u >= 4
        piece = ((2 * u) & 7) | (1 if swap else 0)
        at = (piece ^ (lane >> 3)) << 4
        for j in range(4):
            line = (u >> 2) * 8192 + r0 * 128
            x = 64 if j & 1 else 0
            first, second = (2 * u + 1, 2 * u) if swap else (2 * u, 2 * u + 1)
            out[(r0 + 4 * j, first)] = line + (at ^ x) + j * 512
            out[(r0 + 4 * j, second)] = line + (at ^ 16 ^ x) + j * 512
    return out


def test_converter_writes_the_swizzled_tile():
    """Each 16-byte piece lands where the 128-byte swizzle puts it (piece index xor row mod 8 within
    its 64-column chunk), all distinct, and the lanes that store together use each bank once."""
    layout = _converter_layout()
    assert len(layout) == 64 * 16
    for (row, piece), off in layout.items():
        assert off == (piece // 8) * 8192 + row * 128 + ((piece % 8) ^ (row % 8)) * 16
    for warp, j in itertools.product(range(4), range(4)):
        for group in range(4):  # eight lanes of a quarter warp, one row
            row = warp * 16 + group + 4 * j
            for firsts in (True, False):
                pieces = [(2 * u + 1 if (u >= 4) == firsts else 2 * u) for u in range(8)]
                assert len({(layout[(row, p)] // 16) % 8 for p in pieces}) == 8
