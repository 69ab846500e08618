"""The converters' addresses of the small-tile weight gradient (csrc/ckpt_layout.h), compiled for the
host: every piece of both operands is converted once, lands where the 128-byte swizzle puts it, and
threads that go together touch every bank once."""
import subprocess

import pytest
import torch

from c3_b200.build import CSRC

_LAYOUT = r"""
#include <cstdio>
#include <cstring>
#include "ckpt_layout.h"
using namespace c3cu::ckpt;

// byte offset of 16-byte piece p (of a chunk's eight) of row r under the 128-byte swizzle: address bits
// 4..6 are xored with bits 7..9
static unsigned swizzled(unsigned r, unsigned p) {
  unsigned a = r * 128 + p * 16;
  return a ^ ((a >> 3) & 0x70);
}

static bool banks_once(const unsigned* at) {  // eight 16-byte accesses
  unsigned seen = 0;
  for (int i = 0; i < 8; ++i) seen |= 1u << (at[i] / 16 % 8);
  return seen == 0xff;
}

static int x_tile() {
  static char written[16384 / 16], read[8192 / 16];
  for (int i = 0; i < 4; ++i)
    for (int t = 0; t < 128; ++t) {
      const XUnit x = x_unit(t, i);
      if (x_from(x) % 16 || x_from(x) >= 8192 || read[x_from(x) / 16]++) return 1;
      const unsigned row = x_from(x) / 128, unit = x_from(x) % 128 / 16;  // columns 16 unit .. 16 unit + 15
      for (int second = 0; second < 2; ++second) {
        const bool odd = x.odd_first != (second != 0);  // which half of the unit the kernel stores there
        const unsigned piece = 2 * unit + (odd ? 1 : 0);
        const unsigned want = piece / 8 * kChunkBytes + swizzled(row, piece % 8);
        if (x_to(x, second != 0) != want || written[want / 16]++) return 2;
      }
    }
  for (int i = 0; i < 4; ++i)
    for (int t = 0; t < 128; t += 8)
      for (int second = 0; second < 2; ++second) {
        unsigned from[8], to[8];
        for (int j = 0; j < 8; ++j) {
          from[j] = x_from(x_unit(t + j, i));
          to[j] = x_to(x_unit(t + j, i), second != 0);
        }
        if (!banks_once(from) || !banks_once(to)) return 3;
      }
  for (char c : read)
    if (c != 1) return 4;
  for (char c : written)
    if (c != 1) return 5;
  return 0;
}

template <int T>
static int dz_tile() {
  using U = DzUnits<T>;
  static char seen[U::kChunks][8192 / 16];
  std::memset(seen, 0, sizeof seen);
  static char both[U::kBytes / 16];  // head and tail, as the MMA reads them: column n, then T + n
  std::memset(both, 0, sizeof both);
  for (int c = 0; c < U::kChunks; ++c)
    for (int i = 0; i < U::kRows; ++i) {
      for (int t = 0; t < 128; ++t) {
        const int row = U::row(t, i), piece = U::piece(t);
        if (row < 0 || row >= 64 || piece < 0 || piece >= 8 || 64 * c + 8 * piece >= T) return 1;
        if (piece_at(row, piece) != swizzled(row, piece)) return 2;
        if (seen[c][piece_at(row, piece) / 16]++) return 3;
        for (int tail = 0; tail < 2; ++tail) {
          const int col = tail * T + 64 * c + 8 * piece;
          const unsigned want = col / 64 * kChunkBytes + swizzled(row, col % 64 / 8);
          if ((tail ? U::tail_at(t, i, c) : U::head_at(t, i, c)) != want || both[want / 16]++) return 6;
        }
      }
      for (int t = 0; t < 128; t += 8) {
        unsigned at[8], behind[8];
        for (int j = 0; j < 8; ++j) {
          at[j] = U::head_at(t + j, i, c);
          behind[j] = U::tail_at(t + j, i, c);
        }
        if (!banks_once(at) || !banks_once(behind)) return 4;
      }
    }
  for (char b : both)
    if (b != 1) return 7;
  for (int row = 0; row < 64; ++row)
    for (int col = 0; col < T; col += 8)
      if (seen[col / 64][swizzled(row, col % 64 / 8) / 16] != 1) return 5;
  return 0;
}

int main() {
  if (const int e = x_tile()) return 10 + e;
  if (const int e = dz_tile<32>()) return 20 + e;
  if (const int e = dz_tile<64>()) return 30 + e;
  if (const int e = dz_tile<128>()) return 40 + e;
  return 0;
}
"""


@pytest.fixture(scope="module")
def compiled(tmp_path_factory):
    d = tmp_path_factory.mktemp("layout")
    (d / "layout.cpp").write_text(_LAYOUT)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{CSRC}", str(d / "layout.cpp"), "-o", str(d / "layout")],
                   check=True)
    return d / "layout"


def test_each_piece_is_converted_once_and_lands_in_its_place(compiled):
    r = subprocess.run([str(compiled)])
    assert r.returncode == 0, f"check {r.returncode} failed"


def test_two_bf16_terms_hold_the_product():
    """head and tail of dZ * scale as gemm_ckpt_narrow.cuh makes them (split_scale, split_pair), in fp64 with
    each rounding to bf16: within 2^-14 of the product, worst and over random scales, and their first
    multiply-add is exact."""
    g = torch.Generator().manual_seed(1)

    def bf16(v):
        return v.to(torch.float32).to(torch.bfloat16).double()  # exact in fp32 or far from a tie of both
    z = bf16(torch.randn(400000, generator=g).double())
    s = (torch.rand(400000, generator=g) * torch.exp(4 * torch.randn(400000, generator=g))).double() * 64
    s = s.float().double()
    s_head = bf16(s)
    s_tail = bf16(s - s_head)
    assert float(((s - s_head - s_tail).abs() / s).max()) <= 2.0 ** -16
    head = bf16(z * s_head)
    left = z * s_head - head
    assert torch.equal(bf16(left), left)
    tail = bf16(z * s_tail + left)
    p = z * s
    ok = p.abs() > 1e-30
    assert float(((head + tail - p).abs()[ok] / p.abs()[ok]).max()) <= 2.0 ** -14


def test_workspace_of_a_dw_too_large():
    """More tiles than an int counts: refused, where the count used to wrap around."""
    from c3_b200 import _lib
    lib = _lib.load()
    huge = 2 ** 31 - 1000
    assert lib.c3cu_gemm_dw_int8_workspace(64, huge, huge) == 0 and "too large" in _lib.last_error()
    assert lib.c3cu_gemm_dw_int8_workspace(16384, 4096, 4096) >= 2 * 16384 * (4096 + 4096)
