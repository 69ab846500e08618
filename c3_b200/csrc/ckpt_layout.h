// Who converts what in the small-tile weight gradient (gemm_ckpt_narrow.cuh): the addresses that a
// thread of a converter group reads and writes, shared by the kernel and the host-side test.
//
// A tile holds 64 rows (the sum's index m) of 16-byte pieces of eight bf16, in chunks of 64 columns
// with the 128-byte swizzle: piece j of row r of a chunk lies at 128 r + 16 (j xor r mod 8). A group is
// 128 threads; `t` counts them.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define C3CU_HD __host__ __device__
#else
#define C3CU_HD
#endif

namespace c3cu {
namespace ckpt {

constexpr uint32_t kChunkBytes = 64 * 64 * 2;  // 64 rows of 64 bf16

C3CU_HD constexpr uint32_t piece_at(int row, int piece) {
  return static_cast<uint32_t>(row * 128 + ((piece ^ (row & 7)) << 4));
}

// X: 128 columns, from int8 rows of 128 bytes. In step i (0..3) a thread reads the 16 int8 of unit u of
// its row and writes two pieces of eight bf16. Threads of units 4..7 write their odd piece first, so that
// the eight threads of a row, which store together, touch every bank once.
struct XUnit {
  int row, unit;
  bool odd_first;
};

C3CU_HD constexpr XUnit x_unit(int t, int i) {
  return XUnit{(t >> 5) * 16 + ((t & 31) >> 3) + 4 * i, t & 7, (t & 7) >= 4};
}

C3CU_HD constexpr uint32_t x_from(const XUnit& x) { return static_cast<uint32_t>(x.row * 128 + x.unit * 16); }

// `second`: of the two pieces in the order of their stores.
C3CU_HD constexpr uint32_t x_to(const XUnit& x, bool second) {
  const int piece = 2 * (x.unit & 3) + ((second != x.odd_first) ? 1 : 0);
  return static_cast<uint32_t>(x.unit >> 2) * kChunkBytes + piece_at(x.row, piece);
}

// dZ: T columns, in place. With 64 columns or more a thread has the same piece of four rows of each chunk;
// with 32, of which a row has four pieces, one piece of two rows. Eight neighbouring threads touch every
// bank once: they have the eight pieces of a row, or the four of rows r and r + 4.
template <int T>
struct DzUnits {
  static constexpr int kChunks = (T + 63) / 64;
  static constexpr int kRows = T >= 64 ? 4 : 2;
  static C3CU_HD constexpr int row(int t, int i) {
    return T >= 64 ? (t >> 3) + 16 * i : 8 * (t >> 5) + ((t >> 3) & 3) + 4 * ((t >> 2) & 1) + 32 * i;
  }
  static C3CU_HD constexpr int piece(int t) { return T >= 64 ? t & 7 : t & 3; }

  // Where dZ lies in chunk c of its tile, and later head; and where tail goes, so that the MMA sees one tile
  // of 2 T columns, all of head's before all of tail's: in chunks behind head's, or (32 columns) in the second
  // half of the one chunk.
  static C3CU_HD constexpr uint32_t head_at(int t, int i, int c) {
    return static_cast<uint32_t>(c) * kChunkBytes + piece_at(row(t, i), piece(t));
  }
  static C3CU_HD constexpr uint32_t tail_at(int t, int i, int c) {
    return T >= 64 ? head_at(t, i, c + kChunks) : piece_at(row(t, i), piece(t) + 4);
  }
  static constexpr uint32_t kBytes = T >= 64 ? 2 * kChunks * kChunkBytes : kChunkBytes;  // head and tail
};

}  // namespace ckpt
}  // namespace c3cu
