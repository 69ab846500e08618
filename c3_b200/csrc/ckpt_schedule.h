// Work split of the weight-gradient GEMM over an 8-bit checkpoint (gemm_ckpt.cuh), shared by the
// launcher, the kernel, the kernel that adds the pieces up, and the host-side tests.
//
// `whole` output tiles, a multiple of the cluster count, run from the first K block to the last.
// The tiles left over, too few to occupy every cluster, are cut along K into `pieces` ranges of
// `kb_per_piece` blocks: each piece writes fp32 partial sums to the workspace, and a second kernel
// adds a tile's pieces in order and rounds once. No cluster waits for another.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define C3CU_HD __host__ __device__
#else
#define C3CU_HD
#endif

namespace c3cu {
namespace ckpt {

struct Plan {
  int whole;         // tiles computed in one piece (the first ones)
  int rest;          // tiles cut into pieces
  int pieces;        // >= 2 when rest > 0
  int kb_per_piece;  // K blocks in each piece but perhaps the last
};

struct Item {
  int tile;
  int kb0, kb1;
  int slot;  // partial-sum slot (rest tile * pieces + piece), or -1
};

C3CU_HD inline int item_count(const Plan& p) { return p.whole + p.rest * p.pieces; }

C3CU_HD inline Item item_at(const Plan& p, int index, int k_blocks) {
  Item it;
  if (index < p.whole) {
    it.tile = index;
    it.kb0 = 0;
    it.kb1 = k_blocks;
    it.slot = -1;
    return it;
  }
  const int j = index - p.whole;
  it.tile = p.whole + j / p.pieces;
  it.kb0 = (j % p.pieces) * p.kb_per_piece;
  it.kb1 = it.kb0 + p.kb_per_piece < k_blocks ? it.kb0 + p.kb_per_piece : k_blocks;
  it.slot = j;
  return it;
}

// A K block of a tile takes about 0.27 us; a split costs the second launch (about 2.5 us) and its
// partial sums' way through L2 (256 KiB a piece, about 0.07 us each way over the whole GPU).
inline Plan make_plan(int tiles, int clusters, int k_blocks) {
  Plan p{tiles, 0, 1, k_blocks};
  if (clusters < 1 || tiles < 1 || k_blocks < 1) return p;
  const int rest = tiles % clusters;
  if (rest == 0) return p;
  double best = 0.27 * k_blocks;
  int best_per = k_blocks;
  for (int n = 2; n * rest <= clusters && n <= k_blocks; ++n) {
    const int per = (k_blocks + n - 1) / n;
    const int pieces = (k_blocks + per - 1) / per;
    const double t = 0.27 * per + 2.5 + 0.14 * rest * pieces;
    if (t < best) {
      best = t;
      best_per = per;
    }
  }
  const int pieces = (k_blocks + best_per - 1) / best_per;
  if (pieces < 2) return p;
  p.whole = tiles - rest;
  p.rest = rest;
  p.pieces = pieces;
  p.kb_per_piece = best_per;
  return p;
}

}  // namespace ckpt
}  // namespace c3cu
