// The weight gradient from an 8-bit checkpoint (gemm_ckpt.cuh) in small tiles: 128 columns x T rows of
// dW on one CTA, for the many layers whose dW has too few 256 x 256 tiles to occupy the GPU. The sum's
// K blocks of a tile are split over a cluster, whose CTAs add their fp32 partial sums through distributed
// shared memory, in the order of their ranks: one launch, no workspace, the same bits every time.
//
// A stage of the ring holds a K block's raw int8 (8 KB), the widened tile made of it (16 KB) and dZ. The
// stage is free again when its MMAs are done, so a converter waits for nothing but the loads. What bounds
// a long sum is the converters' arithmetic, 0.35 us a K block: rings of their own for loads and tiles
// (0.40) and twice the converters (0.34) did not shorten it.
// Warps: 0 TMA, 1 MMA, 2..9 converters in two groups of four that take the K blocks in turn, and the
// epilogue after them.
#pragma once

#include "gemm_ckpt.cuh"
#include "igemm.cuh"

namespace c3cu {
namespace ckpt_narrow {

using ckpt::BK;
using ckpt::kConvGroups;
using ckpt::kConvWarps;
using ckpt::MN_CHUNK_BYTES;
using ckpt::RAW_BYTES;
using ckpt::UMMA_K;
constexpr int COLS = ckpt::HN;  // columns of dW per CTA: the MMA's 128 rows
constexpr int kThreads = 32 * (2 + kConvGroups * kConvWarps);
constexpr int kMaxCluster = 8;
constexpr uint32_t WIDE_BYTES = 2 * MN_CHUNK_BYTES;
__host__ __device__ constexpr int chunks(int T) { return (T + 63) / 64; }  // of 64 columns of dZ

template <int T>
struct Ring {
  static constexpr int kStages = T <= 64 ? 6 : 4;
  static constexpr uint32_t kStage = WIDE_BYTES + chunks(T) * MN_CHUNK_BYTES + RAW_BYTES;
  static constexpr uint32_t kSmem = kStages * kStage + (3 * kStages + 1) * 8 + 8 + 1024;
  static_assert(kStages % kConvGroups == 0, "a stage belongs to one group, which so sees each of its phases");
  static_assert(kSmem <= 227 * 1024 && kStages * kStage >= T * COLS * 4, "shared memory");
};

struct Params {
  int32_t M, N, K;  // dW is N x K, the sum runs over M
  __nv_bfloat16* out;
  int64_t ldo;
  const float* scale;  // [M]
  int32_t kb_per_cta;  // K blocks per CTA of a cluster
  int32_t k_tiles;     // tiles of 128 columns
};

template <int T>
__global__ void __launch_bounds__(kThreads)
    dw_narrow_kernel(const __grid_constant__ CUtensorMap tmz, const __grid_constant__ CUtensorMap tmx, const Params p) {
  constexpr int STAGES = Ring<T>::kStages;
  constexpr uint32_t STAGE = Ring<T>::kStage;
  constexpr uint32_t Z_AT = WIDE_BYTES, RAW_AT = Z_AT + chunks(T) * MN_CHUNK_BYTES;
  constexpr uint32_t TMEM = T < 32 ? 32 : T;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE);  // dZ and the int8 block landed
  uint64_t* wide = full + STAGES;                                       // widened
  uint64_t* empty = wide + STAGES;                                      // read by the MMAs
  uint64_t* acc_full = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);

  const uint32_t warp = warp_id_sync();
  const uint32_t lane = lane_id();
  const uint32_t rank = cluster_ctarank();
  uint32_t size;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const int tile = static_cast<int>(blockIdx.x / size);
  const int k0 = (tile % p.k_tiles) * COLS;
  const int n0 = (tile / p.k_tiles) * T;
  const int blocks = (p.M + BK - 1) / BK;
  const int kb0 = min(static_cast<int>(rank) * p.kb_per_cta, blocks);
  const int kb1 = min(kb0 + p.kb_per_cta, blocks);

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&wide[s], kConvWarps);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    fence_mbarrier_init();
    tma_prefetch_desc(&tmz);
    tma_prefetch_desc(&tmx);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, armed = 0u, armed_par = 0u;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[s], ph ^ 1u, kFaultWaitEmpty)) { ok = false; break; }
        uint8_t* at = smem + s * STAGE;
        mbar_arrive_expect_tx(&full[s], chunks(T) * MN_CHUNK_BYTES + RAW_BYTES);
        tma_load_2d(at + RAW_AT, &tmx, &full[s], k0, kb * BK);
#pragma unroll
        for (int c = 0; c < chunks(T); ++c)
          tma_load_2d(at + Z_AT + c * MN_CHUNK_BYTES, &tmz, &full[s], n0 + 64 * c, kb * BK);
        armed |= 1u << s;
        armed_par = (armed_par & ~(1u << s)) | (ph << s);
        if (++s == STAGES) { s = 0; ph ^= 1u; }
      }
      if (!ok || fault_raised())
        for (int t = 0; t < STAGES; ++t)
          if (armed & (1u << t)) gemm::drain_wait(&full[t], (armed_par >> t) & 1u);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t IDESC = make_idesc_bf16_f32(COLS, T, true, true);
      int s = 0;
      uint32_t ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        // dZ landed before the tile was widened, but that was seen by the converters, not by this thread
        if (!mbar_wait(&full[s], ph, kFaultWaitFull) || !mbar_wait(&wide[s], ph, kFaultWaitFull)) break;
        tc_fence_after();
        const uint32_t x = smem_u32(smem + s * STAGE);
        const uint32_t z = x + Z_AT;
#pragma unroll
        for (int kk = 0; kk < BK / UMMA_K; ++kk)
          umma_f16_ss(tmem, make_sw128_desc(x + kk * UMMA_K * 128, MN_CHUNK_BYTES, 1024),
                      make_sw128_desc(z + kk * UMMA_K * 128, MN_CHUNK_BYTES, 1024), IDESC,
                      (kb != kb0 || kk != 0) ? 1u : 0u);
        umma_commit(&empty[s]);
        if (++s == STAGES) { s = 0; ph ^= 1u; }
      }
      umma_commit(acc_full);  // also on a fault: completes when the MMAs issued so far have
      gemm::drain_wait(acc_full, 0u);
    }
    __syncwarp();
  } else {
    const int group = static_cast<int>(warp - 2u) / kConvWarps;
    const ckpt::Widener widen(static_cast<int>(warp - 2u) % kConvWarps, static_cast<int>(lane));
    float next[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = (kb0 + group) * BK + widen.r0 + 4 * j;
      next[j] = m < p.M ? __ldg(p.scale + m) : 0.f;
    }
    int s = group;
    uint32_t ph = 0;
    for (int kb = kb0 + group; kb < kb1; kb += kConvGroups) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full[s], ph, kFaultWaitFull))) break;
      const uint32_t at = smem_u32(smem + s * STAGE);
      uint4 w[4], o[8];
      widen.load(at + RAW_AT, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        widen.convert(w[j], next[j], &o[2 * j]);
        const int m = (kb + kConvGroups) * BK + widen.r0 + 4 * j;
        next[j] = m < p.M ? __ldg(p.scale + m) : 0.f;
      }
      widen.store(at, o);
      fence_proxy_async_shared();  // the MMA reads the tile through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(&wide[s]);
      s += kConvGroups;
      if (s >= STAGES) { s -= STAGES; ph ^= 1u; }
    }
  }

  // ------------------------------------------------------------ epilogue: one column per lane
  const uint32_t q = warp & 3u;               // the lane quarter of a warp
  const int half = warp >= 6 ? 1 : 0;         // the two warps of a quarter share the rows of dW
  const uint32_t in_quarter = (lane + 1u) & 2u ? lane ^ 3u : lane;  // scale8 swapped the middle two of four
  const int k = k0 + static_cast<int>(q * 32 + in_quarter);
  const uint32_t t_row = tmem + ((q * 32u) << 16);
  const int rows = min(T, p.N - n0);
  bool ok = true;
  if (warp >= 2) {
    ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0u, kFaultWaitAccFull));
    tc_fence_after();
  }
  __nv_bfloat16* const out = p.out + static_cast<int64_t>(n0) * p.ldo + k;
  if (size == 1u) {
    if (warp >= 2 && ok) {
#pragma unroll 1
      for (int c = 16 * half; c < rows; c += 32) {
        uint32_t r[16];
        __syncwarp();  // lanes past the last column skip the stores
        tmem_ld_32x32b_x16(t_row + c, r);
        tmem_wait_ld();
        if (k < p.K) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c + j < rows) out[(c + j) * p.ldo] = __float2bfloat16_rn(__uint_as_float(r[j]));
        }
      }
      __syncwarp();
    }
  } else {
    // The ring is free (every MMA has read its stage): it takes this CTA's partial sums [row][column],
    // and each CTA adds up and stores its share of the rows.
    float* part = reinterpret_cast<float*>(smem);
    const bool any = kb0 < kb1;  // the last CTAs may have no K block: their sums are zero
    if (warp >= 2) {
#pragma unroll 1
      for (int c = 16 * half; c < rows; c += 32) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(t_row + c, r);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * COLS + q * 32u + lane] = any ? __uint_as_float(r[j]) : 0.f;
      }
    }
    cluster_sync_all();
    if (warp >= 2 && ok && k < p.K) {
      const uint32_t mine = smem_u32(part) + (q * 32u + lane) * 4u;
      const int share = T / static_cast<int>(size);
      const int first = static_cast<int>(rank) * share;
      const int last = min(first + share, rows);
      constexpr int J = T / kMaxCluster < 8 ? T / kMaxCluster : 8;  // divides every share
#pragma unroll 1
      for (int t = first + J * half; t < last; t += 2 * J) {
        float sum[J];
#pragma unroll
        for (int j = 0; j < J; ++j) sum[j] = 0.f;
#pragma unroll 2
        for (uint32_t r = 0; r < size; ++r) {
          const uint32_t from = mapa_shared(mine + t * (COLS * 4), r);
#pragma unroll
          for (int j = 0; j < J; ++j) sum[j] += __uint_as_float(igemm::ld_shared_cluster(from + j * (COLS * 4)));
        }
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (t + j < last) out[(t + j) * p.ldo] = __float2bfloat16_rn(sum[j]);
      }
    }
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while another reads its sums
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM);
  }
}

}  // namespace ckpt_narrow
}  // namespace c3cu
