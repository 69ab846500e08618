// Weight gradient from an 8-bit checkpoint of the layer's input:
//
//   dW[N][K] = sum_m dZ[m][n] * (q[m][k] * scale[m])        (bf16 out, fp32 sums in TMEM)
//
// dZ is bf16, X is held as int8 rows with one fp32 scale each (c3cu_quantize_rows). The scale runs
// along the sum, so it cannot wait for the epilogue: q * scale is formed in the kernel and rounded
// to bf16, the tensor cores' operand type. That rounding (relative 2^-8 at most, the size of the
// output's own) is the only one besides the output's; q itself would be exact in bf16.
//
// The structure is gemm2_kernel's (256 x 256 tiles on CTA pairs, both operands MN-major, since dZ
// and X are stored with the sum's index as their rows) with one more role: TMA brings X's int8
// block into a raw buffer, and four converter warps widen it into the swizzled bf16 tile that the
// MMA reads. So X crosses HBM and L2 at one byte per element and no bf16 copy of it exists.
//
// Warps: 0 TMA, 1 MMA (leader), 2..9 epilogue, 10..13 converters.
#pragma once

#include "ckpt_schedule.h"
#include "gemm2_tcgen05.cuh"

namespace c3cu {
namespace ckpt {

using gemm2::A_STAGE_BYTES;
using gemm2::B_STAGE_BYTES;
using gemm2::BK;
using gemm2::HM;
using gemm2::HN;
using gemm2::kEpiWarps;
using gemm2::kPairMask;
using gemm2::MN_CHUNK_BYTES;
using gemm2::TM;
using gemm2::TMEM_COLS;
using gemm2::TN;
using gemm2::UMMA_K;
constexpr int STAGES = 5;
constexpr int kConvWarps = 4;
constexpr int kThreads = 64 + 32 * (kEpiWarps + kConvWarps);
constexpr uint32_t RAW_BYTES = BK * HN;  // 64 rows (m) of 128 int8 (k)
constexpr uint32_t STAGE_BYTES = A_STAGE_BYTES + B_STAGE_BYTES + RAW_BYTES;
constexpr uint32_t BAR_BYTES = (3 * STAGES + 5) * 8 + 8;
constexpr uint32_t SMEM_BYTES = STAGES * STAGE_BYTES + BAR_BYTES + 1024;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");

struct Params {
  int32_t M, N, K;     // dW is N x K, the sum runs over M
  __nv_bfloat16* out;
  int64_t ldo;
  const float* scale;  // [M]
  float* partial;      // slots of [256][256] fp32
  int32_t vec_ok;
  Plan plan;
};

// Four int8 in a word -> fp32: the bytes, biased to unsigned, become the low mantissa bits of 2^23.
__device__ __forceinline__ void widen4(uint32_t w, float (&f)[4]) {
  w ^= 0x80808080u;
  constexpr float kBias = 8388608.f + 128.f;
  f[0] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)) - kBias;
  f[1] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441)) - kBias;
  f[2] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)) - kBias;
  f[3] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443)) - kBias;
}

// Eight int8 (two words) times s, as one 16-byte piece of bf16.
__device__ __forceinline__ uint4 scale8(uint32_t w0, uint32_t w1, float s) {
  float a[4], b[4];
  widen4(w0, a);
  widen4(w1, b);
  return make_uint4(pack_bf16x2(a[0] * s, a[1] * s), pack_bf16x2(a[2] * s, a[3] * s),
                    pack_bf16x2(b[0] * s, b[1] * s), pack_bf16x2(b[2] * s, b[3] * s));
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    dw_kernel(const __grid_constant__ CUtensorMap tma, const __grid_constant__ CUtensorMap tmx, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * A_STAGE_BYTES;
  uint8_t* sRaw = sB + STAGES * B_STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  uint64_t* full = bars;                   // A landed and B converted, in both CTAs (leader's is used)
  uint64_t* empty = full + STAGES;
  uint64_t* raw_full = empty + STAGES;     // this CTA's raw block landed
  uint64_t* acc_full = raw_full + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const uint32_t warp = warp_id_sync();
  const uint32_t lane = lane_id();
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0u;
  const int cluster = static_cast<int>(blockIdx.x >> 1);
  const int num_clusters = static_cast<int>(gridDim.x >> 1);
  const int k_tiles = (p.K + TN - 1) / TN;
  const int blocks = (p.M + BK - 1) / BK;
  const int items = item_count(p.plan);

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1 + 2 * kConvWarps);
      mbar_init(&empty[s], 1);
      mbar_init(&raw_full[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kEpiWarps);
    }
    mbar_init(drain, 1);
    fence_mbarrier_init();
    tma_prefetch_desc(&tma);
    tma_prefetch_desc(&tmx);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, armed = 0u, armed_par = 0u;
      bool ok = true;
      for (int i = cluster; ok && i < items; i += num_clusters) {
        const Item it = item_at(p.plan, i, blocks);
        const int n0 = (it.tile / k_tiles) * TM + static_cast<int>(rank) * HM;
        const int k0 = (it.tile % k_tiles) * TN + static_cast<int>(rank) * HN;
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait(&empty[s], ph ^ 1u, kFaultWaitEmpty)) { ok = false; break; }
          mbar_arrive_expect_tx(&raw_full[s], RAW_BYTES);
          tma_load_2d(sRaw + s * RAW_BYTES, &tmx, &raw_full[s], k0, kb * BK);
          if (leader) mbar_arrive_expect_tx(&full[s], 2u * A_STAGE_BYTES);
          const uint32_t bar_leader = mapa_shared(smem_u32(&full[s]), 0u);
          uint8_t* sa = sA + s * A_STAGE_BYTES;
#pragma unroll
          for (int j = 0; j < HM / 64; ++j)
            tma_load_2d_pair(sa + j * MN_CHUNK_BYTES, &tma, bar_leader, n0 + 64 * j, kb * BK);
          armed |= 1u << s;
          armed_par = (armed_par & ~(1u << s)) | (ph << s);
          if (++s == STAGES) { s = 0; ph ^= 1u; }
        }
      }
      if (!ok) {
        for (int t = 0; t < STAGES; ++t)
          if (armed & (1u << t)) gemm::drain_wait(&raw_full[t], (armed_par >> t) & 1u);
        gemm2::settle_inflight_copies();
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (leader && lane == 0) {
      constexpr uint32_t IDESC = make_idesc_bf16_f32(TM, TN, true, true);
      int s = 0;
      uint32_t ph = 0, acc = 0, acc_ph = 0;
      bool ok = true;
      for (int i = cluster; ok && i < items; i += num_clusters) {
        const Item it = item_at(p.plan, i, blocks);
        if (!mbar_wait(&acc_empty[acc], acc_ph ^ 1u, kFaultWaitAccEmpty)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * TN;
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait(&full[s], ph, kFaultWaitFull)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(sA + s * A_STAGE_BYTES);
          const uint32_t b_addr = smem_u32(sB + s * B_STAGE_BYTES);
#pragma unroll
          for (int kk = 0; kk < BK / UMMA_K; ++kk)
            umma_f16_ss_pair(d_tmem, make_sw128_desc(a_addr + kk * UMMA_K * 128, MN_CHUNK_BYTES, 1024),
                             make_sw128_desc(b_addr + kk * UMMA_K * 128, MN_CHUNK_BYTES, 1024), IDESC,
                             (kb != it.kb0 || kk != 0) ? 1u : 0u);
          umma_commit_pair_mc(&empty[s], kPairMask);
          if (++s == STAGES) { s = 0; ph ^= 1u; }
        }
        if (!ok) break;
        umma_commit_pair_mc(&acc_full[acc], kPairMask);
        acc ^= 1u;
        if (acc == 0u) acc_ph ^= 1u;
      }
      umma_commit_pair_mc(drain, 0x1);
      gemm::drain_wait(drain, 0u);
    }
    __syncwarp();
  } else if (warp < 2 + kEpiWarps) {
    // ------------------------------------------------------------ epilogue (warps 2..9)
    const uint32_t q = warp & 3u;
    const int c_lo = static_cast<int>((warp - 2u) >> 2) * (TN / 64);
    gemm::Params g{};
    g.M = p.N;
    g.N = p.K;
    g.out = p.out;
    g.ldo = p.ldo;
    g.vec_ok = p.vec_ok;
    uint32_t acc = 0, acc_ph = 0;
    for (int i = cluster; i < items; i += num_clusters) {
      const Item it = item_at(p.plan, i, blocks);
      const int in_tile = static_cast<int>(rank) * HM + static_cast<int>(q * 32 + lane);
      const int row = (it.tile / k_tiles) * TM + in_tile;
      const int k0 = (it.tile % k_tiles) * TN;
      if (!mbar_wait(&acc_full[acc], acc_ph, kFaultWaitAccFull)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((q * 32u) << 16) + acc * TN;
#pragma unroll 1
      for (int c = c_lo; c < c_lo + TN / 64; ++c) {
        const int col0 = k0 + c * 32;
        if (col0 >= p.K) break;
        uint32_t r[32];
        tmem_ld_32x32b_x32(t_row + c * 32, r);
        tmem_wait_ld();
        if (it.slot < 0) {
          gemm::epilogue_chunk<kEpiStoreBf16>(g, r, row, col0);
        } else if (row < p.N) {
          // slot[column][row]: a warp stores 128 contiguous bytes per column
          float* part = p.partial + static_cast<size_t>(it.slot) * (TM * TN) + in_tile;
          const int cols = min(32, p.K - col0);
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j < cols) __stcg(part + (c * 32 + j) * TM, __uint_as_float(r[j]));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[acc]), 0u));
      acc ^= 1u;
      if (acc == 0u) acc_ph ^= 1u;
    }
  } else {
    // ------------------------------------------------------------ converters (warps 10..13)
    // A warp takes 16 of the block's 64 rows, four at a time: lane = 8 * row + u reads the 16
    // int8 of unit u of its row and writes two 16-byte pieces of the swizzled bf16 tile: chunk
    // u / 4 (64 columns), pieces 2u and 2u + 1 of 8, at position piece ^ (row mod 8). Units 4..7
    // write their odd piece first, so that the eight lanes of a row touch all banks once.
    const int cw = static_cast<int>(warp) - 2 - kEpiWarps;
    const int u = static_cast<int>(lane & 7u);
    const int r0 = cw * 16 + static_cast<int>(lane >> 3);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int i = cluster; ok && i < items; i += num_clusters) {
      const Item it = item_at(p.plan, i, blocks);
      float next[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = it.kb0 * BK + r0 + 4 * j;
        next[j] = m < p.M ? __ldg(p.scale + m) : 0.f;
      }
      for (int kb = it.kb0; kb < it.kb1; ++kb) {
        float sc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sc[j] = next[j];
          const int m = (kb + 1) * BK + r0 + 4 * j;
          next[j] = kb + 1 < it.kb1 && m < p.M ? __ldg(p.scale + m) : 0.f;
        }
        if (!mbar_wait(&raw_full[s], ph, kFaultWaitFull)) { ok = false; break; }
        const uint8_t* raw = sRaw + s * RAW_BYTES;
        uint8_t* dst = sB + s * B_STAGE_BYTES + (u >> 2) * MN_CHUNK_BYTES;
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint4*>(raw + (r0 + 4 * j) * HN + u * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = r0 + 4 * j;
          const uint4 even = scale8(w[j].x, w[j].y, sc[j]);
          const uint4 odd = scale8(w[j].z, w[j].w, sc[j]);
          uint8_t* line = dst + r * 128;
          const int pe = ((2 * u) & 7) ^ (r & 7), po = ((2 * u + 1) & 7) ^ (r & 7);
          const bool swap = u >= 4;
          *reinterpret_cast<uint4*>(line + (swap ? po : pe) * 16) = swap ? odd : even;
          *reinterpret_cast<uint4*>(line + (swap ? pe : po) * 16) = swap ? even : odd;
        }
        fence_proxy_async_shared();  // the MMA reads the tile through the async proxy
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&full[s]), 0u));
        if (++s == STAGES) { s = 0; ph ^= 1u; }
      }
    }
  }

  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// Adds the pieces of the cut tiles in order, rounds once. A block takes 32 rows x 32 columns of a
// tile: partial sums are read along rows ([column][row]) and leave along columns.
__global__ void __launch_bounds__(256) add_pieces_kernel(const Params p) {
  __shared__ float t[32][33];
  const int tile = p.plan.whole + static_cast<int>(blockIdx.y);
  const int k_tiles = (p.K + TN - 1) / TN;
  const int br = static_cast<int>(blockIdx.x) / (TN / 32) * 32, bc = static_cast<int>(blockIdx.x) % (TN / 32) * 32;
  const int row0 = (tile / k_tiles) * TM + br, col0 = (tile % k_tiles) * TN + bc;
  if (row0 >= p.N || col0 >= p.K) return;
  const float* part = p.partial + static_cast<size_t>(blockIdx.y) * p.plan.pieces * (TM * TN);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = warp * 4 + i;
    float sum = 0.f;
    if (row0 + lane < p.N && col0 + c < p.K) {
#pragma unroll 4
      for (int s = 0; s < p.plan.pieces; ++s)
        sum += __ldcg(part + static_cast<size_t>(s) * (TM * TN) + (bc + c) * TM + br + lane);
    }
    t[c][lane] = sum;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = warp * 4 + i;
    if (row0 + r < p.N && col0 + lane < p.K)
      p.out[static_cast<int64_t>(row0 + r) * p.ldo + col0 + lane] = __float2bfloat16_rn(t[lane][r]);
  }
}

}  // namespace ckpt
}  // namespace c3cu
