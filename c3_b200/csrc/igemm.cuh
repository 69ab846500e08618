// Int8 matrix product on the 5th-generation tensor cores (tcgen05.mma kind::i8, int32 sums in
// TMEM) with a scale per row of X (token) and per row of W (channel):
//
//   z[m][n] = fl(fl(float(sum_k X[m][k] W[n][k]) * fl(xs[m] ws[n])) + b[n]),   Y = z or max(z, 0)
//
// The sum is exact (K <= 131071 keeps it inside int32), and the fp32 operations after it are
// separate round-to-nearest operations in this order, so Y and the mask do not depend on the
// kernel or tile that computed them. X and W are row-major [rows][K] (K-major operands): a
// 128-deep K block of a row is one 128-byte swizzled line.
//
// Two kernels (igemv.cuh has a third, for a token or a few). In both the channels are the MMA's rows and
// the tokens its columns, so that few tokens leave no tensor-core rows empty and a warp's stores run
// along a row of Y.
//   igemm_pair_kernel    tiles of 256 channels x 256 tokens on CTA pairs (cta_group::2), persistent:
//                        the structure of gemm2_kernel with int8 K blocks. For many tiles. 8192 x
//                        4096 x 4096: 92 us (3.0 POP/s) on a cool chip, 112 at the power limit. A tile
//                        costs 2.4 us beside its MMAs, at K 16384 as at 256: the epilogue's
//                        arithmetic, mask and stores slow the MMAs that they overlap (78 us without).
//   igemm_narrow_kernel  128 channels x T tokens per CTA (40 x 4096 x 4096: 7.0 us in a graph, of
//                        which reading W once is 2.6). The K blocks of a tile are
//                        split over a cluster whose CTAs add their int32 partial sums through
//                        distributed shared memory: with few tokens the weights are the traffic,
//                        and the split lets all SMs read them.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "gemm2_tcgen05.cuh"

namespace c3cu {
namespace igemm {

struct Params {
  int32_t M, N, K;
  void* out;           // bf16 or fp32 [M][ldo]
  int64_t ldo;
  const float* xs;     // [M]
  const float* ws;     // [N]
  const float* bias;   // [N] or null
  uint32_t* mask;      // [M][ldm] (RELU), may be null
  int64_t ldm;
  int32_t kb_per_cta;  // narrow kernel: K blocks per CTA of a cluster
  int32_t n_tiles;     // narrow kernel: tiles of 128 channels
  int32_t stages;      // narrow kernel: ring depth
};

// kind::i8: signed int8 operands, int32 accumulator without saturation, both operands K-major.
__host__ __device__ constexpr uint32_t make_idesc_s8_s32(uint32_t M, uint32_t N) {
  return (2u << 4)           // D format: S32
         | (1u << 7)         // A format: S8
         | (1u << 10)        // B format: S8
         | ((N >> 3) << 17)  // N / 8
         | ((M >> 4) << 24); // M / 16
}

__device__ __forceinline__ void umma_i8_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void umma_i8_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ float relu_keep_nan(float z) {  // a NaN (a row that was not finite) stays one
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(z));
  return r;
}

// The epilogue of J tokens, one channel per lane: a token's 32 lanes store 32 consecutive channels
// (16-byte stores of a row per lane would touch 32 lines each), and the channel's scale and bias stay
// in registers. `m` is the first token, `count` how many there are, xs(j) their scales. The J tokens'
// arithmetic and stores are independent of one another.
template <int J, bool F32, bool RELU, class Scale>
__device__ __forceinline__ void store_tokens(const Params& p, const uint32_t (&acc)[J], Scale xs, int m, int count,
                                             int n, float ws, float b, uint32_t lane) {
  const bool in = n < p.N;
  float z[J];
  // Scalar intrinsics, which are never contracted: ptxas fused a packed (f32x2) multiply and add.
#pragma unroll
  for (int j = 0; j < J; ++j) {
    z[j] = __fmul_rn(__int2float_rn(static_cast<int>(acc[j])), __fmul_rn(xs(j), ws));
    if (p.bias) z[j] = __fadd_rn(z[j], b);
  }
  if constexpr (RELU) {
    if (p.mask) {
      uint32_t word = 0u;  // of token `lane`
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint32_t bits = __ballot_sync(0xffffffffu, in && z[j] > 0.f);
        if (lane == static_cast<uint32_t>(j)) word = bits;
      }
      const int n0 = n - static_cast<int>(lane);
      if (n0 < p.N && static_cast<int>(lane) < count && lane < J)
        p.mask[static_cast<int64_t>(m + lane) * p.ldm + (n0 >> 5)] = word;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) z[j] = relu_keep_nan(z[j]);
  }
  if (!in) return;
  using Out = typename std::conditional<F32, float, __nv_bfloat16>::type;
  Out* out = static_cast<Out*>(p.out) + static_cast<int64_t>(m) * p.ldo + n;
  Out v[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if constexpr (F32) v[j] = z[j];
    else v[j] = __float2bfloat16_rn(z[j]);
  }
  if (count >= J) {
#pragma unroll
    for (int j = 0; j < J; ++j, out += p.ldo) *out = v[j];
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j, out += p.ldo)
      if (j < count) *out = v[j];
  }
}

// ================================================================ CTA pairs
namespace pair {
using gemm2::A_STAGE_BYTES;
using gemm2::B_STAGE_BYTES;
using gemm2::HM;
using gemm2::HN;
using gemm2::kPairMask;
using gemm2::SMEM_BYTES;
using gemm2::STAGE_BYTES;
using gemm2::STAGES;
using gemm2::TM;
using gemm2::TMEM_COLS;
using gemm2::TN;
constexpr int BK = 128;         // int8 elements: the same 128-byte lines as 64 bf16
constexpr uint32_t KSTEP = 32;  // bytes (elements) of K per MMA
constexpr int kEpiWarps = 8;     // sixteen measured the same
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kWarpTokens = TN / (kEpiWarps / 4);
}  // namespace pair

template <bool F32, bool RELU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::kThreads, 1)
    igemm_pair_kernel(const __grid_constant__ CUtensorMap tmw, const __grid_constant__ CUtensorMap tmx,
                      const Params p) {
  using namespace pair;
  __shared__ __align__(16) float s_xs[kEpiWarps][32];  // each warp's own: the scales of the tokens it works on
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  uint64_t* full = bars;
  uint64_t* empty = bars + STAGES;
  uint64_t* acc_full = bars + 2 * STAGES;
  uint64_t* acc_empty = bars + 2 * STAGES + 2;
  uint64_t* drain = bars + 2 * STAGES + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 5);

  const uint32_t warp = warp_id_sync();
  const uint32_t lane = lane_id();
  const uint32_t rank = cluster_ctarank();  // 0 = leader
  const bool leader = rank == 0u;
  const int cluster = static_cast<int>(blockIdx.x >> 1);
  const int num_clusters = static_cast<int>(gridDim.x >> 1);
  // a tile: 256 channels (the MMA's rows) x 256 tokens
  const int n_tiles = (p.N + TM - 1) / TM;
  const int num_tiles = ((p.M + TN - 1) / TN) * n_tiles;
  const int k_blocks = (p.K + BK - 1) / BK;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kEpiWarps);
    }
    mbar_init(drain, 1);
    fence_mbarrier_init();
    tma_prefetch_desc(&tmw);
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
      for (int tile = cluster; ok && tile < num_tiles; tile += num_clusters) {
        const int n0 = (tile % n_tiles) * TM + static_cast<int>(rank) * HM;
        const int m0 = (tile / n_tiles) * TN + static_cast<int>(rank) * HN;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&empty[s], ph ^ 1u, kFaultWaitEmpty)) { ok = false; break; }
          if (leader) mbar_arrive_expect_tx(&full[s], 2u * STAGE_BYTES);
          const uint32_t bar_leader = mapa_shared(smem_u32(&full[s]), 0u);
          tma_load_2d_pair(sA + s * A_STAGE_BYTES, &tmw, bar_leader, kb * BK, n0);
          tma_load_2d_pair(sB + s * B_STAGE_BYTES, &tmx, bar_leader, kb * BK, m0);
          armed |= 1u << s;
          armed_par = (armed_par & ~(1u << s)) | (ph << s);
          if (++s == STAGES) { s = 0; ph ^= 1u; }
        }
      }
      // No copy outlives the CTA, also where the MMA issuer gave up on a late one after this lane was done
      // (the leader's barriers count both CTAs' copies, and the pair leaves together).
      if (leader) {
        for (int t = 0; t < STAGES; ++t)
          if (armed & (1u << t)) gemm::drain_wait(&full[t], (armed_par >> t) & 1u);
      }
      if (!ok) gemm2::settle_inflight_copies();
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (leader && lane == 0) {
      constexpr uint32_t IDESC = make_idesc_s8_s32(TM, TN);
      int s = 0;
      uint32_t ph = 0, acc = 0, acc_ph = 0;
      bool ok = true;
      for (int tile = cluster; ok && tile < num_tiles; tile += num_clusters) {
        if (!mbar_wait(&acc_empty[acc], acc_ph ^ 1u, kFaultWaitAccEmpty)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * TN;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&full[s], ph, kFaultWaitFull)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(sA + s * A_STAGE_BYTES);
          const uint32_t b_addr = smem_u32(sB + s * B_STAGE_BYTES);
#pragma unroll
          for (int kk = 0; kk < BK / static_cast<int>(KSTEP); ++kk)
            umma_i8_ss_pair(d_tmem, make_sw128_desc(a_addr + kk * KSTEP, 16, 1024),
                            make_sw128_desc(b_addr + kk * KSTEP, 16, 1024), IDESC, (kb != 0 || kk != 0) ? 1u : 0u);
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
  } else {
    // ------------------------------------------------------------ epilogue (warps 2..9)
    const uint32_t q = warp & 3u;
    float* my_xs = s_xs[warp - 2u];
    const int c_lo = static_cast<int>((warp - 2u) >> 2) * kWarpTokens;  // this warp's share of the tokens
    uint32_t acc = 0, acc_ph = 0;
    for (int tile = cluster; tile < num_tiles; tile += num_clusters) {
      const int n = (tile % n_tiles) * TM + static_cast<int>(rank) * HM + static_cast<int>(q * 32 + lane);
      const int m0 = (tile / n_tiles) * TN + c_lo;
      const float ws = n < p.N ? __ldg(p.ws + n) : 0.f;
      const float b = p.bias && n < p.N ? __ldg(p.bias + n) : 0.f;
      float xs[kWarpTokens / 32];  // of token m0 + 32 c + lane
#pragma unroll
      for (int c = 0; c < kWarpTokens / 32; ++c) {
        const int m = m0 + c * 32 + static_cast<int>(lane);
        xs[c] = m < p.M ? __ldg(p.xs + m) : 0.f;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[acc], acc_ph, kFaultWaitAccFull))) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((q * 32u) << 16) + acc * TN + static_cast<uint32_t>(c_lo);
      // two chunks' accumulators in registers, so that one is on its way while the other is worked on
      uint32_t r[2][32];
      tmem_ld_32x32b_x32(t_row, r[0]);
#pragma unroll
      for (int c = 0; c < kWarpTokens / 32; ++c) {
        __syncwarp();  // lanes past the last channel skip the stores
        tmem_wait_ld();
        if (c + 1 < kWarpTokens / 32) {
          tmem_ld_32x32b_x32(t_row + (c + 1) * 32, r[(c + 1) & 1]);
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_leader(&acc_empty[acc]);
        }
        const int m = m0 + c * 32;
        my_xs[lane] = xs[c];
        __syncwarp();
        if (m < p.M)
          store_tokens<32, F32, RELU>(
              p, r[c & 1], [&](int j) { return my_xs[j]; }, m, p.M - m, n, ws, b, lane);
        __syncwarp();
      }
      __syncwarp();
      acc ^= 1u;
      if (acc == 0u) acc_ph ^= 1u;
    }
  }

  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// ================================================================ few tokens
namespace narrow {
constexpr int BN = 128;          // channels per CTA: the MMA's 128 rows
constexpr int BK = 128;
constexpr int kThreads = 320;    // TMA, MMA, eight epilogue warps: two a scheduler, since one alone
                                 // waits out the latency of each of its instructions
constexpr int kMaxStages = 8;
constexpr int kMaxCluster = 8;
constexpr uint32_t W_BYTES = BN * BK;
constexpr uint32_t BAR_BYTES = (2 * kMaxStages + 2) * 8 + 16;
constexpr uint32_t kMaxRing = 200 * 1024;
constexpr int kMaxSmem = static_cast<int>(kMaxRing) + 4096;  // barriers and alignment besides
__host__ __device__ constexpr uint32_t stage_bytes(int T) { return W_BYTES + static_cast<uint32_t>(T) * BK; }
__host__ __device__ constexpr uint32_t partial_bytes(int T) { return static_cast<uint32_t>(T) * BN * 4; }
__host__ __device__ constexpr uint32_t smem_bytes(int T, int stages) {
  const uint32_t ring = stage_bytes(T) * static_cast<uint32_t>(stages);
  return (ring > partial_bytes(T) ? ring : partial_bytes(T)) + BAR_BYTES + 1024;
}
}  // namespace narrow

__device__ __forceinline__ uint32_t ld_shared_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <int T, bool F32, bool RELU>
__global__ void __launch_bounds__(narrow::kThreads)
    igemm_narrow_kernel(const __grid_constant__ CUtensorMap tmw, const __grid_constant__ CUtensorMap tmx,
                        const Params p) {
  using namespace narrow;
  constexpr uint32_t STAGE = stage_bytes(T);
  constexpr uint32_t COLS = T < 32 ? 32 : T;
  __shared__ __align__(16) float s_xs[T];
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const uint32_t ring = STAGE * static_cast<uint32_t>(p.stages);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (ring > partial_bytes(T) ? ring : partial_bytes(T)));
  uint64_t* full = bars;
  uint64_t* empty = bars + kMaxStages;
  uint64_t* acc_full = bars + 2 * kMaxStages;
  uint64_t* drain = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  uint32_t* gave_up = tmem_slot + 1;  // set by the MMA lane
  uint32_t* asked = tmem_slot + 2;    // the TMA lane's stages that were asked for, and their phases

  const uint32_t warp = warp_id_sync();
  const uint32_t lane = lane_id();
  const uint32_t rank = cluster_ctarank();
  uint32_t size;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const int tile = static_cast<int>(blockIdx.x / size);
  const int n0 = (tile % p.n_tiles) * BN;
  const int m0 = (tile / p.n_tiles) * T;
  const int k_blocks = (p.K + BK - 1) / BK;
  const int kb0 = static_cast<int>(rank) * p.kb_per_cta;
  const int kb1 = min(kb0 + p.kb_per_cta, k_blocks);

  if (warp == 0 && lane == 0) {
    *gave_up = 0u;
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(drain, 1);
    fence_mbarrier_init();
    tma_prefetch_desc(&tmw);
    tma_prefetch_desc(&tmx);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, COLS);
    tmem_relinquish();
  }
  // the tokens' scales: fetched now, since in the epilogue every fetch would be waited for
  for (int t = static_cast<int>(threadIdx.x); t < T; t += kThreads) s_xs[t] = m0 + t < p.M ? __ldg(p.xs + m0 + t) : 0.f;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, armed = 0u, armed_par = 0u;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[s], ph ^ 1u, kFaultWaitEmpty)) break;
        mbar_arrive_expect_tx(&full[s], STAGE);
        tma_load_2d(smem + s * STAGE, &tmw, &full[s], kb * BK, n0);
        tma_load_2d(smem + s * STAGE + W_BYTES, &tmx, &full[s], kb * BK, m0);
        armed |= 1u << s;
        armed_par = (armed_par & ~(1u << s)) | (ph << s);
        if (++s == p.stages) { s = 0; ph ^= 1u; }
      }
      asked[0] = armed;
      asked[1] = armed_par;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t IDESC = make_idesc_s8_s32(BN, T);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[s], ph, kFaultWaitFull)) { ok = false; break; }
        tc_fence_after();
        const uint32_t w = smem_u32(smem + s * STAGE);
        const uint32_t x = w + W_BYTES;
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk)
          umma_i8_ss(tmem, make_sw128_desc(w + kk * 32, 16, 1024), make_sw128_desc(x + kk * 32, 16, 1024), IDESC,
                     (kb != kb0 || kk != 0) ? 1u : 0u);
        umma_commit(&empty[s]);
        if (++s == p.stages) { s = 0; ph ^= 1u; }
      }
      // After a fault the epilogue is not told that the sums are there: it gives up as well.
      if (!ok) *gave_up = 1u;
      uint64_t* done = ok ? acc_full : drain;
      umma_commit(done);
      gemm::drain_wait(done, 0u);
    }
    __syncwarp();
  }

  const uint32_t q = warp & 3u;                              // the lane quarter of an epilogue warp
  const int half = warp >= 6 ? 1 : 0;                        // the two warps of a quarter share the tokens
  const int n = n0 + static_cast<int>(q * 32 + lane);
  const uint32_t t_row = tmem + ((q * 32u) << 16);
  float ws = 0.f, b = 0.f;
  bool ok = true;
  if (warp >= 2) {
    if (n < p.N) {
      ws = __ldg(p.ws + n);
      if (p.bias) b = __ldg(p.bias + n);
    }
    ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0u, kFaultWaitAccFull));
    tc_fence_after();
  }
  const int tokens = min(T, p.M - m0);
  if (size == 1u) {
    if (warp >= 2 && ok) {
#pragma unroll 1
      for (int c = 16 * half; c < tokens; c += 32) {
        uint32_t r[16];
        __syncwarp();
        tmem_ld_32x32b_x16(t_row + c, r);
        tmem_wait_ld();
        store_tokens<16, F32, RELU>(p, r, [&](int j) { return s_xs[c + j]; }, m0 + c, tokens - c, n, ws, b, lane);
      }
    }
  } else {
    // The ring is free (every MMA has read its stage): it takes this CTA's partial sums
    // [token][channel], and each CTA adds up and stores its share of the tokens.
    uint32_t* part = reinterpret_cast<uint32_t*>(smem);
    const bool any = kb0 < kb1;  // the last CTAs may have no K block: their sums are zero
    if (warp >= 2 && ok) {
#pragma unroll 1
      for (int c = 16 * half; c < tokens; c += 32) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(t_row + c, r);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * BN + q * 32u + lane] = any ? r[j] : 0u;
      }
    }
    cluster_sync_all();
    if (warp >= 2 && ok) {
      const uint32_t mine = smem_u32(part) + (q * 32u + lane) * 4u;
      const int share = T / static_cast<int>(size);
      const int first = static_cast<int>(rank) * share;
      const int last = min(first + share, tokens);
      constexpr int J = T / kMaxCluster < 8 ? T / kMaxCluster : 8;  // divides every share
#pragma unroll 1
      for (int t = first + J * half; t < last; t += 2 * J) {
        uint32_t sum[J];
#pragma unroll
        for (int j = 0; j < J; ++j) sum[j] = 0u;
#pragma unroll 2
        for (uint32_t r = 0; r < size; ++r) {
          const uint32_t from = mapa_shared(mine + t * (BN * 4), r);
#pragma unroll
          for (int j = 0; j < J; ++j) sum[j] += ld_shared_cluster(from + j * (BN * 4));
        }
        store_tokens<J, F32, RELU>(p, sum, [&](int j) { return s_xs[t + j]; }, m0 + t, last - t, n, ws, b, lane);
      }
    }
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while another reads its sums
  }

  tc_fence_before();
  __syncthreads();
  // No copy outlives the CTA. Where the MMA lane went through all blocks, it saw each of them land; where it
  // gave up on a late one, the TMA lane, which may have been done long before, waits for them here.
  if (threadIdx.x == 0 && *gave_up != 0u)
    for (int t = 0; t < p.stages; ++t)
      if (asked[0] & (1u << t)) gemm::drain_wait(&full[t], (asked[1] >> t) & 1u);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, COLS);
  }
}

}  // namespace igemm
}  // namespace c3cu
