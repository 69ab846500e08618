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
// Two kernels:
//   igemm_pair_kernel    256 x 256 tiles on CTA pairs (cta_group::2), persistent: the structure of
//                        gemm2_kernel with int8 K blocks. For sizes whose tiles fill the GPU.
//   igemm_narrow_kernel  128 channels x T tokens per CTA, the channels as the MMA's rows, so that
//                        few tokens leave no tensor-core rows empty. The K blocks of a tile are
//                        split over a cluster whose CTAs add their int32 partial sums through
//                        distributed shared memory: with few tokens the weights are the traffic,
//                        and the split lets all SMs read them.
#pragma once

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
  int32_t vec_ok;      // every full 32-column chunk may use 16-byte accesses
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

__device__ __forceinline__ float scaled(uint32_t acc, float xs, float ws) {
  return __fmul_rn(__int2float_rn(static_cast<int>(acc)), __fmul_rn(xs, ws));
}

__device__ __forceinline__ float relu_keep_nan(float z) {  // a NaN (a row that was not finite) stays one
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(z));
  return r;
}

// Packed fp32 arithmetic: two elements per instruction, each rounded like its scalar form.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}

// 32 columns of one row of the output (pair kernel: a thread owns a row).
template <bool F32, bool RELU>
__device__ __forceinline__ void store_chunk(const Params& p, const uint32_t (&r)[32], int row, int col0, float xs) {
  if (row >= p.M) return;
  const int ncols = min(32, p.N - col0);
  const bool full = p.vec_ok && ncols == 32;
  float z[32];
  if (full) {
    const float2 xs2 = make_float2(xs, xs);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 w = __ldg(reinterpret_cast<const float4*>(p.ws + col0) + j);
      float2 lo = make_float2(__int2float_rn(static_cast<int>(r[4 * j])), __int2float_rn(static_cast<int>(r[4 * j + 1])));
      float2 hi = make_float2(__int2float_rn(static_cast<int>(r[4 * j + 2])), __int2float_rn(static_cast<int>(r[4 * j + 3])));
      lo = mul2(lo, mul2(xs2, make_float2(w.x, w.y)));
      hi = mul2(hi, mul2(xs2, make_float2(w.z, w.w)));
      if (p.bias) {
        const float4 b = __ldg(reinterpret_cast<const float4*>(p.bias + col0) + j);
        lo = add2(lo, make_float2(b.x, b.y));
        hi = add2(hi, make_float2(b.z, b.w));
      }
      z[4 * j] = lo.x; z[4 * j + 1] = lo.y; z[4 * j + 2] = hi.x; z[4 * j + 3] = hi.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      z[j] = 0.f;
      if (j < ncols) {
        z[j] = scaled(r[j], xs, __ldg(p.ws + col0 + j));
        if (p.bias) z[j] = __fadd_rn(z[j], __ldg(p.bias + col0 + j));
      }
    }
  }
  if constexpr (RELU) {
    if (p.mask) {
      uint32_t bits = 0u;
#pragma unroll
      for (int j = 0; j < 32; ++j) bits |= z[j] > 0.f ? 1u << j : 0u;
      p.mask[static_cast<int64_t>(row) * p.ldm + (col0 >> 5)] = bits;
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) z[j] = relu_keep_nan(z[j]);
  }
  if constexpr (F32) {
    float* out = static_cast<float*>(p.out) + static_cast<int64_t>(row) * p.ldo + col0;
    if (full) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        reinterpret_cast<float4*>(out)[j] = make_float4(z[4 * j], z[4 * j + 1], z[4 * j + 2], z[4 * j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < ncols) out[j] = z[j];
    }
  } else {
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(row) * p.ldo + col0;
    if (full) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        reinterpret_cast<uint4*>(out)[j] =
            make_uint4(pack_bf16x2(z[8 * j], z[8 * j + 1]), pack_bf16x2(z[8 * j + 2], z[8 * j + 3]),
                       pack_bf16x2(z[8 * j + 4], z[8 * j + 5]), pack_bf16x2(z[8 * j + 6], z[8 * j + 7]));
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < ncols) out[j] = __float2bfloat16_rn(z[j]);
    }
  }
}

// Counts an arrival on a barrier of the leader CTA without a release at cluster scope, which would
// wait for the warp's stores to reach memory: what the arrival reports is that the accumulator has
// been read, and the tcgen05 fence orders that.
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(mapa_shared(smem_u32(bar), 0u)) : "memory");
}

// ================================================================ CTA pairs
namespace pair {
using gemm2::A_STAGE_BYTES;
using gemm2::B_STAGE_BYTES;
using gemm2::HM;
using gemm2::HN;
using gemm2::kEpiWarps;
using gemm2::kPairMask;
using gemm2::kThreads;
using gemm2::SMEM_BYTES;
using gemm2::STAGE_BYTES;
using gemm2::STAGES;
using gemm2::TM;
using gemm2::TMEM_COLS;
using gemm2::TN;
constexpr int BK = 128;         // int8 elements: the same 128-byte lines as 64 bf16
constexpr uint32_t KSTEP = 32;  // bytes (elements) of K per MMA
}  // namespace pair

template <bool F32, bool RELU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::kThreads, 1)
    igemm_pair_kernel(const __grid_constant__ CUtensorMap tma, const __grid_constant__ CUtensorMap tmb,
                      const Params p) {
  using namespace pair;
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
  const int n_tiles = (p.N + TN - 1) / TN;
  const int num_tiles = ((p.M + TM - 1) / TM) * n_tiles;
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
    tma_prefetch_desc(&tma);
    tma_prefetch_desc(&tmb);
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
        const int m0 = (tile / n_tiles) * TM + static_cast<int>(rank) * HM;
        const int n0 = (tile % n_tiles) * TN + static_cast<int>(rank) * HN;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&empty[s], ph ^ 1u, kFaultWaitEmpty)) { ok = false; break; }
          if (leader) mbar_arrive_expect_tx(&full[s], 2u * STAGE_BYTES);
          const uint32_t bar_leader = mapa_shared(smem_u32(&full[s]), 0u);
          tma_load_2d_pair(sA + s * A_STAGE_BYTES, &tma, bar_leader, kb * BK, m0);
          tma_load_2d_pair(sB + s * B_STAGE_BYTES, &tmb, bar_leader, kb * BK, n0);
          armed |= 1u << s;
          armed_par = (armed_par & ~(1u << s)) | (ph << s);
          if (++s == STAGES) { s = 0; ph ^= 1u; }
        }
      }
      if (!ok) {
        if (leader) {
          for (int t = 0; t < STAGES; ++t)
            if (armed & (1u << t)) gemm::drain_wait(&full[t], (armed_par >> t) & 1u);
        }
        gemm2::settle_inflight_copies();
      }
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
    const int c_lo = static_cast<int>((warp - 2u) >> 2) * (TN / 64);
    uint32_t acc = 0, acc_ph = 0;
    for (int tile = cluster; tile < num_tiles; tile += num_clusters) {
      const int row = (tile / n_tiles) * TM + static_cast<int>(rank) * HM + static_cast<int>(q * 32 + lane);
      const int n0 = (tile % n_tiles) * TN;
      const float xs = row < p.M ? __ldg(p.xs + row) : 0.f;
      if (!mbar_wait(&acc_full[acc], acc_ph, kFaultWaitAccFull)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((q * 32u) << 16) + acc * TN;
      // two chunks' accumulators in registers, so that one is on its way while the other is worked on
      uint32_t r[2][32];
      tmem_ld_32x32b_x32(t_row + c_lo * 32, r[0]);
#pragma unroll
      for (int c = 0; c < TN / 64; ++c) {
        tmem_wait_ld();
        if (c + 1 < TN / 64) {
          tmem_ld_32x32b_x32(t_row + (c_lo + c + 1) * 32, r[(c + 1) & 1]);
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_leader(&acc_empty[acc]);
        }
        const int col0 = n0 + (c_lo + c) * 32;
        if (col0 < p.N) store_chunk<F32, RELU>(p, r[c & 1], row, col0, xs);
      }
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
constexpr int kThreads = 192;    // TMA, MMA, four epilogue warps
constexpr int kMaxStages = 8;
constexpr int kMaxCluster = 8;
constexpr uint32_t W_BYTES = BN * BK;
constexpr uint32_t BAR_BYTES = (2 * kMaxStages + 1) * 8 + 8;
constexpr uint32_t kMaxRing = 200 * 1024;
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

// One element per lane: 32 consecutive channels of one token.
template <bool F32, bool RELU>
__device__ __forceinline__ void store_token(const Params& p, uint32_t acc, int m, int n, float ws, float b,
                                            uint32_t lane) {
  const bool in = n < p.N;
  float z = scaled(acc, __ldg(p.xs + m), ws);
  if (p.bias) z = __fadd_rn(z, b);
  if constexpr (RELU) {
    const uint32_t bits = __ballot_sync(0xffffffffu, in && z > 0.f);
    if (p.mask && lane == 0 && in) p.mask[static_cast<int64_t>(m) * p.ldm + (n >> 5)] = bits;
    z = relu_keep_nan(z);
  }
  if (!in) return;
  if constexpr (F32) static_cast<float*>(p.out)[static_cast<int64_t>(m) * p.ldo + n] = z;
  else static_cast<__nv_bfloat16*>(p.out)[static_cast<int64_t>(m) * p.ldo + n] = __float2bfloat16_rn(z);
}

template <int T, bool F32, bool RELU>
__global__ void __launch_bounds__(narrow::kThreads)
    igemm_narrow_kernel(const __grid_constant__ CUtensorMap tmw, const __grid_constant__ CUtensorMap tmx,
                        const Params p) {
  using namespace narrow;
  constexpr uint32_t STAGE = stage_bytes(T);
  constexpr uint32_t COLS = T < 32 ? 32 : T;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const uint32_t ring = STAGE * static_cast<uint32_t>(p.stages);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (ring > partial_bytes(T) ? ring : partial_bytes(T)));
  uint64_t* full = bars;
  uint64_t* empty = bars + kMaxStages;
  uint64_t* acc_full = bars + 2 * kMaxStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStages + 1);

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
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    fence_mbarrier_init();
    tma_prefetch_desc(&tmw);
    tma_prefetch_desc(&tmx);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, COLS);
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
        mbar_arrive_expect_tx(&full[s], STAGE);
        tma_load_2d(smem + s * STAGE, &tmw, &full[s], kb * BK, n0);
        tma_load_2d(smem + s * STAGE + W_BYTES, &tmx, &full[s], kb * BK, m0);
        armed |= 1u << s;
        armed_par = (armed_par & ~(1u << s)) | (ph << s);
        if (++s == p.stages) { s = 0; ph ^= 1u; }
      }
      if (!ok)
        for (int t = 0; t < p.stages; ++t)
          if (armed & (1u << t)) gemm::drain_wait(&full[t], (armed_par >> t) & 1u);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t IDESC = make_idesc_s8_s32(BN, T);
      int s = 0;
      uint32_t ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[s], ph, kFaultWaitFull)) break;
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
      umma_commit(acc_full);  // also on a fault: completes when the MMAs issued so far have
      gemm::drain_wait(acc_full, 0u);
    }
    __syncwarp();
  }

  const uint32_t q = warp & 3u;  // the lane quarter of an epilogue warp
  const int n = n0 + static_cast<int>(q * 32 + lane);
  const uint32_t t_row = tmem + ((q * 32u) << 16);
  float ws = 0.f, b = 0.f;
  bool ok = true;
  if (warp >= 2) {
    if (n < p.N) {
      ws = __ldg(p.ws + n);
      if (p.bias) b = __ldg(p.bias + n);
    }
    ok = mbar_wait(acc_full, 0u, kFaultWaitAccFull);
    tc_fence_after();
  }
  if (size == 1u) {
    if (warp >= 2 && ok) {
#pragma unroll 1
      for (int c = 0; c < T; c += 16) {
        if (m0 + c >= p.M) break;
        uint32_t r[16];
        tmem_ld_32x32b_x16(t_row + c, r);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (m0 + c + j < p.M) store_token<F32, RELU>(p, r[j], m0 + c + j, n, ws, b, lane);
      }
    }
  } else {
    // The ring is free (every MMA has read its stage): it takes this CTA's partial sums
    // [token][channel], and each CTA adds up and stores its share of the tokens.
    uint32_t* part = reinterpret_cast<uint32_t*>(smem);
    const int tokens = min(T, p.M - m0);
    const bool any = kb0 < kb1;  // the last CTAs may have no K block: their sums are zero
    if (warp >= 2) {
#pragma unroll 1
      for (int c = 0; c < T; c += 16) {
        if (c >= tokens) break;
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
      for (int t = static_cast<int>(rank); t < tokens; t += static_cast<int>(size)) {
        uint32_t sum = 0u;
        for (uint32_t r = 0; r < size; ++r) sum += ld_shared_cluster(mapa_shared(mine + t * (BN * 4), r));
        store_token<F32, RELU>(p, sum, m0 + t, n, ws, b, lane);
      }
    }
    cluster_sync_all();  // no CTA leaves while another reads its sums
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, COLS);
  }
}

}  // namespace igemm
}  // namespace c3cu
