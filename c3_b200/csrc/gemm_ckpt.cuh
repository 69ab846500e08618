// Weight gradient from an 8-bit checkpoint of the layer's input:
//
//   dW[N][K] = sum_m dZ[m][n] * (q[m][k] * scale[m])        (bf16 out, fp32 sums in TMEM)
//
// dZ is bf16, X is held as int8 rows with one fp32 scale each (c3cu_quantize_rows). The scale runs along
// the sum, so it cannot wait for the epilogue: it goes to an operand. q is exact in the tensor cores' 16-bit
// types, so the scale goes to dZ, and the operand rounding is that of dZ * scale alone. In bf16 that
// rounding (2^-8) would be as large as the output's own; so it is fp16 here (2^-11), and two bf16 terms
// (2^-14) in the small tiles of gemm_ckpt_narrow.cuh. Against fp64 the error of dW is then the output
// rounding's (0.0017 of the norm; 0.0024 with operands in bf16).
//
// fp16 has five bits of exponent where bf16 has eight, so each column of dZ * scale, i.e. each row of dW,
// is brought into its range by a power of two of its own:
//   column_top_kernel  the largest finite |dZ * scale| of each column (in bands of rows; not launched for one)
//   operands_kernel    dZ * scale * 2^(14 - e) in fp16, e the exponent of the column's largest, and q in
//                      fp16, both into the workspace
//   dw_kernel          the product, gemm2_kernel's structure (256 x 256 tiles on CTA pairs, both operands
//                      MN-major, since dZ and X are stored with the sum's index as their rows); its epilogue
//                      multiplies by 2^(e - 14), exactly
// 16384 x 4096 x 4096: 480 to 500 us, of which the product takes 340 and the first two, which read dZ twice,
// about 110. Operands rounded to bf16, for which X alone was rewritten, took 433 to 450.
// An element is rounded by 2^-11 of itself or, from 2^-28 of its column's largest down, by 2^-39 of that
// largest, which is below what fp32 sums over the column lose. What is not finite stays so.
//
// The MMA's rows are the columns of dW, so that a warp's stores run along its rows whatever their
// alignment (2176 x 4822 over 576 rows: 138 us with a row of dW per lane, 27 so).
//
// Warps of dw_kernel: 0 TMA, 1 MMA (leader), 2..9 epilogue.
#pragma once

#include <cuda_fp16.h>

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
using gemm2::kThreads;
using gemm2::MN_CHUNK_BYTES;
using gemm2::SMEM_BYTES;
using gemm2::STAGE_BYTES;
using gemm2::STAGES;
using gemm2::TM;
using gemm2::TMEM_COLS;
using gemm2::TN;
using gemm2::UMMA_K;

struct Params {
  int32_t M, N, K;     // dW is N x K, the sum runs over M
  __nv_bfloat16* out;
  int64_t ldo;
  const float* back;   // [N, padded to 64]: 2^(e - 14) of each row of dW
  float* partial;      // slots of [256 rows][256 columns] fp32, not yet multiplied by it
  Plan plan;
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    dw_kernel(const __grid_constant__ CUtensorMap tmz, const __grid_constant__ CUtensorMap tmx, const Params p) {
  __shared__ float4 s_back[kEpiWarps][8];  // each warp's own: of the 32 rows it works on
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sZ = smem;
  uint8_t* sX = smem + STAGES * A_STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);  // loads of both CTAs (the leader's is used)
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
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
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kEpiWarps);
    }
    mbar_init(drain, 1);
    fence_mbarrier_init();
    tma_prefetch_desc(&tmz);
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
          if (leader) mbar_arrive_expect_tx(&full[s], 2u * STAGE_BYTES);
          const uint32_t bar_leader = mapa_shared(smem_u32(&full[s]), 0u);
          uint8_t* sz = sZ + s * A_STAGE_BYTES;
          uint8_t* sx = sX + s * B_STAGE_BYTES;
#pragma unroll
          for (int j = 0; j < HM / 64; ++j)
            tma_load_2d_pair(sz + j * MN_CHUNK_BYTES, &tmz, bar_leader, n0 + 64 * j, kb * BK);
#pragma unroll
          for (int j = 0; j < HN / 64; ++j)
            tma_load_2d_pair(sx + j * MN_CHUNK_BYTES, &tmx, bar_leader, k0 + 64 * j, kb * BK);
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
      constexpr uint32_t IDESC = make_idesc_f16_f32(TM, TN, true, true);
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
          const uint32_t z_addr = smem_u32(sZ + s * A_STAGE_BYTES);
          const uint32_t x_addr = smem_u32(sX + s * B_STAGE_BYTES);
#pragma unroll
          for (int kk = 0; kk < BK / UMMA_K; ++kk)
            umma_f16_ss_pair(d_tmem, make_sw128_desc(x_addr + kk * UMMA_K * 128, MN_CHUNK_BYTES, 1024),
                             make_sw128_desc(z_addr + kk * UMMA_K * 128, MN_CHUNK_BYTES, 1024), IDESC,
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
  } else {
    // ------------------------------------------------------------ epilogue (warps 2..9)
    const uint32_t q = warp & 3u;
    const int c_lo = static_cast<int>((warp - 2u) >> 2) * (TM / 2);  // this warp's half of the rows of dW
    const int in_tile = static_cast<int>(rank) * HN + static_cast<int>(q * 32u + lane);
    float4* back = s_back[warp - 2u];
    uint32_t acc = 0, acc_ph = 0;
    for (int i = cluster; i < items; i += num_clusters) {
      const Item it = item_at(p.plan, i, blocks);
      const int n0 = (it.tile / k_tiles) * TM + c_lo;
      const int k = (it.tile % k_tiles) * TN + in_tile;
      // asked for while the MMAs run: in the loop below each would be waited for
      const int at = n0 + 4 * static_cast<int>(lane);
      const float4 mine = at < p.N ? __ldg(reinterpret_cast<const float4*>(p.back + at)) : make_float4(0.f, 0.f, 0.f, 0.f);
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[acc], acc_ph, kFaultWaitAccFull))) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((q * 32u) << 16) + acc * TM + static_cast<uint32_t>(c_lo);
#pragma unroll 1
      for (int c = 0; c < TM / 2; c += 32) {
        const int rows = min(32, p.N - n0 - c);
        if (rows <= 0) break;
        uint32_t r[32];
        __syncwarp();  // lanes past the last column skip the stores
        if (static_cast<int>(lane >> 3) == c / 32) back[lane & 7u] = mine;
        tmem_ld_32x32b_x32(t_row + c, r);
        tmem_wait_ld();
        __syncwarp();
        if (k >= p.K) continue;
        if (it.slot < 0) {
          __nv_bfloat16* out = p.out + static_cast<int64_t>(n0 + c) * p.ldo + k;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 f = back[j / 4];
            const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4, out += p.ldo)
              if (j + i4 < rows) *out = __float2bfloat16_rn(__uint_as_float(r[j + i4]) * v[i4]);
          }
        } else {
          float* part = p.partial + static_cast<size_t>(it.slot) * (TM * TN) + (c_lo + c) * TN + in_tile;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j < rows) __stcg(part + j * TN, __uint_as_float(r[j]));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(&acc_empty[acc]);
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

// ---------------------------------------------------------------- fp16 operands
// dZ is walked in items of 64 columns (a 128-byte line of a row: eight lanes, 16 bytes each) by a band of
// rows; bands are few, so that their column maxima are soon put together again.
constexpr int kPrepThreads = 256;
constexpr int kMaxBands = 32;
constexpr int kPrepRows = kPrepThreads / 8;  // rows of an item that a block has at a time

struct Prep {
  const __nv_bfloat16* dz;
  const int8_t* q;
  const float* scale;
  float* top;     // [bands][tiles * 64]
  float* back;    // [tiles * 64]
  __half* z16;    // [M][ldz]
  __half* x16;    // [M][ldx16]
  int64_t lddz, ldq, ldz, ldx16;
  int32_t M, N, K;
  int32_t tiles, bands, band_rows;
};

// Eight columns of a row of dZ from column n on, zeros past N.
__device__ __forceinline__ uint4 load_ragged_dz(const Prep& p, int64_t m, int n) {
  const __nv_bfloat16* at = p.dz + m * p.lddz + n;
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (n + j < p.N) w[j / 2] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const unsigned short*>(at) + j)) << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// f(row, dZ's eight columns from n on, scale) for A of the thread's rows at a time, whose loads go out
// together, while there are A left before m1; returns the next row.
template <int A, class F>
__device__ __forceinline__ int64_t for_rows_by(const Prep& p, int64_t m, int64_t m1, int n, F& f) {
  for (; m + (A - 1) * kPrepRows < m1; m += A * kPrepRows) {
    uint4 w[A];
    float s[A];
#pragma unroll
    for (int a = 0; a < A; ++a) {
      w[a] = __ldg(reinterpret_cast<const uint4*>(p.dz + (m + a * kPrepRows) * p.lddz + n));
      s[a] = __ldg(p.scale + m + a * kPrepRows);
    }
#pragma unroll
    for (int a = 0; a < A; ++a) f(m + a * kPrepRows, w[a], s[a]);
  }
  return m;
}

// The same for all of the thread's rows of a band.
template <class F>
__device__ __forceinline__ void for_rows(const Prep& p, int64_t m, int64_t m1, int n, F f) {
  if (n + 8 <= p.N) {
    m = for_rows_by<8>(p, m, m1, n, f);
    m = for_rows_by<4>(p, m, m1, n, f);
    for_rows_by<1>(p, m, m1, n, f);
  } else {
    for (; m < m1; m += kPrepRows) f(m, load_ragged_dz(p, m, n), __ldg(p.scale + m));
  }
}

// dZ * scale, the product that both kernels take.
__device__ __forceinline__ void scaled8(const uint4& w, float s, float2 (&v)[4]) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = mul2(make_float2(__uint_as_float(x[j] << 16), __uint_as_float(x[j] & 0xffff0000u)), make_float2(s, s));
}

// The larger magnitude; a NaN counts for nothing.
__device__ __forceinline__ float larger(float top, float v) { return fmaxf(top, fabsf(v)); }
__device__ __forceinline__ float larger_finite(float top, float v) {
  return fabsf(v) < __builtin_huge_valf() ? larger(top, v) : top;
}

// The largest finite |dZ * scale| of the tile's column threadIdx.x (below 64) in rows m0.. of a band, by the
// whole block.
struct Tops {
  float of[kPrepThreads / 32][64];
};

__device__ __forceinline__ float column_top(const Prep& p, int tile, int64_t m0, int64_t m1, Tops& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int piece = lane & 7, n = tile * 64 + piece * 8;
  m0 += threadIdx.x >> 3;
  float top[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (n < p.N) {
    const auto walk = [&](auto pick) {
      for_rows(p, m0, m1, n, [&](int64_t, const uint4& w, float scale) {
        float2 v[4];
        scaled8(w, scale, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          top[2 * j] = pick(top[2 * j], v[j].x);
          top[2 * j + 1] = pick(top[2 * j + 1], v[j].y);
        }
      });
    };
    walk([](float t, float v) { return larger(t, v); });
    bool infinite = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) infinite = infinite || top[j] == __builtin_huge_valf();
    if (infinite) {  // again without what is infinite
#pragma unroll
      for (int j = 0; j < 8; ++j) top[j] = 0.f;
      walk([](float t, float v) { return larger_finite(t, v); });
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 8));
    top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 16));
  }
  if (lane < 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s.of[warp][piece * 8 + j] = top[j];
  }
  __syncthreads();
  float t = 0.f;
  if (threadIdx.x < 64) {
#pragma unroll
    for (int w = 0; w < kPrepThreads / 32; ++w) t = fmaxf(t, s.of[w][threadIdx.x]);
  }
  return t;
}

__global__ void __launch_bounds__(kPrepThreads) column_top_kernel(const Prep p) {
  __shared__ Tops s_top;
  pdl_wait();
  pdl_launch_dependents();
  for (int item = blockIdx.x; item < p.tiles * p.bands; item += gridDim.x) {
    const int tile = item % p.tiles, band = item / p.tiles;
    const int64_t m0 = static_cast<int64_t>(band) * p.band_rows;
    const float t = column_top(p, tile, m0, min(static_cast<int64_t>(p.M), m0 + p.band_rows), s_top);
    if (threadIdx.x < 64) p.top[(static_cast<int64_t>(band) * p.tiles + tile) * 64 + threadIdx.x] = t;
    __syncthreads();  // the next item's maxima go to the same place
  }
}

// Four int8 in fp16, exactly: 0x6400 is 1024 with one as its last place, so or-ing q + 128 gives
// 1152 + q.
__device__ __forceinline__ uint2 widen4(uint32_t w) {
  const uint32_t u = w ^ 0x80808080u;
  uint32_t v[2] = {__byte_perm(u, 0x64646464u, 0x4140), __byte_perm(u, 0x64646464u, 0x4342)};
  const __half2 bias = __float2half2_rn(1152.f);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&v[j]), bias);
    v[j] = *reinterpret_cast<const uint32_t*>(&x);
  }
  return make_uint2(v[0], v[1]);
}

constexpr int kWidenAhead = 8;

// Row m of X in fp16 (columns past K zero): a lane has eight columns at a time, so that a warp's stores
// are one run of 512 bytes, eight loads ahead of their use.
__device__ __forceinline__ void widen_row(const Prep& p, int64_t m, int lane) {
  const int units = static_cast<int>(p.ldx16 / 8), whole = p.K / 8;
  const int8_t* from = p.q + m * p.ldq;
  uint4* to = reinterpret_cast<uint4*>(p.x16 + m * p.ldx16);
  for (int u0 = lane; u0 < units; u0 += 32 * kWidenAhead) {
    uint2 w[kWidenAhead];
#pragma unroll
    for (int i = 0; i < kWidenAhead; ++i) {
      const int u = u0 + 32 * i;
      w[i] = make_uint2(0u, 0u);
      if (u < whole) {
        w[i] = __ldcs(reinterpret_cast<const uint2*>(from) + u);
      } else if (u < units) {
        uint32_t x[2] = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (u * 8 + j < p.K) x[j / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(from[u * 8 + j])) << (8 * (j % 4));
        w[i] = make_uint2(x[0], x[1]);
      }
    }
#pragma unroll
    for (int i = 0; i < kWidenAhead; ++i) {
      const int u = u0 + 32 * i;
      if (u >= units) break;
      const uint2 a = widen4(w[i].x), b = widen4(w[i].y);
      to[u] = make_uint4(a.x, a.y, b.x, b.y);
    }
  }
}

// Both operands, as one list of items: first dZ's (from its end: the last that column_top_kernel read are
// still in L2), then X's rows, one a warp.
constexpr int kWidenRows = kPrepThreads / 32;

__global__ void __launch_bounds__(kPrepThreads) operands_kernel(const Prep p) {
  __shared__ Tops s_top;
  __shared__ __align__(16) float s_up[64];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int dz_items = p.tiles * p.bands;
  const int items = dz_items + static_cast<int>((static_cast<int64_t>(p.M) + kWidenRows - 1) / kWidenRows);
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    if (item >= dz_items) {
      const int64_t m = static_cast<int64_t>(item - dz_items) * kWidenRows + warp;
      if (m < p.M) widen_row(p, m, lane);
      continue;
    }
    const int back_item = dz_items - 1 - item;
    const int tile = back_item % p.tiles, band = back_item / p.tiles;
    const int64_t m0 = static_cast<int64_t>(band) * p.band_rows;
    const int64_t m1 = min(static_cast<int64_t>(p.M), m0 + p.band_rows);
    const int c = threadIdx.x & 63;
    float t = 0.f;
    if (p.bands == 1) {  // no kernel before this one
      t = column_top(p, tile, m0, m1, s_top);
    } else {
      for (int b = threadIdx.x >> 6; b < p.bands; b += kPrepThreads / 64)
        t = fmaxf(t, __ldcg(p.top + (static_cast<int64_t>(b) * p.tiles + tile) * 64 + c));
      s_top.of[threadIdx.x >> 6][c] = t;
      __syncthreads();
#pragma unroll
      for (int i = 1; i < kPrepThreads / 64; ++i) t = fmaxf(t, s_top.of[i][c]);
    }
    if (threadIdx.x < 64) {
      // Below 2^-112 the exponent stays there, so that both powers are normal numbers; fp16's last
      // place is then 2^-150, beneath fp32's.
      const int e = max(static_cast<int>(__float_as_uint(t) >> 23) - 127, -112);
      s_up[c] = __uint_as_float(static_cast<uint32_t>(14 - e + 127) << 23);
      if (band == 0) p.back[tile * 64 + c] = __uint_as_float(static_cast<uint32_t>(e - 14 + 127) << 23);
    }
    __syncthreads();
    const int piece = lane & 7, n = tile * 64 + piece * 8;
    if (n < p.N) {
      float2 up[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) up[j] = *reinterpret_cast<const float2*>(&s_up[piece * 8 + 2 * j]);
      for_rows(p, m0 + (threadIdx.x >> 3), m1, n,
               [&](int64_t m, const uint4& w, float s) {
                 float2 v[4];
                 scaled8(w, s, v);
                 uint32_t o[4];
#pragma unroll
                 for (int j = 0; j < 4; ++j) {
                   const float2 x = mul2(v[j], up[j]);
                   const __half2 h = __floats2half2_rn(x.x, x.y);
                   o[j] = *reinterpret_cast<const uint32_t*>(&h);
                 }
                 *reinterpret_cast<uint4*>(p.z16 + m * p.ldz + n) = make_uint4(o[0], o[1], o[2], o[3]);
               });
    }
    __syncthreads();  // the next item's maxima go to the same place
  }
}

// Adds the pieces of the cut tiles in order, rounds once. A block takes eight rows of a tile, a thread
// one column of them.
constexpr int kAddRows = 8;

__global__ void __launch_bounds__(TN) add_pieces_kernel(const Params p) {
  pdl_wait();
  const int tile = p.plan.whole + static_cast<int>(blockIdx.y);
  const int k_tiles = (p.K + TN - 1) / TN;
  const int r0 = static_cast<int>(blockIdx.x) * kAddRows;
  const int n0 = (tile / k_tiles) * TM + r0, k = (tile % k_tiles) * TN + static_cast<int>(threadIdx.x);
  if (n0 >= p.N || k >= p.K) return;
  const float* part = p.partial + static_cast<size_t>(blockIdx.y) * p.plan.pieces * (TM * TN) + r0 * TN + threadIdx.x;
  float sum[kAddRows];
#pragma unroll
  for (int i = 0; i < kAddRows; ++i) sum[i] = 0.f;
#pragma unroll 2
  for (int s = 0; s < p.plan.pieces; ++s) {
#pragma unroll
    for (int i = 0; i < kAddRows; ++i)
      if (n0 + i < p.N) sum[i] += __ldcg(part + static_cast<size_t>(s) * (TM * TN) + i * TN);
  }
  __nv_bfloat16* out = p.out + static_cast<int64_t>(n0) * p.ldo + k;
#pragma unroll
  for (int i = 0; i < kAddRows; ++i)
    if (n0 + i < p.N) out[i * p.ldo] = __float2bfloat16_rn(sum[i] * __ldg(p.back + n0 + i));
}

}  // namespace ckpt
}  // namespace c3cu
