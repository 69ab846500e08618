// The weight gradient from an 8-bit checkpoint (gemm_ckpt.cuh) in small tiles: 128 columns x T rows of
// dW on one CTA, for the many layers whose dW has too few 256 x 256 tiles to occupy the GPU. The sum's
// K blocks of a tile are split over a cluster, whose CTAs add their fp32 partial sums through distributed
// shared memory, in the order of their ranks: one launch, no workspace, the same bits every time.
//
// A stage of the ring holds a K block's raw int8 (8 KB), the widened tile made of it (16 KB), and dZ, which
// the same warps replace by dZ * scale in two bf16 terms (8 KB each per 64 columns): head, the product
// rounded to bf16, and tail, what that took from it. Their sum is the product to 2^-14 of it, at fp32's
// range; q itself is exact in bf16. The MMA takes both as one tile of 2 T columns, so that X's tile is read
// once for the two, and the epilogue adds their sums.
// (One fp16 term needs the columns' largest first, i.e. two launches more.) The stage is free again when
// its MMAs are done, so a converter waits for nothing but the loads. What bounds a long sum is shared
// memory: of a K block of 128 x 128 a copy writes 24 KB, the converters read those and write 48, and the MMAs
// read 48 (about 0.65 us, where twice the converters changed nothing).
// Warps: 0 TMA, 1 MMA, 2..9 converters in two groups of four that take the K blocks in turn, and the
// epilogue after them.
#pragma once

#include "ckpt_layout.h"
#include "gemm_ckpt.cuh"
#include "igemm.cuh"

namespace c3cu {
namespace ckpt_narrow {

using ckpt::BK;
using ckpt::MN_CHUNK_BYTES;
using ckpt::UMMA_K;
constexpr int kConvWarps = 4;   // a group's warps
constexpr int kConvGroups = 2;  // the groups take K blocks in turn
constexpr int COLS = 128;       // columns of dW per CTA: the MMA's 128 rows
constexpr int kThreads = 32 * (2 + kConvGroups * kConvWarps);
constexpr int kMaxCluster = 8;
constexpr uint32_t RAW_BYTES = BK * COLS;  // 64 rows (m) of 128 int8 (k)
constexpr uint32_t WIDE_BYTES = 2 * MN_CHUNK_BYTES;
__host__ __device__ constexpr int chunks(int T) { return (T + 63) / 64; }  // of 64 columns of dZ
static_assert(MN_CHUNK_BYTES == ckpt::kChunkBytes && BK == 64, "ckpt_layout.h");

template <int T, bool READY>
struct Ring {
  static constexpr int kStages = READY ? (T <= 64 ? 8 : 6) : T == 32 ? 6 : 4;
  static constexpr uint32_t kZ = READY ? chunks(T) * MN_CHUNK_BYTES : ckpt::DzUnits<T>::kBytes;
  static constexpr uint32_t kStage = WIDE_BYTES + kZ + (READY ? 0 : RAW_BYTES);
  static constexpr uint32_t kSmem = kStages * kStage + (3 * kStages + 2) * 8 + 16 + 1024;
  static_assert(READY || kStages % kConvGroups == 0, "a stage belongs to one group, which so sees each of its phases");
  static_assert(kSmem <= 227 * 1024 && kStages * kStage >= T * COLS * 4, "shared memory");
};

struct Params {
  int32_t M, N, K;  // dW is N x K, the sum runs over M
  __nv_bfloat16* out;
  int64_t ldo;
  const float* scale;  // [M]; READY: 2^(e - 14) of each row of dW, padded to 64
  int32_t kb_per_cta;  // K blocks per CTA of a cluster
  int32_t k_tiles;     // tiles of 128 columns
};

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// dZ * scale is taken times 2^6 and q times 2^-6: what head and tail lose of a product at the bottom of
// fp32's normal numbers then is no more than of any other (below, a product is held to 2^-138), and the
// scale of a row of fp32's largest numbers, 2^128 / 127, times 2^6 is finite. Products from 2^122 on are not.
constexpr float kUp = 64.f;

// The two int8 in bits 0..7 and 16..23 of w times 2^-6 as two bf16, exactly. 0x4000 is 128 * 2^-6 in bf16,
// with 2^-6 as its last place: or-ing the low seven bits gives (128 + low7) 2^-6, or-ing the sign bit
// 128 or 256 times 2^-6, and the difference is the int8 times 2^-6.
__device__ __forceinline__ uint32_t widen_pair(uint32_t w) {
  const uint32_t a = (w & 0x007f007fu) | 0x40004000u;
  const uint32_t b = (w & 0x00800080u) | 0x40004000u;
  const __nv_bfloat162 q = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                   *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&q);
}

// Eight int8 (two words) as one 16-byte piece of bf16. The middle two of each four trade places (the
// pairs are bytes 0, 2 and 1, 3 of a word); the epilogue trades them back, where it costs nothing.
__device__ __forceinline__ uint4 widen8(uint32_t w0, uint32_t w1) {
  return make_uint4(widen_pair(w0), widen_pair(w0 >> 8), widen_pair(w1), widen_pair(w1 >> 8));
}

// The raw block at `raw` into the tile at `tile`: thread t's share.
__device__ __forceinline__ void widen_x(uint32_t raw, uint32_t tile, int t) {
  uint4 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = ld_shared_v4(raw + ckpt::x_from(ckpt::x_unit(t, i)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const ckpt::XUnit x = ckpt::x_unit(t, i);
    const uint4 even = widen8(w[i].x, w[i].y), odd = widen8(w[i].z, w[i].w);
    st_shared_v4(tile + ckpt::x_to(x, false), x.odd_first ? odd : even);
    st_shared_v4(tile + ckpt::x_to(x, true), x.odd_first ? even : odd);
  }
}

// A row's scale times kUp as two bf16, each twice: the sum is the scale to 2^-16 of it.
struct Scale2 {
  __nv_bfloat162 head, tail;
};

__device__ __forceinline__ Scale2 split_scale(float s) {
  const float up = __fmul_rn(s, kUp);
  const __nv_bfloat16 head = __float2bfloat16_rn(up);
  return {__bfloat162bfloat162(head), __bfloat162bfloat162(__float2bfloat16_rn(__fsub_rn(up, __bfloat162float(head))))};
}

// Two bf16 (w) times s, as head and tail: head is the product with the scale's head, rounded; a fused
// multiply-add gives what that rounding took, exactly (16 bits less their upper 8), and a second one adds
// the product with the scale's tail. |tail| <= 2^-7 of the product, so its one rounding and the scale's
// are 2^-15 + 2^-16 of it in all.
__device__ __forceinline__ void split_pair(uint32_t w, const Scale2& s, uint32_t& head, uint32_t& tail) {
  const __nv_bfloat162 z = *reinterpret_cast<const __nv_bfloat162*>(&w);
  const __nv_bfloat162 h = __hmul2_rn(z, s.head);
  const __nv_bfloat162 t = __hfma2(z, s.tail, __hfma2(z, s.head, __hneg2(h)));
  head = *reinterpret_cast<const uint32_t*>(&h);
  tail = *reinterpret_cast<const uint32_t*>(&t);
}

// What is infinite has no tail (infinity less infinity); NaN is NaN in the head.
__device__ __noinline__ uint32_t finite_pair(uint32_t tail) {
  if ((tail & 0x7f80u) == 0x7f80u) tail &= 0xffff0000u;
  if ((tail & 0x7f800000u) == 0x7f800000u) tail &= 0xffffu;
  return tail;
}

__device__ __forceinline__ void split8(const uint4& w, const Scale2& s, uint4& h, uint4& l) {
  split_pair(w.x, s, h.x, l.x);
  split_pair(w.y, s, h.y, l.y);
  split_pair(w.z, s, h.z, l.z);
  split_pair(w.w, s, h.w, l.w);
  const uint32_t any = l.x | l.y | l.z | l.w;  // all ones in an exponent here: perhaps in one of the tails
  if ((any & 0x7f80u) == 0x7f80u || (any & 0x7f800000u) == 0x7f800000u)
    l = make_uint4(finite_pair(l.x), finite_pair(l.y), finite_pair(l.z), finite_pair(l.w));
}

// dZ at `z` becomes head and tail: thread t's share. scale[i] is that of the thread's i-th row.
template <int T>
__device__ __forceinline__ void split_dz(uint32_t z, int t, const float (&scale)[ckpt::DzUnits<T>::kRows]) {
  using U = ckpt::DzUnits<T>;
#pragma unroll
  for (int c = 0; c < U::kChunks; ++c) {
    uint4 w[U::kRows];
#pragma unroll
    for (int i = 0; i < U::kRows; ++i) w[i] = ld_shared_v4(z + U::head_at(t, i, c));
#pragma unroll
    for (int i = 0; i < U::kRows; ++i) {
      uint4 h, l;
      split8(w[i], split_scale(scale[i]), h, l);
      st_shared_v4(z + U::head_at(t, i, c), h);
      st_shared_v4(z + U::tail_at(t, i, c), l);
    }
  }
}

// Sixteen sums of a lane's column from row c on. Converted tiles have head's and tail's beside each other.
template <int T, bool READY>
__device__ __forceinline__ void load_sums(uint32_t t_row, int c, float (&sum)[16]) {
  uint32_t r[16];
  tmem_ld_32x32b_x16(t_row + c, r);
  if constexpr (READY) {
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) sum[j] = __uint_as_float(r[j]);
  } else {
    uint32_t l[16];
    tmem_ld_32x32b_x16(t_row + T + c, l);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) sum[j] = __uint_as_float(r[j]) + __uint_as_float(l[j]);
  }
}

template <int T, bool READY>
__global__ void __launch_bounds__(kThreads)
    dw_narrow_kernel(const __grid_constant__ CUtensorMap tmz, const __grid_constant__ CUtensorMap tmx, const Params p) {
  constexpr int STAGES = Ring<T, READY>::kStages;
  constexpr uint32_t STAGE = Ring<T, READY>::kStage;
  constexpr uint32_t Z_AT = WIDE_BYTES, RAW_AT = Z_AT + Ring<T, READY>::kZ;
  constexpr uint32_t SUMS = READY ? T : 2 * T;  // columns of the accumulator
  __shared__ float s_back[T];  // READY
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE);  // dZ and the int8 block landed
  uint64_t* wide = full + STAGES;                                       // converted
  uint64_t* empty = wide + STAGES;                                      // read by the MMAs
  uint64_t* acc_full = empty + STAGES;
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
  const int k0 = (tile % p.k_tiles) * COLS;
  const int n0 = (tile / p.k_tiles) * T;
  const int blocks = (p.M + BK - 1) / BK;
  const int kb0 = min(static_cast<int>(rank) * p.kb_per_cta, blocks);
  const int kb1 = min(kb0 + p.kb_per_cta, blocks);

  if (warp == 0 && lane == 0) {
    *gave_up = 0u;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&wide[s], kConvWarps);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(drain, 1);
    fence_mbarrier_init();
    tma_prefetch_desc(&tmz);
    tma_prefetch_desc(&tmx);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, SUMS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if constexpr (READY) {
    pdl_wait();
    pdl_launch_dependents();
  }

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, armed = 0u, armed_par = 0u;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[s], ph ^ 1u, kFaultWaitEmpty)) break;
        uint8_t* at = smem + s * STAGE;
        mbar_arrive_expect_tx(&full[s], chunks(T) * MN_CHUNK_BYTES + (READY ? WIDE_BYTES : RAW_BYTES));
        if constexpr (READY) {
          tma_load_2d(at, &tmx, &full[s], k0, kb * BK);
          tma_load_2d(at + MN_CHUNK_BYTES, &tmx, &full[s], k0 + 64, kb * BK);
        } else {
          tma_load_2d(at + RAW_AT, &tmx, &full[s], k0, kb * BK);
        }
#pragma unroll
        for (int c = 0; c < chunks(T); ++c)
          tma_load_2d(at + Z_AT + c * MN_CHUNK_BYTES, &tmz, &full[s], n0 + 64 * c, kb * BK);
        armed |= 1u << s;
        armed_par = (armed_par & ~(1u << s)) | (ph << s);
        if (++s == STAGES) { s = 0; ph ^= 1u; }
      }
      asked[0] = armed;
      asked[1] = armed_par;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t IDESC = READY ? make_idesc_f16_f32(COLS, SUMS, true, true) : make_idesc_bf16_f32(COLS, SUMS, true, true);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        // dZ and the int8 block were there before they were converted, but the converters saw that, not
        // this thread
        ok = mbar_wait(&full[s], ph, kFaultWaitFull) && (READY || mbar_wait(&wide[s], ph, kFaultWaitFull));
        if (!ok) break;
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
      // After a fault the epilogue is not told that the sums are there: it gives up as well.
      if (!ok) *gave_up = 1u;
      uint64_t* done = ok ? acc_full : drain;
      umma_commit(done);
      gemm::drain_wait(done, 0u);
    }
    __syncwarp();
  } else if constexpr (READY) {
    for (int t = static_cast<int>(threadIdx.x) - 64; t < T; t += kThreads - 64)
      s_back[t] = n0 + t < p.N ? __ldg(p.scale + n0 + t) : 0.f;
  } else {
    const int group = static_cast<int>(warp - 2u) / kConvWarps;
    const int t = static_cast<int>((warp - 2u) % kConvWarps * 32u + lane);
    using U = ckpt::DzUnits<T>;
    float next[U::kRows];
#pragma unroll
    for (int i = 0; i < U::kRows; ++i) {
      const int m = (kb0 + group) * BK + U::row(t, i);
      next[i] = m < p.M ? __ldg(p.scale + m) : 0.f;
    }
    int s = group;
    uint32_t ph = 0;
    for (int kb = kb0 + group; kb < kb1; kb += kConvGroups) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full[s], ph, kFaultWaitFull))) break;
      const uint32_t at = smem_u32(smem + s * STAGE);
      float scale[U::kRows];
#pragma unroll
      for (int i = 0; i < U::kRows; ++i) {
        scale[i] = next[i];
        const int m = (kb + kConvGroups) * BK + U::row(t, i);
        next[i] = m < p.M ? __ldg(p.scale + m) : 0.f;
      }
      widen_x(at + RAW_AT, at, t);
      split_dz<T>(at + Z_AT, t, scale);
      fence_proxy_async_shared();  // the MMA reads the tiles through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(&wide[s]);
      s += kConvGroups;
      if (s >= STAGES) { s -= STAGES; ph ^= 1u; }
    }
  }

  // ------------------------------------------------------------ epilogue: one column per lane
  if constexpr (READY) __syncthreads();  // s_back
  const auto rounded = [&](float sum, int row) { return __float2bfloat16_rn(READY ? sum * s_back[row] : sum); };
  const uint32_t q = warp & 3u;               // the lane quarter of a warp
  const int half = warp >= 6 ? 1 : 0;         // the two warps of a quarter share the rows of dW
  const uint32_t in_quarter = !READY && ((lane + 1u) & 2u) ? lane ^ 3u : lane;  // widen8 swapped the middle two of four
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
        float sum[16];
        __syncwarp();  // lanes past the last column skip the stores
        load_sums<T, READY>(t_row, c, sum);
        if (k < p.K) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c + j < rows) out[(c + j) * p.ldo] = rounded(sum[j], c + j);
        }
      }
      __syncwarp();
    }
  } else {
    // The ring is free (every MMA has read its stage): it takes this CTA's partial sums [row][column],
    // and each CTA adds up and stores its share of the rows.
    float* part = reinterpret_cast<float*>(smem);
    const bool any = kb0 < kb1;  // the last CTAs may have no K block: their sums are zero
    if (warp >= 2 && ok) {
#pragma unroll 1
      for (int c = 16 * half; c < rows; c += 32) {
        float sum[16];
        load_sums<T, READY>(t_row, c, sum);
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * COLS + q * 32u + lane] = any ? sum[j] : 0.f;
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
          if (t + j < last) out[(t + j) * p.ldo] = rounded(sum[j], t + j);
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
    for (int t = 0; t < STAGES; ++t)
      if (asked[0] & (1u << t)) gemm::drain_wait(&full[t], (asked[1] >> t) & 1u);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, SUMS);
  }
}

}  // namespace ckpt_narrow
}  // namespace c3cu
