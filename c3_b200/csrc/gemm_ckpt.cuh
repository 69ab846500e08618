// Weight gradient from an 8-bit checkpoint of the layer's input:
//
//   dW[N][K] = sum_m dZ[m][n] * (q[m][k] * scale[m])        (bf16 out, fp32 sums in TMEM)
//
// dZ is bf16, X is held as int8 rows with one fp32 scale each (c3cu_quantize_rows). The scale runs
// along the sum, so it cannot wait for the epilogue: q * scale is rounded to bf16, the tensor
// cores' operand type, on its way to them. That rounding (relative 2^-8 at most, the size of the
// output's own) is the only one besides the output's; q itself would be exact in bf16.
//
// dw_kernel has gemm2_kernel's structure (256 x 256 tiles on CTA pairs, both operands MN-major,
// since dZ and X are stored with the sum's index as their rows). The MMA's rows are the columns of
// dW, so that a warp's stores run along its rows whatever their alignment (2176 x 4822 over 576 rows:
// 138 us with a row of dW per lane, 27 so). Two forms:
//   RAW   TMA brings X's int8 block into a raw buffer and converter warps widen it into the
//         swizzled bf16 tile that the MMA reads: X crosses HBM and L2 at one byte per element and
//         no bf16 copy of it exists, but it is widened once for every 256 rows of dW.
//   !RAW  X was widened once into a bf16 workspace (widen_kernel), which the kernel reads by TMA.
// Beside the tensor cores the widening runs into the power limit and the shared-memory traffic of
// the tiles (16384 x 4096 x 4096: 505 to 548 us RAW, 424 !RAW, of which widen_kernel 33; the bf16
// gradient from a bf16 X takes 350 to 370 in the same loop). With few K blocks RAW saves the launch
// (in these tiles 128 x 256 x 784 took 10.2 us RAW, 12.3 else; gemm_ckpt_narrow.cuh takes 6.2).
//
// Warps: 0 TMA, 1 MMA (leader), 2..9 epilogue; RAW: 10..17 converters (two groups of four), 18 TMA
// of X.
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
constexpr int kConvWarps = 4;   // a group's warps
constexpr int kConvGroups = 2;  // the groups take K blocks in turn
constexpr int kRawWarp = 2 + kEpiWarps + kConvGroups * kConvWarps;
constexpr uint32_t RAW_BYTES = BK * HN;  // 64 rows (m) of 128 int8 (k)

// Ring depths. RAW: dZ, raw int8 and widened tiles go through rings of their own, so that the
// loads' latency and the conversion's are each hidden by as many stages as they take. !RAW: one
// ring of both operands' stages.
template <bool RAW>
struct Ring {
  static constexpr int kA = RAW ? 5 : 7;
  static constexpr int kB = RAW ? 4 : 7;
  static constexpr int kRaw = RAW ? 8 : 0;
  static constexpr int kThreads = RAW ? 32 * (kRawWarp + 1) : 32 * (2 + kEpiWarps);
  static constexpr uint32_t kBytes = kA * A_STAGE_BYTES + kB * B_STAGE_BYTES + kRaw * RAW_BYTES;
  static constexpr uint32_t kSmem = kBytes + 2 * (kA + kB + kRaw) * 8 + 5 * 8 + 8 + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory");
  static_assert(kB % kConvGroups == 0 || !RAW, "a stage belongs to one group, which so sees each of its phases");
};

struct Params {
  int32_t M, N, K;     // dW is N x K, the sum runs over M
  __nv_bfloat16* out;
  int64_t ldo;
  const float* scale;  // [M]
  float* partial;      // slots of [256 rows][256 columns] fp32
  Plan plan;
};

// A row's scale as two bf16 pairs: s = head + tail to 16 bits (both truncated).
struct Scale2 {
  __nv_bfloat162 head, tail;
};

__device__ __forceinline__ __nv_bfloat162 both_halves(float v) {  // v's upper 16 bits, twice
  const uint32_t b = __byte_perm(__float_as_uint(v), 0u, 0x3232);
  return *reinterpret_cast<const __nv_bfloat162*>(&b);
}

__device__ __forceinline__ Scale2 split_scale(float s) {
  const float head = __uint_as_float(__float_as_uint(s) & 0xffff0000u);
  return {both_halves(s), both_halves(s - head)};
}

// The two int8 in bits 0..7 and 16..23 of w, times the scale, as two bf16 (packed conversions
// from fp32 run at a fraction of this rate). 0x4300 is 128 in bf16, with one as its last place:
// or-ing the low seven bits gives 128 + low7, or-ing the sign bit 128 or 256, and the difference
// is the int8, exactly. q * tail is rounded at 2^-8 of a number 2^-8 of the result, then one fused
// multiply-add rounds the result, so it is q * s rounded to bf16 to within 2^-16; zero stays zero.
__device__ __forceinline__ uint32_t scale_pair(uint32_t w, const Scale2& s) {
  const uint32_t a = (w & 0x007f007fu) | 0x43004300u;
  const uint32_t b = (w & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 q = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                   *reinterpret_cast<const __nv_bfloat162*>(&b));
  const __nv_bfloat162 x = __hfma2(q, s.head, __hmul2(q, s.tail));
  return *reinterpret_cast<const uint32_t*>(&x);
}

// Eight int8 (two words) times s, as one 16-byte piece of bf16. The middle two of each four trade
// places (the pairs are bytes 0, 2 and 1, 3 of a word); the epilogue trades them back, where it
// costs nothing.
__device__ __forceinline__ uint4 scale8(uint32_t w0, uint32_t w1, const Scale2& s) {
  return make_uint4(scale_pair(w0, s), scale_pair(w0 >> 8, s), scale_pair(w1, s), scale_pair(w1 >> 8, s));
}

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// One warp's part in widening a K block: 16 of the block's 64 rows, four at a time. Lane = 8 * row + u
// reads the 16 int8 of unit u of its row and writes two 16-byte pieces of the swizzled bf16 tile:
// chunk u / 4 (64 columns), pieces 2u and 2u + 1 of 8, at position piece ^ (row mod 8). Units 4..7
// write their odd piece first, so that the eight lanes of a row touch all banks once.
struct Widener {
  int r0;             // the lane's rows are r0, r0 + 4, ...
  uint32_t from, to;  // of the lane's first unit and piece's line in the raw block and the tile
  uint32_t at;        // rows r0, r0 + 4, ...: the row modulo 8 alternates between lane / 8 and that plus 4
  bool swap;

  __device__ __forceinline__ Widener(int warp, int lane) {
    const int u = lane & 7;
    r0 = warp * 16 + (lane >> 3);
    swap = u >= 4;
    from = static_cast<uint32_t>(r0 * HN + u * 16);
    const uint32_t piece = static_cast<uint32_t>(((2 * u) & 7) | (swap ? 1 : 0));
    to = static_cast<uint32_t>((u >> 2) * MN_CHUNK_BYTES + r0 * 128);
    at = (piece ^ static_cast<uint32_t>(lane >> 3)) << 4;
  }
  __device__ __forceinline__ void load(uint32_t raw, uint4 (&w)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = ld_shared_v4(raw + from + j * (4 * HN));
  }
  __device__ __forceinline__ void convert(const uint4& w, float scale, uint4* o) const {
    const Scale2 sc = split_scale(scale);
    o[0] = scale8(swap ? w.z : w.x, swap ? w.w : w.y, sc);
    o[1] = scale8(swap ? w.x : w.z, swap ? w.y : w.w, sc);
  }
  __device__ __forceinline__ void store(uint32_t tile, const uint4 (&o)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      st_shared_v4(tile + to + (at ^ ((j & 1) ? 64u : 0u)) + j * 512, o[2 * j]);
      st_shared_v4(tile + to + (at ^ 16u ^ ((j & 1) ? 64u : 0u)) + j * 512, o[2 * j + 1]);
    }
  }
};

// Counts an arrival on a barrier of the leader CTA. The writes it publishes were made visible to
// the async proxy, which alone reads them, by the writers' proxy fences; a release at cluster
// scope stalled the warp for a round trip to memory (16384 x 4096 x 4096: 743 us, 527 without).
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(mapa_shared(smem_u32(bar), 0u)) : "memory");
}

template <bool RAW>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Ring<RAW>::kThreads, 1)
    dw_kernel(const __grid_constant__ CUtensorMap tma, const __grid_constant__ CUtensorMap tmx, const Params p) {
  constexpr int A_STAGES = Ring<RAW>::kA, B_STAGES = Ring<RAW>::kB, RAW_STAGES = Ring<RAW>::kRaw;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + A_STAGES * A_STAGE_BYTES;
  uint8_t* sRaw = sB + B_STAGES * B_STAGE_BYTES;
  uint64_t* a_full = reinterpret_cast<uint64_t*>(smem + Ring<RAW>::kBytes);  // loads of both CTAs (the leader's is used)
  uint64_t* a_empty = a_full + A_STAGES;
  uint64_t* b_full = a_empty + A_STAGES;      // RAW: widened, in both CTAs (the leader's is used)
  uint64_t* b_empty = b_full + B_STAGES;
  uint64_t* raw_full = b_empty + B_STAGES;    // this CTA's int8 block landed
  uint64_t* raw_empty = raw_full + RAW_STAGES;
  uint64_t* acc_full = raw_empty + RAW_STAGES;
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
    for (int s = 0; s < A_STAGES; ++s) {
      mbar_init(&a_full[s], 1);
      mbar_init(&a_empty[s], 1);
    }
    for (int s = 0; s < B_STAGES; ++s) {
      mbar_init(&b_full[s], 2 * kConvWarps);
      mbar_init(&b_empty[s], 1);
    }
    for (int s = 0; s < RAW_STAGES; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], kConvWarps);
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
        [[maybe_unused]] const int k0 = (it.tile % k_tiles) * TN + static_cast<int>(rank) * HN;
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait(&a_empty[s], ph ^ 1u, kFaultWaitEmpty)) { ok = false; break; }
          if (leader) mbar_arrive_expect_tx(&a_full[s], 2u * (A_STAGE_BYTES + (RAW ? 0u : B_STAGE_BYTES)));
          const uint32_t bar_leader = mapa_shared(smem_u32(&a_full[s]), 0u);
          uint8_t* sa = sA + s * A_STAGE_BYTES;
#pragma unroll
          for (int j = 0; j < HM / 64; ++j)
            tma_load_2d_pair(sa + j * MN_CHUNK_BYTES, &tma, bar_leader, n0 + 64 * j, kb * BK);
          if constexpr (!RAW) {
            uint8_t* sb = sB + s * B_STAGE_BYTES;
#pragma unroll
            for (int j = 0; j < HN / 64; ++j)
              tma_load_2d_pair(sb + j * MN_CHUNK_BYTES, &tmx, bar_leader, k0 + 64 * j, kb * BK);
          }
          armed |= 1u << s;
          armed_par = (armed_par & ~(1u << s)) | (ph << s);
          if (++s == A_STAGES) { s = 0; ph ^= 1u; }
        }
      }
      if (!ok || fault_raised()) {
        if (leader) {
          for (int t = 0; t < A_STAGES; ++t)
            if (armed & (1u << t)) gemm::drain_wait(&a_full[t], (armed_par >> t) & 1u);
        }
        gemm2::settle_inflight_copies();
      }
    }
    __syncwarp();
  } else if (RAW && warp == kRawWarp) {
    // ------------------------------------------------------------ TMA producer of the int8 blocks
    if constexpr (RAW) if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, armed = 0u, armed_par = 0u;
      bool ok = true;
      for (int i = cluster; ok && i < items; i += num_clusters) {
        const Item it = item_at(p.plan, i, blocks);
        const int k0 = (it.tile % k_tiles) * TN + static_cast<int>(rank) * HN;
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait(&raw_empty[s], ph ^ 1u, kFaultWaitEmpty)) { ok = false; break; }
          mbar_arrive_expect_tx(&raw_full[s], RAW_BYTES);
          tma_load_2d(sRaw + s * RAW_BYTES, &tmx, &raw_full[s], k0, kb * BK);
          armed |= 1u << s;
          armed_par = (armed_par & ~(1u << s)) | (ph << s);
          if (++s == RAW_STAGES) { s = 0; ph ^= 1u; }
        }
      }
      if (!ok || fault_raised()) {
        for (int t = 0; t < RAW_STAGES; ++t)
          if (armed & (1u << t)) gemm::drain_wait(&raw_full[t], (armed_par >> t) & 1u);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (leader && lane == 0) {
      constexpr uint32_t IDESC = make_idesc_bf16_f32(TM, TN, true, true);
      int sa = 0, sb = 0;
      uint32_t pa = 0, pb = 0, acc = 0, acc_ph = 0;
      bool ok = true;
      for (int i = cluster; ok && i < items; i += num_clusters) {
        const Item it = item_at(p.plan, i, blocks);
        if (!mbar_wait(&acc_empty[acc], acc_ph ^ 1u, kFaultWaitAccEmpty)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * TN;
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait(&a_full[sa], pa, kFaultWaitFull) ||
              (RAW && !mbar_wait(&b_full[sb], pb, kFaultWaitFull))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(sA + sa * A_STAGE_BYTES);
          const uint32_t b_addr = smem_u32(sB + sb * B_STAGE_BYTES);
#pragma unroll
          for (int kk = 0; kk < BK / UMMA_K; ++kk)
            umma_f16_ss_pair(d_tmem, make_sw128_desc(b_addr + kk * UMMA_K * 128, MN_CHUNK_BYTES, 1024),
                             make_sw128_desc(a_addr + kk * UMMA_K * 128, MN_CHUNK_BYTES, 1024), IDESC,
                             (kb != it.kb0 || kk != 0) ? 1u : 0u);
          if constexpr (RAW) umma_commit_pair_mc(&b_empty[sb], kPairMask);
          umma_commit_pair_mc(&a_empty[sa], kPairMask);
          if (++sa == A_STAGES) { sa = 0; pa ^= 1u; }
          if (++sb == B_STAGES) { sb = 0; pb ^= 1u; }
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
    const int c_lo = static_cast<int>((warp - 2u) >> 2) * (TM / 2);  // this warp's half of the rows of dW
    // the column within the CTA's 128: RAW tiles hold the middle two of each four swapped (scale8)
    const uint32_t l = RAW && ((lane + 1u) & 2u) ? lane ^ 3u : lane;
    const int in_tile = static_cast<int>(rank) * HN + static_cast<int>(q * 32u + l);
    uint32_t acc = 0, acc_ph = 0;
    for (int i = cluster; i < items; i += num_clusters) {
      const Item it = item_at(p.plan, i, blocks);
      const int n0 = (it.tile / k_tiles) * TM + c_lo;
      const int k = (it.tile % k_tiles) * TN + in_tile;
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[acc], acc_ph, kFaultWaitAccFull))) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((q * 32u) << 16) + acc * TM + static_cast<uint32_t>(c_lo);
#pragma unroll 1
      for (int c = 0; c < TM / 2; c += 32) {
        const int rows = min(32, p.N - n0 - c);
        if (rows <= 0) break;
        uint32_t r[32];
        __syncwarp();  // lanes past the last column skip the stores
        tmem_ld_32x32b_x32(t_row + c, r);
        tmem_wait_ld();
        if (k >= p.K) continue;
        if (it.slot < 0) {
          __nv_bfloat16* out = p.out + static_cast<int64_t>(n0 + c) * p.ldo + k;
#pragma unroll
          for (int j = 0; j < 32; ++j, out += p.ldo)
            if (j < rows) *out = __float2bfloat16_rn(__uint_as_float(r[j]));
        } else {
          float* part = p.partial + static_cast<size_t>(it.slot) * (TM * TN) + (c_lo + c) * TN + in_tile;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j < rows) __stcg(part + j * TN, __uint_as_float(r[j]));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_leader(&acc_empty[acc]);
      acc ^= 1u;
      if (acc == 0u) acc_ph ^= 1u;
    }
  } else if constexpr (RAW) {
    // ------------------------------------------------------------ converters (warps 10..17)
    const int cw = static_cast<int>(warp) - 2 - kEpiWarps;
    const int group = cw / kConvWarps;
    const Widener widen(cw % kConvWarps, static_cast<int>(lane));
    int turn = 0;  // K blocks of earlier items, modulo the groups
    uint32_t sr = group, sb = group, pr = 0, pb = 0;
    bool ok = true;
    for (int i = cluster; ok && i < items; i += num_clusters) {
      const Item it = item_at(p.plan, i, blocks);
      const int first = it.kb0 + (group - turn + kConvGroups) % kConvGroups;
      turn = (turn + it.kb1 - it.kb0) % kConvGroups;
      float next[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = first * BK + widen.r0 + 4 * j;
        next[j] = m < p.M ? __ldg(p.scale + m) : 0.f;
      }
      for (int kb = first; kb < it.kb1; kb += kConvGroups) {
        ok = __all_sync(0xffffffffu, mbar_wait(&raw_full[sr], pr, kFaultWaitFull));
        if (!ok) break;
        uint4 w[4], o[8];
        widen.load(smem_u32(sRaw) + sr * RAW_BYTES, w);
        __syncwarp();
        if (lane == 0) mbar_arrive(&raw_empty[sr]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          widen.convert(w[j], next[j], &o[2 * j]);
          const int m = (kb + kConvGroups) * BK + widen.r0 + 4 * j;
          next[j] = m < p.M ? __ldg(p.scale + m) : 0.f;
        }
        // only now: the conversion runs while the MMAs still read the stage's last tile
        ok = __all_sync(0xffffffffu, mbar_wait(&b_empty[sb], pb ^ 1u, kFaultWaitEmpty));
        if (!ok) break;
        widen.store(smem_u32(sB) + sb * B_STAGE_BYTES, o);
        fence_proxy_async_shared();  // the MMA reads the tile through the async proxy
        __syncwarp();
        if (lane == 0) arrive_leader(&b_full[sb]);
        sr += kConvGroups;
        if (sr >= RAW_STAGES) { sr -= RAW_STAGES; pr ^= 1u; }
        sb += kConvGroups;
        if (sb >= B_STAGES) { sb -= B_STAGES; pb ^= 1u; }
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

// X in bf16: out[m][k] = bf16(q * scale), rows of `ldo` elements (a multiple of 8, columns past K
// zero). A warp takes rows, a lane eight columns at a time (so that a warp's stores are one run of
// 512 bytes), eight loads ahead of their use.
constexpr int kWidenWarps = 8;
constexpr int kWidenAhead = 8;

__global__ void __launch_bounds__(32 * kWidenWarps)
    widen_kernel(const int8_t* __restrict__ q, int64_t ldq, const float* __restrict__ scale,
                 __nv_bfloat16* __restrict__ out, int64_t ldo, int M, int K) {
  pdl_wait();
  pdl_launch_dependents();
  const int units = static_cast<int>(ldo / 8), whole = K / 8;
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * kWidenWarps;
  for (int64_t m = static_cast<int64_t>(blockIdx.x) * kWidenWarps + (threadIdx.x >> 5); m < M; m += warps) {
    const float s = __ldg(scale + m);
    const int8_t* from = q + m * ldq;
    uint4* to = reinterpret_cast<uint4*>(out + m * ldo);
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
            if (u * 8 + j < K) x[j / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(from[u * 8 + j])) << (8 * (j % 4));
          w[i] = make_uint2(x[0], x[1]);
        }
      }
#pragma unroll
      for (int i = 0; i < kWidenAhead; ++i) {
        const int u = u0 + 32 * i;
        if (u >= units) break;
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t v = (j < 2 ? w[i].x : w[i].y) >> (16 * (j % 2));
          o[j] = pack_bf16x2(static_cast<float>(static_cast<int8_t>(v)) * s,
                             static_cast<float>(static_cast<int8_t>(v >> 8)) * s);
        }
        to[u] = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
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
    if (n0 + i < p.N) out[i * p.ldo] = __float2bfloat16_rn(sum[i]);
}

}  // namespace ckpt
}  // namespace c3cu
